"""Pages more than 4 GiB into a cache and rows of logits more than 2^31 elements apart: the same bits as near the start."""
import numpy as np
import pytest
import torch

from test_q8_gpu import DEV, Step, i32, tables
from test_verify_gpu import call, case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,past", [([1, 1, 1], [70, 2300, 0]), ([3, 6], [500, 64]), ([100, 40], [0, 1000]), ([20], [3000]), ([600], [0])])
def test_pages_far_into_a_cache(q_lens, past):
    H, KV, hd = 8, 2, 64
    s = Step(q_lens, past, H, KV, hd, seed=sum(past))
    s.fill()
    cos, sin = tables(max(p + q for p, q in zip(past, q_lens)), hd)
    unrotated = s.storage.clone()
    want_q = s.store(cos=cos, sin=sin)
    want = s.attend(want_q)
    # the same pages, a long way apart and in the opposite order: the first one ends 5.4 GB into the cache
    page, n = s.stride, s.n_pages
    stride = ((5400 << 20) // (n - 1)) // 16 * 16
    far = torch.empty((n - 1) * stride + page, dtype=torch.uint8, device=DEV)
    assert far.numel() > 5 << 30

    def at(i):
        return far[(n - 1 - i) * stride:][:page]

    def fill():
        for i in range(n):
            at(i).copy_(unrotated[i * page:(i + 1) * page])
    table = np.where(s.table >= 0, n - 1 - s.table, -1)
    fill()
    s.storage, s.cache, s.stride, s.table, near = far, far, stride, table, s.storage
    got_q = s.store(cos=cos, sin=sin)
    assert torch.equal(got_q, want_q)
    assert all(torch.equal(at(i), near[i * page:(i + 1) * page]) for i in range(n))
    assert torch.equal(s.attend(got_q), want)
    if max(q_lens) == 1:                                 # rotated and stored on the way
        fill()
        assert torch.equal(s.attend(s.qkv, out=torch.empty_like(want), rotation=(cos, sin)), want)
        assert all(torch.equal(at(i), near[i * page:(i + 1) * page]) for i in range(n))


@pytest.mark.parametrize("model_drafts", [True, False])
def test_rows_of_logits_far_apart(model_drafts):
    logits, drafts, k, t, u, ld = case([2, 0, 1], 5000, 6, model_drafts)
    want = call(logits.to(DEV), drafts, k, t, u, ld.to(DEV) if model_drafts else None)
    ldl = (1 << 29) + 64
    far = torch.empty((logits.shape[0] - 1) * ldl + 5000, device=DEV).as_strided(logits.shape, (ldl, 1))
    assert (logits.shape[0] - 1) * ldl > 1 << 31
    far.copy_(logits)
    fard = None
    if model_drafts:
        fard = torch.empty((ld.shape[0] - 1) * ldl + 5000, device=DEV).as_strided(ld.shape, (ldl, 1))
        fard.copy_(ld)
    got = call(far, drafts, k, t, u, fard)
    assert got[0] == want[0] and got[1] == want[1] and torch.equal(got[2], want[2])
