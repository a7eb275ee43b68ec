"""Windows that no sequence outgrows, up to the largest number there is: as good as none."""
import ctypes

import pytest
import torch

from test_operators_host import lib_of


@pytest.mark.parametrize("rows,n_seq,q,kv", [(1, 1, 1, 131072), (4, 4, 1, 32768), (17, 1, 17, 16401), (96, 16, 6, 4096)])
def test_they_are_dealt_as_without_one(rows, n_seq, q, kv):
    need = lib_of("attention_q8", HEAD_DIM=64).dlgo_attention_q8_scratch
    without = need(rows, n_seq, 32, 8, q, kv, 0)
    assert without > 0
    for window in (kv, 2 ** 30, 2 ** 31 - 100, 2 ** 31 - 1):
        assert need(rows, n_seq, 32, 8, q, kv, ctypes.c_int(window)) == without


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,past", [([1], [20000]), ([17], [9000]), ([1, 5], [200, 70])])
def test_they_are_attended_as_without_one(q_lens, past):
    from test_q8_gpu import Step
    s = Step(q_lens, past, 8, 2, 64)
    s.fill()
    q = torch.randn(s.rows, 8 * 64, generator=s.gen).bfloat16().to("cuda:0")
    want = s.attend(q)
    s.check(want, q)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40):
        assert torch.equal(s.attend(q, window), want)
