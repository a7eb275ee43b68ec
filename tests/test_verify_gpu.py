"""The verification of drafted tokens (verify_drafts) against a plain computation in 64 bits.

Kept drafts and tokens are whole numbers and have to be equal: both sides decide with 64-bit sums.  The kernel's weights are
off by at most 1.1 * 10^-12 of themselves, each differently, so a border between two tokens moves by at most that much of the
whole, and a draw over a few thousand tokens meets a border that moved for one uniform number in 10^8.  Probabilities are 64-bit values rounded to
float32 once: 2^-24 of themselves, 2^-23 allowed."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _ops():
    from dlgo_amd.kernels import ops
    return ops


def i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32), device=DEV)


def plain(logits, drafts, k, temperature, uniform, draft_logits):
    """Lists of kept counts, tokens and probabilities.  logits, draft_logits: float64 on the host."""
    accepted, token, probs = [], [], []
    row = at = 0
    for n, t in zip(k, temperature):
        x = logits[row:row + n + 1]
        if t > 0:
            p = torch.softmax(x / t, -1)
            q = torch.softmax(draft_logits[at:at + n] / t, -1) if draft_logits is not None else None
        j, refused = 0, False
        for m in range(n):
            tok = drafts[at + m]
            inside = 0 <= tok < x.shape[1]
            pt = 0.0 if not inside else (float(int(x[m].argmax()) == tok) if t <= 0 else p[m, tok].item())
            probs.append(pt)
            if not refused:
                qt = 1.0 if t <= 0 or q is None else (q[m, tok].item() if inside else 0.0)
                keep = pt > 0 if t <= 0 else uniform[row + m] * qt < pt
                if keep:
                    j += 1
                else:
                    refused = True
        accepted.append(j)
        if t <= 0:
            token.append(int(x[j].argmax()))
        else:
            w = p[j].clone()
            if refused and q is not None:
                w = (w - q[j]).clamp(min=0)
            elif refused and 0 <= drafts[at + j] < x.shape[1]:
                w[drafts[at + j]] = 0.0
            if not w.sum() > 0:
                w = p[j]
            c = torch.cumsum(w, 0)
            hit = int((c <= uniform[row + n] * c[-1].item()).sum())
            token.append(min(hit, x.shape[1] - 1))
        row += n + 1
        at += n
    return accepted, token, probs


def call(logits, drafts, k, temperature, uniform, draft_logits, most=None, **kw):
    n, d = len(k), sum(k)
    acc, tok = torch.full((n,), -9, dtype=torch.int32, device=DEV), torch.full((n,), -9, dtype=torch.int32, device=DEV)
    probs = torch.full((d,), -1.0, device=DEV)
    _ops().verify_drafts(logits, i32(drafts), i32(np.concatenate([[0], np.cumsum(k)])), torch.tensor(temperature, dtype=torch.float32, device=DEV),
                         torch.tensor(uniform, dtype=torch.float32, device=DEV), acc, tok, max(k + [0]) if most is None else most,
                         draft_logits=draft_logits, probs=probs, **kw)
    return acc.tolist(), tok.tolist(), probs


def f32(v):
    return [float(np.float32(x)) for x in v]


def case(k, vocab, seed, model_drafts, spread=2.0, apart=0.5, temps=(0.8, 1.0, 0.0, 0.3)):
    g = torch.Generator().manual_seed(seed)
    n, d = len(k), sum(k)
    logits = spread * torch.randn(d + n, vocab, generator=g)
    rows = [c + i + j for i, (c, m) in enumerate(zip(np.cumsum([0] + list(k)), k)) for j in range(m)]
    t = f32([temps[i % len(temps)] for i in range(n)])
    seq = [i for i, m in enumerate(k) for _ in range(m)]
    ld = logits[rows] + apart * torch.randn(d, vocab, generator=g) if model_drafts else None
    src = ld if model_drafts else logits[rows]
    noise = -torch.log(-torch.log(torch.rand(d, vocab, generator=g).clamp(1e-9, 1 - 1e-7)))
    scale = torch.tensor([max(t[i], 1e-3) for i in seq]).view(-1, 1) if d else torch.ones(0, 1)
    drafts = (src / scale + noise).argmax(-1).tolist() if d else []
    u = f32(torch.rand(d + n, generator=g).tolist())
    return logits, drafts, list(k), t, u, ld


@pytest.mark.parametrize("model_drafts", [True, False])
@pytest.mark.parametrize("k,vocab", [([4], 384), ([0], 7), ([0, 3, 1, 0, 8, 2, 5], 1001), ([1], 1), ([2, 2], 4096), ([3, 0, 4, 1], 4097),
                                     ([5] * 12, 20011), ([7, 3], 128256), ([1] * 300, 130), ([0, 0, 0, 0], 5000), ([40, 3], 300)])
def test_verify(k, vocab, model_drafts):
    for seed, spread in ((1, 2.0), (2, 0.05), (3, 12.0)):
        logits, drafts, k_, t, u, ld = case(k, vocab, seed, model_drafts, spread)
        dev, ldev = logits.to(DEV), None if ld is None else ld.to(DEV)
        acc, tok, probs = call(dev, drafts, k_, t, u, ldev)
        want = plain(logits.double(), drafts, k_, t, u, None if ld is None else ld.double())
        assert acc == want[0] and tok == want[1]
        w = torch.tensor(want[2], dtype=torch.float64)
        assert ((probs.double().cpu() - w).abs() <= 2.0 ** -23 * w + 1e-44).all()


@pytest.mark.parametrize("model_drafts", [True, False])
@pytest.mark.parametrize("t", [1e-2, 1e-4, 1e-7, 1e-20, 1e-38, 1e6])
def test_temperatures_near_zero_and_far_above(t, model_drafts):
    """Near zero the maximum has all the weight, and equal maxima share it; far above every token has as much."""
    logits, drafts, k, _, u, ld = case([3, 0, 2], 5000, 11, model_drafts, spread=8.0)
    t = f32([t] * 3)
    logits += 25.0                                        # far from zero, where a difference of products would lose it
    if model_drafts:
        ld += 25.0
    logits[:, 17] = logits[:, 4321] = logits.amax(-1) + 0.25
    got = call(logits.to(DEV), drafts, k, t, u, ld.to(DEV) if model_drafts else None)
    want = plain(logits.double(), drafts, k, t, u, ld.double() if model_drafts else None)
    assert got[0] == want[0] and got[1] == want[1]
    assert torch.allclose(got[2].double().cpu(), torch.tensor(want[2], dtype=torch.float64), rtol=2.0 ** -23, atol=1e-37)


def test_rows_further_apart_than_they_are_long_and_not_aligned():
    logits, drafts, k, t, u, ld = case([3, 2, 6], 1003, 5, True)
    want = call(logits.to(DEV), drafts, k, t, u, ld.to(DEV))
    for pad, first in ((5, 1), (8, 4), (1, 0)):
        a = torch.full((logits.shape[0], 1003 + pad), math.nan, device=DEV)
        b = torch.full((ld.shape[0], 1003 + pad), math.nan, device=DEV)
        a[:, first:first + 1003] = logits.to(DEV)
        b[:, first:first + 1003] = ld.to(DEV)
        got = call(a[:, first:first + 1003], drafts, k, t, u, b[:, first:first + 1003])
        assert got[0] == want[0] and got[1] == want[1] and torch.equal(got[2], want[2])


def test_drafts_from_the_targets_own_distribution_are_all_kept():
    logits, drafts, k, t, u, _ = case([6, 6, 6], 5003, 7, False, temps=(1.0, 0.5, 2.0))
    rows = [c + i + j for i, (c, m) in enumerate(zip(np.cumsum([0] + k), k)) for j in range(m)]
    u = f32([1 - 2.0 ** -24] * len(u))
    acc, tok, _ = call(logits.to(DEV), drafts, k, t, u, logits[rows].contiguous().to(DEV))
    assert acc == [6, 6, 6]
    want = plain(logits.double(), drafts, k, t, u, logits[rows].double())
    assert tok == want[1]


def test_the_ends_of_the_uniform_numbers_and_draws_at_the_edges():
    vocab = 9000
    logits = torch.full((2, vocab), -math.inf)
    logits[0, [3, 4500, 8999]] = 0.0
    logits[1, [0, 8998]] = 0.0
    # no drafts: two plain draws each
    for u, want in (([0.0, 0.0], [3, 0]), ([0.34, 0.5], [4500, 8998]), ([1 - 2.0 ** -24] * 2, [8999, 8998])):
        acc, tok, _ = call(logits.to(DEV), [], [0, 0], [1.0, 1.0], u, None)
        assert acc == [0, 0] and tok == want
    # the draft is refused (u = 0 keeps nothing that has no probability) and what is left is drawn from
    acc, tok, probs = call(logits.to(DEV), [7], [1], [1.0], [0.0, 0.5], None)
    assert acc == [0] and tok == [4500] and probs.tolist() == [0.0]
    acc, tok, probs = call(logits.to(DEV), [4500], [1], [1.0], [0.99, 0.6], None)
    assert acc == [0] and tok == [8999]
    acc, tok, probs = call(logits.to(DEV), [4500], [1], [1.0], [0.3, 0.6], None)
    assert acc == [1] and tok == [8998]


def test_infinite_logits_nan_and_greedy_ties():
    vocab = 5000
    logits = torch.randn(3, vocab, generator=torch.Generator().manual_seed(0))
    logits[0, [10, 4999]] = 50.0                    # greedy: the lowest of equals
    logits[1, 77] = math.nan                        # no weight
    logits[2, :] = torch.finfo(torch.float32).min   # masked with the type's lowest value, but for two
    logits[2, [40, 41]] = 1.0
    acc, tok, probs = call(logits.to(DEV), [4999, 77], [2], [0.0], [0.5] * 3, None)
    assert acc == [0] and tok == [10] and probs.tolist() == [0.0, 0.0]
    acc, tok, probs = call(logits[1:].contiguous().to(DEV), [77], [1], [0.7], [0.0, 0.5], None)
    assert acc == [0] and probs.tolist() == [0.0] and tok[0] != 77
    acc, tok, _ = call(logits[2:].contiguous().to(DEV), [], [0], [1.0], [0.75], None)
    assert tok == [41]
    inf = logits[1:2].clone()
    inf[0, [5, 900]] = math.inf
    assert call(inf.to(DEV), [], [0], [1.0], [0.75], None)[1] == [900]
    assert call(inf.to(DEV), [], [0], [0.0], [0.75], None)[1] == [5]
    none = torch.full((2, vocab), math.nan, device=DEV)
    acc, tok, _ = call(none, [3], [1], [1.0], [0.5, 0.5], None)
    assert acc == [0] and 0 <= tok[0] < vocab


def test_tokens_outside_the_vocabulary_and_more_drafts_than_are_looked_at():
    logits, drafts, k, t, u, ld = case([3, 3], 700, 9, True, temps=(1.0,))
    drafts = [700, -1, 5, 2 ** 30, 6, 7]
    acc, tok, probs = call(logits.to(DEV), drafts, k, t, u, ld.to(DEV))
    want = plain(logits.double(), drafts, k, t, u, ld.double())
    assert acc == want[0] == [0, 0] and tok == want[1] and probs[0] == 0 and probs[3] == 0
    lo, dr, k, t, u, _ = case([5, 2], 300, 4, False, temps=(0.0,))
    dr = [int(lo[0].argmax()), int(lo[1].argmax()), int(lo[2].argmax()), 0, 0, int(lo[6].argmax()), int(lo[7].argmax())]
    acc, _, _ = call(lo.to(DEV), dr, k, t, u, None, most=2)
    assert acc == [2, 2]


def test_same_bits_on_another_stream_and_replayed():
    logits, drafts, k, t, u, ld = case([3, 5, 0, 4] * 5, 50257, 3, True)
    dev, ldev = logits.to(DEV), ld.to(DEV)
    first = call(dev, drafts, k, t, u, ldev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = call(dev, drafts, k, t, u, ldev)
    assert first[0] == again[0] and first[1] == again[1] and torch.equal(first[2], again[2])
    n, d = len(k), sum(k)
    args = (dev, i32(drafts), i32(np.concatenate([[0], np.cumsum(k)])), torch.tensor(t, device=DEV), torch.tensor(u, device=DEV))
    acc, tok, probs = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(d, device=DEV)
    work = torch.empty(1 << 22, dtype=torch.uint8, device=DEV)
    _ops().verify_drafts(*args, acc, tok, 5, draft_logits=ldev, probs=probs, scratch=lambda m: work)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _ops().verify_drafts(*args, acc, tok, 5, draft_logits=ldev, probs=probs, scratch=lambda m: work)
    for seed in range(3):
        args[4].copy_(torch.rand(d + n, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = plain(logits.double(), drafts, k, t, args[4].tolist(), ld.double())
        assert acc.tolist() == want[0] and tok.tolist() == want[1]


def test_refusals():
    ops = _ops()
    logits, drafts, k, t, u, ld = case([3, 2], 100, 9, True)
    ok = dict(logits=logits.to(DEV), draft_tokens=i32(drafts), cu_drafts=i32([0, 3, 5]), temperature=torch.tensor(t, device=DEV),
              uniform=torch.tensor(u, device=DEV), accepted=i32([0, 0]), token=i32([0, 0]), max_drafts=3, draft_logits=ld.to(DEV))
    ops.verify_drafts(**ok)
    bad = [dict(logits=ok["logits"][:6]), dict(logits=ok["logits"].double()), dict(logits=ok["logits"].cpu()), dict(draft_tokens=i32(drafts).long()),
           dict(draft_tokens=i32(drafts[:4])), dict(cu_drafts=i32([0, 5])), dict(temperature=ok["temperature"].double()),
           dict(uniform=ok["uniform"][:5]), dict(accepted=i32([0])), dict(token=i32([0, 0, 0])), dict(max_drafts=-1),
           dict(draft_logits=ok["draft_logits"][:, :99]), dict(draft_logits=ok["draft_logits"][:4]), dict(probs=torch.zeros(4, device=DEV)),
           dict(uniform=torch.zeros(14, device=DEV)[::2]), dict(scratch=lambda n: torch.empty(n - 1, dtype=torch.uint8, device=DEV)),
           dict(scratch=lambda n: torch.empty(n, dtype=torch.float32, device=DEV)), dict(logits=torch.zeros(100, 7, device=DEV).t())]
    for kw in bad:
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**ok, **kw})
