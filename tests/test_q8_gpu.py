"""The 8-bit cache: the kernel that rotates and stores (rope_kv_q8) and the attention that reads (attention_q8), each alone
against a plain float64 computation that goes by the documented place of every byte.

Tolerances.  Rounding to a format is off by at most eps / 2 of the value: 2^-4 for e4m3 (2^-10 times the power of two below
its smallest normal number), 2^-8 for bfloat16.  A rotated element is two float32 products and a sum: 2^-22 of the head's
largest element covers its three roundings.  A result of the attention is sum(p v) / sum(p): p is rounded to bfloat16 in the
numerator (2^-8 of sum(p |v|)), the result to bfloat16 (2^-8 of itself), and scores are float32 sums: with the magnitudes
used here (|q||k| * scale below 2^5) they are off by less than head size * 2^-23 * 2^5 <= 2^-10 at a head size of 256, which moves
every p by as much."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PAGE = 64


def _ops():
    from dlgo_amd.kernels import ops
    return ops


def i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32), device=DEV)


def places(hd):
    """Offsets in a head's part of a page of every key byte, value byte [64, hd] and scale byte [64]."""
    tok, d = torch.arange(PAGE)[:, None], torch.arange(hd)[None]
    t, i, g, r = tok // 16, tok % 16, tok % 16 // 4, tok % 4
    k = (t * (hd // 16) + d // 16) * 256 + 16 * i + d % 16
    v = PAGE * hd + (d // 16 * 4 + g) * 256 + d % 16 * 16 + 4 * t + r
    return k, v, (2 * PAGE * hd + 4 * i + t)[:, 0], (2 * PAGE * hd + PAGE + 16 * g + 4 * t + r)[:, 0]


E4M3 = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()


def unpack(storage, off, stride, pages, kv, hd):
    """Keys and values [pages, kv, 64, hd] float64 and their scale bytes of a unit whose pages begin `off` bytes into
    storage, `stride` apart."""
    raw = storage.cpu().view(-1)
    k, v, ks, vs = places(hd)
    nb = 128 * (hd + 1)
    at = torch.as_tensor(pages)[:, None] * stride + off + torch.arange(kv)[None] * nb
    kb, vb = raw[at[..., None, None] + k].long(), raw[at[..., None, None] + v].long()
    ks, vs = raw[at[..., None] + ks].long(), raw[at[..., None] + vs].long()
    p = lambda b: torch.exp2(b.double() - 127)[..., None]     # noqa: E731
    return E4M3[kb] * p(ks), E4M3[vb] * p(vs), ks, vs


class Step:
    """A paged 8-bit cache with sequences at random pages, and a step's rows for them."""

    def __init__(self, q_lens, past, H, KV, hd, units=1, unit=0, seed=0, extra_rows=0, width=None, pad_cols=0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.past, self.H, self.KV, self.hd = list(q_lens), list(past), H, KV, hd
        n = len(q_lens)
        held = [(p + q + PAGE - 1) // PAGE for p, q in zip(past, q_lens)]
        self.n_pages = sum(held) + 2
        page = KV * 128 * (hd + 1)
        self.stride, self.off = units * page, unit * page
        ids = torch.randperm(self.n_pages, generator=g)[:sum(held)].tolist()
        self.slots = torch.randperm(n + 2, generator=g)[:n].tolist()
        width = width or max(held + [1]) + 1
        self.table = np.full((n + 2, width), -1, dtype=np.int32)
        self.pages = []
        for s, h in zip(self.slots, held):
            mine = [ids.pop() for _ in range(h)]
            self.pages.append(mine)
            self.table[s, :h] = mine
        # what was there before is anybody's, NaN codes among it
        self.storage = torch.randint(0, 256, (self.n_pages * self.stride,), generator=g, dtype=torch.int32).to(torch.uint8).to(DEV)
        self.cache = self.storage[self.off:]
        self.rows = sum(q_lens)
        self.cu = np.concatenate([[0], np.cumsum(q_lens)])
        self.pos = np.concatenate([np.arange(p, p + q) for p, q in zip(past, q_lens)] or [[]])
        self.seq = np.repeat(np.arange(n), q_lens)
        self.gen = g
        wide = (H + 2 * KV) * hd + pad_cols
        self.qkv_all = (torch.randn(self.rows + extra_rows, wide, generator=g) * torch.exp(0.7 * torch.randn(self.rows + extra_rows, 1, generator=g))).bfloat16().to(DEV)
        self.qkv = self.qkv_all[:self.rows, :(H + 2 * KV) * hd]

    def arrays(self):
        return i32(self.pos), i32(self.seq), i32(self.slots), i32(self.table)

    def store(self, q_out=None, rot=None, inter=False, cos=None, sin=None, **kw):
        pos, seq, slots, table = self.arrays()
        q_out = torch.empty(self.rows, self.H * self.hd, dtype=torch.bfloat16, device=DEV) if q_out is None else q_out
        _ops().rope_kv_q8(self.qkv, q_out, self.H, self.KV, self.hd, self.hd if rot is None else rot, inter, cos, sin, pos, seq, slots,
                          table, self.cache, self.stride, **kw)
        return q_out

    def fill(self):
        """Keys and values of every token that the sequences hold, stored through the kernel without a rotation."""
        lens = [p + q for p, q in zip(self.past, self.q_lens)]
        rows = sum(lens)
        kv = torch.randn(rows, (self.H + 2 * self.KV) * self.hd, generator=self.gen)
        kv *= torch.exp(0.5 * torch.randn(rows, 1, generator=self.gen))
        pos, seq = np.concatenate([np.arange(m) for m in lens] or [[]]), np.repeat(np.arange(len(lens)), lens)
        q = torch.empty(rows, self.H * self.hd, dtype=torch.bfloat16, device=DEV)
        _ops().rope_kv_q8(kv.bfloat16().to(DEV), q, self.H, self.KV, self.hd, 0, False, None, None, i32(pos), i32(seq), i32(self.slots),
                          i32(self.table), self.cache, self.stride)

    def attend(self, q, window=0, scale=None, out=None, bound_len=None, bound_q=None, **kw):
        out = torch.full_like(q, 7.0) if out is None else out
        _ops().attention_q8(q, out, self.H, self.KV, self.hd, i32(self.cu), i32(self.past), kw.pop("slots", i32(self.slots)),
                            kw.pop("table", i32(self.table)), self.cache, self.stride,
                            bound_q or max(self.q_lens + [0]), bound_len or max([p + x for p, x in zip(self.past, self.q_lens)] + [0]),
                            window=window, scale=scale, **kw)
        return out

    def wanted(self, q, window=0, scale=None):
        """(results, sum(p |v|)) in float64."""
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        group = self.H // self.KV
        out = torch.zeros(self.rows, self.H, self.hd, dtype=torch.float64)
        mag = torch.zeros_like(out)
        qd = q[:self.rows].double().cpu().view(self.rows, self.KV, group, self.hd)
        for s, (p0, n) in enumerate(zip(self.past, self.q_lens)):
            if n == 0:
                continue
            k, v, _, _ = unpack(self.storage, self.off, self.stride, self.pages[s], self.KV, self.hd)
            k = k.transpose(0, 1).reshape(self.KV, -1, self.hd)[:, :p0 + n]
            v = v.transpose(0, 1).reshape(self.KV, -1, self.hd)[:, :p0 + n]
            a = torch.einsum("tkgd,kld->tkgl", qd[self.cu[s]:self.cu[s + 1]], k) * scale
            pos, key = p0 + torch.arange(n)[:, None], torch.arange(p0 + n)[None]
            hidden = key > pos
            if window:
                hidden |= key <= pos - window
            w = torch.softmax(a.masked_fill(hidden[:, None, None], -math.inf), -1)
            out[self.cu[s]:self.cu[s + 1]] = torch.einsum("tkgl,kld->tkgd", w, v).reshape(n, self.H, self.hd)
            mag[self.cu[s]:self.cu[s + 1]] = torch.einsum("tkgl,kld->tkgd", w, v.abs()).reshape(n, self.H, self.hd)
        return out.view(self.rows, -1), mag.view(self.rows, -1)

    def check(self, got, q, window=0, scale=None):
        want, mag = self.wanted(q, window, scale)
        err = (got[:self.rows].double().cpu() - want).abs()
        allowed = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mag + 1e-30
        assert torch.isfinite(got[:self.rows]).all()
        worst = (err / allowed).max().item()
        assert worst <= 1.0, f"off by {worst:.2f} of what is allowed"


def tables(n, rot, theta=10000.0):
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return torch.cos(a).float().to(DEV), torch.sin(a).float().to(DEV)


def turned(x, pos, cos, sin, rot, inter):
    """x [T, heads, hd] float64, rotated."""
    c, s = cos.double().cpu()[pos][:, None], sin.double().cpu()[pos][:, None]
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    lo, hi = a * c - b * s, a * s + b * c
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = lo, hi
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = lo, hi
    return y


STORES = [   # q_lens, past, H, KV, hd, rot, interleaved
    ([1], [0], 4, 2, 16, 16, False),
    ([1, 1, 1], [63, 64, 129], 6, 3, 48, 48, True),
    ([1] * 9, [5 + 31 * i for i in range(9)], 8, 1, 128, 128, False),
    ([1, 4, 2], [62, 127, 0], 32, 8, 64, 64, False),
    ([3, 5], [61, 1], 4, 2, 32, 10, False),                # a rotated width that is no whole number of pieces
    ([130, 70], [0, 61], 4, 2, 64, 64, False),
    ([64, 64, 65], [0, 64, 63], 3, 3, 16, 8, True),
    ([200], [3], 8, 2, 80, 64, False),
    ([129, 1, 17], [2, 700, 30], 5, 1, 256, 256, False),
    ([300], [1], 2, 1, 32, 6, True),
    ([1] * 140, [(37 * i) % 200 for i in range(140)], 4, 2, 64, 32, False),      # many rows, each of another sequence
    # from 512 rows on another kernel, with every offset in a page and a word
    ([600], [0], 4, 2, 64, 64, False),
    ([130, 70, 400], [1, 62, 3], 8, 2, 128, 128, False),
    ([64, 64, 65, 3, 500], [0, 64, 63, 6, 1], 3, 3, 16, 8, True),
    ([513], [2], 5, 1, 256, 256, False),
    ([300, 300], [61, 7], 2, 1, 32, 6, True),
    ([600], [3], 9, 2, 80, 64, False),
    ([700], [64], 6, 3, 48, 48, False),
    ([1] * 530, [(37 * i) % 200 for i in range(530)], 4, 2, 64, 32, False),
    ([1, 5, 2] * 70, [(41 * i) % 130 for i in range(210)], 4, 1, 32, 32, True),
]


@pytest.mark.parametrize("q_lens,past,H,KV,hd,rot,inter", STORES)
def test_store(q_lens, past, H, KV, hd, rot, inter):
    s = Step(q_lens, past, H, KV, hd, units=3, unit=1, seed=hd + rot, extra_rows=2, pad_cols=8)
    cos, sin = tables(max(p + q for p, q in zip(past, q_lens)), rot)
    before = s.storage.clone()
    q = s.store(rot=rot, inter=inter, cos=cos, sin=sin)
    x = s.qkv.double().cpu().view(s.rows, H + 2 * KV, hd)
    y = turned(x[:, :H + KV], s.pos, cos, sin, rot, inter)
    big = y[:, :H].abs().amax(-1, keepdim=True)
    err = (q.double().cpu().view(s.rows, H, hd) - y[:, :H]).abs()
    assert (err <= 2.0 ** -8 * y[:, :H].abs() + 2.0 ** -22 * big).all()
    kp, vp, kso, vso = places(hd)
    touched = torch.zeros(s.storage.numel(), dtype=torch.bool)
    for i in range(len(q_lens)):
        k, v, ks, vs = unpack(s.storage, s.off, s.stride, s.pages[i], KV, hd)
        rows = slice(s.cu[i], s.cu[i + 1])
        at = torch.as_tensor(s.pos[rows])
        pg, tok = at // PAGE, at % PAGE
        for got, sc, want in ((k, ks, y[rows, H:H + KV]), (v, vs, x[rows, H + KV:])):
            got, sc = got[pg, :, tok], sc[pg, :, tok].double()             # [rows, KV, hd], [rows, KV]
            power = torch.exp2(sc - 127)[..., None]
            big = want.abs().amax(-1, keepdim=True)
            assert (got.isfinite()).all()
            assert (big <= 448 * power * (1 + 2.0 ** -22)).all() and (big * (1 + 2.0 ** -22) > 224 * power).all(), "not the least power of two"
            assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * power) + 2.0 ** -22 * big).all()
        # values are not rotated: their bits are what one rounding gives
        bits = (x[rows, H + KV:] / torch.exp2(vs[pg, :, tok].double() - 127)[..., None]).float().to(torch.float8_e4m3fn).double()
        assert torch.equal(bits * torch.exp2(vs[pg, :, tok].double() - 127)[..., None], v[pg, :, tok])
        base = torch.as_tensor(s.pages[i])[pg] * s.stride + s.off
        for h in range(KV):
            b = (base + h * 128 * (hd + 1))[:, None]
            for o in (kp[tok], vp[tok], kso[tok][:, None], vso[tok][:, None]):
                touched[(b + o).view(-1)] = True
    same = s.storage.cpu() == before.cpu()
    assert same[~touched].all(), "bytes of other tokens were written"


@pytest.mark.parametrize("q_lens", [[70, 90], [400, 190]])
def test_store_in_place_and_queries_only(q_lens):
    s = Step(q_lens, [10, 0], 8, 2, 64, seed=3)
    cos, sin = tables(500, 64)
    q = s.store(cos=cos, sin=sin)
    pages = s.storage.clone()
    kv = s.qkv[:, 8 * 64:].clone()
    s.store(q_out=s.qkv[:, :8 * 64], cos=cos, sin=sin)       # into their own place
    assert torch.equal(s.qkv[:, :8 * 64], q) and torch.equal(s.qkv[:, 8 * 64:], kv) and torch.equal(s.storage, pages)
    s2 = Step(q_lens, [10, 0], 8, 2, 64, seed=3)
    before = s2.storage.clone()
    q2 = torch.empty_like(q)
    _ops().rope_kv_q8(s2.qkv, q2, 8, 2, 64, 64, False, cos, sin, i32(s2.pos), None, None, None, None, 0, write_kv=False)
    assert torch.equal(q2, q) and torch.equal(s2.storage, before)


@pytest.mark.parametrize("runs", [1, 2, 4, 5, 9])
@pytest.mark.parametrize("q_lens,hd,rot,inter,write", [([1, 3, 1], 64, 64, False, True), ([90], 48, 32, True, True), ([40, 2], 80, 64, False, True),
                                                       ([300, 250], 128, 128, False, True), ([7], 256, 256, False, False), ([5], 32, 0, False, True)])
def test_store_of_rows_that_a_product_left_unsummed(runs, q_lens, hd, rot, inter, write):
    """Planes whose sum in their order is exactly the row (in any other order it is not): the same bits as from the row."""
    H, KV = 6, 2
    s = Step(q_lens, [60] * len(q_lens), H, KV, hd, units=2, unit=1, seed=runs)
    cos, sin = tables(700, rot) if rot else (None, None)
    kw = dict(rot=rot, inter=inter, cos=cos, sin=sin, write_kv=write)
    before = s.storage.clone()
    q = s.store(**kw)
    kept = s.storage.clone()
    s.storage.copy_(before)
    rows = s.qkv.float()
    width = rows.shape[1] + 8                                   # columns that are nobody's
    planes = torch.full((runs, s.rows, width), math.nan, device=DEV)
    planes[:, :, :rows.shape[1]] = 0.0
    if runs == 1:
        planes[0, :, :rows.shape[1]] = rows
    else:                                                       # 2^30 swallows what is added before it goes again
        planes[0, :, :rows.shape[1]], planes[runs - 1, :, :rows.shape[1]] = rows / 2, rows / 2
        if runs >= 4:
            planes[0, :, :rows.shape[1]], planes[1, :, :rows.shape[1]], planes[2, :, :rows.shape[1]] = 2.0 ** 30, -2.0 ** 30, rows / 2
    from dlgo_amd.kernels.ops import UnsummedRows
    s.qkv.fill_(math.nan)
    assert torch.equal(s.store(unsummed=UnsummedRows(planes.view(-1), runs, s.rows, width), **kw), q)
    assert torch.equal(s.storage, kept)
    with pytest.raises(_ops().KernelError, match="unsummed"):
        s.store(unsummed=UnsummedRows(planes.view(-1), runs, s.rows + 1, width), **kw)


@pytest.mark.parametrize("rows", [3, 150, 520])
def test_store_of_zeros_tiny_huge_and_what_is_not_finite(rows):
    H, KV, hd = 2, 2, 32
    s = Step([rows], [0], H, KV, hd, seed=11)
    x = s.qkv.float().view(rows, H + 2 * KV, hd)
    x[0, H:] = 0.0                                   # a token of zeros
    x[1, H] = 1e-39                                  # below float32's normal numbers
    x[1, H + 1, :] = 3e38
    x[1, H + KV, 0] = -448.0
    x[1, H + KV, 1:] = 447.0
    x[2, H, 5] = math.inf                            # a key that is not finite, and a value of the other head
    x[2, H + KV + 1, 7] = math.nan
    s.qkv.copy_(x.view(rows, -1).bfloat16())
    s.store(rot=0)
    k, v, ks, vs = unpack(s.storage, s.off, s.stride, s.pages[0], KV, hd)
    raw = s.storage.cpu()
    kp, vp, _, _ = places(hd)
    assert (k[0, :, 0] == 0).all() and (v[0, :, 0] == 0).all()
    want = s.qkv.double().cpu().view(rows, H + 2 * KV, hd)[1]
    assert ks[0, 0, 1] == 1 and ((k[0, 0, 1] - want[H]).abs() <= 2.0 ** -10 * 2.0 ** -126).all()
    assert ((k[0, 1, 1] - want[H + 1]).abs() <= 2.0 ** -4 * want[H + 1]).all()
    assert vs[0, 0, 1] == 127 and v[0, 0, 1, 0] == -448.0 and (v[0, 0, 1, 1:] == 448.0).all()
    # the token is marked in its keys' scale, in both heads here, and its bytes are zeros
    for h in range(KV):
        assert ks[0, h, 2] == 255 and vs[0, h, 2] == 127
        b = s.pages[0][0] * s.stride + s.off + h * 128 * (hd + 1)
        assert (raw[b + kp[2]] == 0).all() and (raw[b + vp[2]] == 0).all()


def test_store_writes_nothing_where_there_is_no_page():
    for rows in (5, 140, 600):
        s = Step([rows, 7], [0, 0], 4, 2, 64, seed=rows)
        table = s.table.copy()
        s.table[s.slots[0], 0] = -1                       # a hole
        s.table[s.slots[1], 0] = s.n_pages + 3            # a page that the cache does not hold
        before = s.storage.clone()
        s.store(rot=0)
        inside = torch.zeros(s.n_pages, dtype=torch.bool)
        inside[s.pages[0][1:]] = True
        changed = (s.storage != before).view(s.n_pages, -1).any(-1).cpu()
        assert not (changed & ~inside).any()
        s.table = table
        s.slots[0] = 10 ** 6                              # a slot that the table does not have
        s.slots[1] = -1
        before = s.storage.clone()
        s.store(rot=0)
        assert torch.equal(before, s.storage)


ATTENDS = [   # q_lens, past, H, KV, hd, window
    ([1], [0], 4, 2, 16, 0),
    ([1, 1, 1], [62, 63, 64], 4, 2, 32, 0),
    ([1, 1], [400, 3], 6, 3, 48, 0),
    ([1, 1, 1], [127, 700, 2300], 32, 8, 64, 0),
    ([1] * 5, [1, 100, 1000, 1900, 64], 8, 1, 80, 0),
    ([1, 1], [511, 3000], 32, 8, 128, 0),
    ([1, 1], [5, 1300], 8, 4, 256, 0),
    ([1, 1], [700, 90], 40, 1, 64, 0),                    # more heads than 16 columns
    ([1, 1], [300, 65], 100, 2, 16, 0),                   # 50 heads a group
    ([1, 1, 1], [10, 64, 1000], 8, 2, 64, 33),            # windows
    ([1, 1], [1000, 4095], 4, 4, 128, 1),
    ([3, 0, 1, 5], [60, 10, 0, 500], 8, 2, 64, 0),        # drafted tokens; a sequence that brings none
    ([6, 2], [1200, 61], 32, 8, 64, 0),
    ([4, 4], [126, 1], 28, 4, 128, 0),
    ([2, 5], [300, 60], 6, 2, 256, 40),
    ([9, 7], [64, 250], 14, 2, 48, 100),
    ([65], [0], 4, 2, 64, 0),                             # prompts
    ([200, 17, 1], [0, 130, 777], 32, 8, 64, 0),
    ([333], [77], 6, 2, 128, 0),                          # a group of three
    ([129, 64], [1, 63], 8, 8, 16, 0),
    ([150], [40], 8, 2, 256, 0),
    ([70, 260], [500, 0], 10, 2, 80, 0),
    ([90, 130], [200, 0], 8, 2, 32, 50),
    ([257], [300], 12, 4, 64, 64),
    ([40], [0], 100, 1, 64, 0),
]


@pytest.mark.parametrize("q_lens,past,H,KV,hd,window", ATTENDS)
def test_attention(q_lens, past, H, KV, hd, window):
    s = Step(q_lens, past, H, KV, hd, units=2, unit=1, seed=hd + H)
    s.fill()
    wide = torch.randn(s.rows + 2, H * hd + 16, generator=s.gen).bfloat16().to(DEV)      # rows further apart than they are long
    q = wide[:, :H * hd]
    out_wide = torch.full_like(wide, 7.0)
    s.attend(q, window, out=out_wide[:, :H * hd])
    s.check(out_wide[:, :H * hd], q, window)
    assert (out_wide[s.rows:] == 7.0).all() and (out_wide[:, H * hd:] == 7.0).all(), "rows or columns that are nobody's were written"
    # the same step as a recorded launch sees it, with bounds for longer sequences: another dealing of the pages
    far = s.attend(q.contiguous(), window, bound_len=s.table.shape[1] * PAGE + 5000)
    s.check(far, q, window)
    # tables by sequence instead of by slot
    by_seq = s.attend(q.contiguous(), window, slots=None, table=i32(s.table[s.slots]))
    assert torch.equal(by_seq[:s.rows], out_wide[:s.rows, :H * hd])


@pytest.mark.parametrize("q_lens,past,H,KV,hd,window", [
    ([17], [3000], 32, 8, 64, 0), ([40, 70], [2000, 5], 8, 2, 128, 0), ([130], [1500], 8, 4, 48, 0), ([90, 1, 0, 20], [900, 1800, 40, 700], 10, 2, 80, 0),
    ([70], [4000], 6, 3, 32, 1200), ([66], [1100], 2, 2, 256, 0), ([35], [2500], 24, 3, 16, 0), ([33, 33], [1000, 3300], 100, 1, 64, 0)])
def test_a_few_tiles_behind_a_long_past(q_lens, past, H, KV, hd, window):
    """A tile's pages dealt to several blocks, evenly and with less for the last; tiles and sequences that are not dealt beside
    them; launches sized for more rows and for longer sequences."""
    s = Step(q_lens, past, H, KV, hd, units=2, unit=1, seed=hd)
    s.fill()
    q = torch.randn(s.rows, H * hd, generator=s.gen).bfloat16().to(DEV)
    for kw in (dict(), dict(bound_len=64 * s.table.shape[1] + 900), dict(bound_len=64 * s.table.shape[1], bound_q=min(s.rows, max(q_lens) + 30))):
        out = s.attend(q, window, **kw)
        s.check(out, q, window)
    big = s.attend(q, window, scratch=lambda n: torch.full((n + 8,), math.nan, device=DEV))      # what is in the scratch before
    assert torch.equal(big, s.attend(q, window))


def test_attention_with_a_table_for_far_longer_sequences():
    """Pages of each sequence dealt to many blocks or to one, whatever the launch was sized for."""
    for width, H, KV, hd in ((600, 8, 2, 64), (1500, 4, 1, 128)):
        s = Step([1, 1, 1, 3], [5, 64 * 9, 64 * 70 + 1, 200], H, KV, hd, seed=width, width=width)
        s.fill()
        q = torch.randn(s.rows, H * hd, generator=s.gen).bfloat16().to(DEV)
        for bound in (64 * 71, 64 * 300, 64 * width):
            s.check(s.attend(q, bound_len=bound), q)


UNEQUAL = [   # sequences, rows each, the longest pasts, H, KV, hd, window
    (150, (1,), [1300, 40], 3, 1, 16, 0),
    (130, (0, 1, 2), [700, 650, 5], 6, 1, 32, 90),
    (20, (1,), [9000, 300], 32, 8, 64, 0),
    (40, (2, 1), [2100, 100], 8, 4, 48, 0),
    (17, (1,), [1500, 900], 160, 4, 64, 0),               # two blocks for a group's heads
    (70, (1,), [7000, 130], 8, 8, 16, 0),                 # the sequences alone fill the chip, one is far longer
    (33, (3, 1), [500, 2500], 8, 4, 256, 0),
]


@pytest.mark.parametrize("n,rows,longest,H,KV,hd,window", UNEQUAL)
def test_attention_over_many_unequal_sequences(n, rows, longest, H, KV, hd, window):
    rng = np.random.default_rng(n + hd)
    past = rng.integers(0, 130, size=n).tolist()
    for i, p in zip(rng.permutation(n), longest):
        past[i] = p
    s = Step([rows[i % len(rows)] for i in range(n)], past, H, KV, hd, seed=n)
    s.fill()
    q = torch.randn(s.rows, H * hd, generator=s.gen).bfloat16().to(DEV)
    s.check(s.attend(q, window), q, window)
    # bounds for longer sequences and more rows
    s.check(s.attend(q, window, bound_len=s.table.shape[1] * PAGE, bound_q=max(rows) + 1), q, window)


@pytest.mark.parametrize("rows,n,window", [(1, 3, 10), (1, 3, 0), (1, 40, 10), (40, 2, 10)])
def test_positions_behind_the_table(rows, n, window):
    """Nothing is read past the table's end: with a window such a row sees nothing and gets zeros.  (Without one it sees what
    the table holds, places that nothing was stored in among it, so its numbers are anybody's.)"""
    s = Step([rows] * n, [70] * n, 8, 4, 64, seed=rows)
    s.fill()
    q = torch.randn(s.rows, 8 * 64, generator=s.gen).bfloat16().to(DEV)
    past = list(s.past)
    s.past = [p if i % 2 else 64 * s.table.shape[1] + 500 for i, p in enumerate(past)]
    out = s.attend(q, window, bound_len=20000)
    s.past = past
    out = out.view(n, rows, -1)
    for i in range(0, n, 2):
        assert not window or (out[i] == 0).all()
    want, mag = s.wanted(q, window)
    for i in range(1, n, 2):
        off = (out[i].double().cpu() - want.view(n, rows, -1)[i]).abs()
        assert (off <= 2.0 ** -8 * want.view(n, rows, -1)[i].abs() + (2.0 ** -8 + 2.0 ** -10) * mag.view(n, rows, -1)[i] + 1e-30).all()


def test_attention_scales_of_either_sign_and_peaked_scores():
    for q_lens, hd in (([1, 2], 64), ([80], 64), ([3], 128)):
        s = Step(q_lens, [300] * len(q_lens), 8, 2, hd, seed=5)
        s.fill()
        q = torch.randn(s.rows, 8 * hd, generator=s.gen).bfloat16().to(DEV)
        for scale in (-0.1, 0.02, 0.25):
            s.check(s.attend(q, scale=scale), q, scale=scale)
        with pytest.raises(_ops().KernelError, match="scale"):
            s.attend(q, scale=0.0)
        with pytest.raises(_ops().KernelError, match="scale"):
            s.attend(q, scale=math.inf)


@pytest.mark.parametrize("q_lens", [[1, 1], [4, 1], [90, 1]])
def test_what_a_row_must_not_see_does_not_reach_it(q_lens):
    """A token that is not finite, later than a row or before its window, and bytes of NaN behind the sequence."""
    hd, H, KV = 64, 8, 2
    s = Step(q_lens, [100, 70], H, KV, hd, seed=9)
    s.fill()
    q = torch.randn(s.rows, H * hd, generator=s.gen).bfloat16().to(DEV)
    clean = s.attend(q)
    kp, vp, ks, vs = places(hd)
    for i in range(2):          # everything behind the sequences: keys, values and scales of all ones (NaN)
        n = s.past[i] + q_lens[i]
        for tok in range(n % PAGE, PAGE if n % PAGE else 0):
            for h in range(KV):
                b = s.pages[i][-1] * s.stride + s.off + h * 128 * (hd + 1)
                for o in (kp[tok], vp[tok], ks[tok:tok + 1], vs[tok:tok + 1]):
                    s.storage[(b + o).to(DEV)] = 255
    assert torch.equal(s.attend(q), clean)
    # the last token of the first sequence is not finite in head 1: its own row is NaN there, the others are as before
    last = s.past[0] + q_lens[0] - 1
    b = s.pages[0][last // PAGE] * s.stride + s.off + 128 * (hd + 1)
    s.storage[b + ks[last % PAGE]] = 255
    for o in (kp[last % PAGE], vp[last % PAGE]):
        s.storage[(b + o).to(DEV)] = 0
    got = s.attend(q).view(s.rows, H, hd)
    r = q_lens[0] - 1
    assert got[r, H // KV:].isnan().all() and torch.equal(got[r, :H // KV], clean.view(s.rows, H, hd)[r, :H // KV])
    keep = [i for i in range(s.rows) if i != r]
    assert torch.equal(got[keep], clean.view(s.rows, H, hd)[keep])
    # a token before the window
    s.storage[b + ks[last % PAGE]] = 127
    windowed = s.attend(q, window=20)
    tok = s.past[0] - 30
    b = s.pages[0][tok // PAGE] * s.stride + s.off
    s.storage[b + ks[tok % PAGE]] = 255
    assert torch.equal(s.attend(q, window=20), windowed)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 1, 2], [70, 80, 1]])
def test_pages_that_are_missing_count_nothing(q_lens):
    hd, H, KV = 64, 4, 2
    s = Step(q_lens, [200, 10, 70], H, KV, hd, seed=21)
    s.fill()
    q = torch.randn(s.rows, H * hd, generator=s.gen).bfloat16().to(DEV)
    clean = s.attend(q)
    table = s.table.copy()
    table[s.slots[0], :] = [-1, s.n_pages] * (table.shape[1] // 2) + [-5] * (table.shape[1] % 2)      # no page at all
    got = s.attend(q, table=i32(table))
    assert (got[:q_lens[0]] == 0).all() and torch.equal(got[q_lens[0]:], clean[q_lens[0]:])
    got = s.attend(q, slots=i32([-1, s.slots[1], 99]))
    assert (got[:q_lens[0]] == 7).all() and (got[s.cu[2]:] == 7).all()       # no such slot: not a row of a sequence
    assert torch.equal(got[s.cu[1]:s.cu[2]], clean[s.cu[1]:s.cu[2]])


def test_the_same_call_gives_the_same_bits_and_replays():
    """Also captured into a graph, replayed with other work between, with sequences that have grown since."""
    hd, H, KV = 64, 32, 8
    s = Step([1] * 6, [70, 800, 64, 2000, 5, 1023], H, KV, hd, seed=2, width=40)
    s.fill()
    cos, sin = tables(2600, hd)
    pos, seq, slots, table = s.arrays()
    cu, start = i32(s.cu), i32(s.past)
    q, out = torch.empty(6, H * hd, dtype=torch.bfloat16, device=DEV), torch.empty(6, H * hd, dtype=torch.bfloat16, device=DEV)
    part = {}

    def scratch(n):
        if "p" not in part:
            part["p"] = torch.empty(n, dtype=torch.float32, device=DEV)
        return part["p"]

    def step():
        ops = _ops()
        ops.rope_kv_q8(s.qkv, q, H, KV, hd, hd, False, cos, sin, pos, seq, slots, table, s.cache, s.stride)
        ops.attention_q8(q, out, H, KV, hd, cu, start, slots, table, s.cache, s.stride, 1, 40 * PAGE, scratch=scratch)
    step()
    first = out.clone()
    step()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        s.qkv.normal_()
        if k == 2:                       # shorter sequences: other pages, another dealing
            pos.copy_(i32([3, 100, 63, 64, 4, 500]))
            start.copy_(pos)
        out.zero_()
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        step()
        assert torch.equal(out, replayed)


def test_on_another_stream():
    s = Step([70, 1], [30, 500], 8, 2, 64, seed=4)
    s.fill()
    q = torch.randn(s.rows, 512, generator=s.gen).bfloat16().to(DEV)
    want = s.attend(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = s.attend(q)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    ops = _ops()
    s = Step([1, 2], [70, 3], 4, 2, 64, seed=1)
    q = torch.zeros(3, 256, dtype=torch.bfloat16, device=DEV)
    pos, seq, slots, table = s.arrays()

    def store(qkv=s.qkv, q_out=q, H=4, KV=2, hd=64, rot=0, cos=None, sin=None, pos=pos, seq=seq, slots=slots, table=table,
              cache=s.cache, stride=s.stride):
        ops.rope_kv_q8(qkv, q_out, H, KV, hd, rot, False, cos, sin, pos, seq, slots, table, cache, stride)

    def attend(q=q, out=q, H=4, KV=2, hd=64, cu=i32(s.cu), start=i32(s.past), slots=slots, table=table, cache=s.cache,
               stride=s.stride, mq=2, mk=80, **kw):
        ops.attention_q8(q, out, H, KV, hd, cu, start, slots, table, cache, stride, mq, mk, **kw)
    bad_store = [dict(qkv=s.qkv.float()), dict(q_out=q[:2]), dict(q_out=q.float()), dict(hd=40), dict(hd=512), dict(KV=0), dict(KV=3),
                 dict(pos=pos[:2]), dict(pos=pos.long()), dict(seq=seq[:1]), dict(table=table.t()), dict(table=table[0]),
                 dict(cache=s.cache.view(torch.int8)), dict(cache=s.cache[:100]), dict(cache=s.cache[1:]), dict(stride=s.stride - 16),
                 dict(stride=s.stride + 8), dict(rot=3), dict(rot=66), dict(cos=torch.zeros(80, 32, device=DEV)),
                 dict(rot=64, cos=torch.zeros(80, 16, device=DEV), sin=torch.zeros(80, 16, device=DEV)), dict(pos=pos.cpu()), dict(cache=s.cache.cpu())]
    for kw in bad_store:
        with pytest.raises(ops.KernelError):
            store(**kw)
    bad_attend = [dict(q=q.float()), dict(out=q.float()), dict(H=3), dict(KV=3), dict(hd=40), dict(cu=i32([0, 3])), dict(start=i32([1])),
                  dict(cu=i32(s.cu).long()), dict(slots=i32([1])), dict(slots=None, table=table[:1]), dict(table=table.t()), dict(mq=-1),
                  dict(mk=-1), dict(window=-2), dict(cache=s.cache[:50]), dict(stride=16), dict(stride=s.stride + 4), dict(cache=s.cache[8:]),
                  dict(q=torch.zeros(3, 258, dtype=torch.bfloat16, device=DEV)[:, :256]), dict(q=torch.zeros(257, 3, dtype=torch.bfloat16, device=DEV).t()[:, :256])]
    for kw in bad_attend:
        with pytest.raises(ops.KernelError):
            attend(**kw)
    for scratch in (lambda n: torch.empty(n - 1, device=DEV), lambda n: torch.empty(n, dtype=torch.uint8, device=DEV), lambda n: torch.empty(n)):
        with pytest.raises(ops.KernelError):
            attend(mk=4096, table=i32(np.zeros((5, 64))), scratch=scratch)
    # nothing to do is no error
    store(qkv=s.qkv[:0], q_out=q[:0], pos=pos[:0], seq=seq[:0])
    attend(q=q[:0], out=q[:0])
    attend(cu=i32([0]), start=i32([]), slots=i32([]))
    attend(mq=0)


FUSED = [   # past, H, KV, hd, window: single tokens
    ([0], 4, 2, 32, 0), ([5, 63, 64, 700], 32, 8, 64, 0), ([127, 2300], 8, 1, 32, 0), ([1, 15, 16, 17, 31, 48, 130], 6, 3, 128, 0),
    ([400, 3], 16, 1, 64, 0), ([500, 64], 8, 4, 32, 0), ([1000, 10, 4095], 8, 2, 64, 70), ([90] * 40, 4, 2, 64, 0), ([64 * i for i in range(20)], 16, 8, 128, 0),
    ([20000], 8, 2, 32, 0),
]


@pytest.mark.parametrize("past,H,KV,hd,window", FUSED)
def test_single_tokens_rotated_and_stored_on_the_way(past, H, KV, hd, window):
    """The same bits, in the cache and in the result, as from the two kernels; a token whose page is missing, one that is not
    finite and what lies around them as there."""
    ops = _ops()
    n = len(past)
    assert ops.attention_q8_fuses_rotation(hd, H // KV, 1, hd, False, n, KV) == (n * KV * max(hd, 64) <= 128 * ops.compute_units())
    s = Step([1] * n, past, H, KV, hd, units=2, unit=1, seed=hd, pad_cols=8)
    s.fill()
    cos, sin = tables(max(past) + 1, hd)
    if n > 3:
        s.qkv[1, H * hd + 3] = math.inf                         # a key, and another token's value
        s.qkv[2, -1] = math.nan
        s.table[s.slots[3], past[3] // PAGE] = -1               # nowhere to store it
    before = s.storage.clone()
    q = s.store(cos=cos, sin=sin)
    for bound in (None, 64 * s.table.shape[1] + 3000):
        want = s.attend(q, window, bound_len=bound)
        kept = s.storage.clone()
        s.storage.copy_(before)
        out = torch.full_like(want, 7.0)
        got = s.attend(s.qkv, window, out=out, bound_len=bound, rotation=(cos, sin))
        assert torch.equal(s.storage, kept)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    if n > 3:
        rows = want.view(n, KV, -1).isnan().all(-1).cpu()
        assert rows[1, 0] and not rows[1, 1:].any() and rows[2, KV - 1] and not rows[2, :KV - 1].any() and not rows[0].any()


def test_refusals_of_rows_to_be_rotated():
    ops = _ops()
    s = Step([1, 1], [3, 70], 4, 2, 64)
    cos, sin = tables(100, 64)
    s.attend(s.qkv, out=torch.empty(2, 256, dtype=torch.bfloat16, device=DEV), rotation=(cos, sin))
    for kw in (dict(rotation=(cos, sin), bound_q=2), dict(rotation=(cos[:, :16], sin[:, :16])), dict(rotation=(cos, sin[:50])), dict(rotation=(cos.double(), sin)),
               dict(rotation=(cos.cpu(), sin.cpu()))):
        with pytest.raises(ops.KernelError):
            s.attend(s.qkv, out=torch.empty(2, 256, dtype=torch.bfloat16, device=DEV), **kw)
    with pytest.raises(ops.KernelError, match="single tokens"):
        s.attend(s.qkv[:, :256], out=torch.empty(2, 256, dtype=torch.bfloat16, device=DEV), rotation=(cos, sin))
    odd = Step([1], [3], 4, 2, 48)
    with pytest.raises(ops.KernelError, match="steps of 32"):
        odd.attend(odd.qkv, out=torch.empty(1, 192, dtype=torch.bfloat16, device=DEV), rotation=tables(100, 48))
    many = Step([1], [3], 34, 2, 64)
    with pytest.raises(ops.KernelError, match="up to 16 heads"):
        many.attend(many.qkv, out=torch.empty(1, 34 * 64, dtype=torch.bfloat16, device=DEV), rotation=(cos, sin))
