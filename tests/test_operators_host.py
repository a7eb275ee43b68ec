"""What the launchers of the 8-bit cache's kernels and of the verification refuse before they touch a device, and how they
size their scratch.  These need the compiler (the libraries are built at first use) but no GPU; no call here launches."""
import ctypes

import pytest

from dlgo_amd.kernels import build

P, NONE, LL = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), ctypes.c_longlong


def lib_of(module, **defines):
    lib = build.load(module, tuple(defines.items()))
    for name in ("dlgo_rope_kv_q8", "dlgo_attention_q8", "dlgo_verify_drafts"):
        if hasattr(lib, name):
            getattr(lib, name).restype = ctypes.c_char_p
    for name in ("dlgo_attention_q8_scratch", "dlgo_verify_drafts_scratch"):
        if hasattr(lib, name):
            getattr(lib, name).restype = LL
    return lib


def rope(**kw):
    a = dict(qkv=P, ld=384, q_out=P, ldq=256, t=3, H=4, KV=1, hd=64, rot=64, inter=0, cos=P, sin=P, table=100, pos=P, tok_seq=P, slots=P, n_seq=3, pages=P,
             n_slots=3, max_pages=4, cache=P, stride=LL(128 * 65), n_pages=9, write=1, part=NONE, runs=0, plane=LL(0), part_ld=0, stream=NONE)
    a.update(kw)
    return lib_of("kv_q8").dlgo_rope_kv_q8(*a.values())


@pytest.mark.parametrize("kw,why", [
    (dict(hd=24), b"head sizes"), (dict(hd=272), b"head sizes"), (dict(t=-1), b"rows"), (dict(rot=63), b"even"), (dict(rot=66), b"at most"),
    (dict(ld=383), b"shorter"), (dict(ldq=255), b"shorter"), (dict(sin=NONE), b"together"), (dict(table=0), b"empty"),
    (dict(cache=NONE), b"missing"), (dict(pages=NONE), b"missing"), (dict(slots=NONE), b"missing"), (dict(tok_seq=NONE), b"missing"), (dict(n_pages=0), b"missing"),
    (dict(KV=0), b"missing"), (dict(stride=LL(128 * 65 - 16)), b"bytes apart"), (dict(stride=LL(128 * 65 + 8)), b"bytes apart"),
    (dict(cache=ctypes.c_void_p((1 << 20) + 4)), b"bytes apart"), (dict(t=2 ** 31 - 1, H=4000, ld=4002 * 64, ldq=4000 * 64), b"too many"),
    (dict(part=P, runs=0, plane=LL(3 * 384), part_ld=384), b"unsummed"), (dict(part=P, runs=2, plane=LL(3 * 384 - 4), part_ld=384), b"unsummed"),
    (dict(part=P, runs=2, plane=LL(3 * 384), part_ld=380), b"unsummed"), (dict(part=P, runs=2, plane=LL(3 * 384), part_ld=384, rot=10), b"unsummed"),
])
def test_the_store_refuses(kw, why):
    assert why in rope(**kw)


def test_a_store_of_no_rows_is_nothing():
    assert rope(t=0) is None


def attend(hd=64, **kw):
    a = dict(q=P, ldq=2048, out=P, ldo=2048, rows=2, n_seq=2, H=32, KV=8, hd=hd, cu=P, start=P, slots=P, pages=P, n_slots=4, max_pages=100, cache=P,
             stride=LL(8 * 128 * (hd + 1)), n_pages=50, max_q=1, max_kv=5000, window=0, scale=ctypes.c_float(0.1), part=P, part_n=LL(1 << 30),
             cos=NONE, sin=NONE, table=0, stream=NONE)
    a.update(kw)
    return lib_of("attention_q8", HEAD_DIM=hd).dlgo_attention_q8(*a.values())


@pytest.mark.parametrize("kw,why", [
    (dict(KV=5), b"over 5 kv heads"), (dict(H=0), b"heads"), (dict(n_seq=-1), b"heads"), (dict(H=258, KV=2, ldq=258 * 64, ldo=258 * 64), b"at most 128"),
    (dict(max_kv=0), b"bounds"), (dict(n_pages=0), b"bounds"), (dict(max_pages=0), b"bounds"), (dict(n_slots=0), b"bounds"),
    (dict(scale=ctypes.c_float(0.0)), b"scale"), (dict(scale=ctypes.c_float(float("inf"))), b"scale"), (dict(scale=ctypes.c_float(float("nan"))), b"scale"),
    (dict(ldq=2044), b"aligned"), (dict(ldo=2046), b"aligned"), (dict(ldq=2040), b"aligned"), (dict(q=ctypes.c_void_p((1 << 20) + 8)), b"aligned"),
    (dict(stride=LL(8 * 128 * 65 - 16)), b"bytes apart"), (dict(n_seq=70000), b"65535"),
    (dict(part_n=LL(10)), b"scratch"), (dict(part=NONE), b"scratch"), (dict(rows=40, max_q=20, part=NONE), b"scratch"),
    (dict(cos=P), b"rotates"), (dict(cos=P, sin=P, table=9), b"rotates"), (dict(cos=P, sin=P, table=9, ldq=48 * 64, max_q=2), b"rotates"),
    (dict(cos=P, sin=P, table=9, ldq=50 * 64, H=34, KV=2, ldo=34 * 64, stride=LL(2 * 128 * 65)), b"rotates"),
])
def test_the_attention_refuses(kw, why):
    assert why in attend(**kw)


def test_the_attention_of_nothing_and_of_another_head_size():
    assert attend(rows=0) is None and attend(n_seq=0) is None and attend(max_q=0) is None
    lib = lib_of("attention_q8", HEAD_DIM=64)
    assert lib.dlgo_attention_q8_head_dim() == 64
    assert b"built for a head size of 64" in lib.dlgo_attention_q8(P, 2048, P, 2048, 2, 2, 32, 8, 128, P, P, P, P, 4, 100, P, LL(8 * 128 * 129), 50, 1, 5000, 0,
                                                                   ctypes.c_float(0.1), P, LL(1 << 30), NONE, NONE, 0, NONE)


def test_how_the_attention_deals_pages():
    """Nothing is dealt, and no scratch needed, where sequences are short or there are enough of them; one sequence is dealt to
    what fills the chip at most, many long ones to eight blocks each at most."""
    need = lib_of("attention_q8", HEAD_DIM=64).dlgo_attention_q8_scratch
    row = 64 + 4
    assert need(1, 1, 32, 8, 1, 300, 0) == need(1, 1, 32, 8, 1, 24 * 64, 0) == 0
    assert need(1, 1, 32, 8, 1, 2304, 0) == 9 * 32 * row                    # 36 pages, a page a wave at least
    assert need(1, 1, 32, 8, 1, 131072, 0) == 64 * 32 * row                 # 64 blocks for each of 8 heads
    assert need(16, 16, 32, 8, 1, 4096, 0) == need(32, 32, 32, 8, 1, 8192, 0) == need(64, 64, 32, 8, 1, 8192, 0) == 0
    assert need(96, 16, 32, 8, 6, 4096, 0) == 96 * 4 * 32 * row             # drafts: a page takes a wave longer
    assert need(32, 32, 32, 8, 1, 131072, 0) == 32 * 8 * 32 * row
    assert need(1, 1, 32, 8, 1, 131072, 100) == 0                           # a window of two or three pages
    assert need(2048, 1, 32, 8, 2048, 2048, 0) == 0                         # a prompt fills the chip with tiles
    assert need(17, 1, 32, 8, 17, 16401, 0) == 17 * 64 * 32 * row           # one tile a head behind a long past
    assert need(17, 1, 32, 8, 17, 400, 0) == 0
    for bad in ((0, 1, 32, 8, 1, 100, 0), (1, 0, 32, 8, 1, 100, 0), (1, 1, 4, 8, 1, 100, 0), (1, 1, 32, 8, 0, 100, 0), (1, 1, 32, 8, 1, 0, 0)):
        assert need(*bad) == 0


def verify(**kw):
    a = dict(logits=P, ldl=LL(1000), tokens=P, drafts=P, ldd=LL(1000), cu=P, temperature=P, uniform=P, n=2, d=6, vocab=1000, most=4, accepted=P, token=P,
             probs=NONE, scratch=P, size=LL(1 << 30), stream=NONE)
    a.update(kw)
    return lib_of("verify").dlgo_verify_drafts(*a.values())


@pytest.mark.parametrize("kw,why", [
    (dict(n=-1), b"sizes"), (dict(d=-1), b"sizes"), (dict(vocab=0), b"sizes"), (dict(most=-1), b"sizes"), (dict(most=1025), b"1024"),
    (dict(ldl=LL(999)), b"shorter"), (dict(ldd=LL(999)), b"shorter"), (dict(scratch=NONE), b"scratch"), (dict(size=LL(100)), b"scratch"),
    (dict(scratch=ctypes.c_void_p((1 << 20) + 8)), b"scratch"), (dict(n=70000, size=LL(1 << 40)), b"too many"),
])
def test_the_verification_refuses(kw, why):
    assert why in verify(**kw)


def test_the_verification_of_nothing_and_its_scratch():
    assert verify(n=0) is None
    need = lib_of("verify").dlgo_verify_drafts_scratch
    assert need(0, 0, 1000, 0) == need(2, -1, 1000, 0) == need(2, 0, 0, 0) == 0
    assert 0 < need(2, 0, 1000, 0) < need(2, 6, 1000, 0) < need(2, 6, 1000, 1) < need(2, 6, 128256, 1)
