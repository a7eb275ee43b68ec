"""Heads of 96 over the 8-bit cache: six pieces of 16, so that of the two loads that bring 16 keys the second is half full, also
where the kernel rotates and stores single tokens by itself.  The checks and tolerances are those of the other sizes."""
import pytest
import torch

from test_q8_gpu import (DEV, PAGE, Step, test_a_few_tiles_behind_a_long_past as few_tiles, test_attention as attention,
                         test_attention_over_many_unequal_sequences as unequal, test_single_tokens_rotated_and_stored_on_the_way as fused, tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("past,H,KV,window", [
    ([0], 4, 2, 0), ([63], 16, 1, 0), ([5, 63, 64, 700], 12, 4, 0), ([127, 2300], 8, 1, 0), ([1, 15, 16, 17, 31, 48, 130], 6, 3, 0),
    ([1000, 10, 4095], 8, 2, 70), ([64 * i for i in range(20)], 16, 4, 0), ([20000], 8, 2, 0)])
def test_single_tokens_rotated_and_stored_on_the_way(past, H, KV, window):
    fused(past, H, KV, 96, window)


@pytest.mark.parametrize("q_lens,past,H,KV,window", [
    ([1], [0], 4, 2, 0), ([1, 1, 1], [127, 700, 2300], 32, 8, 0), ([1, 1], [300, 65], 40, 2, 0), ([3, 0, 1, 5], [60, 10, 0, 500], 8, 2, 0),
    ([6, 2], [1200, 61], 6, 2, 45), ([65], [0], 4, 2, 0), ([200, 17, 1], [0, 130, 777], 24, 8, 0), ([257], [300], 12, 4, 64)])
def test_attention(q_lens, past, H, KV, window):
    attention(q_lens, past, H, KV, 96, window)


@pytest.mark.parametrize("q_lens,past,H,KV,window", [([17], [3000], 32, 8, 0), ([40, 70], [2000, 5], 6, 2, 0), ([70], [4000], 6, 3, 1200)])
def test_a_few_tiles_behind_a_long_past(q_lens, past, H, KV, window):
    few_tiles(q_lens, past, H, KV, 96, window)


def test_many_unequal_sequences():
    unequal(70, (1, 3), [3000, 130], 8, 2, 96, 0)


@pytest.mark.parametrize("n", [1, 8, 600])
def test_what_is_stored_is_what_is_read(n):
    """One head, values that name their token and element: every place of a page comes back from where it went."""
    s = Step([n], [0], 1, 1, 96, seed=n)
    s.qkv[:] = 0
    s.qkv[:, 192:] = torch.randint(-14, 15, (n, 96), generator=s.gen).to(DEV)       # whole numbers that four bits hold, twice some
    cos, sin = tables(n + PAGE, 96)
    q = s.store(cos=cos, sin=sin)
    want, _ = s.wanted(q)                                # all scores equal: the running mean of the values
    mean = s.qkv[:, 192:].double().cpu().cumsum(0) / torch.arange(1, n + 1)[:, None]
    assert torch.allclose(want, mean, rtol=1e-12, atol=1e-12)
    s.check(s.attend(q), q)
