"""A refused step leaves the sequences as they were (no GPU: the engine's checks over a cache on the host)."""
import random

import pytest
import torch

from dlgo_amd.cache import PAGE, Cache
from dlgo_amd.engine.engine import Engine, EngineError, Entry
from dlgo_amd.parts import CacheNeed

FULL, WINDOWED = CacheNeed("kv", 1, 16), CacheNeed("kv", 2, 16, window=100)


def engine_over(cache):
    """The engine's bookkeeping without a device: what its checks read."""
    eng = object.__new__(Engine)
    eng.cache, eng.max_ctx, eng.max_step_tokens, eng.vocab, eng.steps_run, eng.graph_max_batch = cache, cache.max_ctx, 64, 10, 0, 8
    return eng


@pytest.mark.parametrize("call", ["step", "decode"])
def test_drafts_can_be_rewound_after_a_step_that_was_refused(call):
    """158 tokens and 34 drafts behind them: a token at 158 sees page 0, one at 192 does not.  The step after is refused for
    want of pages, and the drafts are still to be taken back."""
    c = Cache([[FULL], [WINDOWED]], 5 * PAGE, 5 * PAGE, torch.bfloat16, "cpu", max_slots=2, max_step_tokens=64)
    eng = engine_over(c)
    s, other = c.alloc_slot(), c.alloc_slot()
    for n in (64, 64, 30):
        c.reserve([(s, c.length(s) + n)])
        c.advance(s, n)
    c.reserve([(s, 192)])
    c.advance(s, 34, sure=158)
    c.reserve([(other, 128)])                                 # the last pages of the group without a window
    c.advance(other, 128)
    before = [dict(c.held_pages(s, g)) for g in (0, 1)]
    assert sorted(before[1]) == [0, 1, 2]
    with pytest.raises(EngineError, match="cache full"):
        eng.step([Entry(s, [1, 2], (0, 1), undecided=1)]) if call == "step" else eng.decode([s], [1])
    assert [c.held_pages(s, g) for g in (0, 1)] == before and c.length(s) == 192
    c.check_consistent()
    eng.rewind(s, 158)
    assert c.length(s) == 158 and sorted(c.held_pages(s, 1)) == [0, 1, 2]


def test_what_settling_would_free_is_counted():
    """can_reserve(settled=True) says what settle() and then can_reserve() say, over random drafting in a tight cache."""
    rng = random.Random(3)
    c = Cache([[FULL], [CacheNeed("kv", 2, 16, window=70)]], 9 * PAGE, 6 * PAGE, torch.bfloat16, "cpu", max_slots=3, max_step_tokens=64)
    slots = [c.alloc_slot() for _ in range(3)]
    refused = freed = 0
    for _ in range(3000):
        some = rng.sample(slots, rng.randint(1, 3))
        wants = [(s, c.length(s) + rng.choice([1, 2, 9, 64])) for s in some]
        before = [c.held_pages(s, 1) for s in slots]
        early = c.can_reserve(wants, settled=True)
        assert [c.held_pages(s, 1) for s in slots] == before
        c.settle(some)
        freed += [c.held_pages(s, 1) for s in slots] != before
        why = c.can_reserve(wants)
        assert early == why
        if why:
            refused += 1
            s = rng.choice(slots)
            c.free_slot(s)
            assert c.alloc_slot() == s
            continue
        c.reserve(wants)
        for s, n in wants:
            k = n - c.length(s)
            u = rng.randint(0, k)
            c.advance(s, k, n - u)
            if rng.random() < 0.5:
                c.rewind(s, n - rng.randint(0, u))
        c.check_consistent()
    assert refused > 50 and freed > 50
