"""Drafted tokens without a GPU: what a text's own repetitions propose, the loop that has them verified (with stand-ins for
the engine and the sampler), the cache that takes refused ones back, and the sizes of a cache of 8-bit keys and values."""
import random

import numpy as np
import pytest
import torch

from dlgo_amd.cache import PAGE, Cache, CacheError
from dlgo_amd.cache.cache import kv_bytes_per_token
from dlgo_amd.engine.generate import FILL_ROWS, GenerationError, LookupDrafts, fill_drafts, generate
from dlgo_amd.parts import CacheNeed
from dlgo_amd.sampling import GenerateConfig, SamplerConfig, apply_options, with_lookup_drafts, with_temperature
from test_cache_and_loop import FakeEngine, ScriptSampler


# -- proposals ---------------------------------------------------------------------
def test_lookup_of_the_last_three_then_two_tokens():
    t = LookupDrafts([1, 2, 3, 4, 5, 1, 2, 3])
    assert t.propose(2) == [4, 5] and t.propose(10) == [4, 5, 1, 2, 3] and t.propose(0) == []
    t.extend([9])
    assert t.propose(4) == []                        # (2, 3, 9) and (3, 9) stood nowhere before
    t.extend([2, 3])
    assert t.propose(1) == [9]                       # three (9, 2, 3) nowhere; two: the latest (2, 3) was followed by 9
    assert LookupDrafts([]).propose(3) == [] and LookupDrafts([7]).propose(3) == [] and LookupDrafts([7, 7]).propose(3) == []
    assert LookupDrafts([7, 7, 7]).propose(3) == [7]           # (7, 7) was followed by 7; there is no more text


def test_small_steps_are_filled_to_one_shape():
    assert fill_drafts([[], []], [3, 3], [8, 9]) == [[], []]                                     # nobody drafts: single tokens
    assert fill_drafts([[1], [], [4, 5, 6]], [3, 2, 3], [7, 8, 9]) == [[1, 7, 7], [8, 8], [4, 5, 6]]
    assert fill_drafts([[1], []], [3, 0], [7, 8]) == [[1, 7, 7], []]                             # no room, or does not draft
    n = FILL_ROWS // 8
    assert all(len(x) == 7 for x in fill_drafts([[1]] + [[]] * (n - 1), [7] * n, [0] * n))
    assert fill_drafts([[1]] + [[]] * n, [7] * (n + 1), [0] * (n + 1)) == [[1]] + [[]] * n       # too many rows


# -- the loop ------------------------------------------------------------------------
class DraftEngine(FakeEngine):
    """One row per wanted place: (slot, tokens held up to and with that place).  Keeps what every slot holds."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.text, self.rewinds = {}, []

    def _run(self, rows):
        super()._run(rows)
        out = []
        for slot, tokens, want in rows:
            text = self.text.setdefault(slot, [])
            text += tokens
            assert len(text) == self.held[slot]
            out += [(slot, len(text) - len(tokens) + w + 1) for w in want]
        return np.array(out)

    def step(self, entries):
        for e in entries:
            assert e.undecided == (len(e.tokens) - 1 if self.text.get(e.slot) else 0)
        return super().step(entries)

    def rewind(self, slot, length):
        assert length < self.held[slot]
        self.rewinds.append((slot, self.held[slot], length))
        self.held[slot] = length
        del self.text[slot][length:]

    def close(self, slots):
        super().close(slots)
        for s in slots:
            self.text.pop(s, None)


class DraftSampler(ScriptSampler):
    """The target's token after n tokens of a slot is say(slot, n); drafts are kept as long as they are that."""

    def __init__(self, say):
        super().__init__()
        self.say, self.verified = say, []

    def verify(self, logits, drafts, configs, uniforms):
        assert len(drafts) == len(configs) == len(uniforms) and all(len(u) == len(x) + 1 for u, x in zip(uniforms, drafts))
        assert len(logits) == sum(len(x) + 1 for x in drafts)
        kept, tokens, row = [], [], 0
        for x in drafts:
            rows = logits[row:row + len(x) + 1]
            row += len(x) + 1
            assert len({int(s) for s, _ in rows}) == 1 and [int(n) for _, n in rows] == list(range(rows[0][1], rows[0][1] + len(rows)))
            want = [self.say(int(s), int(n)) for s, n in rows]
            k = next((j for j, t in enumerate(x) if t != want[j]), len(x))
            kept.append(k)
            tokens.append(want[k])
        self.verified.append(([list(x) for x in drafts], [list(u) for u in uniforms]))
        return kept, tokens


def plain_run(say, slot, prompt, max_tokens, max_ctx, stop=()):
    out = []
    while True:
        if len(out) >= max_tokens:
            return out, "length"
        if len(prompt) + len(out) >= max_ctx - 1:
            return out, "context"
        t = say(slot, len(prompt) + len(out))
        if t in stop:
            return out, "stop"
        out.append(t)


def cfg(n, drafts, **kw):
    return GenerateConfig(max_tokens=n, sampler=SamplerConfig(temperature=0), lookup_drafts=drafts, **kw)


@pytest.mark.parametrize("drafts", [1, 2, 3, 7])
def test_drafted_loop_emits_what_the_plain_one_does(drafts):
    """Texts that repeat every few tokens, with a break now and then: drafts are kept up to the break."""
    say = lambda slot, n: 50 + n % (3 + slot) + (20 if n % 17 == 0 else 0)       # noqa: E731
    prompts = [[50 + n % 3 for n in range(7)], [50 + n % 4 for n in range(9)], [1]]
    lens = [30, 25, 1]
    eng, samp, seen = DraftEngine(max_ctx=64), DraftSampler(say), []
    results, stats = generate(eng, samp, prompts, [cfg(n, drafts) for n in lens], on_token=lambda i, t: seen.append((i, t)))
    for i, (p, n, r) in enumerate(zip(prompts, lens, results)):
        assert (r.tokens, r.finish_reason) == plain_run(say, i, p, n, 64)
        assert [t for j, t in seen if j == i] == r.tokens
    assert stats.output_tokens == 56 and 0 < stats.kept_drafts < stats.drafted_tokens
    assert stats.steps == len(eng.steps) < 30 and len(stats.step_ms) == 1 + len(samp.verified)
    assert eng.rewinds and not eng.held and sorted(eng.closed) == [0, 1, 2]
    assert all(len(x) <= drafts for xs, _ in samp.verified for x in xs)


def test_drafted_loop_ends_where_the_plain_one_ends():
    """The last token, the context's end and stop tokens, met inside a run of kept drafts or by the token after it."""
    say = lambda slot, n: 10 + n % 4                                             # noqa: E731
    prompt = [10 + n % 4 for n in range(9)]
    for n in range(1, 12):
        eng = DraftEngine(max_ctx=64)
        (r,), stats = generate(eng, DraftSampler(say), [prompt], [cfg(n, 5)])
        assert (r.tokens, r.finish_reason) == plain_run(say, 0, prompt, n, 64) and stats.output_tokens == n
        assert max(len(t) for s in eng.steps for _, t, _ in s[:1]) <= max(9, n)
    for ctx in range(10, 22):                        # from no room for a single token on
        eng = DraftEngine(max_ctx=ctx)
        (r,), _ = generate(eng, DraftSampler(say), [prompt], [cfg(50, 4)])
        assert (r.tokens, r.finish_reason) == plain_run(say, 0, prompt, 50, ctx) and r.finish_reason == "context"
    for at in range(9, 24):
        stopping = lambda slot, n: 99 if n == at else say(slot, n)               # noqa: E731
        (r,), stats = generate(DraftEngine(max_ctx=64), DraftSampler(stopping), [prompt], [cfg(40, 4)], default_stop=(99,))
        assert (r.tokens, r.finish_reason) == plain_run(stopping, 0, prompt, 40, 64, stop=(99,)) and r.finish_reason == "stop"
        (r,), _ = generate(DraftEngine(max_ctx=64), DraftSampler(say), [prompt], [cfg(40, 4, stop_tokens=(12,))], default_stop=(99,))
        assert (r.tokens, r.finish_reason) == ([11], "stop")          # 12 would be the first draft's successor


def test_uniform_numbers_are_not_used_twice():
    """Every decision that counts has a number of its own: the token drawn at a place, and whether the draft there is kept."""
    say = lambda slot, n: 10 + n % 4 + (n % 9 == 0)                              # noqa: E731
    samp = DraftSampler(say)
    c = cfg(40, 4, seed=3)
    generate(DraftEngine(max_ctx=64), samp, [[10 + n % 4 for n in range(9)]], [c])
    drawn, decided, place = {}, {}, 0
    for (x,), (u,) in samp.verified:
        k = next((j for j, t in enumerate(x) if t != say(0, 9 + place + j)), len(x))
        for j in range(min(k + 1, len(x))):
            assert place + j not in decided
            decided[place + j] = u[j]
        drawn[place] = u[-1]
        place += k + 1
    every = list(drawn.values()) + list(decided.values())
    assert len(set(every)) == len(every) and all(0 <= v < 1 for v in every)


def test_a_batch_mixes_requests_that_draft_and_that_do_not():
    say = lambda slot, n: 5 + n % 3                                              # noqa: E731
    samp, eng = DraftSampler(say), DraftEngine(max_ctx=64)
    prompts = [[5 + n % 3 for n in range(8)]] * 2
    results, _ = generate(eng, samp, prompts, [cfg(9, 3), cfg(9, 0)])
    assert [r.tokens for r in results] == [plain_run(say, 0, prompts[0], 9, 64)[0]] * 2
    assert all(not xs[-1] for xs, _ in samp.verified if len(xs) == 2) and any(xs[0] for xs, _ in samp.verified)
    # one whose distribution is cut cannot be verified: nobody drafts beside it, everyone gets the plain loop
    samp, eng = DraftSampler(say), DraftEngine(max_ctx=64)
    results, stats = generate(eng, samp, prompts, [cfg(4, 3), GenerateConfig(max_tokens=4)])
    assert not samp.verified and [len(r.tokens) for r in results] == [4, 4] and stats.drafted_tokens == 0


def test_options_and_refusals():
    c = apply_options([with_lookup_drafts(4), with_temperature(0)])
    assert c.lookup_drafts == 4 and c.sampler.temperature_alone
    with pytest.raises(ValueError, match="lookup_drafts"):
        apply_options([with_lookup_drafts(-1)])
    alone = dict(temperature=0.8, top_k=0, top_p=1.0, min_p=0.0, repetition_penalty=1.0)
    assert SamplerConfig(**alone).temperature_alone and SamplerConfig(temperature=0).temperature_alone
    for cut in (dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(repetition_penalty=1.2)):
        s = SamplerConfig(**{**alone, **cut})
        assert not s.temperature_alone
        eng = DraftEngine()
        with pytest.raises(GenerationError, match="request 1: drafts"):
            generate(eng, DraftSampler(lambda s, n: 1), [[1], [2]], [cfg(2, 0), GenerateConfig(sampler=s, lookup_drafts=2)])
        assert not eng.steps and eng.free_slots() == 3
    eng = DraftEngine()
    eng.can_rewind = False                            # a model with state that no length determines
    with pytest.raises(GenerationError, match="cannot be taken back"):
        generate(eng, DraftSampler(lambda s, n: 1), [[1]], [cfg(2, 1)])
    # a failure on the way gives the slots back
    eng, samp = DraftEngine(), DraftSampler(lambda s, n: 1 // 0)
    with pytest.raises(ZeroDivisionError):
        generate(eng, samp, [[1], [2]], [cfg(2, 1)] * 2)
    assert eng.free_slots() == 3


# -- taking tokens back -----------------------------------------------------------------
KV = CacheNeed("kv", 2, 16)


def make(needs, **kw):
    kw.setdefault("max_slots", 4)
    return Cache(needs, 64 * PAGE, 16 * PAGE, torch.bfloat16, "cpu", **kw)


def test_rewind_gives_back_the_pages_that_held_nothing_else():
    c = make([[KV], [CacheNeed("kv", 1, 32)]])
    s = c.alloc_slot()
    c.reserve([(s, 130)])
    c.advance(s, 130)
    c.rewind(s, 130)
    assert len(c.held_pages(s, 0)) == 3
    c.rewind(s, 128)
    assert sorted(c.held_pages(s, 0)) == sorted(c.held_pages(s, 1)) == [0, 1] and c.length(s) == 128
    assert all(g.table_host[s, 2] == -1 for g in c.groups)
    c.check_consistent()
    c.rewind(s, 65)
    assert sorted(c.held_pages(s, 0)) == [0, 1]
    c.reserve([(s, 129)])
    c.advance(s, 64)
    assert sorted(c.held_pages(s, 1)) == [0, 1, 2]
    c.rewind(s, 0)
    assert not c.held_pages(s, 0) and c.length(s) == 0 and all(g.pool.n_free == g.pool.n_pages for g in c.groups)
    for bad in (-1, 1):
        with pytest.raises(CacheError, match="rewind"):
            c.rewind(s, bad)
    c.free_slot(s)
    with pytest.raises(CacheError, match="not in use"):
        c.rewind(s, 0)
    st = make([[KV, CacheNeed("state", state_shape=(3,))]])
    s = st.alloc_slot()
    st.reserve([(s, 4)])
    st.advance(s, 4)
    with pytest.raises(CacheError, match="state"):
        st.rewind(s, 3)
    assert st.length(s) == 4


def test_windows_keep_what_a_rewound_slot_sees():
    """A window of 100: after 164 tokens the next one sees places 65 on, so page 0 is gone; after 163 it sees 64 on.  With
    the last tokens undecided, the pages that a token at the length before them sees stay until the next step."""
    c = make([[CacheNeed("kv", 2, 16, window=100)]], max_step_tokens=64)
    for kept in range(0, 41):
        s = c.alloc_slot()
        for n in (64, 64, 30):
            c.reserve([(s, c.length(s) + n)])
            c.advance(s, n)
        assert sorted(c.held_pages(s)) == [0, 1, 2]
        c.reserve([(s, 158 + 40)])
        c.advance(s, 40, sure=158)                            # 198 tokens: alone they would have let page 0 go
        assert sorted(c.held_pages(s)) == [0, 1, 2, 3]
        c.rewind(s, 158 + kept)
        c.settle([s])
        assert sorted(c.held_pages(s)) == list(range((158 + kept - 99) // 64, (158 + kept - 1) // 64 + 1))
        c.check_consistent()
        c.free_slot(s)
    s = c.alloc_slot()
    c.reserve([(s, 64)])
    c.advance(s, 64)
    c.reserve([(s, 128)])
    c.advance(s, 64)
    c.reserve([(s, 192)])
    c.advance(s, 64)
    with pytest.raises(CacheError, match="no longer holds"):
        c.rewind(s, 150)
    assert c.length(s) == 192
    c.check_consistent()


def test_random_drafting_keeps_the_books():
    rng = random.Random(1)
    c = make([[KV], [CacheNeed("kv", 2, 16, window=70)]], max_step_tokens=64)
    slots = [c.alloc_slot() for _ in range(4)]
    for _ in range(800):
        s = rng.choice(slots)
        n = c.length(s)
        k = rng.choice([1, 1, 2, 5, 9, 64])
        if n + k > c.max_ctx:
            c.rewind(s, n)
            c.free_slot(s)
            assert c.alloc_slot() == s
            continue
        c.settle([s])
        assert c.can_reserve([(s, n + k)]) is None
        c.reserve([(s, n + k)])
        undecided = rng.randrange(k + 1)
        c.advance(s, k, n + k - undecided)
        if rng.random() < 0.7:
            c.rewind(s, n + k - rng.randrange(undecided + 1))
        c.check_consistent()
        assert sorted(c.held_pages(s, 0)) == list(range((c.length(s) + 63) // 64))
        assert set(c.held_pages(s, 1)) >= set(range(max(0, c.length(s) - 69) // 64, (c.length(s) + 63) // 64))


# -- 8-bit keys and values -----------------------------------------------------------------
@pytest.mark.parametrize("heads,hd", [(2, 16), (8, 64), (1, 80), (4, 128), (3, 256)])
def test_sizes_of_an_8_bit_cache(heads, hd):
    need = [[CacheNeed("kv", heads, hd)]] * 3
    c = make(need, kv_dtype="e4m3")
    g = c.groups[0]
    unit = heads * 128 * (hd + 1)                      # 64 tokens of keys, values and a scale byte for each
    assert g.storage.dtype == torch.uint8 and g.page_stride == 3 * unit and g.storage.numel() == g.pool.n_pages * 3 * unit
    assert kv_bytes_per_token(need, torch.bfloat16, "e4m3") == 3 * heads * 2 * (hd + 1)
    assert kv_bytes_per_token(need, torch.bfloat16, None) == 3 * heads * 2 * hd * 2
    views = [c.kv_view(u) for u in range(3)]
    assert all(v.q8 for v in views) and not make(need).kv_view(0).q8
    base = g.storage.data_ptr()
    assert [v.cache.data_ptr() - base for v in views] == [0, unit, 2 * unit] and all(v.page_stride == 3 * unit for v in views)


def test_what_an_8_bit_cache_refuses():
    with pytest.raises(CacheError, match="int4"):
        make([[KV]], kv_dtype="int4")
    for hd in (24, 272):
        with pytest.raises(CacheError, match="head"):
            make([[CacheNeed("kv", 2, hd)]], kv_dtype="e4m3")


def test_a_copied_slot_has_the_bytes():
    c = make([[KV]], kv_dtype="e4m3")
    a = c.alloc_slot()
    c.reserve([(a, 100)])
    c.advance(a, 100)
    g = c.groups[0]
    g.storage.copy_(torch.arange(g.storage.numel()) % 251)
    b = c.copy_slot(a)
    rows = g.storage.view(-1, g.page_stride)
    assert all(torch.equal(rows[c.held_pages(b)[i]], rows[p]) for i, p in c.held_pages(a).items())
