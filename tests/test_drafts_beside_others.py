"""What drafting does to whom (no GPU: stand-ins for the engine and the sampler)."""
import numpy as np
import pytest

from dlgo_amd.engine.generate import generate
from dlgo_amd.sampling import GenerateConfig, SamplerConfig, uniform
from test_drafts import DraftEngine, DraftSampler

ALONE = dict(top_k=0, top_p=1.0, min_p=0.0, repetition_penalty=1.0)


class TwoSums(DraftSampler):
    """The sampler and the verification sum a row differently: with the same number they may draw neighbours."""

    def choose_async(self, logits, configs, uniforms, recent=None, keys=None):
        super().choose_async(logits, configs, uniforms, recent, keys)
        ids = [self.say(int(s), int(n)) if c.greedy else 1000 + int(1e6 * u) for (s, n), c, u in zip(logits, configs, uniforms)]
        return np.array(ids), lambda: ids

    def verify(self, logits, drafts, configs, uniforms):
        kept, tokens = super().verify(logits, drafts, configs, uniforms)
        return kept, [t if c.greedy else 1001 + int(1e6 * u[-1]) for t, c, u in zip(tokens, configs, uniforms)]


@pytest.mark.parametrize("mates", [1, 2])
@pytest.mark.parametrize("first", [False, True])
def test_a_request_that_does_not_draft_gets_the_same_tokens_beside_one_that_does(first, mates):
    """Its draws are the sampler's, number by number, whoever shares its batch; rows and keys stay in step."""
    say = lambda slot, n: 5 + n % 3                                              # noqa: E731
    plain = GenerateConfig(max_tokens=9, sampler=SamplerConfig(temperature=0.7, **ALONE), seed=11)
    prompt = [5 + n % 3 for n in range(8)]
    at = 0 if first else mates
    runs = []
    for drafts in (0, 3):
        mate = GenerateConfig(max_tokens=12, sampler=SamplerConfig(temperature=0), lookup_drafts=drafts)
        configs = [mate] * mates
        configs.insert(at, plain)
        samp, eng = TwoSums(say), DraftEngine(max_ctx=64)
        results, stats = generate(eng, samp, [prompt] * (mates + 1), configs)
        runs.append([r.tokens for r in results])
        assert (stats.kept_drafts > 0) == (drafts > 0) and not eng.held
    assert runs[0] == runs[1]
    assert runs[1][at] == [1000 + int(1e6 * uniform(11, at, j)) for j in range(9)]


def test_a_batch_where_only_a_drawn_request_is_left():
    """The drafting one ends first: nothing is left to verify."""
    say = lambda slot, n: 5 + n % 3                                              # noqa: E731
    plain = GenerateConfig(max_tokens=12, sampler=SamplerConfig(temperature=0.7, **ALONE), seed=4)
    drafting = GenerateConfig(max_tokens=3, sampler=SamplerConfig(temperature=0), lookup_drafts=2)
    samp = TwoSums(say)
    results, _ = generate(DraftEngine(max_ctx=64), samp, [[5, 6, 7, 5, 6, 7]] * 2, [plain, drafting])
    assert results[0].tokens == [1000 + int(1e6 * uniform(4, 0, j)) for j in range(12)] and len(results[1].tokens) == 3
    assert all(xs for xs, _ in samp.verified)


def test_what_fills_a_step_up_is_not_counted_as_drafts():
    """Two requests, one whose text repeats three tokens and one whose text never does: the second one's rows fill the step."""
    say = lambda slot, n: 5 + n % 3 if slot == 0 else 100 + n                    # noqa: E731
    draft = GenerateConfig(max_tokens=20, sampler=SamplerConfig(temperature=0), lookup_drafts=5)
    samp = DraftSampler(say)
    _, stats = generate(DraftEngine(max_ctx=64), samp, [[5, 6, 7] * 3, [1, 2, 3, 4]], [draft, draft])
    rows = sum(len(x) for xs, _ in samp.verified for x in xs)
    looked_up = sum(min(3, len(xs[0])) for xs, _ in samp.verified if len(xs) == 2)       # the text behind the last match is three tokens long
    assert any(len(xs) == 2 and len(xs[1]) == 5 for xs, _ in samp.verified)
    assert stats.drafted_tokens == looked_up < rows and 0 < stats.kept_drafts <= looked_up
