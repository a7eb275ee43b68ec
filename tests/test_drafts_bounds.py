"""How many tokens a step drafts at most, whatever a request asks for (no GPU: stand-ins for the engine and the sampler)."""
import pytest

from dlgo_amd.engine.generate import generate
from test_drafts import DraftEngine, DraftSampler, cfg, plain_run


class Strict(DraftSampler):
    """Refuses what the kernel refuses."""

    def verify(self, logits, drafts, configs, uniforms):
        assert max(len(x) for x in drafts) <= 1024
        return super().verify(logits, drafts, configs, uniforms)


class Rows(DraftEngine):
    """Refuses what the engine refuses: more undecided tokens than a step's rows."""

    def __init__(self, rows=None, **kw):
        super().__init__(max_ctx=8192, pages=400, **kw)
        self.most = 0
        if rows is not None:
            self.logits_rows = rows

    def step(self, entries):
        drafting = [e for e in entries if self.text.get(e.slot)]
        if drafting:
            self.most = max(self.most, sum(len(e.tokens) for e in drafting))
            assert getattr(self, "logits_rows", None) is None or len(drafting) > self.logits_rows or sum(len(e.tokens) for e in drafting) <= self.logits_rows
        return super().step(entries)


@pytest.mark.parametrize("rows,ask", [(None, 2000), (1024, 2000), (5000, 2000), (3000, 1024), (64, 40), (3, 5), (2, 1), (1, 7)])
@pytest.mark.parametrize("n", [1, 3])
def test_a_request_for_more_drafts_than_a_step_takes(rows, ask, n):
    """A text that repeats 3,000 tokens proposes as many as it is asked for: all the same the generation ends as without."""
    say = lambda slot, k: k % 1500                                               # noqa: E731
    prompt = [k % 1500 for k in range(3001)]
    eng, samp = Rows(rows), Strict(say)
    results, stats = generate(eng, samp, [prompt] * n, [cfg(2500, ask)] * n)
    assert all(r.tokens == plain_run(say, 0, prompt, 2500, 8192)[0] for r in results)
    assert eng.most == n * max(1, min(ask + 1, 1025, (rows or 1024) // n)) and not eng.held
    assert stats.kept_drafts <= stats.drafted_tokens


def test_a_request_of_its_own_numbers():
    """A configuration made by hand, without the options' checks, drafts nothing below zero."""
    say = lambda slot, k: 5 + k % 3                                              # noqa: E731
    eng = DraftEngine(max_ctx=64)
    results, _ = generate(eng, DraftSampler(say), [[5 + k % 3 for k in range(8)]] * 2, [cfg(9, 3), cfg(9, -2)])
    assert [r.tokens for r in results] == [plain_run(say, 0, [0] * 8, 9, 64)[0]] * 2
