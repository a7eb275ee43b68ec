"""A request that asks for no drafts beside one that does, through the whole library on the GPU."""
import pytest

from test_drafts_gpu import TINY_B, folders, repeating, texts_of  # noqa: F401  (folders is a fixture)

pytestmark = pytest.mark.gpu


def test_a_drawn_request_keeps_its_tokens_beside_one_that_drafts(folders):  # noqa: F811
    """In float32, where a step's shape changes logits by rounding alone: the same seed, the same tokens."""
    import dlgo_amd
    from dlgo_amd.engine.generate import generate
    from dlgo_amd.sampling import GenerateConfig, SamplerConfig
    llm = dlgo_amd.load_llm(folders["B", "float32"], dtype="float32", max_tokens=1024)
    prompts = [texts_of(TINY_B, [5], 21)[0], repeating(TINY_B, 22, 30, 5), texts_of(TINY_B, [17], 23)[0]]
    drawn = GenerateConfig(max_tokens=24, sampler=SamplerConfig(temperature=0.6, top_k=0, top_p=1.0, min_p=0.0, repetition_penalty=1.0),
                           seed=5, ignore_eos=True)
    runs = []
    for drafts in (0, 4):
        mate = GenerateConfig(max_tokens=40, sampler=SamplerConfig(temperature=0), ignore_eos=True, lookup_drafts=drafts)
        results, stats = generate(llm.engine, llm.sampler, prompts, [drawn, mate, drawn])
        runs.append([r.tokens for r in results])
        assert (stats.drafted_tokens > 0) == (drafts > 0) and [len(t) for t in runs[-1]] == [24, 40, 24]
    assert runs[0] == runs[1]
    llm.engine.cache.check_consistent()
