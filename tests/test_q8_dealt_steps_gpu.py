"""The engine's recorded steps over an 8-bit cache where a launch deals a sequence's pages to several blocks: partial results
in a scratch buffer, and the kernel that joins them.  (The other engine tests' contexts are too short for that.)"""
import numpy as np
import pytest
import torch

from conftest import TINY_B, make_folder
from test_drafts_gpu import TOL, plain_q8, rel_err, texts_of  # noqa: F401  (plain_q8 is a fixture)

pytestmark = pytest.mark.gpu
CTX = 4096


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("dealt"))
    make_folder({**TINY_B, "max_position_embeddings": CTX}, 47, path, dtype="bfloat16", norm_jitter=0.1, std=0.08)
    return path


def partials(eng):
    return eng.workspace._bufs["flat:attention.partials", 0, torch.float32]


def test_recorded_steps_deal_pages(folder, plain_q8):  # noqa: F811
    """Steps of drafts and of single tokens, two sequences (one grows past the 16 pages from which on a sequence is dealt,
    while it is drafted for), the third time and later by replay: the plain implementation's logits, and the bits of the
    same launches made one by one.  What a recording writes its partial results to was there before it and stays."""
    from dlgo_amd.engine import Engine, Entry
    from dlgo_amd.kernels import ops
    made = [Engine.from_folder(folder, "bfloat16", max_tokens=2 * CTX, max_ctx=CTX, max_step_tokens=1024, cache_dtype="e4m3") for _ in range(2)]
    H, KV, hd = TINY_B["num_attention_heads"], TINY_B["num_key_value_heads"], TINY_B["head_dim"]
    for rows, q in ((10, 5), (2, 1)):
        assert ops._attention_q8_scratch(hd, rows, 2, H, KV, q, CTX, 0) > 0
    texts = texts_of(TINY_B, [1360, 300], seed=2)
    cfg, w = plain_q8.read_model(folder)
    want = [plain_q8.forward(cfg, w, t) for t in texts]
    pos = [1002, 31]
    slots = [eng.open(2) for eng in made]
    for eng, s in zip(made, slots):
        for i in (0, 1):
            eng.step([Entry(s[i], texts[i][:pos[i]], (pos[i] - 1,))])

    def both(call):
        out = [call(eng, s) for eng, s in zip(made, slots)]
        assert torch.equal(*out)
        return out[0]

    wrong = lambda t: (t + 1) % TINY_B["vocab_size"]         # noqa: E731
    for turn in range(8):
        drafts = [texts[i][pos[i]:pos[i] + 3] + [wrong(t) for t in texts[i][pos[i] + 3:pos[i] + 5]] for i in (0, 1)]
        made[1]._prompt_seen.clear()                          # never the second time: launch by launch
        buffer = partials(made[0]) if turn else None
        out = both(lambda eng, s: eng.step([Entry(s[i], drafts[i], range(5), undecided=4) for i in (0, 1)]))
        assert buffer is None or partials(made[0]) is buffer
        for i in (0, 1):
            assert rel_err(out[5 * i:5 * i + 3], want[i][pos[i]:pos[i] + 3]) <= TOL["B"], (turn, i)
            pos[i] += 3
            for eng, s in zip(made, slots):
                eng.rewind(s[i], pos[i])
        if turn == 5:                                         # far ahead: more pages than the recording ever saw
            for eng, s in zip(made, slots):
                eng.step([Entry(s[0], texts[0][pos[0]:pos[0] + 300], (0,))])
            pos[0] += 300
        torch.cuda.synchronize()
    assert [sum(not k[2] for k in eng._prompt_graphs) for eng in made] == [1, 0]
    for turn in range(6):
        buffer = partials(made[0]) if turn else None
        out = both(lambda eng, s: eng.decode(s, [texts[i][pos[i]] for i in (0, 1)], replay=eng is made[0]).clone())
        assert buffer is None or partials(made[0]) is buffer
        for i in (0, 1):
            assert rel_err(out[i], want[i][pos[i]]) <= TOL["B"], (turn, i)
            pos[i] += 1
        torch.cuda.synchronize()
    assert pos[0] > 16 * 64 and [len(eng._graphs) for eng in made] == [1, 0]
    # the steps of drafts again, recorded before the single tokens asked for scratch of their own
    for _ in range(2):
        made[1]._prompt_seen.clear()
        out = both(lambda eng, s: eng.step([Entry(s[i], texts[i][pos[i]:pos[i] + 5], range(5), undecided=4) for i in (0, 1)]))
        for i in (0, 1):
            assert rel_err(out[5 * i:5 * i + 5], want[i][pos[i]:pos[i] + 5]) <= TOL["B"]
            for eng, s in zip(made, slots):
                eng.rewind(s[i], pos[i] + 2)
            pos[i] += 2
    for eng in made:
        eng.cache.check_consistent()


def test_a_next_turn_behind_a_long_past(folder, plain_q8):  # noqa: F811
    """Tiles of a prompt's piece dealt to several blocks, in an engine's step, eager."""
    from dlgo_amd.engine import Engine, Entry
    from dlgo_amd.kernels import ops
    eng = Engine.from_folder(folder, "bfloat16", max_tokens=CTX, max_ctx=CTX, max_step_tokens=1024, cache_dtype="e4m3")
    (text,) = texts_of(TINY_B, [2300], seed=3)
    assert ops._attention_q8_scratch(TINY_B["head_dim"], 40, 1, TINY_B["num_attention_heads"], TINY_B["num_key_value_heads"], 40, 2300, 0) > 0
    cfg, w = plain_q8.read_model(folder)
    want = plain_q8.forward(cfg, w, text, rows=range(2260, 2300))
    (s,) = eng.open(1)
    eng.step([Entry(s, text[:2260], (0,))])
    got = eng.step([Entry(s, text[2260:], range(40))])
    assert rel_err(got, want) <= TOL["B"]
    assert np.abs(want).max() > 0 and eng.length(s) == 2300
