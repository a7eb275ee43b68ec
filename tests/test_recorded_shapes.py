"""Which steps are recorded, and which recordings stay (no GPU: the engine's own bookkeeping)."""
from types import SimpleNamespace

import pytest

from dlgo_amd.engine.engine import Engine, Entry


def engine(**kw):
    eng = object.__new__(Engine)
    eng.__dict__.update(dict(use_graphs=True, max_step_tokens=512, prompt_graph_max_tokens=256, prompt_graph_bytes=1 << 20, prompt_graph_limit=3,
                             graph_max_batch=32, vocab=500, _prompt_graphs={}), **kw)
    return eng


def shape(eng, q_lens, starts, undecided=None, want=None):
    entries, wanted, row = [], [], 0
    for i, n in enumerate(q_lens):
        places = range(n) if want is None else want[i]
        entries.append(Entry(i, [1] * n, list(places), undecided[i] if undecided else 0))
        wanted += [row + w for w in places]
        row += n
    return eng._shape_to_record(entries, q_lens, starts, wanted)


def test_steps_of_drafts_and_fresh_prompts_are_recorded():
    eng = engine()
    drafts = shape(eng, [5, 5], [7, 90], [4, 4])
    assert drafts == ((5, 5), tuple(range(10)), False) == shape(eng, [5, 5], [1, 2], [1, 5])
    assert shape(eng, [5, 9], [0, 0], want=[[4], [8]]) == ((5, 9), (4, 13), True)
    assert shape(eng, [5, 5], [0, 0], [4, 4])[2]                       # fresh: sized by its own lengths
    for q, u in (([5, 4], [4, 3]), ([11] * 3, [10] * 3)):              # unequal, and more rows than graph_max_batch
        assert shape(eng, q, [9] * len(q), u) is None
    assert shape(eng, [5, 5], [7, 90], [4, 4], want=[[4], [4]]) is None
    assert shape(engine(use_graphs=False), [5], [7], [4]) is None and shape(engine(vocab=10 ** 6), [5], [7], [4]) is None
    assert shape(eng, [257], [0], want=[[256]]) is None and shape(eng, [5], [0], want=[[]]) is None


@pytest.mark.parametrize("undecided", [None, [0, 0], [4, 0]])
def test_other_steps_behind_a_past_are_not(undecided):
    """Pieces of prompts with every row wanted, of equal length or not: nothing is taken back, so nothing says that the shape
    comes again, and the step is sized by its own lengths."""
    assert shape(engine(), [5, 5], [7, 90], undecided) is None
    assert shape(engine(), [5], [7], undecided and undecided[1:]) is None


def keep(eng, key, mb=0.1):
    eng._prompt_graphs.pop(key, None)
    eng._prompt_graphs[key] = SimpleNamespace(logits=SimpleNamespace(numel=lambda: int(mb * (1 << 20)) // 4))
    eng._drop_recordings()


def test_shapes_of_drafts_do_not_push_out_prompts():
    """Three places for either kind: ten shapes of drafts (a batch that thins out) leave the prompts' recordings."""
    eng = engine()
    prompts = [((n,), (n - 1,), True) for n in (5, 6, 7)]
    drafts = [((n,), tuple(range(n)), False) for n in range(2, 12)]
    for k in prompts + drafts:
        keep(eng, k)
    assert list(eng._prompt_graphs) == prompts + drafts[-3:]
    keep(eng, ((9,), (8,), True))
    assert list(eng._prompt_graphs) == prompts[1:] + drafts[-3:] + [((9,), (8,), True)]


def test_recordings_that_keep_too_much_go_whatever_they_are():
    eng = engine()
    keys = [((5,), (4,), True), ((2,), (0, 1), False), ((6,), (5,), True), ((3,), (0, 1, 2), False)]
    for k in keys:
        keep(eng, k, 0.4)
    assert list(eng._prompt_graphs) == keys[-2:]             # 1 MB in all
    keep(eng, keys[0], 5)
    assert list(eng._prompt_graphs) == keys[:1]              # the newest one stays
