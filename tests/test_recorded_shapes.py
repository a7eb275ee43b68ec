"""Which steps are recorded (no GPU: the engine's own bookkeeping)."""
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
