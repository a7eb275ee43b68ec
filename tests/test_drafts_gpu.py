"""The 8-bit cache and drafted tokens through the library's entry points, on the GPU.

Tolerances of the 8-bit runs.  The plain implementation rounds keys and values as the cache does, so what is left is the
run's own bfloat16 (3e-2 of the largest logit, as over a bfloat16 cache) and the elements that it puts on the other side of
a border of the 8-bit grid.  Through a few layers of bfloat16 an element is off by about d = 1e-2 (what plain.forward gives
when every product's result, norm and gate is rounded to bfloat16: 0.6e-2 to 1.6e-2 of the largest logit for these models).
The grid's steps are s = 2^-3 to 2^-4 of an element; d / s of the elements move, by s each: sqrt(d / s) * s = sqrt(d s) =
sqrt(1e-2 * 2^-3.5) = 3e-2 in the root mean square, in every layer's values, and a row that sees one token has nothing to
average over.  So 3e-2 for each layer more.  (2^-8, the rounding of the stored element alone, in place of d gave 3e-2 for
all layers together; the plain implementation itself, rounded to bfloat16 as above, is off by up to 7.9e-2 for model C.)"""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_llama as plain
from conftest import ROOT, TINY_A, TINY_B, TINY_C, TINY_D, make_folder
from test_verify_gpu import plain as plain_verify

pytestmark = pytest.mark.gpu

CONFIGS = {"A": (TINY_A, dict(std=0.1)), "B": (TINY_B, dict(norm_jitter=0.1, std=0.08)), "C": (TINY_C, dict(norm_jitter=0.1, std=0.12)),
           "D": (TINY_D, dict(norm_jitter=0.2, std=0.08))}
TOL = {name: 3e-2 + 3e-2 * raw["num_hidden_layers"] for name, (raw, _) in CONFIGS.items()}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for name, (raw, kw) in CONFIGS.items():
        for dtype in ("bfloat16", "float32"):
            out[name, dtype] = str(tmp_path_factory.mktemp(f"drafts{name}"))
            make_folder(raw, 31 + len(out), out[name, dtype], dtype=dtype, **kw)
    return out


def rounded(x, heads, hd):
    """Rows of a cache of 8 bits: e4m3 times the least power of two that holds a head's largest element."""
    x = torch.as_tensor(x).view(-1, heads, hd)
    m = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(m.clamp(min=2.0 ** -200) / 448)).clamp(min=-126)
    e = torch.where(m > 448 * torch.exp2(e), e + 1, e)
    return ((x / torch.exp2(e)).float().to(torch.float8_e4m3fn).double() * torch.exp2(e)).view(len(x), heads * hd).numpy()


@pytest.fixture
def plain_q8(monkeypatch):
    """plain.forward over rounded keys and values."""
    exact = plain.attention

    def attention(q, k, v, H, KV, hd, window=None):
        return exact(q, rounded(k, KV, hd), rounded(v, KV, hd), H, KV, hd, window)
    monkeypatch.setattr(plain, "attention", attention)
    return plain


def rel_err(got, want):
    return np.abs(got.double().cpu().numpy() - want).max() / np.abs(want).max()


def texts_of(raw, lens, seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, raw["vocab_size"], size=n).tolist() for n in lens]


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_an_8_bit_cache_under_every_kind_of_step(folders, plain_q8, name, graphs):
    """Prompts whole and in pieces, single tokens (recorded from the second on), a few tokens at once, a copied sequence,
    unequal batches in slots that were used before."""
    from dlgo_amd.engine import Engine, Entry
    raw = CONFIGS[name][0]
    eng = Engine.from_folder(folders[name, "bfloat16"], "bfloat16", max_tokens=2048, max_step_tokens=96, use_graphs=graphs, cache_dtype="e4m3")
    assert eng.cache.groups[0].storage.dtype == torch.uint8
    cfg, w = plain.read_model(folders[name, "bfloat16"])
    for turn in range(2):
        texts = texts_of(raw, [120, 9, 70], seed=turn)
        want = [plain_q8.forward(cfg, w, t) for t in texts]
        slots = eng.open(3)
        first = [len(t) - 6 for t in texts]
        out = eng.step([Entry(s, t[:n], range(n)) for s, t, n in zip(slots, texts, first)])
        for o, x, n in zip(torch.split(out, first), want, first):
            assert rel_err(o, x[:n]) <= TOL[name]
        for j in range(3):
            out = eng.decode(slots, [t[n + j] for t, n in zip(texts, first)])
            for i, n in enumerate(first):
                assert rel_err(out[i], want[i][n + j]) <= TOL[name], (turn, i, j)
        twin = eng.fork(slots[0])
        out = eng.step([Entry(s, t[n + 3:], (0, 1, 2)) for s, t, n in zip(slots, texts, first)])
        alone = eng.step([Entry(twin, texts[0][first[0] + 3:], (0, 1, 2))])
        for i, n in enumerate(first):
            assert rel_err(out[3 * i:3 * i + 3], want[i][n + 3:]) <= TOL[name]
        assert rel_err(alone, want[0][first[0] + 3:]) <= TOL[name]
        eng.close(slots + [twin])
    eng.cache.check_consistent()


@pytest.mark.parametrize("cache_dtype", [None, "e4m3"])
@pytest.mark.parametrize("window", [None, 70])
def test_a_rewound_sequence_goes_on_as_if_nothing_had_been_there(folders, monkeypatch, window, cache_dtype):
    """Wrong drafts behind a sequence, taken back, then the right tokens: the same bits as without the drafts, around the
    ends of pages and with layers that see a window only."""
    from dlgo_amd.engine import Engine, EngineError, Entry
    from dlgo_amd.parts.attention import Attention
    if window:
        init = Attention.__init__
        monkeypatch.setattr(Attention, "__init__", lambda self, *a, **kw: init(self, *a, **{**kw, "window": window}))
    eng = Engine.from_folder(folders["B", "bfloat16"], "bfloat16", max_tokens=1024, max_ctx=256, max_step_tokens=64, cache_dtype=cache_dtype)
    assert eng.can_rewind and (eng.cache.has_windows == bool(window))
    (text,) = texts_of(TINY_B, [200], seed=5)
    a, b = eng.open(2)
    pos = 0
    for n in (50, 9, 3, 1, 4, 60, 5, 12, 2, 33, 8):
        piece = text[pos:pos + n]
        wrong = [(t + 1) % TINY_B["vocab_size"] for t in text[pos:pos + min(9, 64 - n)]]
        if pos:
            eng.step([Entry(a, [text[pos]] + wrong, range(len(wrong) + 1), undecided=len(wrong) + 1)])
            eng.rewind(a, pos)
        x = eng.step([Entry(a, piece, range(n))])
        y = eng.step([Entry(b, piece, range(n))])
        assert torch.equal(x, y) and torch.isfinite(x).all()
        pos += n
        eng.cache.check_consistent()
    with pytest.raises(EngineError, match="rewind"):
        eng.rewind(a, pos + 1)
    with pytest.raises(EngineError, match="undecided"):
        eng.step([Entry(a, [1, 2], (1,), undecided=3)])
    eng.close([a])
    with pytest.raises(EngineError, match="not in use"):
        eng.rewind(a, 0)


@pytest.mark.parametrize("seed", [0, 1])
def test_random_traffic_over_an_8_bit_cache(folders, plain_q8, seed):
    """Sequences opened, closed and copied; prompts, pieces, single tokens and drafts that are taken back in part, several
    sequences a step: every logit that is asked for is the plain implementation's for that text."""
    from dlgo_amd.engine import Engine, Entry
    rng = np.random.default_rng(seed)
    name = "AB"[seed]
    raw = CONFIGS[name][0]
    eng = Engine.from_folder(folders[name, "bfloat16"], "bfloat16", max_tokens=640, max_ctx=128, max_slots=5, max_step_tokens=48, cache_dtype="e4m3")
    cfg, w = plain.read_model(folders[name, "bfloat16"])
    token = lambda n: rng.integers(0, raw["vocab_size"], size=n).tolist()        # noqa: E731
    texts, checked = {}, 0

    def check(slot, rows, got):
        nonlocal checked
        assert rel_err(got, plain_q8.forward(cfg, w, texts[slot], rows=rows)) <= TOL[name]
        checked += len(rows)
    for turn in range(90):
        kind = rng.choice(["open", "step", "step", "decode", "decode", "drafts", "drafts", "fork", "close"])
        live = [s for s in texts if len(texts[s]) < 100]
        if kind == "open" and eng.free_slots() and eng.free_pages()[0] >= 3:
            texts[eng.open(1)[0]] = []
        elif kind == "close" and texts:
            s = rng.choice(list(texts))
            eng.close([int(s)])
            del texts[s]
        elif kind == "fork" and live and eng.free_slots() and eng.free_pages()[0] >= 3:
            s = int(rng.choice(live))
            texts[eng.fork(s)] = list(texts[s])
        elif kind in ("step", "decode", "drafts") and live:
            mates = [int(s) for s in rng.permutation(live)[:rng.integers(1, 4)]]
            if kind == "decode":
                mates = [s for s in mates if texts[s]] or mates[:1]
                new = [token(1) for _ in mates]
                out = eng.decode(mates, [t[0] for t in new])
                for s, t, x in zip(mates, new, out.clone()):
                    texts[s] += t
                    check(s, [len(texts[s]) - 1], x[None])
                continue
            n = int(rng.integers(2, 7))
            new = [token(n if kind == "drafts" else int(rng.integers(1, 25))) for _ in mates]
            out = eng.step([Entry(s, t, range(len(t)), undecided=n - 1 if kind == "drafts" else 0) for s, t in zip(mates, new)])
            for s, t, x in zip(mates, new, torch.split(out, [len(t) for t in new])):
                texts[s] += t
                check(s, list(range(len(texts[s]) - len(t), len(texts[s]))), x)
                if kind == "drafts":
                    texts[s] = texts[s][:len(texts[s]) - int(rng.integers(0, n))]
                    eng.rewind(s, len(texts[s]))
        eng.cache.check_consistent()
    assert checked > 200


@pytest.mark.parametrize("dtype,cache_dtype", [("bfloat16", "e4m3"), ("bfloat16", None), ("float32", None)])
def test_steps_of_drafts_are_recorded(folders, dtype, cache_dtype):
    """A shape's third step and those after it are replayed, at lengths that had not been reached when it was recorded, with
    other sequences in other slots, and give the bits that the launches one by one give."""
    from dlgo_amd.engine import Engine, Entry
    folder = folders["B", dtype]
    made = [Engine.from_folder(folder, dtype, max_tokens=1024, max_ctx=512, use_graphs=g, cache_dtype=cache_dtype) for g in (True, False)]
    texts = texts_of(TINY_B, [400, 390], seed=8)
    pos = [12, 3]
    slots = [eng.open(3) for eng in made]
    for eng, s in zip(made, slots):
        eng.step([Entry(s[i], texts[i][:pos[i]], (pos[i] - 1,)) for i in (0, 1)])
        eng.step([Entry(s[2], texts[1][:70], (69,))])
    for turn in range(16):
        take = (0, 1) if turn % 4 < 3 else (1, 0)
        outs = [eng.step([Entry(s[i], texts[i][pos[i]:pos[i] + 5], range(5), undecided=4) for i in take]) for eng, s in zip(made, slots)]
        assert torch.equal(*outs), turn
        for eng, s in zip(made, slots):
            for i in take:
                eng.rewind(s[i], pos[i] + 2 + 3 * i)
        pos = [pos[0] + 2, pos[1] + 5]
        if turn == 9:                                        # far ahead: pages and lengths the recording never saw
            for eng, s in zip(made, slots):
                eng.step([Entry(s[i], texts[i][pos[i]:pos[i] + 250], (0,)) for i in (0, 1)])
            pos = [p + 250 for p in pos]
        torch.cuda.synchronize()
    assert [len(eng._prompt_graphs) for eng in made] == [1, 0]
    for eng in made:
        eng.cache.check_consistent()


def repeating(raw, seed, n=30, period=7):
    return (texts_of(raw, [period], seed)[0] * n)[:n]


def test_greedy_with_drafts_is_greedy(folders):
    """In float32 the tokens are the plain implementation's, drafts or none; where the text repeats, in fewer steps."""
    import dlgo_amd
    folder = folders["A", "float32"]
    cfg, w = plain.read_model(folder)
    llm = dlgo_amd.load_llm(folder, dtype="float32", max_tokens=1024, max_batch=3)
    prompts = [repeating(TINY_A, 3), texts_of(TINY_A, [1], 4)[0], repeating(TINY_A, 5, 20, 3), repeating(TINY_A, 6, 9, 4), [7, 7, 7]]
    want = [plain.greedy_generate(cfg, w, p, 40) for p in prompts]
    for n in (1, 4, 15):
        got = llm.generate(prompts, dlgo_amd.with_greedy(), dlgo_amd.with_max_tokens(40), dlgo_amd.with_ignore_eos(), dlgo_amd.with_lookup_drafts(n))
        assert [r.tokens for r in got] == want and all(r.finish_reason == "length" for r in got)
    # up to the context's end, and a stop token among what would be emitted
    long = llm.generate(prompts[0], dlgo_amd.with_greedy(), dlgo_amd.with_max_tokens(500), dlgo_amd.with_ignore_eos(), dlgo_amd.with_lookup_drafts(6))
    assert long.finish_reason == "context" and len(prompts[0]) + len(long.tokens) == TINY_A["max_position_embeddings"] - 1
    assert long.tokens == plain.greedy_generate(cfg, w, prompts[0], len(long.tokens))
    stop = want[0][9]
    r = llm.generate(prompts[0], dlgo_amd.with_greedy(), dlgo_amd.with_max_tokens(40), dlgo_amd.with_stop_tokens([stop]), dlgo_amd.with_lookup_drafts(6))
    assert r.tokens == plain.greedy_generate(cfg, w, prompts[0], 40, stop_tokens=(stop,)) and r.finish_reason == "stop"
    llm.engine.cache.check_consistent()
    assert llm.engine.free_slots() == llm.engine.cache.max_slots


def test_sampling_with_drafts_is_what_the_formulas_say(folders):
    """The whole loop again with the plain model and the plain verification, number by number; and the same twice."""
    import dlgo_amd
    from dlgo_amd.engine.generate import _VERIFY_STREAM, LookupDrafts, fill_drafts
    from dlgo_amd.sampling import uniform
    folder = folders["B", "float32"]
    cfg, w = plain.read_model(folder)
    llm = dlgo_amd.load_llm(folder, dtype="float32", max_tokens=1024)
    prompts = [repeating(TINY_B, 8, 25, 5), texts_of(TINY_B, [3], 9)[0], repeating(TINY_B, 10, 40, 4)]
    opts = [dlgo_amd.with_temperature(0.25), dlgo_amd.with_top_k(0), dlgo_amd.with_top_p(1.0), dlgo_amd.with_repetition_penalty(1.0),
            dlgo_amd.with_seed(77), dlgo_amd.with_max_tokens(20), dlgo_amd.with_ignore_eos(), dlgo_amd.with_lookup_drafts(3)]
    got = llm.generate(prompts, *opts)
    assert [r.tokens for r in llm.generate(prompts, *opts)] == [r.tokens for r in got]
    t = float(np.float32(0.25))
    decided = 0
    out, drafts, texts = [[] for _ in prompts], [[] for _ in prompts], [LookupDrafts(p) for p in prompts]
    while any(len(o) < 20 for o in out):
        live = [i for i, o in enumerate(out) if len(o) < 20]
        for i in live:
            u = [uniform(77 ^ _VERIFY_STREAM, i, len(out[i]) + j) for j in range(len(drafts[i]))] + [uniform(77, i, len(out[i]))]
            at = len(prompts[i]) + len(out[i]) - 1
            logits = torch.as_tensor(plain.forward(cfg, w, prompts[i] + out[i] + drafts[i], rows=range(at, at + len(drafts[i]) + 1)))
            (kept,), (token,), _ = plain_verify(logits, drafts[i], [len(drafts[i])], [t], u, None)
            decided += len(drafts[i])
            new = drafts[i][:kept] + [token]
            out[i] += new
            texts[i].extend(new)
        live = [i for i in live if len(out[i]) < 20]
        room = [min(3, 20 - len(out[i]) - 1) for i in live]
        for i, x in zip(live, fill_drafts([texts[i].propose(r) for i, r in zip(live, room)], room, [out[i][-1] for i in live])):
            drafts[i] = x
    assert [r.tokens for r in got] == out
    assert decided >= 6, "too few drafts: the check says little"


def test_drafts_over_an_8_bit_cache_keep_to_the_margins(folders, plain_q8):
    """The three operators together as a server runs them: prompts stored and attended in 8 bits, tokens drafted, verified and
    taken back.  Every emitted token is the plain maximum, or within the tolerance of it."""
    import dlgo_amd
    folder = folders["A", "bfloat16"]
    cfg, w = plain.read_model(folder)
    llm = dlgo_amd.load_llm(folder, dtype="bfloat16", max_tokens=2048, cache_dtype="e4m3")
    assert "e4m3" in llm.model_info()
    prompts = [repeating(TINY_A, 13), texts_of(TINY_A, [2], 14)[0], repeating(TINY_A, 15, 61, 3), repeating(TINY_A, 16, 66, 5)]
    results = llm.generate(prompts, dlgo_amd.with_greedy(), dlgo_amd.with_max_tokens(30), dlgo_amd.with_ignore_eos(), dlgo_amd.with_lookup_drafts(5))
    for p, r in zip(prompts, results):
        assert len(r.tokens) == 30
        x = plain_q8.forward(cfg, w, p + r.tokens)[len(p) - 1:-1]
        off = x.max(-1) - x[np.arange(30), r.tokens]
        assert (off <= 2 * TOL["A"] * np.abs(x).max()).all()
    llm.engine.cache.check_consistent()


def test_what_does_not_go_together_is_refused(folders, monkeypatch):
    import dlgo_amd
    from dlgo_amd.engine import Engine, EngineError
    from dlgo_amd.sampling import SamplerConfig
    from dlgo_amd.sampling.sampler import Sampler
    with pytest.raises(EngineError, match="bfloat16 run"):
        Engine.from_folder(folders["A", "float32"], "float32", max_tokens=128, cache_dtype="e4m3")
    with pytest.raises(EngineError, match="e5m2"):
        Engine.from_folder(folders["A", "bfloat16"], "bfloat16", max_tokens=128, cache_dtype="e5m2")
    from dlgo_amd.parts.attention import Attention
    with monkeypatch.context() as m, pytest.raises(EngineError, match="self_attn.*not something this part reads"):
        m.setattr(Attention, "cache_kernel_variants", lambda self, kv_dtype: ())
        Engine.from_folder(folders["A", "bfloat16"], "bfloat16", max_tokens=128, cache_dtype="e4m3")
    llm = dlgo_amd.load_llm(folders["A", "bfloat16"], dtype="bfloat16", max_tokens=128)
    with pytest.raises(ValueError, match="drafts are verified"):
        llm.generate([1, 2], dlgo_amd.with_lookup_drafts(2))               # the default options cut the distribution
    s = Sampler(256, "cuda:0")
    greedy, logits = SamplerConfig(temperature=0), torch.randn(3, 256, device="cuda:0")
    assert s.verify(logits, [[logits[0].argmax().item()], []], [greedy] * 2, [[0.5, 0.5], [0.5]]) == ([1, 0], logits.argmax(-1)[1:].tolist())
    assert s.verify(logits[:0], [], [], []) == ([], [])
    for args in [([[1], []], [greedy], [[0.5, 0.5], [0.5]]), ([[1], []], [greedy] * 2, [[0.5], [0.5]]), ([[1]], [greedy], [[0.5, 0.5]]),
                 ([[1], []], [greedy, SamplerConfig()], [[0.5, 0.5], [0.5]])]:
        with pytest.raises(ValueError, match="sampler"):
            s.verify(logits, *args)


def test_the_replay_program_takes_an_8_bit_cache(folders, plain_q8, tmp_path):
    cfg, w = plain.read_model(folders["A", "bfloat16"])
    (text,) = texts_of(TINY_A, [75], seed=20)
    steps = [{"step": 0, "entries": [{"id": "x", "tokens": text[:60], "want": [59]}], "end": []},
             {"step": 1, "entries": [{"id": "x", "tokens": text[60:], "want": list(range(15))}], "end": ["x"]}]
    p = subprocess.run([os.path.join(ROOT, "bin", "trace_run"), "--model", folders["A", "bfloat16"], "--dtype", "bfloat16", "--cache-dtype", "e4m3",
                        "--out", str(tmp_path), "--max-tokens", "128"], input="".join(json.dumps(s) + "\n" for s in steps),
                       capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr
    got = np.fromfile(tmp_path / "1.f32", dtype="<f4").reshape(15, -1)
    assert rel_err(torch.from_numpy(got), plain_q8.forward(cfg, w, text)[60:]) <= TOL["A"]


def test_the_command_line_takes_both(folders):
    cmd = [sys.executable, "-m", "dlgo_amd", folders["A", "bfloat16"], "--greedy", "--max-tokens", "8", "--ignore-eos",
           "--prompt-ids", "5,6,7,5,6,7,5,6", "--ctx", "128", "--cache-dtype", "e4m3", "--lookup-drafts", "3"]
    p = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr
    lines = p.stdout.splitlines()
    assert "e4m3" in lines[0]
    assert len(json.loads(next(x for x in lines if x.startswith("{")))["tokens"]) == 8
