"""Sequences forked from one another, through the engine, the generation loop and trace replay: their steps read shared pages once, and
give what the same tokens give in a sequence of their own."""
import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from helpers import TINY, TOL_BF16, TOL_F32, make_model_dir, random_ids
from helpers import rel_err as _rel_err
from scriptling_llm_lib_b200 import llm
from scriptling_llm_lib_b200.cache import CacheFull
from scriptling_llm_lib_b200.engine import Engine, StepEntry
from scriptling_llm_lib_b200.engine.step import StepError

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

# every earlier key seen, grouped heads of 64 and 128, and a width off the tensor-core kernels' steps
LLAMA = dict(TINY["D"][0], sliding_window=None, max_position_embeddings=2048)
WIDE = dict(TINY["E"][0], sliding_window=None, max_position_embeddings=2048)
ODD = dict(TINY["C"][0], sliding_window=None, max_position_embeddings=2048, head_dim=20)
WINDOW = dict(TINY["D"][0], max_position_embeddings=2048)


def other_architectures():
    import importlib
    return {name: importlib.import_module(f"test_{name}_cpu").RAW for name in ("sozilix", "muvorax", "belasun", "tufazen", "fopezen", "debusun")}


def engine(tmp_path, raw, dtype, max_tokens=8192, max_seqs=32, **kw):
    path = tmp_path / "config.json"
    path.write_text(json.dumps(raw))
    return Engine.from_folder(f"random:{path}:3", dtype, max_tokens=max_tokens, max_seqs=max_seqs, **kw)


@pytest.fixture(autouse=True)
def shares_whatever_it_costs(monkeypatch, request):
    """The tests' models are too small for shared reading to pay: here it does wherever sequences share a page."""
    if "by_the_estimate" not in request.node.name:
        monkeypatch.setattr("scriptling_llm_lib_b200.engine.step.share_pays", lambda tree, *a: bool(tree and tree[1]))


def rel_err(got, want):
    return _rel_err(got.cpu(), want.cpu())


def tol(dtype):
    return TOL_F32 if dtype == "float32" else TOL_BF16


def alone(eng, tokens):
    s = eng.open()
    out = eng.step([StepEntry(s, tokens)])[0]
    s.close()
    return out


def follow(eng, dtype, vocab, prompt, depth, n=5, steps=4):
    """A prompt, forks of it, forks of a fork, runs of tokens and single ones in turn; every step's logits against the tokens alone."""
    held = {}
    root = eng.open()
    eng.step([StepEntry(root, prompt)])
    held[root] = list(prompt)
    for k, s in enumerate(root.fork(n)):
        held[s] = list(prompt)
    for k in range(steps):
        entries = []
        for j, s in enumerate(held):
            new = random_ids(1 if k % 2 == 0 else 1 + (7 * j + k) % 9, vocab, 1000 * k + j)
            entries.append(StepEntry(s, new))
        logits = eng.step(entries)
        eng.check_errors()
        for e, row in zip(entries, logits):
            held[e.sequence] += e.tokens
            if (k + len(held[e.sequence])) % 3 == 0:
                assert rel_err(row, alone(eng, held[e.sequence])) < tol(dtype)
        if k == depth:
            some = list(held)[1]
            for s in some.fork(2):
                held[s] = list(held[some])
            list(held)[2].close()
            del held[list(held)[2]]
    for s, tokens in held.items():
        assert s.length == len(tokens)
        s.close()
    assert eng.cache.slots.n_held == 0 and all(g.pool.n_held == 0 and g.pool.n_shared == 0 for g in eng.cache.groups)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False], ids=["replayed", "launched"])
@pytest.mark.parametrize("raw", [LLAMA, WIDE, ODD, WINDOW], ids=["grouped64", "one128", "odd20", "window"])
def test_forks_go_on_as_sequences_of_their_own(tmp_path, raw, dtype, graphs):
    eng = engine(tmp_path, raw, dtype, use_graphs=graphs)
    for n in (700, 64 * 8, 64 * 9 + 1):
        follow(eng, dtype, raw["vocab_size"], random_ids(n, raw["vocab_size"], n), depth=1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["sozilix", "muvorax", "belasun", "tufazen", "fopezen", "debusun"])
def test_forks_of_every_architecture(tmp_path, name, dtype):
    raw = other_architectures()[name]
    eng = engine(tmp_path, raw, dtype, max_tokens=4096, max_seqs=12)
    vocab = eng.layout.vocab_size
    follow(eng, dtype, vocab, random_ids(min(330, eng.max_positions - 40), vocab, 5), depth=1, n=3)


def test_the_captured_step_reads_shared_pages_once(tmp_path):
    """The captured step of forked sequences launches the shared kernel in the layers that see every key, and keeps doing so as the
    batch changes; a batch that shares nothing keeps the step it had."""
    eng = engine(tmp_path, LLAMA, "bfloat16")
    V = LLAMA["vocab_size"]
    root = eng.open()
    eng.step([StepEntry(root, random_ids(900, V, 1))])
    others = [eng.open() for _ in range(4)]
    for i, s in enumerate(others):
        eng.step([StepEntry(s, random_ids(900, V, 2 + i))])
    eng.step([StepEntry(s, [1]) for s in others])
    assert ["shared" in k for k in eng.decode_graphs.graphs] == [False]
    forks = root.fork(7)
    for i in range(70):                                  # past the ends of pages: the plan is laid out again
        eng.step([StepEntry(s, [(i + j) % V]) for j, s in enumerate([root] + forks)])
    assert ["shared" in k for k in eng.decode_graphs.graphs] == [False, True]
    graph = eng.decode_graphs.last_graph
    assert graph.ctx.share is not None and any(p is not None for p in graph.ctx.share.plans.values())
    want = [alone(eng, random_ids(900, V, 1) + [(i + j) % V for i in range(70)] + [5]) for j in (0, 3, 7)]
    got = eng.step([StepEntry(s, [5]) for s in [root] + forks])
    assert all(rel_err(got[j], w) < TOL_BF16 for j, w in zip((0, 3, 7), want))
    three = eng.step([StepEntry(s, [6]) for s in forks[:3]])            # fewer than the captured rows: the batch is filled up
    assert rel_err(three[1], alone(eng, random_ids(900, V, 1) + [(i + 2) % V for i in range(70)] + [5, 6])) < TOL_BF16
    for s in [root] + forks + others:
        s.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_compaction_leaves_sequences_as_they_are(tmp_path, dtype):
    eng = engine(tmp_path, WINDOW if dtype == "float32" else LLAMA, dtype, max_tokens=6400, max_seqs=16)
    V = LLAMA["vocab_size"]
    seqs = [eng.open() for _ in range(8)]
    tokens = {s: random_ids(100 + 70 * i, V, i) for i, s in enumerate(seqs)}
    eng.step([StepEntry(s, t) for s, t in tokens.items()])
    for s in seqs[::2]:
        s.close()
        del tokens[s]
    for s in seqs[1].fork(2):
        tokens[s] = list(tokens[seqs[1]])

    def go_on(k):
        rows = eng.step([StepEntry(s, [k]) for s in tokens])
        eng.check_errors()
        for (s, t), row in zip(tokens.items(), rows):
            t.append(k)
            assert rel_err(row, alone(eng, t)) < tol(dtype)
    go_on(3)
    assert eng.compact() > 0 and eng.compact() == 0
    go_on(4)
    bytes_before = sum(g.k.numel() for g in eng.cache.groups)
    held = max(g.pool.n_held for g in eng.cache.groups)
    eng.compact((held + 20) * 64)                          # smaller
    assert sum(g.k.numel() for g in eng.cache.groups) < bytes_before and eng.cache.n_pages == held + 20
    go_on(5)
    eng.compact(9600)                                      # larger
    go_on(6)
    for wrong, error in ((64, (StepError, CacheFull)), (64 * (held - 1), (StepError, CacheFull))):
        with pytest.raises(error):
            eng.compact(wrong)
    go_on(7)
    for s in tokens:
        s.close()


def test_a_step_shares_by_the_estimate_alone(tmp_path):
    """A tiny model's forks go on by the steps they had; with the weight of a long context the estimate turns."""
    from scriptling_llm_lib_b200.cache import share_pays
    eng = engine(tmp_path, LLAMA, "bfloat16")
    root = eng.open()
    eng.step([StepEntry(root, random_ids(900, LLAMA["vocab_size"], 1))])
    seqs = [root] + root.fork(5)
    eng.step([StepEntry(s, [i]) for i, s in enumerate(seqs)])
    assert ["shared" in k for k in eng.decode_graphs.graphs] == [False]
    tree = eng.cache.share_tree(0, [s.slot for s in seqs])
    assert not share_pays(tree, [901] * 6, [1] * 6, 4, 2, 128, False) and share_pays(tree, [901] * 6, [1] * 6, 128, 128, 256, False)
    for s in seqs:
        s.close()


def test_refusals_of_forks(tmp_path):
    eng, other = engine(tmp_path, LLAMA, "bfloat16", max_seqs=4), engine(tmp_path, LLAMA, "bfloat16", max_seqs=4)
    s = eng.open()
    with pytest.raises(StepError):
        other.fork(s)
    with pytest.raises(CacheFull):
        s.fork(4)
    assert eng.cache.slots.n_held == 1
    a = s.fork()[0]                                        # of an empty sequence
    out = eng.step([StepEntry(s, [1, 2]), StepEntry(a, [1, 2])])
    assert rel_err(out[0], out[1]) < TOL_BF16
    s.close()
    with pytest.raises(StepError):
        s.fork()
    assert rel_err(eng.step([StepEntry(a, [3])])[0], alone(eng, [1, 2, 3])) < TOL_BF16


# --------------------------------------------------------------------------- generation, command line, trace replay
def test_continuations_and_shared_prefixes_through_the_entry_point(tmp_path):
    d = make_model_dir(tmp_path / "m", LLAMA, 3)
    V = LLAMA["vocab_size"]
    front = random_ids(300, V, 1)
    prompts = [front + random_ids(n, V, 50 + n) for n in (5, 90, 17)] + [random_ids(40, V, 9)]
    llm.unload()
    kw = dict(dtype="float32", stop_ids=[], seed=4)
    sampled = dict(strategy="temperature", temperature=1.0, repeat_penalty=0.0)
    for how in (dict(temperature=0.0), sampled):
        flat = llm.generate(d, [p for p in prompts for _ in range(3)], 9, **how, **kw)
        got, st = llm.generate(d, prompts, 9, n=3, stats=True, **how, **kw)
        assert [o for outs in got for o in outs] == flat and st["prompt_tokens"] == [[len(p)] * 3 for p in prompts]
        assert llm.generate(d, prompts, 9, share_prefix=True, **how, **kw) == llm.generate(d, prompts, 9, **how, **kw)
        both = llm.generate(d, prompts, 9, n=3, share_prefix=True, max_batch=5, **how, **kw)
        assert [o for outs in both for o in outs] == flat
    assert len({tuple(o) for o in flat[:3]}) == 3                          # three streams, three continuations
    one, st = llm.generate(d, prompts[0], 9, n=2, stats=True, **sampled, **kw)
    assert one == flat[:2] and st["generated_tokens"] == [9, 9]
    eng, _ = llm.load(d, "float32")
    assert eng.cache.slots.n_held == 0 and all(g.pool.n_held == 0 for g in eng.cache.groups)
    with pytest.raises(ValueError):
        llm.generate(d, prompts[0], 9, n=0, **kw)
    low = llm.generate(d, prompts, 6, n=8, share_prefix=True, dtype="bfloat16", stop_ids=[], temperature=0.0)
    assert all(len(o) == 6 for outs in low for o in outs)
    llm.unload()


def test_the_command_line_prints_every_continuation(tmp_path):
    d = make_model_dir(tmp_path / "m", LLAMA, 3)
    prompt = " ".join(str(t) for t in random_ids(130, LLAMA["vocab_size"], 8))
    run = subprocess.run([sys.executable, str(ROOT / "bin" / "sllm-b200"), "-model", str(d), "-prompt", f"{prompt};{prompt} 7", "-tokens", "4", "-n", "3",
                          "-share-prefix", "-strategy", "temperature", "-stop", ""], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    lines = run.stdout.strip().splitlines()
    assert len(lines) == 6 and all(len(line.split()) == 4 for line in lines) and "generated   24 tokens" in run.stderr


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replay_of_a_trace_that_forks(tmp_path, dtype):
    d = make_model_dir(tmp_path / "m", LLAMA, 3)
    V = LLAMA["vocab_size"]
    a = random_ids(200, V, 3)
    records = [{"step": 0, "entries": [{"id": "a", "tokens": a, "want": [199]}]},
               {"step": 1, "fork": [{"id": "b", "of": "a"}, {"id": "c", "of": "b"}],
                "entries": [{"id": i, "tokens": [t], "want": [0]} for i, t in (("a", 4), ("b", 5), ("c", 6))], "end": ["b"]},
               {"step": 2, "entries": [{"id": "c", "tokens": [7, 8], "want": [0, 1]}, {"id": "a", "tokens": [9], "want": [0]}], "end": ["a", "c"]},
               {"step": 3, "entries": [{"id": "x", "tokens": a + [5], "want": [200]}], "end": ["x"]},
               {"step": 4, "entries": [{"id": "x", "tokens": a + [6, 7, 8], "want": [200, 201, 202]}], "end": ["x"]}]
    run = subprocess.run([sys.executable, str(ROOT / "bin" / "trace_run"), "--model", str(d), "--dtype", dtype, "--out", str(tmp_path / "o"), "--max-tokens",
                          "1200"], input="\n".join(json.dumps(r) for r in records), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    rows = [torch.from_file(str(tmp_path / "o" / f"{i}.f32"), size=n * V).view(n, V) for i, n in enumerate((1, 3, 3, 1, 3))]
    assert rel_err(rows[1][1], rows[3][0]) < tol(dtype) and rel_err(rows[1][2], rows[4][0]) < tol(dtype) and rel_err(rows[2][:2], rows[4][1:]) < tol(dtype)
