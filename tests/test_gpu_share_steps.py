"""Steps of sequences that share pages, and which of them the shared kernel ran in: its calls are counted."""
import pytest
import torch

from helpers import random_ids
from scriptling_llm_lib_b200.csrc.bindings import SharedAttention
from scriptling_llm_lib_b200.engine import StepEntry
from test_gpu_fork import LLAMA, alone, engine, rel_err, tol

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def shares_whatever_it_costs(monkeypatch):
    monkeypatch.setattr("scriptling_llm_lib_b200.engine.step.share_pays", lambda tree, *a: bool(tree and tree[1]))


@pytest.fixture
def calls(monkeypatch):
    """(rows, sequences) of every call of the shared kernel."""
    seen, attn = [], SharedAttention.attn

    def counted(self, q, out, tok_pos, block_table, kpages, vpages, plan, *a, **k):
        seen.append((plan.n_rows, plan.n_seqs))
        return attn(self, q, out, tok_pos, block_table, kpages, vpages, plan, *a, **k)
    monkeypatch.setattr(SharedAttention, "attn", counted)
    return seen


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_batch_whose_partial_results_do_not_fit_goes_in_portions_that_share(tmp_path, monkeypatch, calls, dtype):
    eng = engine(tmp_path, LLAMA, dtype, max_tokens=16384, max_seqs=40)
    V, layers = LLAMA["vocab_size"], LLAMA["num_hidden_layers"]
    front = random_ids(700, V, 1)
    root = eng.open()
    eng.step([StepEntry(root, front)])
    seqs = [root] + root.fork(23)
    entries = [StepEntry(s, random_ids(11 + i, V, 100 + i)) for i, s in enumerate(seqs)]
    rows = sum(len(e.tokens) for e in entries)
    key = next(iter(eng._share_groups(False)))
    takes = lambda some: dict(eng._gains([e.sequence.slot for e in some], [700] * len(some), [len(e.tokens) for e in some]))[key]      # noqa: E731
    assert takes(entries[:18]) < takes(entries)
    monkeypatch.setattr(SharedAttention, "SCRATCH_BYTES", takes(entries[:18]))
    logits, _ = eng.prompt_step(entries)
    steps = [c for i, c in enumerate(calls) if i % layers == 0]
    assert 2 <= len(steps) <= 3 and sum(r for r, _ in steps) == rows and len(calls) == layers * len(steps)
    for i in (0, 7, 23):
        assert rel_err(logits[i], alone(eng, front + entries[i].tokens)) < tol(dtype)
    calls.clear()
    monkeypatch.setattr(SharedAttention, "SCRATCH_BYTES", 1000)          # nothing fits: each for itself, and no second capture
    before = len(eng.decode_graphs.graphs)
    out = eng.step([StepEntry(s, [1 + i]) for i, s in enumerate(seqs)])
    assert not calls and ["shared" in k for k in eng.decode_graphs.graphs][before:] == [False]
    assert rel_err(out[7], alone(eng, front + entries[7].tokens + [8])) < tol(dtype)
    for s in seqs:
        s.close()


def test_a_trace_that_forks_what_is_not_live_ends_with_a_message(tmp_path):
    import json
    import subprocess
    import sys
    from pathlib import Path
    from helpers import make_model_dir
    d = make_model_dir(tmp_path / "m", LLAMA, 3)
    records = [{"step": 0, "entries": [{"id": "a", "tokens": [1, 2], "want": []}], "end": ["a"]}, {"step": 1, "fork": [{"id": "b", "of": "a"}]}]
    run = subprocess.run([sys.executable, str(Path(__file__).resolve().parent.parent / "bin" / "trace_run"), "--model", str(d), "--dtype", "float32", "--out",
                          str(tmp_path / "o"), "--max-tokens", "640"], input="\n".join(json.dumps(r) for r in records), capture_output=True, text=True, timeout=300)
    assert run.returncode != 0 and "done 0" in run.stdout
    assert "the request 'a' to fork is not live" in run.stderr and "Traceback" not in run.stderr


def test_a_plan_goes_to_the_device_without_waiting_for_what_is_queued():
    from scriptling_llm_lib_b200.cache import SharePlan
    from scriptling_llm_lib_b200.csrc.bindings import KernelSet
    from test_gpu_share import B16, Case
    c = Case("runs", (16, 4, 64, 64), B16)
    want, shape = c.run(), KernelSet(B16).shared.shape(64, 64)
    done = torch.cuda.Event()
    torch.cuda._sleep(400_000_000)                                     # about 0.2 s
    done.record()
    plan = SharePlan.build(c.table, c.held, c.new, 16, 4, shape, "cuda", queued=True)
    assert not done.query()
    others = [torch.zeros(n, dtype=torch.int32).pin_memory() for n in (plan.dev.numel(),) * 4]      # (its pinned memory is not handed on meanwhile)
    for t in others:
        t.fill_(-1)
    assert torch.equal(c.run(plan), want)


def followed(calls, eng, dtype, vocab, prompt, n=5):
    """What `follow` of test_gpu_fork.py checks, and the calls for steps of single tokens and for steps of runs."""
    from test_gpu_fork import follow
    follow(eng, dtype, vocab, prompt, depth=1, n=n)
    single = sum(rows == seqs for rows, seqs in calls)
    return single, len(calls) - single


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False], ids=["replayed", "launched"])
@pytest.mark.parametrize("name", ["LLAMA", "WIDE", "ODD", "WINDOW"])
def test_every_layer_that_sees_all_keys_reads_shared_pages_once(tmp_path, calls, name, dtype, graphs):
    import test_gpu_fork
    raw = getattr(test_gpu_fork, name)
    eng = engine(tmp_path, raw, dtype, use_graphs=graphs)
    single, runs = followed(calls, eng, dtype, raw["vocab_size"], random_ids(700, raw["vocab_size"], 7))
    if name == "WINDOW":
        assert single == runs == 0
    else:
        layers = raw["num_hidden_layers"]
        assert runs == 2 * layers                                  # two steps of runs, not captured
        assert single > 0 and single % layers == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["sozilix", "muvorax", "belasun", "tufazen", "fopezen", "debusun"])
def test_architectures_whose_layers_see_all_keys_share_them(tmp_path, calls, name, dtype):
    """Two of them: the others' layers have windows or chunks, latent keys, or widths that the shared kernels do not take."""
    from test_gpu_fork import other_architectures
    raw = other_architectures()[name]
    eng = engine(tmp_path, raw, dtype, max_tokens=4096, max_seqs=12)
    vocab = eng.layout.vocab_size
    single, runs = followed(calls, eng, dtype, vocab, random_ids(min(330, eng.max_positions - 40), vocab, 5), n=3)
    assert (single > 0, runs > 0) == (name in ("belasun", "tufazen"),) * 2


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_of_requests_that_share_reads_shared_pages_once(tmp_path, calls, dtype):
    from helpers import make_model_dir
    from scriptling_llm_lib_b200 import llm
    d = make_model_dir(tmp_path / "m", LLAMA, 3)
    V = LLAMA["vocab_size"]
    front = random_ids(300, V, 1)
    prompts = [front + random_ids(n, V, 50 + n) for n in (5, 90, 17)]
    llm.unload()
    kw = dict(dtype=dtype, stop_ids=[], temperature=0.0)
    llm.generate(d, prompts, 6, **kw)
    assert not calls
    llm.generate(d, prompts, 6, share_prefix=True, **kw)
    assert any(rows > seqs for rows, seqs in calls) and any(rows == seqs for rows, seqs in calls)      # the questions, then their answers
    calls.clear()
    llm.unload()                                                      # (its captured steps with it)
    llm.generate(d, prompts[0], 6, n=4, **kw)
    assert any(rows == seqs for rows, seqs in calls)
    llm.unload()


def test_a_plan_that_is_not_queued_is_there_for_any_stream():
    from scriptling_llm_lib_b200.cache import SharePlan
    from scriptling_llm_lib_b200.csrc.bindings import KernelSet
    from test_gpu_share import B16, Case
    c = Case("runs", (16, 4, 64, 64), B16)
    want, shape, side = c.run(), KernelSet(B16).shared.shape(64, 64), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)                                     # the current stream is busy; the other one is not
    plan = SharePlan.build(c.table, c.held, c.new, 16, 4, shape, "cuda")
    with torch.cuda.stream(side):
        got = c.run(plan)
    side.synchronize()
    assert torch.equal(got, want)


def test_prompts_of_closed_or_foreign_sequences_are_refused_beside_shared_ones(tmp_path):
    from scriptling_llm_lib_b200.engine.step import StepError
    eng, other = engine(tmp_path, LLAMA, "bfloat16", max_seqs=6), engine(tmp_path, LLAMA, "bfloat16", max_seqs=6)
    root = eng.open()
    eng.step([StepEntry(root, random_ids(300, LLAMA["vocab_size"], 1))])
    seqs = [root] + root.fork(3)
    seqs[2].close()
    for wrong in (seqs[2], other.open()):
        for budget in (None, 3):
            with pytest.raises(StepError, match="closed or belongs to another engine"):
                eng.prompt_step([StepEntry(seqs[0], [1, 2]), StepEntry(wrong, [3, 4])], budget)
