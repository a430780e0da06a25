"""Which form a step takes whose sequences share pages, and what it keeps, without a GPU: the launches are recorded, not made."""
from types import SimpleNamespace

import pytest
import torch

from scriptling_llm_lib_b200.csrc.bindings import KernelError, SharedAttention
from scriptling_llm_lib_b200.parts.attention import Attention


def layer(heads, kv, dim, v_dim=None, **more):
    return Attention(heads * dim, heads, kv, dim, None, "q", "k", "v", "o", v_dim=v_dim, **more)


# (layer, rounds its weights in a decode step, in a step of runs), as the kernels that read each sequence for itself do
WEIGHTS = [(layer(32, 8, 64), True, True), (layer(32, 8, 128), True, True),       # grouped heads: tensor cores in either
           (layer(32, 32, 64), False, True),                                      # a head of its own: float32 in decode steps
           (layer(12, 3, 96), False, False), (layer(16, 4, 32), False, False),    # widths of which prompts keep 24 bits
           (layer(16, 4, 64, v_dim=128), False, False), (layer(10, 2, 48, v_dim=40), False, False),
           (layer(4, 2, 256), False, False),
           (layer(16, 4, 64, v_dim=128, softcap=30.0), True, True),               # capped scores: tensor cores at any such widths
           (layer(4, 2, 256, v_dim=200, softcap=30.0), False, False), (layer(4, 2, 100, softcap=30.0), False, False)]


@pytest.mark.parametrize("part, decode, runs", WEIGHTS)
def test_a_step_that_shares_pages_keeps_the_weights_that_each_sequence_for_itself_has(part, decode, runs):
    seen = []
    ctx = SimpleNamespace(kernels=SimpleNamespace(shared=SimpleNamespace(attn=lambda *a, **k: seen.append(k["exact_weights"]))), tok_pos=None, err_flag=None)
    plan = SimpleNamespace(part_floats=lambda v_dim: 4)
    for ctx.is_decode in (True, False):
        part._attend_shared(plan, torch.zeros(3, part.n_heads * part.head_dim), ctx, None, None, None)
    assert seen == [not decode, not runs]


@pytest.mark.parametrize("scale, softcap", [(0.0, None), (-0.125, None), (float("nan"), None), (float("inf"), None), (0.125, -30.0),
                                            (0.125, float("nan")), (0.125, float("inf"))])
def test_scales_and_caps_that_are_no_numbers_above_zero_are_refused(scale, softcap):
    ops = SharedAttention.__new__(SharedAttention)            # (no library is loaded for a refusal)
    with pytest.raises(KernelError, match="scale above 0"):
        ops.attn(None, None, None, None, None, None, None, None, scale, None, softcap=softcap)


BF16, F32 = torch.bfloat16, torch.float32
# (layer, shares pages in bfloat16 decode steps, in steps of runs)
SHARES = [(layer(32, 8, 64), True, True), (layer(16, 4, 64, v_dim=128, softcap=30.0), True, True), (layer(10, 2, 48, v_dim=40), True, True),
          (layer(32, 8, 192, v_dim=128), True, False),                            # runs for themselves on the tensor cores, single tokens not
          (layer(32, 8, 192, v_dim=128, softcap=30.0), False, False),             # either for itself on the tensor cores
          (layer(16, 4, 256), True, True), (layer(32, 8, 100), True, True), (layer(16, 16, 192), True, True),      # all on FMA
          (layer(16, 4, 64, window=100), False, False)]


@pytest.mark.parametrize("part, decode, runs", SHARES)
def test_pages_are_not_shared_on_slower_units_than_each_sequence_for_itself_has(part, decode, runs):
    widths = (part.n_heads, part.head_dim, part.v_dim)
    assert part.shares_pages(BF16, True) == (widths if decode else None) and part.shares_pages(BF16, False) == (widths if runs else None)
    assert part.shares_pages(F32, True) == part.shares_pages(F32, False) == (None if part.span else widths)
    asked = []
    ctx = SimpleNamespace(share_plan=lambda unit, *w: asked.append(w), dtype=BF16)
    for ctx.is_decode in (True, False):
        part._share_plan(ctx, 0)
    assert asked == [widths] * (decode + runs)


def engine(parts, dtype, tables, held, kv_heads):
    """An engine of these layers whose sequences hold these pages, as far as its choices go."""
    import numpy as np
    from scriptling_llm_lib_b200.cache.share import share_tree
    from scriptling_llm_lib_b200.engine.step import Engine
    need = SimpleNamespace(kind="full", kv_heads=kv_heads)
    groups = [SimpleNamespace(need=need, pool=SimpleNamespace(n_shared=1)) for _ in tables]
    trees = [share_tree(np.asarray(t, dtype=np.int32), np.asarray(held) // 64) for t in tables]
    eng = Engine.__new__(Engine)
    eng.dtype, eng._sharing, eng.sm_count, eng.kernels = dtype, {}, 148, SimpleNamespace(shared=SharedAttention.__new__(SharedAttention))
    eng.kernels.shared.dtype = dtype
    eng.cache = SimpleNamespace(groups=groups, group_of_unit={i: min(i, len(tables) - 1) for i in range(len(parts))}, shares_pages=True,
                                share_tree=lambda g, slots: trees[g])
    eng.layout = SimpleNamespace(schedule=[SimpleNamespace(cache_unit=i, layer=i) for i in range(len(parts))])
    eng.model = SimpleNamespace(blocks=[SimpleNamespace(parts=lambda p=p: [p]) for p in parts])
    return eng


def table(n, shared, own):
    return [list(range(shared)) + list(range(shared + i * own, shared + (i + 1) * own)) for i in range(n)]


def test_wide_bfloat16_runs_are_not_charged_the_tensor_cores_price():
    """16 runs of 150 tokens behind 8,000, keys of 192 and values of 128: on FMA about four times what each for itself takes. Single tokens
    behind as many go by 32-bit's line: 64 of them, not 4."""
    for n, new, part, want in ((16, 150, layer(32, 8, 192, v_dim=128), False), (64, 1, layer(32, 8, 192, v_dim=128), True),
                               (16, 150, layer(32, 8, 128), True), (4, 1, layer(32, 8, 192, v_dim=128), False)):
        held = [8040] * n
        eng = engine([part] * 24, BF16, [table(n, 125, 4)], held, 8)
        assert bool(eng._shares(list(range(n)), held, [new] * n, kept=new == 1)) is want


def test_each_layer_shares_pages_by_its_own_gain():
    """Two kinds of layers in a step: eight keys a token that 16 sequences share, and one. Reading the one once for all is worth less than the
    partial results that it leaves; only the layers that gain have a plan, and only they are captured for it."""
    from scriptling_llm_lib_b200.engine.step import SharedStep
    n, held = 16, [4040] * 16
    eng = engine([layer(32, 32, 64), layer(32, 1, 64)], BF16, [table(n, 62, 4)] * 2, held, 32)
    eng.cache.groups[1].need = SimpleNamespace(kind="full", kv_heads=1)
    shared = eng._shares(list(range(n)), held, [1] * n, kept=True)
    assert shared == ((0, 32, 64, 64),)
    step = SharedStep(eng, shared, list(range(n)), held, [1] * n)
    step._build = lambda key: SimpleNamespace(part_floats=lambda v_dim: 0, key=key)
    assert step.plan(0, 32, 64, 64).key == (0, 32, 64, 64) and step.plan(1, 32, 64, 64) is None


def test_the_scratch_of_a_plan_is_known_before_it_is_laid_out():
    import random
    from scriptling_llm_lib_b200.cache import SharePlan, TileShape, most_part_rows, share_tree
    from test_share_cpu import _batch
    import numpy as np
    rng = random.Random(5)
    for shape in (TileShape(256, 148, True, 5.0, ((128, 0.85),), 2, 16, 8, 0.3, 1.0, 4.0), TileShape(64, 296, min_pages=1), TileShape(64, 148, costs=((4, 0.25),)), TileShape(16, 40, True)):
        for n in (1, 2, 5, 23, 60, 200):
            for runs in (False, True):
                G, rep = rng.choice([1, 2, 8]), rng.choice([1, 3, 4, 8])
                tables, held, new = _batch(rng, n, rep, runs)
                tree = share_tree(tables, np.asarray(held) // 64)
                rows = SharePlan.build(tables, held, new, G * rep, G, shape, None).part_rows
                most = most_part_rows(tree, new, G * rep, G, shape)
                assert rows <= most <= rows + shape.workers * (shape.rows + shape.thin_rows * shape.thin_warps)


def prompts(n, new, prefix, part, kv, layers):
    """An engine of such layers, entries of `new` tokens for each of `n` sequences behind a common prefix."""
    held = [prefix + 40] * n
    eng = engine([part] * layers, BF16, [table(n, prefix // 64, 2)], held, kv)
    full = eng.cache.groups[0]
    from scriptling_llm_lib_b200.cache.share import share_tree
    import numpy as np
    t = np.asarray(table(n, prefix // 64, 2), dtype=np.int32)
    eng.cache.share_tree = lambda g, slots: share_tree(t[list(slots)], np.full(len(slots), held[0] // 64))
    assert full.pool.n_shared
    return eng, [SimpleNamespace(sequence=SimpleNamespace(slot=i, length=held[0], closed=False, engine=eng), tokens=list(range(new))) for i in range(n)], held


@pytest.mark.parametrize("n, new, prefix", [(200, 32, 4096), (250, 32, 16384), (256, 40, 16384), (400, 40, 16384)])
def test_long_batches_of_questions_go_in_portions_whose_partial_results_fit(n, new, prefix):
    """32 heads of 128 on 8, 32 layers: 320 to 526 MB of partial results in one step, which is then each sequence for itself."""
    from scriptling_llm_lib_b200.cache import SharePlan
    import numpy as np
    eng, entries, held = prompts(n, new, prefix, layer(32, 8, 128), 8, 32)
    assert eng._gains(range(n), held, [new] * n) and not eng._shares(range(n), held, [new] * n)
    done, first, steps = [0] * n, 0, 0
    while first < n:
        takes = eng._portion(entries, done, first, 16384)
        slots, new_here = [i for i, _ in takes], [k for _, k in takes]
        assert slots == list(range(first, first + len(takes))) and all(k > 0 for k in new_here)
        assert eng._shares(slots, [held[0]] * len(slots), new_here) == ((0, 32, 128, 128),)
        plan = SharePlan.build(np.asarray(table(n, prefix // 64, 3), dtype=np.int32)[slots], [held[0]] * len(slots), new_here, 32, 8,
                               eng.kernels.shared.shape(128, 128, 148), None)
        assert 4 * plan.part_floats(128) <= SharedAttention.SCRATCH_BYTES
        for i, k in takes:
            done[i] += k
        while first < n and done[first] == new:
            first += 1
        steps += 1
    assert done == [new] * n and 2 <= steps <= 5


def test_a_captured_step_whose_partial_results_do_not_fit_is_not_captured_again():
    eng, _, held = prompts(1024, 1, 4096, layer(64, 8, 128), 8, 32)
    assert eng._gains(range(1024), held, [1] * 1024, kept=True) and eng._shares(range(1024), held, [1] * 1024, kept=True) == ()
    assert eng._shares(range(256), held[:256], [1] * 256, kept=True) == ((0, 64, 128, 128),)


def test_prompts_that_share_nothing_go_in_portions_of_the_budget():
    eng, entries, _ = prompts(6, 100, 4096, layer(32, 8, 128), 8, 32)
    eng.cache.shares_pages = False
    assert eng._portion(entries, [0, 30, 0, 0, 0, 0], 1, 250) == [(1, 70), (2, 100), (3, 80)]
    assert eng._portion(entries, [0] * 6, 0, 10 ** 6) == [(i, 100) for i in range(6)] and eng._portion(entries, [0] * 6, 5, 1) == [(5, 1)]


def test_only_requests_that_share_pages_keep_room_for_their_partial_results(monkeypatch):
    """The cache of requests that share nothing is as large as it would be without shared attention."""
    from scriptling_llm_lib_b200 import llm
    from scriptling_llm_lib_b200.engine.step import Engine
    part = layer(32, 8, 64)
    eng = engine([part] * 2, BF16, [table(2, 4, 1)], [300] * 2, 8)
    eng.model.parts, eng.use_graphs = lambda: [part], False
    eng.layout.hidden_size, eng.layout.vocab_size, eng.layout.max_positions = 2048, 512, 4096
    plain = Engine.activation_reserve_bytes(eng)
    assert Engine.activation_reserve_bytes(eng, sharing=True) == plain + SharedAttention.SCRATCH_BYTES and part.scratch_bytes(16384) == 0
    window = layer(32, 8, 64, window=128)
    other = engine([window], BF16, [table(2, 4, 1)], [300] * 2, 8)
    other.model.parts, other.use_graphs, other.layout.hidden_size, other.layout.vocab_size = lambda: [window], False, 2048, 512
    assert Engine.activation_reserve_bytes(other, sharing=True) == Engine.activation_reserve_bytes(other) == plain
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (1 << 30, 1 << 31))
    eng.device, eng.cache.n_pages, eng.cache.n_slots, sizes = None, 1, 1, []
    eng.bytes_per_page = lambda: 1 << 16
    eng.activation_reserve_bytes = lambda sharing=False: (1 << 28) + (SharedAttention.SCRATCH_BYTES if sharing else 0)
    eng.resize_cache = lambda tokens, seqs: sizes.append(tokens // 64)
    for how in (dict(), dict(n=2), dict(share_prefix=True)):
        llm._fit_cache(eng, [[1] * 4000] * 1000, 50, None, **how)
    assert sizes[0] > sizes[1] == sizes[2]


def test_a_plan_on_the_host_alone_is_refused():
    import numpy as np
    from scriptling_llm_lib_b200.cache import SharePlan, TileShape
    plan = SharePlan.build(np.zeros((2, 3), dtype=np.int32), [10, 20], [1, 1], 4, 2, TileShape(64, 10), None)
    ops = SharedAttention.__new__(SharedAttention)
    with pytest.raises(KernelError, match="host alone"):
        ops.attn(None, None, None, None, None, None, plan, None, 0.125, None)
