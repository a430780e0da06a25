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
    eng.dtype, eng._sharing = dtype, {}
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
