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
