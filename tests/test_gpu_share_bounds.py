"""Attention over shared pages where a position is outside the block table, or a row sees nothing at all."""
import numpy as np
import pytest
import torch

from scriptling_llm_lib_b200.cache import SharePlan
from scriptling_llm_lib_b200.csrc.bindings import KernelSet
from test_gpu_share import B16, F, Case, path

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("batch", ["nested", "runs"])
@pytest.mark.parametrize("layout", [(16, 4, 64, 64), (16, 4, 64, 128), (32, 8, 128, 128)], ids=str)
def test_a_position_outside_the_table_is_reported_and_the_other_rows_go_on(dtype, batch, layout):
    """Below 0 and past the last page, up to the largest 32-bit number: no page that is not there is looked for, however far."""
    c = Case(batch, layout, dtype, junk=False)
    good, plan, ops = c.run(), c.plan(), KernelSet(dtype).shared
    b = 3
    rows = slice(sum(c.new[:b]), sum(c.new[:b + 1]))
    other = torch.ones(c.T, dtype=torch.bool, device="cuda")
    other[rows] = False
    table = torch.from_numpy(c.table).cuda()
    for bad in (-1, -40, -64, -(1 << 31), 64 * c.width + c.new[b], 1 << 30, (1 << 31) - 1):
        pos = c.pos.clone()
        pos[rows] = bad
        err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty_like(good)
        ops.attn(c.q, out, pos, table, c.k, c.v, plan, torch.empty(plan.part_floats(c.vd), device="cuda"), c.scale, err)
        assert int(err) != 0 and torch.equal(out[other], good[other])
