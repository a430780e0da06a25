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


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("seqs", [3, 620])
def test_a_row_that_sees_nothing_is_zero_however_deep_its_sink(dtype, seqs):
    """Keys of minus infinity weigh nothing; the sink is all there is. Few outputs (a block each) and many (a warp each)."""
    c = Case([(path(), 3 + i % 5, 1) for i in range(seqs)], (16, 4, 64, 64), dtype, junk=False)
    blind = torch.arange(c.T, device="cuda") % 3 == 0
    for b in np.flatnonzero(blind.cpu()):
        c.k[c.table[b, 0], :, :, 0] = -torch.inf
    c.q.view(c.T, 16, 64)[..., 0] = 1.0
    for depth in (-3.0, -80.0, -200.0, -1e30):
        sink = torch.full((16,), depth, device="cuda")
        got = c.run(sink=sink)
        assert torch.isfinite(got.float()).all() and not got[blind].float().any()
        want, mean, S, n = c.formula(sink=sink)
        off = (got.double().view_as(want) - want).abs()[~blind]
        u = 2.0 ** -24
        slack = 4 * u * ((64 + 8) * S[..., None] + n[:, None, None] + 8) * mean + (2.0 ** -8 * (mean + want.abs()) if dtype == B16 else 0) + 1e-30
        assert bool((off <= slack[~blind]).all())


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_a_block_table_narrower_than_the_plan_is_refused(dtype):
    from scriptling_llm_lib_b200.csrc.bindings import KernelError
    c = Case("nested", (16, 4, 64, 64), dtype)
    good, plan = c.run(), c.plan()
    wide = c.table
    c.table = np.ascontiguousarray(wide[:, :-1])
    with pytest.raises(KernelError, match="pages"):
        c.run(plan)
    c.table = np.concatenate([wide, np.full((len(wide), 3), -1, dtype=np.int32)], axis=1)
    assert torch.equal(c.run(plan), good)
