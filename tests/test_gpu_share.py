"""Attention over pages that sequences share, and copies of pages and slots, against plain statements in 64 bits.

Tolerances follow from the roundings. Scores: a dot product of d terms in float32 is off by at most d u sum|q_i k_i| (u = 2^-24), and
three more roundings (scale, log2 e, the difference with the maximum); a weight 2^x is off by 2 units and by what its score is off; a sum
of n weights by n u. So the output is off by at most (2 (d + 8) u S + 2 (n + 8) u) times the weighted mean of |v|, S the largest
sum|q_i k_i| * scale of the row. In bfloat16 the weights enter the product with the values rounded (2^-8 of each at most, so 2^-8 of the
weighted mean of |v|) and the output is rounded (2^-8 of itself).
"""
import math

import numpy as np
import pytest
import torch

from scriptling_llm_lib_b200.cache import PAGE, SharePlan, TileShape
from scriptling_llm_lib_b200.csrc.bindings import KernelError, KernelSet, PageKernels

pytestmark = pytest.mark.gpu
F, B16 = torch.float32, torch.bfloat16
LAYOUTS = [(16, 4, 64, 64), (32, 32, 64, 64), (32, 8, 128, 128), (16, 4, 64, 128), (10, 2, 48, 40), (12, 3, 96, 96), (8, 1, 128, 64), (3, 3, 8, 16)]
WIDE = [(4, 2, 256, 256), (4, 1, 192, 128), (6, 2, 100, 20)]          # widths that only the FMA form takes


def path(*runs):
    return tuple(runs)


# name -> [(runs of shared pages (name, pages), tokens held, tokens new)]
BATCHES = {
    "one": [(path(), 130, 1)],
    "one-token": [(path(), 0, 1), (path(), 0, 1)],
    "two": [(path(("a", 3)), 200, 1), (path(("a", 3)), 260, 1)],
    "edge": [(path(("a", 5)), 320, 1), (path(("a", 5)), 383, 1), (path(("a", 5)), 384, 1), (path(("a", 5)), 321, 1)],
    "nested": [(path(("a", 7), ("b", 4)), 750, 1), (path(("a", 7), ("c", 6)), 840, 1), (path(("a", 7), ("b", 4)), 704, 1), (path(("a", 7)), 449, 1),
               (path(("a", 7), ("c", 6)), 833, 1), (path(), 77, 1)],
    "many": [(path(("a", 9)), 576 + 13 * i % 100, 1) for i in range(70)],
    "runs": [(path(("a", 6)), 384 + i, 1 + 17 * i % 40) for i in range(9)],
    "long-runs": [(path(("a", 10)), 650, 300), (path(("a", 10)), 640, 1), (path(), 0, 200), (path(("a", 10)), 700, 129)],
    "empty": [(path(("a", 4)), 256, 0), (path(("a", 4)), 270, 3), (path(("a", 4)), 300, 1), (path(), 50, 0)],
    "long": [(path(("a", 130)), 8320 + 70 * i, 1) for i in range(5)],
}


class Case:
    def __init__(self, batch, layout, dtype, seed=0, q_extra=0, junk=True):
        self.H, self.G, self.hd, self.vd = layout
        self.spec, self.dtype = BATCHES[batch] if isinstance(batch, str) else batch, dtype
        gen = torch.Generator().manual_seed(seed)
        ids, n = {}, 0
        rows = []
        for runs, held, new in self.spec:
            pages = []
            for name, k in runs:
                for i in range(k):
                    if (name, i) not in ids:
                        ids[name, i] = n
                        n += 1
                    pages.append(ids[name, i])
            more = -(-(held + new) // PAGE) - len(pages)
            assert len(pages) * PAGE <= held and more >= 0
            rows.append(pages + list(range(n, n + more)))
            n += more
        self.n_pages = n + 3
        order = torch.randperm(self.n_pages, generator=gen).tolist()
        self.width = max(1, max(len(r) for r in rows))
        self.table = np.full((len(rows), self.width), -1, dtype=np.int32)
        for b, r in enumerate(rows):
            self.table[b, :len(r)] = [order[i] for i in r]
        self.held, self.new = [h for _, h, _ in self.spec], [k for _, _, k in self.spec]
        self.T = sum(self.new)
        k = torch.randn(self.n_pages, self.G, PAGE, self.hd, generator=gen)
        v = torch.randn(self.n_pages, self.G, PAGE, self.vd, generator=gen)
        if junk:          # what no sequence holds may be anything
            used = torch.zeros(self.n_pages, PAGE, dtype=torch.bool)
            for b in range(len(rows)):
                for i in range(self.held[b] + self.new[b]):
                    used[self.table[b, i // PAGE], i % PAGE] = True
            k = torch.where(used[:, None, :, None], k, torch.tensor(math.nan))
            v = torch.where(used[:, None, :, None], v, torch.tensor(math.inf))
        self.k, self.v = k.to(dtype).cuda(), v.to(dtype).cuda()
        self.q = (1.5 * torch.randn(self.T, self.H * self.hd + q_extra, generator=gen)).to(dtype).cuda()
        self.pos = torch.tensor([h + i for h, k in zip(self.held, self.new) for i in range(k)], dtype=torch.int32).cuda()
        self.scale = self.hd ** -0.5

    def plan(self, **more):
        ops = KernelSet(self.dtype).shared
        return SharePlan.build(self.table, self.held, self.new, self.H, self.G, ops.shape(self.hd, self.vd), "cuda", **more)

    def run(self, plan=None, out=None, **options):
        ops, plan = KernelSet(self.dtype).shared, plan or self.plan()
        out = torch.full((self.T, self.H * self.vd), 7.0, dtype=self.dtype, device="cuda") if out is None else out
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        part = torch.full((plan.part_floats(self.vd),), math.nan, device="cuda")
        ops.attn(self.q, out, self.pos, torch.from_numpy(self.table).cuda(), self.k, self.v, plan, part, self.scale, err, **options)
        assert int(err) == 0
        return out

    def formula(self, softcap=None, sink=None):
        """(the output, the weighted mean of |v|, S, keys) of every row, in 64 bits."""
        outs, means, tops, keys, row = [], [], [], [], 0
        R = self.H // self.G
        for b, (held, new) in enumerate(zip(self.held, self.new)):
            n = held + new
            pages = torch.from_numpy(self.table[b, :-(-n // PAGE)]).long().cuda()
            k = self.k[pages].double().transpose(1, 2).reshape(-1, self.G, self.hd)[:n].repeat_interleave(R, 1)
            v = self.v[pages].double().transpose(1, 2).reshape(-1, self.G, self.vd)[:n].repeat_interleave(R, 1)
            q = self.q[row:row + new, :self.H * self.hd].double().view(new, self.H, self.hd)
            s = torch.einsum("nhd,mhd->nhm", q, k) * self.scale
            S = (torch.einsum("nhd,mhd->nhm", q.abs(), k.abs()) * self.scale).amax(-1)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            late = torch.arange(n, device="cuda")[None] > torch.arange(held, n, device="cuda")[:, None]
            s = s.masked_fill(late[:, None], -math.inf)
            if sink is not None:
                s = torch.cat([s, sink.double()[None, :, None].expand(new, -1, 1)], -1)
            w = torch.softmax(s, -1)[..., :n]
            outs.append(torch.einsum("nhm,mhd->nhd", w, v))
            means.append(torch.einsum("nhm,mhd->nhd", w, v.abs()))
            tops.append(S)
            keys.append(torch.full((new,), float(n), device="cuda", dtype=torch.float64))
            row += new
        return torch.cat(outs), torch.cat(means), torch.cat(tops), torch.cat(keys)

    def check(self, got, **options):
        want, mean, S, n = self.formula(**options)
        u, d = 2.0 ** -24, self.hd
        slack = 2 * u * ((d + 8) * S[..., None] + (n[:, None, None] + 8)) * mean + 1e-30
        if self.dtype == B16:
            slack = slack + 2.0 ** -8 * mean + 2.0 ** -8 * want.abs()
        off = (got.double().view_as(want) - want).abs()
        assert bool((off <= slack).all()), float((off / slack).max())


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[2]], ids=str)
def test_attention_of_every_kind_of_batch(batch, dtype, layout):
    c = Case(batch, layout, dtype)
    c.check(c.run())


@pytest.mark.parametrize("batch", ["nested", "runs"])
@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS + WIDE, ids=str)
def test_attention_of_every_head_layout(batch, dtype, layout):
    c = Case(batch, layout, dtype, seed=3)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", [(16, 4, 64, 64), (16, 4, 64, 128), (4, 2, 256, 256)], ids=str)
def test_capped_scores_and_sinks(dtype, layout):
    c = Case("nested", layout, dtype, seed=5)
    sink = torch.linspace(-3, 40, layout[0]).cuda()
    for options in ({"softcap": 2.5}, {"sink": sink}, {"softcap": 30.0, "sink": sink}):
        c.check(c.run(**options), **options)


@pytest.mark.parametrize("layout", [(48, 1, 64, 64), (64, 1, 128, 128), (64, 1, 32, 32), (40, 2, 16, 200)], ids=str)
@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_many_query_heads_on_a_key_value_head(dtype, layout):
    c = Case("nested", layout, dtype, seed=9)
    c.check(c.run())
    c = Case("runs", layout, dtype, seed=9)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_more_items_than_a_block_or_a_warp_holds_at_a_time(dtype):
    """Over 64 tiles a block and over 32 thin ones a warp."""
    c = Case([(path(("a", 2)) if i % 3 else path(), 128 + i % 70, 1) for i in range(620)], (64, 64, 16, 16), dtype, seed=4)
    plan = c.plan()
    assert max(np.diff(plan.parts["first"]).max(), np.diff(plan.parts["thin_first"]).max(initial=0)) > 32
    c.check(c.run(plan))
    c = Case([(path(("a", 1)), 64 + i % 3, 5 + i % 2) for i in range(150)], (64, 16, 24, 24), dtype, seed=4)      # 20 and 24 rows: not thin
    plan = c.plan()
    assert dtype == F or np.diff(plan.parts["first"]).max() > 8
    c.check(c.run(plan))


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_a_step_of_no_tokens_writes_nothing(dtype):
    c = Case([(path(("a", 3)), 200, 0), (path(("a", 3)), 210, 0)], (16, 4, 64, 64), dtype)
    assert c.run().shape == (0, 1024)


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_rows_that_stand_apart_and_the_same_result_again(dtype):
    c = Case("nested", (16, 4, 64, 64), dtype, q_extra=72)
    plan = c.plan()
    a, b = c.run(plan), c.run(plan)
    c.check(a)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", [(16, 4, 64, 64), (16, 4, 64, 128), (32, 8, 128, 128)], ids=str)
def test_what_is_not_finite_stays_with_the_rows_that_see_it(dtype, layout):
    """A value of infinity at a position: the rows at or behind it that see it are not finite, all others as without it. A query of NaN
    spoils its own row."""
    c = Case("runs", layout, dtype, junk=False)
    b = 4
    at, page = c.held[b] + 2, c.table[b, (c.held[b] + 2) // PAGE]
    first = sum(c.new[:b])
    clean = c.run()
    c.v[page, :, at % PAGE] = math.inf
    c.q[first + c.new[b] + 1] = math.nan                                   # a row of the sequence behind
    got = c.run()
    seen = torch.zeros(c.T, dtype=torch.bool)
    seen[first + 2:first + c.new[b]] = True
    seen[first + c.new[b] + 1] = True
    assert not torch.isfinite(got[seen.cuda()].float()).all(-1).any()
    assert torch.isfinite(got[~seen.cuda()].float()).all()
    other = ~seen.cuda()
    assert (got[other].double() - clean[other].double()).abs().max() <= (2.0 ** -7 if dtype == B16 else 1e-5) * clean.double().abs().max()


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_a_plan_serves_the_steps_behind_it_replayed(dtype):
    """Captured with one plan; replayed as the sequences grow by a page and more, with the plan of the first step, then with a new one."""
    from scriptling_llm_lib_b200.cache import PlanCapacity
    c = Case([(path(("a", 5)), 330 + 60 * i, 1) for i in range(6)], (16, 4, 64, 64), dtype, junk=False)
    ops = KernelSet(dtype).shared
    shape = ops.shape(64, 64)
    cap = PlanCapacity.of_decode(6, 16, 4, shape)
    grown = Case([(path(("a", 5)), 330 + 60 * i + 150, 1) for i in range(6)], (16, 4, 64, 64), dtype, junk=False)
    plan = SharePlan.build(grown.table, c.held, c.new, 16, 4, shape, "cuda", capacity=cap)
    pos, table, err = c.pos.clone(), torch.from_numpy(grown.table).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty((6, 16 * 64), dtype=dtype, device="cuda")
    call = lambda part: ops.attn(grown.q, out, pos, table, grown.k, grown.v, plan, part, grown.scale, err)      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(torch.empty((plan.part_floats(64),), device="cuda"))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.empty((plan.part_floats(64),), device="cuda"))
    for more in (0, 1, 40, 150):
        pos.copy_(c.pos + more)
        if more == 150:
            new = SharePlan.build(grown.table, [h + more for h in c.held], c.new, 16, 4, shape, None, capacity=cap)
            plan.dev.copy_(torch.from_numpy(new.host()))
        graph.replay()
        grown.held = [h + more for h in c.held]
        grown.check(out)
    assert int(err) == 0


def test_a_bad_page_is_reported_and_the_others_go_on():
    for dtype in (F, B16):
        c = Case("two", (16, 4, 64, 64), dtype, junk=False)
        good = c.run()
        plan, ops = c.plan(), KernelSet(dtype).shared
        for bad in (-1, c.n_pages, 1 << 30):
            table = c.table.copy()
            table[1, 3] = bad
            err, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty_like(good)
            ops.attn(c.q, out, c.pos, torch.from_numpy(table).cuda(), c.k, c.v, plan, torch.empty(plan.part_floats(64), device="cuda"), c.scale, err)
            assert int(err) != 0 and torch.equal(out[0], good[0])


def test_on_a_stream_of_its_own():
    c = Case("nested", (16, 4, 64, 64), B16)
    plan = c.plan()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = c.run(plan)
    s.synchronize()
    c.check(out)


@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
def test_pages_behind_four_gigabytes_of_a_storage(dtype):
    """Elements past 2^31 (bytes past 2^32), of attention and of copies: the same results as from a small storage."""
    c = Case("runs", (32, 8, 128, 128), dtype, junk=False)
    want, far = c.run(), 33_900
    k, v = (torch.empty((far + 100, *t.shape[1:]), dtype=dtype, device="cuda") for t in (c.k, c.v))
    k[far:far + c.n_pages], v[far:far + c.n_pages] = c.k, c.v
    small, c.k, c.v = (c.k, c.v), k, v
    c.table = np.where(c.table < 0, c.table, c.table + far).astype(np.int32)
    assert torch.equal(c.run(), want)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    src, dst = (torch.arange(a, a + c.n_pages, dtype=torch.int32, device="cuda") for a in (far, 0))
    PageKernels().copy_pages([(k[None], k[None]), (v[None], v[None])], src, dst, None, err)
    assert int(err) == 0 and torch.equal(k[:c.n_pages], small[0]) and torch.equal(v[:c.n_pages], small[1])
    k[far:].zero_()
    PageKernels().copy_pages([(k[None], k[None])], dst, src, None, err)
    assert int(err) == 0 and torch.equal(k[far:far + c.n_pages], small[0])


def test_two_calls_at_once_with_one_plan():
    """Calls on two streams, with a scratch each, share nothing that they write."""
    c = Case("many", (32, 8, 128, 128), B16)
    plan, streams, outs = c.plan(), [torch.cuda.Stream() for _ in range(2)], []
    want = c.run(plan)
    ops, table, err = KernelSet(B16).shared, torch.from_numpy(c.table).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([])
            part = torch.empty((plan.part_floats(128),), device="cuda")
            for _ in range(20):
                out = torch.zeros_like(want)
                ops.attn(c.q, out, c.pos, table, c.k, c.v, plan, part, c.scale, err)
                outs[-1].append(out)
    torch.cuda.synchronize()
    assert int(err) == 0 and all(torch.equal(o, want) for some in outs for o in some)


def test_refusals():
    c = Case("two", (16, 4, 64, 64), B16)
    ops, plan = KernelSet(B16).shared, c.plan()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    part = torch.empty((plan.part_floats(64),), device="cuda")
    out = torch.empty((2, 1024), dtype=B16, device="cuda")
    table = torch.from_numpy(c.table).cuda()
    good = dict(q=c.q, out=out, tok_pos=c.pos, block_table=table, kpages=c.k, vpages=c.v, plan=plan, part=part, scale=0.125, err_flag=err)
    for change in (dict(q=c.q[:1]), dict(q=c.q.float()), dict(q=c.q[:, :1000]), dict(out=out[:, :1000]), dict(out=out.float()), dict(tok_pos=c.pos[:1]),
                   dict(block_table=table[:1]), dict(block_table=table.long()), dict(kpages=c.k[:, :2]), dict(kpages=c.k.float()), dict(part=part[:-1]),
                   dict(sink=torch.zeros(8, device="cuda")), dict(q=c.q.cpu()), dict(kpages=torch.zeros(5, 4, 64, 6, dtype=B16, device="cuda"))):
        with pytest.raises(KernelError):
            ops.attn(**{**good, **change})
    ops.attn(**good)
    with pytest.raises(KernelError, match="laid out for"):
        other = SharePlan.build(c.table, c.held, c.new, 16, 4, TileShape(rows=32, workers=7), "cuda")       # no kernel's
        ops.attn(**{**good, "plan": other, "part": torch.empty((other.part_floats(64),), device="cuda")})


# --------------------------------------------------------------------------- copies
@pytest.mark.parametrize("dtype", [F, B16], ids=["f32", "bf16"])
@pytest.mark.parametrize("units,heads,widths", [(1, 1, (64, 64)), (3, 4, (128, 64)), (2, 5, (36, 20)), (2, 3, (10, 7)), (1, 2, (1, 3))], ids=str)
def test_copies_of_pages(dtype, units, heads, widths):
    gen = torch.Generator().manual_seed(7)
    rows = [64, 1, 0, 63, 17, 64]
    src, dst = [2, 2, 5, 0, 7, 9], [11, 1, 3, 4, 6, 8]
    at = lambda ids: torch.tensor(ids, dtype=torch.int32).cuda()                                     # noqa: E731
    for same in (True, False):
        a = [torch.randn(units, 13, heads, PAGE, w, generator=gen).to(dtype).cuda() for w in widths]
        b = a if same else [torch.randn(units, 17, heads, PAGE, w, generator=gen).to(dtype).cuda() for w in widths]
        want = [t.clone() for t in b]
        for x, y in zip(a, want):
            for s, d, n in zip(src, dst, rows):
                y[:, d, :, :n] = x[:, s, :, :n]
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        PageKernels().copy_pages(list(zip(a, b)), at(src), at(dst), at(rows), err)
        assert all(torch.equal(x, y) for x, y in zip(b, want)) and int(err) == 0
        for x, y in zip(a, want):
            y[:, 12] = x[:, 0]
        PageKernels().copy_pages(list(zip(a, b)), at([0]), at([12]), None, err)
        assert all(torch.equal(x, y) for x, y in zip(b, want)) and int(err) == 0


def test_copies_of_many_tensors_and_of_slots():
    """More tensors than one launch takes, of every element width; ids and counts out of range are reported and left alone."""
    tensors = [torch.arange(9 * n, device="cuda").view(9, n).to(t) for n in (1, 3, 64, 1000, 4096) for t in (F, B16, torch.int32, torch.uint8)]
    want = [t.clone() for t in tensors]
    for t in want:
        t[[1, 4, 8]] = t[6].clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    at = lambda ids: torch.tensor(ids, dtype=torch.int32).cuda()                                     # noqa: E731
    PageKernels().copy_slots([(t, t) for t in tensors], at([6, 6, 6]), at([1, 4, 8]), err)
    assert all(torch.equal(x, y) for x, y in zip(tensors, want)) and int(err) == 0
    PageKernels().copy_slots([(t, t) for t in tensors[:2]], at([9, 0, -1]), at([0, 9, 1]), err)
    assert all(torch.equal(x, y) for x, y in zip(tensors, want)) and int(err) != 0
    pages = torch.randn(1, 4, 2, PAGE, 8, device="cuda")
    before = pages.clone()
    for n in (65, -1):
        err.zero_()
        PageKernels().copy_pages([(pages, pages)], at([0]), at([1]), at([n]), err)
        assert torch.equal(pages, before) and int(err) != 0
    PageKernels().copy_pages([(pages, pages)], at([]), at([]), at([]), err)
    PageKernels().copy_pages([], at([0]), at([1]), at([2]), err)
    with pytest.raises(KernelError):
        PageKernels().copy_pages([(pages, pages)], at([0, 1]), at([1]), None, err)
    with pytest.raises(KernelError):
        PageKernels().copy_pages([(pages, pages[..., :4].contiguous())], at([0]), at([1]), None, err)
    with pytest.raises(KernelError):
        PageKernels().copy_slots([(pages.cpu(), pages.cpu())], at([0]), at([1]), err)
