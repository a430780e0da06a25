"""Sequences that share pages, without a GPU: pools with several holders, forks and their copies on writing, compaction, the tree of shared
pages and the plan that is laid out from it, prompts that begin alike, and what the kernels' wrappers refuse."""
import random

import numpy as np
import pytest
import torch

from scriptling_llm_lib_b200.cache import (PAGE, CacheFull, CacheNeed, FreeList, PlanCapacity, SequenceCache, SharePlan, StateNeed, TileShape,
                                           pages_for, share_pays, share_tree)
from scriptling_llm_lib_b200.csrc import bindings
from scriptling_llm_lib_b200.engine.generate import Generator, plan_batches, request_pages, shared_runs


def test_an_id_with_several_holders_is_free_when_the_last_gives_it_back():
    fl = FreeList(3, "thing")
    a, b = fl.alloc(), fl.alloc()
    fl.share(a)
    fl.share(a)
    assert fl.holders(a) == 3 and fl.holders(b) == 1 and fl.n_shared == 1 and fl.n_held == 2
    fl.free(a)
    fl.free(a)
    assert fl.is_held(a) and fl.n_shared == 0 and fl.n_free == 1
    fl.free(a)
    assert not fl.is_held(a) and fl.n_free == 2
    for bad in (a, 2, -1, 3):
        with pytest.raises(ValueError):
            fl.share(bad)
        with pytest.raises(ValueError):
            fl.free(bad)
    assert fl.alloc() == a
    fl.renumber({a: 2, b: 0}, 4)
    assert fl.n == 4 and fl.n_held == 2 and [fl.is_held(i) for i in range(4)] == [True, False, True, False] and fl.alloc() == 1
    with pytest.raises(ValueError):
        fl.renumber({0: 0, 1: 1})


# --------------------------------------------------------------------------- the cache, with contents
def _cache(n_slots=8, n_pages=30):
    needs = {0: CacheNeed("full", 2, 3), 1: CacheNeed("window", 1, 2, 70, keep=5), 2: CacheNeed("full", 1, 4, v_dim=0)}
    return SequenceCache(needs, {0: StateNeed((2, 3)), 1: {"conv": StateNeed((4,), torch.bfloat16)}, 2: None}, n_slots, n_pages, torch.float32, "cpu")


def _write(c, slot, tokens):
    """A step's tokens into every group at their places."""
    c.reserve([(slot, len(tokens))])
    at = c.length[slot]
    for g in c.groups:
        for i, t in enumerate(tokens):
            page = g.pages[slot][(at + i) // PAGE]
            assert g.pool.holders(page) == 1                       # what is written belongs to the writer alone
            g.k[:, page, :, (at + i) % PAGE] = float(t)
            g.v[:, page, :, (at + i) % PAGE] = -float(t)
    c.advance([(slot, len(tokens))])


def _check(c, slot, tokens):
    assert c.length[slot] == len(tokens)
    for g in c.groups:
        first = max(0, g.need.first_needed(len(tokens)))
        table = c.block_table(c.groups.index(g), [slot])[0]
        for p, t in enumerate(tokens):
            if p >= first or p < g.need.keep:
                page = g.pages[slot][p // PAGE]
                assert page == table[p // PAGE] and g.pool.is_held(page)
                assert float(g.k[0, page, 0, p % PAGE, 0]) == t and (g.v.numel() == 0 or float(g.v[0, page, 0, p % PAGE, 0]) == -t)


def _consistent(c):
    for g in c.groups:
        count = {}
        for lst in g.pages.values():
            for pg in lst:
                if pg >= 0:
                    count[pg] = count.get(pg, 0) + 1
        assert all(g.pool.holders(i) == count.get(i, 0) for i in range(g.pool.n))
        assert g.pool.n_held == len(count) and g.pool.n_shared == sum(n > 1 for n in count.values())


def test_a_random_life_of_forks_writes_closes_and_compactions():
    rng = random.Random(4)
    c, held, full = _cache(), {}, 0
    for step in range(900):
        what = rng.random()
        try:
            if what < 0.15 or not held:
                held[c.open()] = []
            elif what < 0.35:
                s, n = rng.choice(sorted(held)), rng.randint(0, 3)
                for new in c.fork(s, n):
                    assert new not in held
                    held[new] = list(held[s])
                    assert torch.equal(c.seq_state[new], c.seq_state[s]) and torch.equal(c.state[0][new], c.state[0][s])
                    assert torch.equal(c.state[1]["conv"][new], c.state[1]["conv"][s])
            elif what < 0.8:
                s = rng.choice(sorted(held))
                tokens = [rng.randint(1, 9999) for _ in range(rng.choice([1, 1, 2, 40, 64, 150]))]
                if len(held[s]) + len(tokens) < 600:
                    _write(c, s, tokens)
                    held[s] += tokens
                    c.seq_state[s, 0], c.state[0][s], c.state[1]["conv"][s] = tokens[0], float(tokens[0]), float(tokens[-1])
            elif what < 0.95:
                s = rng.choice(sorted(held))
                c.close(s)
                del held[s]
            else:
                n = rng.choice([None, None, 30, 34, max(g.pool.n_held for g in c.groups) or 1])
                c.compact(n)
                assert all(not g.pool.is_held(i) for g in c.groups for i in range(g.pool.n_held, g.pool.n))
                assert all(g.k.shape[1] == c.n_pages + 1 == g.pool.n + 1 for g in c.groups)
        except CacheFull:
            full += 1
        _consistent(c)
        if step % 5 == 0:
            for s, tokens in held.items():
                _check(c, s, tokens)
    assert full > 5
    for s in sorted(held):
        c.close(s)
    assert all(g.pool.n_free == g.pool.n and g.pool.n_shared == 0 for g in c.groups)


def test_a_new_storage_that_finds_no_memory_changes_nothing(monkeypatch):
    c = _cache()
    slot, tokens = c.open(), list(range(1, 200))
    _write(c, slot, tokens)
    fork = c.fork(slot)[0]
    before, pages, made = [(g.k, g.v) for g in c.groups], c.n_pages, []

    def empty(*args, **kwargs):
        made.append(1)
        if len(made) == 4:                  # the second group's values
            raise torch.OutOfMemoryError("no memory")
        return torch.zeros(*args, **kwargs)

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        with pytest.raises(torch.OutOfMemoryError):
            c.compact(40)
    assert len(made) == 4 and c.n_pages == pages and all(g.k is k and g.v is v and g.pool.n == pages for g, (k, v) in zip(c.groups, before))
    _consistent(c)
    for s in (slot, fork):
        _check(c, s, tokens)
    c.compact(40)
    assert c.n_pages == 40
    for s in (slot, fork):
        _check(c, s, tokens)


def test_the_writers_of_a_shared_page_get_their_own_and_the_last_keeps_it():
    c = _cache()
    a = c.open()
    _write(c, a, list(range(1, 101)))
    b, d = c.fork(a, 2)
    g = c.groups[0]
    whole, tail = g.pages[a]
    assert g.pages[b] == g.pages[d] == [whole, tail] and g.pool.n_held == 2 and g.pool.holders(tail) == 3
    for s, t in ((a, 7), (b, 8), (d, 9)):
        _write(c, s, [t])
    assert g.pages[a][0] == g.pages[b][0] == g.pages[d][0] == whole and g.pool.holders(whole) == 3
    assert len({g.pages[s][1] for s in (a, b, d)}) == 3 and g.pages[d][1] == tail and g.pool.n_held == 4
    for s, t in ((a, 7), (b, 8), (d, 9)):
        _check(c, s, list(range(1, 101)) + [t])
    before, free = [list(g.pages[s]) for s in (a, b, d)], g.pool.n_free
    e = c.fork(a, 1)[0]
    c.length[a] = c.length[e] = 64 - 10                               # taken back into a page that all of them share
    c.reserve([(a, 30), (b, 1)])
    assert g.pages[a][0] != whole and g.pages[b] == before[1] and g.pages[e][0] == whole     # the write went nowhere else
    assert g.pool.n_free == free - 2                                                          # its first page and the one shared with e


def test_a_fork_is_all_or_nothing_and_a_step_that_must_copy_too():
    c = _cache(n_slots=3, n_pages=3)
    a = c.open()
    _write(c, a, [1] * 70)
    with pytest.raises(CacheFull):
        c.fork(a, 3)
    assert c.slots.n_held == 1 and c.groups[0].pool.n_shared == 0 and c.fork(a, 0) == []
    b, d = c.fork(a, 2)
    with pytest.raises(CacheFull):
        c.reserve([(a, 1), (b, 1), (d, 1)])                           # two copies of the second page, one page free
    assert c.groups[0].pages[a] == c.groups[0].pages[b] == c.groups[0].pages[d]
    c.reserve([(a, 1)])
    for bad in (3, 7, -1):
        with pytest.raises(ValueError):
            c.fork(bad)
    with pytest.raises(ValueError):
        c.fork(a, -1)
    with pytest.raises(CacheFull):
        c.compact(2)
    with pytest.raises(ValueError):
        c.compact(0)
    assert c.n_pages == 3


def test_the_tree_is_made_again_when_pages_change_hands():
    c = _cache()
    a = c.open()
    _write(c, a, [1] * 300)
    assert c.share_tree(0, [a]) is None and not c.shares_pages
    b = c.fork(a)[0]
    order, nodes, own = c.share_tree(0, [a, b])
    assert nodes == [(0, 2, 0, 4)] and list(own) == [4, 4] and c.share_tree(0, [a, b])[1] is nodes
    d = c.open()
    _write(c, d, [2] * 300)
    order, nodes, own = c.share_tree(0, [d, b, a])
    assert len(nodes) == 1 and sorted(order[nodes[0][0]:nodes[0][1]]) == [1, 2]
    c.close(b)
    b2 = c.fork(d)[0]
    assert b2 == b and sorted(c.share_tree(0, [d, b2, a])[0][:2].tolist()) in ([0, 1], [0, 2])
    assert [sorted(t[0][lo:hi].tolist()) for t in (c.share_tree(0, [d, b2, a]),) for lo, hi, _, _ in t[1]] == [[0, 1]]


# --------------------------------------------------------------------------- trees and plans
def _batch(rng, n, rep, runs):
    """Tables of sequences with shared fronts, nested."""
    ids, tables, held, new = iter(rng.sample(range(100000), 60000)), [], [], []
    fronts = [[next(ids) for _ in range(rng.choice([0, 3, 9, 40]))]]
    for _ in range(rng.randint(0, 4)):
        fronts.append(list(rng.choice(fronts)) + [next(ids) for _ in range(rng.choice([1, 4, 11]))])
    for _ in range(n):
        front = rng.choice(fronts)
        h, k = PAGE * len(front) + rng.choice([0, 1, 63, 64, 200]), 1 if not runs else rng.choice([0, 1, 5, 64, 150])
        tables.append(front + [next(ids) for _ in range(pages_for(h + k) - len(front))])
        held.append(h)
        new.append(k)
    width = max(1, max(len(t) for t in tables))
    table = np.full((n, width), -1, dtype=np.int32)
    for b, t in enumerate(tables):
        table[b, :len(t)] = t
    return table, held, new


@pytest.mark.parametrize("shape", [TileShape(256, 148, True, 1.0, ((128, 0.7),)), TileShape(64, 296), TileShape(64, 7, costs=((4, 0.2), (16, 0.5)), min_pages=1), TileShape(16, 40, True),
                                   TileShape(256, 148, True, 2.0, ((128, 0.7),), 2, 16, 8, 0.4, 0.2)], ids=str)
@pytest.mark.parametrize("runs", [False, True])
def test_a_plan_covers_every_key_of_every_row_once(shape, runs):
    rng = random.Random(11)
    for n in (1, 2, 3, 17, 40, 60 if not runs else 9):
        G, rep = rng.choice([1, 2, 5]), rng.choice([1, 3, 4, 8])
        table, held, new = _batch(rng, n, rep, runs)
        plan = SharePlan.build(table, held, new, G * rep, G, shape, None)
        p, T = plan.parts, sum(new)
        pos = [h + i for h, k in zip(held, new) for i in range(k)]
        seq = [b for b, k in enumerate(new) for _ in range(k)]
        assert plan.n_rows == T and sorted(p["toks"].tolist()) == list(range(T))
        pages, owner, rows_of = {}, {}, {}
        for tok0, n_tok, last, g, a, b, part0, row in p["items"].tolist():
            end = pos[last] // PAGE + 1 if last >= 0 else b
            b = end if b < 0 else min(b, end)
            assert 1 <= n_tok * rep <= shape.rows and a < b and (last < 0 or p["toks"][tok0 + n_tok - 1] == last)
            if last >= 0:                                   # of one sequence, one behind the other
                assert [pos[int(p["toks"][tok0 + i])] for i in range(n_tok)] == list(range(pos[last] - n_tok + 1, pos[last] + 1))
            else:                                           # a node: every one of its keys is in front of all its tokens
                assert all(pos[int(p["toks"][tok0 + i])] >= b * PAGE for i in range(n_tok))
            for i in range(n_tok):
                t = int(p["toks"][tok0 + i])
                pages.setdefault((t, g), []).extend((j, int(table[row, j])) for j in range(a, b))
                for half in range(2 if shape.halves and shape.thin_rows < n_tok * rep <= shape.rows // 2 else 1):
                    at = part0 + half * n_tok * rep + i * rep
                    assert at not in owner
                    owner[at] = (t, g)
                    rows_of.setdefault((t, g), []).append(at)
        assert len(owner) * rep == plan.part_rows and (not owner or max(owner) + rep <= plan.part_rows)
        for t in range(T):
            for g in range(G):
                seen = dict(pages[t, g])
                assert len(seen) == len(pages[t, g])                                            # no page twice
                assert all(seen[j] == table[seq[t], j] for j in range(pos[t] // PAGE + 1))     # every page that it sees, as its own table has it
                mine = p["list"][p["list_first"][t * G + g]:p["list_first"][t * G + g + 1]]
                assert len(mine) and sorted(int(e) for e in mine) == sorted(rows_of[t, g])
        first, thin = p["first"], p["thin_first"]
        assert first[0] == 0 and first[-1] == thin[0] and thin[-1] == len(p["items"]) and (np.diff(first) >= 0).all() and (np.diff(thin) >= 0).all()
        rows = p["items"][:, 1] * rep
        assert (rows[:thin[0]] > shape.thin_rows).all() and (rows[thin[0]:] <= shape.thin_rows).all()
        if not runs:
            cap = PlanCapacity.of_decode(n, G * rep, G, shape)
            assert plan.fits(cap)
            roomy = SharePlan.build(table, held, new, G * rep, G, shape, None, capacity=cap)
            assert len(roomy.again(plan_with(roomy, plan))) == len(roomy.host())


def plan_with(roomy, plan):
    return SharePlan(plan.n_seqs, plan.n_rows, plan.n_heads, plan.n_kv, plan.shape, plan.width, plan.parts, None, roomy.capacity)


def test_plans_share_the_work_evenly_among_blocks():
    table = np.arange(64 * 200, dtype=np.int32).reshape(64, 200)
    table[:, :128] = np.arange(128)
    held = np.asarray([8192 + 40 * i for i in range(64)])
    for thin in (0, 16):
        shape = TileShape(256, 148, True, 1.0, ((128, 0.7),), 2, thin, 8 if thin else 0, 0.5, 0.25)
        plan = SharePlan.build(table, held, [1] * 64, 32, 8, shape, None)
        items, first, warps = plan.parts["items"], plan.parts["first"], plan.parts["thin_first"]
        end = np.where(items[:, 5] < 0, held[items[:, 2]] // PAGE + 1, items[:, 5])
        cost = (end - items[:, 4]) * np.where(items[:, 1] * 4 <= 128, 0.7, 1.0) + 1.0
        load = np.asarray([cost[a:b].sum() for a, b in zip(first, first[1:])])
        if thin:
            cost = (end - items[:, 4]) * 0.5 + 0.25
            load += np.asarray([max(cost[a:b].sum() * 8 for a, b in zip(w, w[1:])) for w in (warps[8 * k:8 * k + 9] for k in range(148))])
        assert max(load) < 1.7 * sum(load) / 148


def test_plans_refuse_what_does_not_fit_together():
    shape, table = TileShape(64, 10), np.zeros((2, 3), dtype=np.int32)
    good = dict(table=table, held=[10, 20], new=[1, 1], n_heads=4, n_kv=2, shape=shape, device=None)
    SharePlan.build(**good)
    for bad in (dict(table=table[0]), dict(table=table.astype(float)), dict(held=[10]), dict(held=[10, -1]), dict(new=[1, -1]), dict(n_kv=3), dict(n_kv=0),
                dict(n_heads=130), dict(held=[10, 192]), dict(table=table[:0], held=[], new=[]), dict(capacity=PlanCapacity(1, 1, 1))):
        with pytest.raises(ValueError):
            SharePlan.build(**{**good, **bad})
    plan = SharePlan.build(**good)
    with pytest.raises(ValueError):
        plan.again(SharePlan.build(**{**good, "new": [1, 2]}))


def test_equal_page_ids_are_shared_only_where_both_hold_the_whole_page():
    table = np.tile(np.arange(10, dtype=np.int32), (3, 1))
    assert share_tree(table, np.asarray([10, 10, 10]))[1] == [(0, 3, 0, 10)]
    order, nodes, own = share_tree(table, np.asarray([4, 10, 10]))
    assert (own[list(order).index(0)], sorted(own.tolist())) == (4, [4, 10, 10]) and len(nodes) == 2
    assert share_tree(table, np.asarray([0, 0, 0]))[1] == []
    assert share_tree(np.full((3, 10), -1, dtype=np.int32), np.asarray([5, 5, 5]))[1] == []


def test_which_steps_read_shared_pages_once():
    """Around the lines that the measurements draw (bfloat16 / 32-bit, tokens each, 32 heads of 64)."""
    def pays(n, prefix, new, kv, floats, own=100, layers=0):
        pages = pages_for(prefix + own + new)
        table = np.arange(n * pages, dtype=np.int32).reshape(n, pages)
        table[:, :prefix // PAGE] = np.arange(prefix // PAGE) + 10 ** 6
        held = np.full(n, prefix + own)
        return share_pays(share_tree(table, held // PAGE), held, [new] * n, 32, kv, 128, floats, layers)
    assert [pays(8, p, 1, 8, False) for p in (300, 1000, 4000, 16000)] == [False, False, False, True]
    assert [pays(n, 1000, 1, 32, False) for n in (2, 4, 32, 64)] == [False, False, True, True]
    assert [pays(n, 4000, 1, 8, True) for n in (2, 16, 64)] == [False, True, True]
    assert [pays(64, p, 1, 32, True) for p in (300, 1000)] == [False, False]
    assert [pays(16, p, 20, 8, False) for p in (100, 2000, 8000)] == [False, True, True]
    assert [pays(16, p, 150, 8, False) for p in (300, 8000)] == [False, True] and pays(4, 600, 30, 8, True)
    assert [pays(8, 4000, 20, 32, False, layers=n) for n in (0, 1, 24)] == [True, False, False] and pays(32, 4000, 20, 8, False, layers=24)
    assert not share_pays(None, [1], [1], 4, 4, 128, False) and not pays(1, 8000, 1, 8, False)


# --------------------------------------------------------------------------- prompts that begin alike
def test_runs_that_prompts_share():
    a = list(range(1000, 1200))
    assert shared_runs([a, a, a]) == [(0, [0, 1, 2], 0, 199)]                       # each keeps its last token
    assert shared_runs([a[:64], a[:64]]) == [] and shared_runs([a[:65], a[:65]]) == [(0, [0, 1], 0, 64)]
    b = a[:100] + [5] * 80
    runs = shared_runs([a, b, [1, 2], a + [9], b])
    assert runs[0][0] == 0 and sorted(runs[0][1]) == [0, 1, 3, 4] and runs[0][2:] == (0, 100)
    assert sorted((sorted(m), s, e) for _, m, s, e in runs[1:]) == [([0, 3], 100, 199), ([1, 4], 100, 179)]
    assert shared_runs([a, a, a, a], [0, 0, 1, 1]) == [(0, [0, 1], 0, 199), (0, [2, 3], 0, 199)] or \
        sorted(r[1] for r in shared_runs([a, a, a, a], [0, 0, 1, 1])) == [[0, 1], [2, 3]]


def test_continuations_hold_their_prompt_once():
    assert request_pages(200, 10, 1000) == (1, 3) and request_pages(64, 1, 1000) == (1, 0) and request_pages(5000, 10, 640) == (1, 9)
    assert plan_batches([200] * 6, 10, 8, 9, 1000, n=3) == [[0, 1, 2], [3, 4, 5]]   # 4 + 1 + 1 pages each
    assert plan_batches([200] * 6, 10, 8, 12, 1000, n=3) == [list(range(6))]
    assert plan_batches([200] * 6, 10, 8, 9, 1000) == [[0, 1], [2, 3], [4, 5]]
    assert plan_batches([200] * 3, 10, 2, 100, 1000, n=3) == [[0, 1], [2]]


class _Seq:
    def __init__(self, eng, slot):
        self.eng, self.slot, self.closed = eng, slot, False

    def close(self):
        if not self.closed:
            self.eng.cache.close(self.slot)
            self.closed = True


class _Engine:
    """Keeps the tokens themselves in its cache and answers with all that a sequence holds."""
    use_graphs = False

    class layout:
        stop_ids = ()

    def __init__(self, n_slots, n_pages):
        self.cache = SequenceCache({0: CacheNeed("full", 1, 1)}, {0: None}, n_slots, n_pages, torch.float32, "cpu")
        self.max_positions, self.rows = n_pages * PAGE, 0

    def open(self):
        return _Seq(self, self.cache.open())

    def fork(self, s, n=1):
        return [_Seq(self, x) for x in self.cache.fork(s.slot, n)]

    def new_event(self):
        class Event:
            record = synchronize = lambda self: None      # noqa: E731
            elapsed_time = lambda self, other: 0.0        # noqa: E731
        return Event()

    def prompt_step(self, entries):
        growth = [(e.sequence.slot, len(e.tokens)) for e in entries]
        assert all(n > 0 for _, n in growth) and len({s for s, _ in growth}) == len(growth)
        self.cache.reserve(growth)
        g, out = self.cache.groups[0], []
        for e in entries:
            s, at = e.sequence.slot, self.cache.length[e.sequence.slot]
            for i, t in enumerate(e.tokens):
                g.k[0, g.pages[s][(at + i) // PAGE], 0, (at + i) % PAGE] = float(t)
            self.rows += len(e.tokens)
            out.append([int(g.k[0, g.pages[s][p // PAGE], 0, p % PAGE, 0]) for p in range(at + len(e.tokens))])
        self.cache.advance(growth)
        return out, None

    def step(self, entries):
        return self.prompt_step(entries)[0]


class _Sampler:
    def sample(self, logits, options, seeds, counts, recent):
        return torch.tensor([(sum(t) * 31 + len(t) * 7 + s) % 1000 for t, s in zip(logits, seeds)])


def test_requests_that_share_give_what_they_give_alone():
    rng, saved = random.Random(2), 0
    for _ in range(60):
        front = [rng.randrange(50) for _ in range(rng.choice([0, 10, 64, 100, 300]))]
        middles = [[rng.randrange(50) for _ in range(rng.choice([0, 1, 64, 129]))] for _ in range(3)]
        prompts = [front + rng.choice(middles) + [rng.randrange(50) for _ in range(rng.randint(1, 150))] for _ in range(rng.randint(1, 7))]
        prompts += [list(prompts[0])] * rng.randint(0, 1)
        n, share = rng.choice([1, 1, 2, 3]), rng.random() < 0.7
        alone = _Engine(40, 400)
        want = Generator(alone, _Sampler()).generate([p for p in prompts for _ in range(n)], 5, seed=9)
        least = max(pages_for(len(p) + 4) for p in prompts)
        eng = _Engine(rng.choice([3, 8, 40]), rng.choice([least, least + 3, 400]))
        got = Generator(eng, _Sampler()).generate(prompts, 5, seed=9, n=n, share_prefix=share)
        assert [r.tokens for r in got] == [r.tokens for r in want]
        assert eng.cache.slots.n_held == 0 and eng.cache.groups[0].pool.n_held == 0 and eng.rows <= alone.rows
        saved += alone.rows - eng.rows
    assert saved > 0
    with pytest.raises(ValueError):
        Generator(_Engine(4, 40), _Sampler()).generate([[1]], 2, n=0)


def test_the_command_line_takes_continuations_and_shared_prefixes():
    from scriptling_llm_lib_b200.cli import build_parser
    args = build_parser().parse_args(["-model", "m", "-prompt", "1 2;1 3", "-n", "4", "-share-prefix"])
    assert args.n == 4 and args.share_prefix
    args = build_parser().parse_args(["-model", "m", "-prompt", "1"])
    assert args.n == 1 and not args.share_prefix


# --------------------------------------------------------------------------- what the wrappers refuse
def test_widths_and_shapes_of_the_attention():
    takes = bindings.SharedAttention.takes
    assert takes(64, 64) and takes(4, 256, 64) and not takes(66, 64) and not takes(64, 260) and not takes(64, 0) and not takes(64, 64, 65) and not takes(64, 64, 0)


def test_copies_refuse_what_is_not_on_a_device():
    k = bindings.PageKernels.__new__(bindings.PageKernels)            # (no library is loaded for a refusal)
    k.lib = None
    pages, ids, err = torch.zeros(1, 4, 2, PAGE, 8), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for pair in ((pages, pages), (pages, pages[..., :4]), (pages[0], pages[0]), (pages, pages.double())):
        with pytest.raises(bindings.KernelError):
            k.copy_pages([pair], ids, ids, None, err)
    for pair in ((pages, pages), (pages, pages[:, :2]), (torch.zeros(()), torch.zeros(()))):
        with pytest.raises(bindings.KernelError):
            k.copy_slots([pair], ids, ids, err)
