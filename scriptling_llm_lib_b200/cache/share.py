"""Which pages the sequences of a step have in common, and how attention goes over them once for all.

The reference holds one sequence (model_f32.go:310-317) and has nothing of the kind. Sequences that were forked from one
another hold the same pages at their front. `share_tree` finds them from the block table alone: two sequences share a page
where their page ids are the same from the front on, as far as both hold the whole page before the step. The result is a tree:
a node is a run of pages that two or more sequences share, a leaf what one sequence has for itself. Softmax attention over a
sequence's keys splits exactly over the nodes on its path (each gives a maximum, a sum and a weighted sum of values, which are
joined at the end), so a node's pages are read once, with the queries of all its members as the rows of one product.

`SharePlan` lays that work out for the kernels: a tile is a few tokens of a node with all the query heads of one key/value head,
an item a tile with a run of the node's pages, and every block has a list of items of about the same cost. An item leaves its
rows' partial results in a scratch buffer; a list says which of them belong to a token and key/value head.
"""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

import numpy as np
import torch

from .needs import PAGE

MAX_DEPTH = 4       # levels of shared runs; what lies deeper is read by each sequence for itself
MOST_PIECES = 64    # that a thin tile's pages are cut into: each is an entry for the joining kernel
MIN_SAVED = 4       # pages that a node must save its members to be worth another partial result for each row
ITEM_WORDS = 8      # int32 words of an item: first token in the list, tokens, last token (-1: of a node, all of whose keys all its tokens
                    # see), kv head, first page, page end (-1: to the last token), first row of the scratch, row of the block table


@dataclass(frozen=True)
class TileShape:
    """What a kernel works on: rows (tokens x query heads of a key/value head) of a tile, blocks that stay and walk their lists.
    `halves`: a tile of at most half the rows is worked on twice, by pages of either parity, and leaves two partial results.
    `thin_rows`: tiles of at most so many rows are thin: they stand behind the others in a block's list, each with one of its
    `thin_warps` warps."""
    rows: int
    workers: int
    halves: bool = False
    item_pages: float = 1.0      # what an item costs beside its pages, in pages
    costs: tuple = ()            # (rows, what a page of a tile of at most so many rows costs), fewest rows first; a full tile's is 1
    min_pages: int = 2           # an item is not cut to fewer
    thin_rows: int = 0
    thin_warps: int = 0
    thin_cost: float = 0.0       # what a page of a thin tile costs the block
    thin_item: float = 0.0       # and an item
    thin_start: float = 0.0      # and having any behind others


def share_tree(table: np.ndarray, whole: np.ndarray):
    """`table` [seqs, width] page ids (-1: none), `whole` [seqs]: pages that each holds wholly before the step. Returns the order of the
    sequences in which every node's members stand side by side, the nodes [(first, end, first page, end page)] in that order, parents
    first, and for every place of the order the first page that the sequence there has for itself."""
    n, width = table.shape
    if n == 1:
        return np.zeros(1, dtype=np.int64), [], np.zeros(1, dtype=np.int64)
    # rows as byte strings: equal fronts come to stand side by side, whatever the order between different pages
    order = np.argsort(np.ascontiguousarray(table).view(f"S{4 * width}").ravel(), kind="stable")
    t, w = table[order], np.asarray(whole, dtype=np.int64)[order]
    differ = (t[1:] != t[:-1]) | (t[1:] < 0)
    same = np.where(differ.any(1), differ.argmax(1), width)
    lcp = np.minimum(np.minimum(same, w[1:]), w[:-1]).tolist()
    nodes, own = [], [0] * n
    stack = [(0, n, 0, 0)]
    while stack:
        lo, hi, page, depth = stack.pop()
        if hi - lo == 1:
            own[lo] = page
            continue
        m = min(lcp[lo:hi - 1])
        if m > page and (m - page) * (hi - lo - 1) >= MIN_SAVED:
            nodes.append((lo, hi, page, m))
            page, depth = m, depth + 1
        if depth == MAX_DEPTH:
            own[lo:hi] = [page] * (hi - lo)
            continue
        at = lo
        for i in range(lo, hi):
            if i == hi - 1 or lcp[i] == m:
                stack.append((at, i + 1, page, depth))
                at = i + 1
    return order, nodes, np.asarray(own, dtype=np.int64)


def share_pays(tree, held, new, n_heads: int, n_kv: int, width: int, floats: bool, layers: int = 0) -> bool:
    """Whether a step of these sequences is estimated to be faster by the tree than each sequence for itself; `width`: of a key and a
    value together; `floats`: the shared pages go on FP32 FMA, in 32-bit and for bfloat16 widths that the tensor-core form does not take; `layers`:
    those that go by a plan made for this step alone (0: the plan is kept for more steps), which is counted as 1.2 ms of the host's and 0.1 us
    for each row and key/value head (728 rows on 8 take it 0.9 ms, 15,000 7 ms). The answer leans to each for itself: 32-bit steps of a token
    each have to be estimated 1.4 times as fast by the tree, and bfloat16 ones to save 80 MB a layer. Measured on 148 SMs, each for itself /
    by the tree, us:
    bfloat16, a token each (bound by the bytes, and the rotation and the cache write become a kernel of their own: in whole steps the
    line is between 50 and 100 MB saved a layer): 32 heads of 64 on 8, 8 sequences behind 1,000 tokens 12.5 / 13.3 (14 MB saved), 32
    behind 1,000 18.8 / 15.5 (61), 8 behind 16,000 41 / 20 (229), 64 behind 300 11.7 / 18.4 (33); 32 heads of 128 on 8, 64 behind 300
    24 / 24 (66).
    32-bit, a token each: each for itself costs a row, head and page 2.1 ns, the tree a key/value head of a sequence 56 ns and a
    tile's page 24: 32 heads of 64 on 8, 64 behind 1,000 72 / 59, 16 behind 4,000 77 / 43; on 32, 64 behind 1,000 110 / 117.
    Runs of tokens: tiles of 128 rows (64 in 32-bit) of a sequence and head, 4 ns a page (24) but no less than the 0.7 us (7) that a page
    takes one tile, against tiles of 256 (64) rows of a node and key/value head, 7.5 ns a page (17), and 50 ns an item: bfloat16, 32 heads of
    64 on 8, 16 of 20 tokens behind 300 18 / 22, behind 2,000 58 / 29, 8 of 60 behind 2,000 32 / 28; 16 of 150 behind 300 29 / 38,
    behind 8,000 312 / 173."""
    if tree is None or not tree[1]:
        return False
    order, nodes, own = tree
    held, new = np.asarray(held, dtype=np.int64)[order], np.asarray(new, dtype=np.int64)[order]
    rep, pages = n_heads // n_kv, (held + new - 1) // PAGE + 1
    ends = np.concatenate([[0], np.cumsum(new)])
    by_plan = (1200.0 + 0.1 * n_kv * int(ends[-1])) / layers if layers else 0.0
    if new.max() <= 1:
        if not floats:
            saved = sum((int(ends[hi] - ends[lo]) - 1) * (b - a) for lo, hi, a, b in nodes)
            return saved * n_kv * PAGE * width * 2 >= 80e6 + (by_plan * 6.5e6 if layers else 0.0)
        alone = 8.0 + 0.0021 * n_heads * float(pages[new > 0].sum())
        tiles = sum(-(-int(ends[hi] - ends[lo]) * rep // 64) * (b - a) for lo, hi, a, b in nodes)
        return (1.4 * (14.0 + 0.04 * n_kv * int(new.sum()) + 0.017 * n_kv * tiles) - alone) * width / 128 + by_plan < 0.0
    rows, page, wide_rows, wide_page, item = (64, 0.024, 64, 0.017, 0.05) if floats else (128, 0.0042, 256, 0.0075, 0.05)
    scale = width / 128 if floats else 0.4 + 0.6 * width / 128
    alone = max(scale * page * n_heads * float((-(-new // rows) * pages).sum()), scale * (7.0 if floats else 0.7) * int(pages.max())) + 4.0
    by_tree = 14.0 + by_plan + item * n_kv * int((-(-new * rep // wide_rows)).sum())
    by_tree += scale * wide_page * n_kv * float((-(-new * rep // wide_rows) * (pages - own)).sum())
    by_tree += scale * wide_page * n_kv * sum(-(-int(ends[hi] - ends[lo]) * rep // wide_rows) * (b - a) for lo, hi, a, b in nodes)
    return by_tree < 0.9 * alone


def scratch_rows(rows: int) -> int:
    """Rows of the scratch that `rows` partial results take: whole groups of 32."""
    return -(-max(1, rows) // 32) * 32


def most_part_rows(tree, new, n_heads: int, n_kv: int, shape: TileShape) -> int:
    """Partial results that a plan for these sequences leaves at most: those of every tile, and of a tile more for each place that a
    block's or a warp's list is cut at."""
    order, nodes, _ = tree
    new, rep = np.asarray(new, dtype=np.int64)[order], n_heads // n_kv
    ends = np.concatenate([[0], np.cumsum(new)])
    n = np.concatenate([new, [ends[hi] - ends[lo] for lo, hi, _, _ in nodes]]).astype(np.int64)
    per = shape.rows // rep
    rest = n % per * rep                       # rows of the tile that is not full; a full one leaves a result for each row unless it is half
    twice = lambda rows: np.where((rows > shape.thin_rows) & (rows <= shape.rows // 2) & shape.halves, 2 * rows, rows)      # noqa: E731
    tiles = n // per * int(twice(np.int64(per * rep))) + twice(rest)
    return int(n_kv * tiles.sum()) + shape.workers * (min(shape.rows, 2 * int(n.max(initial=0)) * rep) + shape.thin_warps * shape.thin_rows)


class SharePlan:
    """The items of one attention over a step's rows, in one int32 buffer on the device. Good for every layer of the step with these
    head counts, and for later steps of the same sequences with as many new tokens each: a leaf's last item goes on to where its
    tokens stand now. `width`: pages of the block table that the layout reaches."""

    def __init__(self, n_seqs: int, n_rows: int, n_heads: int, n_kv: int, shape: TileShape, width: int, parts: dict, device,
                 capacity: "PlanCapacity | None" = None, queued: bool = False):
        self.n_seqs, self.n_rows, self.n_heads, self.n_kv, self.shape, self.width = n_seqs, n_rows, n_heads, n_kv, shape, width
        self.n_items, self.n_list, self.part_rows = len(parts["items"]), len(parts["list"]), parts["part_rows"]
        self.parts = parts
        cap = capacity or PlanCapacity(self.n_items, self.n_list, self.part_rows)
        self.capacity = cap
        if not self.fits(cap):
            raise ValueError(f"a plan of {self.n_items} items, {self.n_list} list entries and {self.part_rows} rows of scratch; there is "
                             f"room for {cap.items}, {cap.entries} and {cap.rows}")
        self.dev, self.address = None, 0              # (a plan that is to take another's place, or to be looked at, is on the host alone)
        if device is not None:
            host = torch.from_numpy(self.host())
            self.dev = host.pin_memory().to(device, non_blocking=True) if queued else host.to(device)
            self._views()

    def again(self, other: "SharePlan") -> np.ndarray:
        """Take the layout of another plan of the same rows, heads, shape and capacity; the words for the device's buffer."""
        same = lambda p: (p.n_seqs, p.n_rows, p.n_heads, p.n_kv, p.shape, p.capacity)        # noqa: E731
        if same(other) != same(self):
            raise ValueError(f"a plan of {same(other)} cannot stand where one of {same(self)} does")
        self.parts, self.n_items, self.n_list, self.part_rows, self.width = other.parts, other.n_items, other.n_list, other.part_rows, other.width
        return self.host()

    def fits(self, cap: "PlanCapacity") -> bool:
        return self.n_items <= cap.items and self.n_list <= cap.entries and self.part_rows <= cap.rows

    def _sizes(self):
        s, c = self.shape, self.capacity
        # (items start at a multiple of four words: they are read sixteen bytes at a time)
        return [-(-(s.workers + 1) // 4) * 4, -(-(s.workers * s.thin_warps + 1) // 4) * 4, ITEM_WORDS * c.items, self.n_rows,
                self.n_rows * self.n_kv + 1, c.entries]

    def host(self) -> np.ndarray:
        """The buffer's words: where each block's items begin, where each of its warps' thin items do, the items, the tokens in the tree's
        order, where each token and key/value head's entries begin, the entries (rows of the scratch)."""
        sizes, p = self._sizes(), self.parts
        out, off = np.zeros(sum(sizes), dtype=np.int32), 0
        for n, part in zip(sizes, (p["first"], p["thin_first"], p["items"].ravel(), p["toks"], p["list_first"], p["list"])):
            out[off:off + len(part)] = part
            off += n
        return out

    def _views(self):
        at, views = 0, []
        for n in self._sizes():
            views.append(self.dev[at:at + n])
            at += n
        self.first, self.thin_first, self.items, self.toks, self.list_first, self.list = views
        # what the kernels' launchers read (SharePlanDev): six addresses, then the scratch's rows and the sizes
        s = self.shape
        self._struct = ctypes.create_string_buffer(struct.pack("6q q 5i 4x", *(v.data_ptr() for v in views), self.scratch_rows, self.n_rows, self.n_heads,
                                                               self.n_kv, s.workers, s.thin_warps))
        self.address = ctypes.addressof(self._struct)

    def part_floats(self, v_dim: int) -> int:
        """float32 elements of the scratch for values `v_dim` wide: the rows' sums over the values, then their maxima and sums."""
        return self.scratch_rows * (v_dim + 2)

    @property
    def scratch_rows(self) -> int:
        return scratch_rows(self.capacity.rows)

    @classmethod
    def build(cls, table, held, new, n_heads: int, n_kv: int, shape: TileShape, device, capacity=None, tree=None, queued: bool = False) -> "SharePlan":
        """`table` [seqs, width] page ids on the host; `held` and `new`: tokens that each sequence holds before the step and brings (0:
        none). `tree`: what `share_tree` gave for these sequences, if it is at hand. The plan is on the device when this returns, for any
        stream; `queued`: its copy is one more operation of the current stream, for calls on this stream (or on one that waits for it),
        and nothing that is queued is waited for."""
        table = np.asarray(table)
        if table.ndim != 2 or table.dtype.kind not in "iu" or table.shape[0] == 0:
            raise ValueError(f"a block table of page ids [sequences, pages], not {table.dtype} {table.shape}")
        table = np.ascontiguousarray(table, dtype=np.int32)
        held, new = np.asarray(held, dtype=np.int64), np.asarray(new, dtype=np.int64)
        n_seqs, width = table.shape
        if held.shape != (n_seqs,) or new.shape != (n_seqs,) or held.min() < 0 or new.min() < 0:
            raise ValueError(f"{n_seqs} sequences need as many counts of tokens held and new, none negative")
        if n_kv < 1 or n_heads % n_kv:
            raise ValueError(f"{n_heads} heads cannot share {n_kv} key/value heads")
        rep = n_heads // n_kv
        if rep > shape.rows:
            raise ValueError(f"{rep} query heads on one key/value head; a tile has {shape.rows} rows")
        if np.any(-(-(held + new) // PAGE) > width):
            raise ValueError(f"a sequence of {int((held + new).max())} tokens does not fit {width} pages")
        if tree is None or any(held[tree[0][lo:hi]].min() < PAGE * end for lo, hi, _, end in tree[1]):     # (or one that was taken back)
            tree = share_tree(table, held // PAGE)
        order, nodes, own = tree
        parts = _lay_out(order, nodes, own, held, new, rep, n_kv, shape)
        return cls(n_seqs, int(new.sum()), n_heads, n_kv, shape, parts["width"], parts, device, capacity, queued)


@dataclass(frozen=True)
class PlanCapacity:
    """Room for plans that take one another's place at the same addresses (a captured step's)."""
    items: int
    entries: int      # of the list
    rows: int         # of the scratch

    @classmethod
    def of_decode(cls, n_seqs: int, n_heads: int, n_kv: int, shape: TileShape) -> "PlanCapacity":
        """What any plan of one token for each of `n_seqs` sequences needs at most: every level of the tree has each token once, in
        at most one tile more than its nodes need, and every block, and every warp with thin tiles, cuts one tile at most."""
        rep = n_heads // n_kv
        per = max(1, shape.rows // rep)
        tiles = n_seqs + MAX_DEPTH * (n_seqs // 2 + -(-n_seqs // per))
        twice = 2 if shape.halves else 1
        thin = shape.workers * shape.thin_warps
        cuts = twice * shape.workers * min(per, n_seqs) + thin * min(shape.thin_rows // rep, n_seqs)
        entries = twice * n_kv * n_seqs * (1 + MAX_DEPTH) + cuts
        return cls(n_kv * tiles + shape.workers + thin, entries, entries * rep)


def _cut(cost, pages, marks, least, grain):
    """Units that stand in a line, each as long as its cost, cut where the line is marked, at a multiple of `grain` pages and into no
    pieces of fewer than `least` (a number for each unit): (unit, first page, page end, the number of marks in front of its middle) of
    every piece, in the line's order."""
    ends = np.cumsum(cost)
    at = ends - cost
    k0, k1 = np.searchsorted(marks, at, "right"), np.searchsorted(marks, ends - 1e-6, "left")
    n = np.maximum(0, k1 - k0)
    cu = np.repeat(np.arange(len(cost)), n)
    k = np.arange(len(cu)) - np.repeat(np.cumsum(n) - n, n) + k0[cu]
    cut = np.rint((marks[k] - at[cu]) / cost[cu] * pages[cu]).astype(np.int64) if len(cu) else cu
    cut = np.rint(cut / grain[cu]).astype(np.int64) * grain[cu]
    fine = (cut >= least[cu]) & (pages[cu] - cut >= least[cu])
    fine[1:] &= (cu[1:] != cu[:-1]) | (cut[1:] - cut[:-1] >= least[cu[1:]])
    cu, cut = cu[fine], cut[fine]
    iu, begin = np.concatenate([np.arange(len(cost)), cu]), np.concatenate([np.zeros(len(cost), dtype=np.int64), cut])
    by = np.lexsort((begin, iu))
    iu, begin = iu[by], begin[by]
    stop = np.append(begin[1:], 0)
    last = np.append(iu[1:] != iu[:-1], np.ones(min(1, len(iu)), dtype=bool))
    stop = np.where(last, pages[iu], stop[:len(iu)])
    middle = at[iu] + cost[iu] * (begin + stop) / (2.0 * np.maximum(1, pages[iu]))
    return iu, begin, stop, np.searchsorted(marks, middle, "right")


def _lay_out(order, nodes, own, held, new, rep: int, n_kv: int, shape: TileShape) -> dict:
    starts = np.cumsum(new) - new                                # first row of every sequence in the packed step
    n_o = new[order]
    ends_o = np.cumsum(n_o)
    T = int(ends_o[-1])
    first_o = ends_o - n_o
    toks = np.repeat(starts[order] - first_o, n_o) + np.arange(T)          # rows of the step in the tree's order
    # ---- nodes and leaves alike: tokens [off, off + n) of `toks` over pages [page, end) of sequence `seq`'s table
    lo = np.asarray([a for a, _, _, _ in nodes], dtype=np.int64)
    hi = np.asarray([b for _, b, _, _ in nodes], dtype=np.int64)
    off = np.concatenate([first_o[lo], first_o])
    n = np.concatenate([ends_o[hi - 1] - first_o[lo], n_o])
    page = np.concatenate([np.asarray([a for _, _, a, _ in nodes], dtype=np.int64), own])
    end = np.concatenate([np.asarray([b for _, _, _, b in nodes], dtype=np.int64), np.full(len(order), -1)])
    seq = np.concatenate([order[lo], order])
    # ---- tiles: a few tokens each, all query heads of a key/value head
    per = shape.rows // rep
    n_tiles = -(-n // per)
    s = np.repeat(np.arange(len(n)), n_tiles)
    i = np.arange(len(s)) - np.repeat(np.cumsum(n_tiles) - n_tiles, n_tiles)
    t_off = off[s] + i * per
    t_n = np.minimum(per, n[s] - i * per)
    t_last = toks[t_off + t_n - 1] if len(s) else np.zeros(0, dtype=np.int64)
    seq_of_row = np.repeat(np.arange(len(new)), new)
    last_pos = held[seq_of_row[t_last]] + t_last - starts[seq_of_row[t_last]] if len(s) else t_last
    t_end = np.where(end[s] < 0, last_pos // PAGE + 1, end[s])
    t_pages = t_end - page[s]
    thin = t_n * rep <= shape.thin_rows
    half = (t_n * rep <= shape.rows // 2) & ~thin if shape.halves else np.zeros(len(s), dtype=bool)
    cost = np.ones(len(s))
    for rows, page_cost in reversed(shape.costs):
        cost[t_n * rep <= rows] = page_cost
    cost = t_pages * cost + shape.item_pages
    cost[thin] = t_pages[thin] * shape.thin_cost + shape.thin_item
    # ---- a tile for every key/value head, the thin ones behind the others
    by = np.argsort(thin, kind="stable")
    u = np.repeat(by, n_kv)
    g = np.tile(np.arange(n_kv), len(s))
    c, pages_u = cost[u], t_pages[u]
    n_thick = n_kv * int((~thin).sum())
    share = max(float(c.sum()) / shape.workers, shape.min_pages + shape.item_pages)      # of a block
    # the line of the tiles' costs is cut into equal lengths, one for each block; what is left of each block's share is the warps'
    i1, b1, e1, w1 = _cut(c[:n_thick], pages_u[:n_thick], share * np.arange(1, shape.workers), np.full(n_thick, shape.min_pages),
                          np.where(half[u[:n_thick]], 2, 1))         # (the halves of a block that take pages in turn have as many each)
    if n_thick < len(u):
        load = np.bincount(w1, weights=c[i1] * (e1 - b1) / np.maximum(1, pages_u[i1]), minlength=shape.workers)
        left = np.maximum(share - load - np.where(load > 0, shape.thin_start, 0.0), 0.0)
        left = np.repeat((left if left.any() else np.ones_like(left)) / shape.thin_warps, shape.thin_warps)
        line = np.cumsum(left)
        least = np.maximum(1, -(-pages_u[n_thick:] // MOST_PIECES))
        i2, b2, e2, w2 = _cut(c[n_thick:], pages_u[n_thick:], line[:-1] * (float(c[n_thick:].sum()) / line[-1]), least, least)
    else:
        i2 = b2 = e2 = w2 = np.zeros(0, dtype=np.int64)
    iu, begin, stop = np.concatenate([i1, i2 + n_thick]), np.concatenate([b1, b2]), np.concatenate([e1, e2])
    last = stop == pages_u[iu]
    tile = u[iu]
    rows = t_n[tile] * rep * np.where(half[tile], 2, 1)
    part0 = np.cumsum(rows) - rows
    items = np.empty((len(iu), ITEM_WORDS), dtype=np.int32)
    leaf = end[s[tile]] < 0
    items[:, 0], items[:, 1], items[:, 2], items[:, 3] = t_off[tile], t_n[tile], np.where(leaf, t_last[tile], -1), g[iu]
    items[:, 4] = page[s[tile]] + begin
    items[:, 5] = np.where(last & leaf, -1, page[s[tile]] + stop)
    items[:, 6], items[:, 7] = part0, seq[s[tile]]
    first = np.searchsorted(w1, np.arange(shape.workers + 1))
    thin_first = len(i1) + np.searchsorted(w2, np.arange(shape.workers * shape.thin_warps + 1))
    # ---- which rows of the scratch belong to a token and key/value head
    n_i = t_n[tile]
    it = np.repeat(np.arange(len(iu)), n_i)
    inside = np.arange(len(it)) - np.repeat(np.cumsum(n_i) - n_i, n_i)
    key = toks[t_off[tile][it] + inside] * n_kv + g[iu][it]
    entry = part0[it] + inside * rep
    if shape.halves:
        twice = half[tile][it]
        key = np.concatenate([key, key[twice]])
        entry = np.concatenate([entry, entry[twice] + (n_i * rep)[it][twice]])
    by = np.argsort(key, kind="stable")
    list_first = np.zeros(T * n_kv + 1, dtype=np.int64)
    np.cumsum(np.bincount(key, minlength=T * n_kv), out=list_first[1:])
    return {"first": first, "thin_first": thin_first, "items": items, "toks": toks, "list_first": list_first, "list": entry[by], "part_rows": int(rows.sum()),
            "width": int(t_end.max(initial=0))}
