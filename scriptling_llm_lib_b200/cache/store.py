"""The cache: a slot for each live sequence, paged keys and values for each cache unit, and
per-sequence state of fixed size beside them.

The reference keeps, per layer and KV head, one growing array of rotated keys and one of values
for its single sequence (float32_ops.go:11-14, model_f32.go:310-317, :445-448). Here a *cache
unit* is what one entry of the model's schedule writes; units with the same need (all keys / a
window of them, same head count and width) form a *group* with storage of its own:
`k, v: [unit, page, kv_head, PAGE, head_dim]`. A sequence holds a slot; in each group the slot owns
a list of pages, position p living in page p // PAGE. One page id serves all units of the group.
Pages come from the group's pool as the sequence grows and go back when it is closed, or, in a
window group, as soon as no later query can see them. Nothing relies on cleared memory: every read
is bounded by the sequence's length.

A sequence can be forked: the new slots hold the same pages (a page's id then has several holders in its pool) and copies of the
fixed-size states. A page that several hold is never written: the step that would write its free positions first gives the
writer a page of its own with the positions held so far (`reserve`). Pages can be moved to the front of their storage, or into a
storage of another size, while sequences hold them (`compact`).
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from .needs import PAGE, CacheNeed, StateNeed
from .share import share_tree

SEQ_STATE_WORDS = 8      # int32 words of a sequence's record (lib_sampling.cu has the same layout)
SEQ_POS, SEQ_GENERATED, SEQ_LAST_TOKEN, SEQ_FLAGS, SEQ_KEY, SEQ_COUNTER = 0, 1, 2, 3, 4, 6
SEQ_FLAG_FINISHED = 1
from .pool import CacheFull, FreeList


def pages_for(n_tokens: int) -> int:
    return (n_tokens + PAGE - 1) // PAGE


@dataclass
class KVGroup:
    need: CacheNeed
    units: list[int]
    pool: FreeList
    k: torch.Tensor            # [len(units), n_pages, kv_heads, PAGE, head_dim]
    v: torch.Tensor
    pages: dict[int, list[int]] = field(default_factory=dict)   # slot -> page id per page index (-1: given back)
    behind: dict[int, int] = field(default_factory=dict)        # slot -> page indices below this one are settled: given back or kept
    table: np.ndarray | None = None    # [slots, pages so far] int32: the same ids as `pages` (-1: none), a step's block tables are cut from it

    def unit_storage(self, unit: int):
        i = self.units.index(unit)
        return self.k[i], self.v[i]

    def pages_needed(self, slot: int, new_len: int) -> int:
        return max(0, pages_for(new_len) - len(self.pages[slot]))

    def grow(self, slot: int, new_len: int) -> None:
        lst = self.pages[slot]
        n = pages_for(new_len)
        if n > self.table.shape[1]:
            more = np.full((self.table.shape[0], max(n, 2 * self.table.shape[1]) - self.table.shape[1]), -1, dtype=np.int32)
            self.table = np.concatenate([self.table, more], axis=1)
        while len(lst) < n:
            page = self.pool.alloc()
            self.table[slot, len(lst)] = page
            lst.append(page)

    def open(self, slot: int) -> None:
        self.pages[slot] = []
        self.behind[slot] = pages_for(self.need.keep)

    def release_unseen(self, slot: int, length: int) -> None:
        """Give back the pages no query at a position >= length can see (the need's kind says which; pages that hold one of
        the kept first positions stay)."""
        first_seen = self.need.first_needed(length)
        if first_seen <= 0:
            return
        lst, i = self.pages[slot], self.behind[slot]
        while i < len(lst) and (i + 1) * PAGE - 1 < first_seen:
            self.pool.free(lst[i])
            lst[i] = self.table[slot, i] = -1
            i += 1
        self.behind[slot] = i

    def fork(self, slot: int, new: int, length: int) -> None:
        """The new slot holds what `slot` holds of its first `length` positions: the same pages."""
        lst = self.pages[slot][:pages_for(length)]
        for pg in lst:
            if pg >= 0:
                self.pool.share(pg)
        self.pages[new] = lst
        self.table[new, :len(lst)] = lst
        self.behind[new] = self.behind[slot]

    def shared_written(self, slot: int, length: int, n: int) -> list[int]:
        """Places of the slot's pages that `n` tokens behind `length` would be written to and that others hold too."""
        lst = self.pages[slot]
        return [i for i in range(length // PAGE, min(len(lst), pages_for(length + n))) if lst[i] >= 0 and self.pool.holders(lst[i]) > 1]

    def copies_needed(self, growth, length) -> int:
        """Pages that a step which adds to these slots has to make its own first: every writer of a shared page needs one, but where all
        its holders write the last of them keeps it."""
        if not self.pool.n_shared:
            return 0
        writers: dict[int, int] = {}
        for slot, n in growth:
            for i in self.shared_written(slot, length[slot], n):
                page = self.pages[slot][i]
                writers[page] = writers.get(page, 0) + 1
        return sum(min(k, self.pool.holders(page) - 1) for page, k in writers.items())

    def own_written(self, slot: int, length: int, n: int) -> list[tuple[int, int, int, int, int]]:
        """Give the slot pages of its own where it would write shared ones: (from, to, positions held, slot, place) of each."""
        out = []
        for i in self.shared_written(slot, length, n):
            page, mine = self.pages[slot][i], self.pool.alloc()
            self.pool.free(page)
            self.pages[slot][i] = self.table[slot, i] = mine
            out.append((page, mine, max(0, length - i * PAGE), slot, i))
        return out

    def disown(self, own) -> None:
        """What `own_written` gave, taken back: the copies were not made."""
        for page, mine, _, slot, i in reversed(own):
            self.pool.share(page)
            self.pool.free(mine)
            self.pages[slot][i] = self.table[slot, i] = page

    def renumber(self, to: dict[int, int], n: int | None = None) -> None:
        self.pool.renumber(to, n)
        for slot, lst in self.pages.items():
            lst[:] = [to[pg] if pg >= 0 else -1 for pg in lst]
            self.table[slot, :len(lst)] = lst

    def release_all(self, slot: int) -> None:
        lst = self.pages.pop(slot)
        for pg in lst:
            if pg >= 0:
                self.pool.free(pg)
        self.table[slot, :len(lst)] = -1
        del self.behind[slot]


class SequenceCache:
    """Slots, page groups and fixed-size state for one model on one device."""

    def __init__(self, cache_needs: dict[int, CacheNeed | None], state_needs: dict[int, StateNeed | None],
                 n_slots: int, n_pages: int, dtype: torch.dtype, device):
        if n_slots < 1 or n_pages < 1:
            raise ValueError("the cache needs at least one slot and one page")
        self.n_slots, self.n_pages, self.dtype, self.device = n_slots, n_pages, dtype, torch.device(device)
        self.slots = FreeList(n_slots, "cache slot")
        self.length = [0] * n_slots
        self.version = 0          # changes whenever slots come to hold other pages than they did, but for pages added at their end
        self._trees: dict = {}
        self._kernels = None
        self.err_flag = None      # where the copying kernels report (an engine's; made on first use else)
        by_need: dict[CacheNeed, list[int]] = {}
        for unit, need in cache_needs.items():
            if need is not None:
                by_need.setdefault(need, []).append(unit)
        self.groups: list[KVGroup] = []
        self.group_of_unit: dict[int, int] = {}
        for need, units in by_need.items():
            # one page more than the pool hands out: padded rows of a replayed decode step write there
            shape = (len(units), n_pages + 1, need.kv_heads, PAGE, need.head_dim)
            v_shape = shape[:-1] + (need.value_dim,)
            g = KVGroup(need, units, FreeList(n_pages, f"cache page ({need.kind})"),
                        torch.empty(shape, dtype=dtype, device=device), torch.empty(v_shape, dtype=dtype, device=device),
                        table=np.full((n_slots, 16), -1, dtype=np.int32))
            for u in units:
                self.group_of_unit[u] = len(self.groups)
            self.groups.append(g)
        # the fixed-size record of every sequence, on the device: tokens held, tokens generated, last token,
        # flags, sampling key (2 words), draw counter (2 words). The sampler's kernel reads key and counter
        # from it and advances it; `length` above and the generation loop's bookkeeping are its host mirror.
        # One spare row serves the padding rows of replayed decode steps.
        self.seq_state = torch.zeros((n_slots + 1, SEQ_STATE_WORDS), dtype=torch.int32, device=device)
        def make(need):                                 # last row: spare, for padding
            if isinstance(need, dict):
                return {name: make(n) for name, n in need.items()}
            return torch.zeros((n_slots + 1, *need.shape), dtype=need.dtype, device=device)
        self.state: dict[int, torch.Tensor | dict] = {unit: make(need) for unit, need in state_needs.items() if need is not None}

    # ------------------------------------------------------------------ slots
    def open(self) -> int:
        slot = self.slots.alloc()
        self.length[slot] = 0
        self.version += 1
        for g in self.groups:
            g.open(slot)
        def zero(st):
            if isinstance(st, dict):
                for t in st.values():
                    zero(t)
            else:
                st[slot].zero_()
        zero(self.state)
        self.seq_state[slot].zero_()
        return slot

    def seed(self, slots: list[int], seeds: list[int]) -> None:
        """Start the sampling streams of freshly opened sequences: key = the sequence's 64-bit seed,
        draw counter 0 (one small copy for the batch)."""
        rec = np.zeros((len(slots), SEQ_STATE_WORDS), dtype=np.int64)
        for i, sd in enumerate(seeds):
            rec[i, SEQ_KEY], rec[i, SEQ_KEY + 1] = sd & 0xFFFFFFFF, (sd >> 32) & 0xFFFFFFFF
        rec = torch.from_numpy(rec.astype(np.uint32).view(np.int32))
        self.seq_state.index_copy_(0, torch.as_tensor(slots, dtype=torch.long, device=self.device), rec.to(self.device))

    def close(self, slot: int) -> None:
        if not self.slots.is_held(slot):
            raise ValueError(f"cache slot {slot} is not held; it cannot be closed")
        for g in self.groups:
            g.release_all(slot)
        self.slots.free(slot)
        self.length[slot] = 0
        self.version += 1

    # ------------------------------------------------------------------ copies
    def _ids(self, *lists):
        """Lists of numbers as int32 tensors on the cache's device, in one copy."""
        host = torch.tensor(list(lists), dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        return host.to(self.device, non_blocking=True)

    def _copy(self, pairs, src, dst, rows=None, slots=False) -> None:
        """Copies of pages (the first `rows` positions of each, None: all) or of slots, from one tensor to another or within one. A cache
        that is not on a CUDA device does bookkeeping alone (its tests); its few bytes go by indexing."""
        if not src or not pairs:
            return
        if self.device.type != "cuda":
            for a, b in pairs:
                for i, (s, d) in enumerate(zip(src, dst)):
                    if slots:
                        b[d] = a[s]
                    else:
                        n = PAGE if rows is None else rows[i]
                        b[:, d, :, :n] = a[:, s, :, :n]
            return
        if self._kernels is None:
            from ..csrc.bindings import PageKernels
            self._kernels = PageKernels()
        if self.err_flag is None:
            self.err_flag = torch.zeros(1, dtype=torch.int32, device=self.device)
        ids = self._ids(src, dst, *([rows] if rows is not None else []))
        if slots:
            self._kernels.copy_slots(pairs, ids[0], ids[1], self.err_flag)
        else:
            self._kernels.copy_pages(pairs, ids[0], ids[1], ids[2] if rows is not None else None, self.err_flag)

    def _states(self) -> list[torch.Tensor]:
        out, todo = [self.seq_state], list(self.state.values())
        while todo:
            st = todo.pop()
            if isinstance(st, dict):
                todo.extend(st.values())
            else:
                out.append(st)
        return out

    def fork(self, slot: int, n: int = 1) -> list[int]:
        """`n` new slots that hold what `slot` holds: the same pages, copies of its states and of its record (its sampling stream goes on
        in each: `seed` starts others). All, or an error (CacheFull, or what the copy of the states met) and none."""
        if not self.slots.is_held(slot):
            raise ValueError(f"cache slot {slot} is not held; it cannot be forked")
        if n < 0:
            raise ValueError(f"{n} forks of a sequence")
        if n > self.slots.n_free:
            raise CacheFull(f"{n} forks of a sequence; {self.slots.n_free} of {self.slots.n} cache slots are free")
        new = [self.slots.alloc() for _ in range(n)]
        for s in new:
            self.length[s] = self.length[slot]
            for g in self.groups:
                g.fork(slot, s, self.length[slot])
        self.version += 1
        try:
            self._copy([(t, t) for t in self._states()], [slot] * n, new, slots=True)
        except BaseException:
            for s in new:
                self.close(s)
            raise
        return new

    def compact(self, n_pages: int | None = None) -> int:
        """Move the held pages of every group to the front of its storage; with `n_pages`, into a new storage of that many (fewer give
        memory back, more make room; both are held until the copies are done). Returns the number of pages that were copied; CacheFull,
        with nothing changed, where more are held, and the allocator's error where there is no memory for the new storage. Kernels that were captured with the old storage's addresses are the caller's to drop."""
        if n_pages is not None:
            if n_pages < 1:
                raise ValueError("the cache needs at least one page")
            for g in self.groups:
                if g.pool.n_held > n_pages:
                    raise CacheFull(f"{g.pool.n_held} pages of the {g.need.kind} group are held; {n_pages} are to be kept")
            fresh = [[torch.empty((t.shape[0], n_pages + 1, *t.shape[2:]), dtype=t.dtype, device=t.device) for t in (g.k, g.v)] for g in self.groups]
        moved = 0
        for at, g in enumerate(self.groups):
            held = [i for i in range(g.pool.n) if g.pool.is_held(i)]
            if n_pages is None:
                k = len(held)
                to = {i: i for i in held if i < k}
                room = [i for i in range(k) if i not in to]
                to.update(zip((i for i in held if i >= k), room))
                src = [i for i in held if i >= k]
                self._copy([(g.k, g.k), (g.v, g.v)], src, [to[i] for i in src])
            else:
                to, src = {i: j for j, i in enumerate(held)}, held
                self._copy([(g.k, fresh[at][0]), (g.v, fresh[at][1])], src, [to[i] for i in src])
                g.k, g.v = fresh[at]
            g.renumber(to, n_pages)
            moved += len(src)
        if n_pages is not None:
            self.n_pages = n_pages
        self.version += 1
        return moved

    # ------------------------------------------------------------------ what sequences share
    @property
    def shares_pages(self) -> bool:
        return any(g.pool.n_shared for g in self.groups)

    def share_tree(self, group: int, slots: list[int]):
        """`share_tree` of these slots' pages, kept until slots come to hold other pages."""
        if not self.groups[group].pool.n_shared:
            return None
        if self._trees.get("version") != self.version or len(self._trees) > 64:
            self._trees = {"version": self.version}
        key = (group, tuple(slots))
        if key not in self._trees:
            whole = np.asarray([self.length[s] // PAGE for s in slots], dtype=np.int64)
            self._trees[key] = share_tree(np.ascontiguousarray(self.block_table(group, slots)), whole)
        return self._trees[key]

    # ------------------------------------------------------------------ growth
    def reserve(self, growth: list[tuple[int, int]]) -> None:
        """Pages for `n_new` more tokens of each (slot, n_new); either all are had or CacheFull is
        raised and nothing has changed. A slot that would write a page that others hold too gets a copy of its own (where that
        copy meets an error, the slots hold the pages that they held)."""
        for g in self.groups:
            want = sum(g.pages_needed(slot, self.length[slot] + n) for slot, n in growth) + g.copies_needed(growth, self.length)
            if want > g.pool.n_free:
                raise CacheFull(f"the step needs {want} more cache pages of {PAGE} tokens in the {g.need.kind} group; "
                                f"{g.pool.n_free} of {g.pool.n} are free")
        for g in self.groups:
            if g.pool.n_shared:
                own = [c for slot, n in growth for c in g.own_written(slot, self.length[slot], n)]
                if own:
                    self.version += 1
                    try:
                        self._copy([(g.k, g.k), (g.v, g.v)], *(list(c) for c in list(zip(*own))[:3]))
                    except BaseException:
                        g.disown(own)
                        raise
            for slot, n in growth:
                g.grow(slot, self.length[slot] + n)

    def advance(self, growth: list[tuple[int, int]]) -> None:
        for slot, n in growth:
            self.length[slot] += n
            for g in self.groups:
                g.release_unseen(slot, self.length[slot])

    # ------------------------------------------------------------------ views for a step
    def block_table(self, group: int, slots: list[int], width: int | None = None) -> np.ndarray:
        g = self.groups[group]
        w = max(1, max(len(g.pages[s]) for s in slots)) if width is None else width
        if w <= g.table.shape[1]:
            return g.table[slots, :w]
        bt = np.full((len(slots), w), -1, dtype=np.int32)
        bt[:, :g.table.shape[1]] = g.table[slots]
        return bt

    def tokens_capacity(self) -> int:
        return self.n_pages * PAGE
