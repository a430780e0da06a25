"""Host-side bookkeeping of pages and slots: nothing is lost, held twice or freed twice."""
from __future__ import annotations


class CacheFull(RuntimeError):
    """The step needs more pages or slots than are free; nothing was changed."""


class FreeList:
    """Ids 0..n-1, handed out lowest first; `free` refuses an id that is not held. An id may have several holders (`share`): it is free
    again when the last of them has given it back."""

    def __init__(self, n: int, what: str):
        self.n = n
        self.what = what
        self._free = list(range(n - 1, -1, -1))
        self._held = [0] * n          # holders of every id
        self.n_shared = 0             # ids with more than one holder

    @property
    def n_free(self) -> int:
        return len(self._free)

    @property
    def n_held(self) -> int:
        return self.n - len(self._free)

    def alloc(self) -> int:
        if not self._free:
            raise CacheFull(f"no free {self.what} (all {self.n} are held)")
        i = self._free.pop()
        self._held[i] = 1
        return i

    def share(self, i: int) -> None:
        """One more holder of an id that is held."""
        if not self.is_held(i):
            raise ValueError(f"{self.what} {i} is not held; it cannot be shared")
        self._held[i] += 1
        self.n_shared += self._held[i] == 2

    def free(self, i: int) -> None:
        if not self.is_held(i):
            raise ValueError(f"{self.what} {i} is not held; it cannot be freed")
        self._held[i] -= 1
        self.n_shared -= self._held[i] == 1
        if self._held[i] == 0:
            self._free.append(i)

    def is_held(self, i: int) -> bool:
        return 0 <= i < self.n and self._held[i] > 0

    def holders(self, i: int) -> int:
        return self._held[i] if 0 <= i < self.n else 0

    def renumber(self, to: dict[int, int], n: int | None = None) -> None:
        """Every held id i becomes to[i], of n ids in all; the free ones are handed out lowest first again."""
        n = self.n if n is None else n
        held = [0] * n
        for i, j in to.items():
            held[j] = self._held[i]
        if len(to) != self.n_held or len(set(to.values())) != len(to) or any(c == 0 for c in (held[j] for j in to.values())):
            raise ValueError(f"{self.what}s: a renumbering names every held id once")
        self.n, self._held, self._free = n, held, [i for i in range(n - 1, -1, -1) if not held[i]]
