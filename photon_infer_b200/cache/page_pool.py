"""Free list of cache pages.

Same contract as the reference's ``BlockManager`` (include/photon/runtime/
block_manager.hpp:39-157, src/runtime/block_manager.cpp:14-182): a stack of free page
ids and a record of which are out, exhaustion is an ``OUT_OF_MEMORY`` error, a page
freed twice is detected.  Pages are handed out in a fixed order (lowest id first, a
freed page is the next to be reused), so a replayed trace gets the same pages.

A page may have several holders (requests that forked from one another); it is free again when the last
of them has freed it.
"""
from __future__ import annotations

from typing import Dict, List

from ..errors import ErrorCode, PhotonError


class PagePool:
    def __init__(self, num_pages: int):
        if num_pages <= 0:
            raise PhotonError(ErrorCode.INVALID_ARGUMENT, "a page pool needs at least one page")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages - 1, -1, -1))   # pop() gives the lowest id first
        self._holders = [0] * num_pages
        self.high_water = 0

    @property
    def num_free(self) -> int:
        return len(self._free)

    @property
    def num_allocated(self) -> int:
        return self.num_pages - len(self._free)

    def allocate(self) -> int:
        if not self._free:
            raise PhotonError(ErrorCode.OUT_OF_MEMORY, f"no free cache page (all {self.num_pages} are in use)")
        page = self._free.pop()
        self._holders[page] = 1
        self.high_water = max(self.high_water, self.num_allocated)
        return page

    def allocate_many(self, n: int) -> List[int]:
        if n > len(self._free):
            raise PhotonError(ErrorCode.OUT_OF_MEMORY,
                              f"{n} cache pages wanted, {len(self._free)} of {self.num_pages} free")
        return [self.allocate() for _ in range(n)]

    def free(self, page: int) -> None:
        if not 0 <= page < self.num_pages:
            raise PhotonError(ErrorCode.INVALID_INDEX, f"page {page} is outside the pool of {self.num_pages}")
        if not self._holders[page]:
            raise PhotonError(ErrorCode.DOUBLE_FREE, f"page {page} is freed but not held")
        self._holders[page] -= 1
        if not self._holders[page]:
            self._free.append(page)

    def share(self, page: int) -> int:
        """One more holder for a page that is out."""
        if not 0 <= page < self.num_pages or not self._holders[page]:
            raise PhotonError(ErrorCode.INVALID_STATE, f"page {page} is shared but not held")
        self._holders[page] += 1
        return page

    def holders(self, page: int) -> int:
        return self._holders[page]

    def is_allocated(self, page: int) -> bool:
        return self._holders[page] > 0

    def pack(self) -> Dict[int, int]:
        """Where the pages that are out would have to go so that they are the lowest ids: old id -> new id of those that move.
        The pool takes the new ids at once; the caller moves the contents."""
        live = self.num_allocated
        gaps = [i for i in range(live) if not self._holders[i]]
        moves = dict(zip((i for i in range(live, self.num_pages) if self._holders[i]), gaps))
        for old, new in moves.items():
            self._holders[new], self._holders[old] = self._holders[old], 0
        self._free = list(range(self.num_pages - 1, live - 1, -1))
        return moves

    def utilization(self) -> float:
        return self.num_allocated / self.num_pages
