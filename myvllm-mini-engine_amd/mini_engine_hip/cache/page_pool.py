"""Refcounted physical pages, including shared read-only prefix pages.

Restates the ownership semantics of the reference's ``BlockManager``
(mini_engine/cache/block_manager.py:10-166) that decide which physical page
ids appear in the block tables the kernels read: private pages are
refcount 1, a cached prefix attached to several requests appears in each of
their tables (refcount = number of holders), and a request can be given
retained pages only (``attach``, block_manager.py:83-97 — the prefix cache's
whole-prompt hit, prefix_cache.py:45-48), so its table holds no private
page at all.  Host-side only.

``fork``, ``make_writable`` and ``compact`` return the page copies that have
to follow on the device, as (source, destination) pairs: ``copy_pages`` and
``compact_pages`` of the cache pools run them.
"""

from __future__ import annotations


class PagePool:
    def __init__(self, num_blocks: int, block_size: int, order=None):
        """``order`` (optional) is the sequence in which free pages are handed out."""
        if num_blocks <= 0 or block_size <= 0:
            raise ValueError("num_blocks and block_size must be positive")
        self.num_blocks = num_blocks
        self.block_size = block_size
        order = list(range(num_blocks)) if order is None else [int(p) for p in order]
        if sorted(order) != list(range(num_blocks)):
            raise ValueError("order must be a permutation of the page ids")
        self._free = order[::-1]
        self._refs = [0] * num_blocks
        self._owned: dict[str, list[int]] = {}

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    def blocks_required(self, token_count: int) -> int:
        if token_count < 0:
            raise ValueError("token_count cannot be negative")
        return -(-token_count // self.block_size)

    def refcount(self, block: int) -> int:
        return self._refs[block]

    def _take(self, count: int) -> list[int]:
        if count > len(self._free):
            raise MemoryError(f"need {count} blocks, only {len(self._free)} free")
        pages = [self._free.pop() for _ in range(count)]
        for page in pages:
            self._refs[page] = 1
        return pages

    def _check_live(self, pages, what="prefix") -> None:
        if len(set(pages)) != len(pages):
            raise ValueError(f"{what} pages must be distinct")
        for page in pages:
            if page < 0 or page >= self.num_blocks or self._refs[page] <= 0:
                raise ValueError(f"cannot attach unallocated block: {page}")

    def allocate(self, request_id: str, token_count: int) -> list[int]:
        return self.allocate_with_prefix(request_id, token_count, ())

    def allocate_with_prefix(self, request_id: str, token_count: int, prefix) -> list[int]:
        """Attach shared prefix pages, then allocate private pages for the rest."""
        if request_id in self._owned:
            raise ValueError(f"request already owns blocks: {request_id}")
        prefix = list(prefix)
        self._check_live(prefix)
        required = self.blocks_required(token_count)
        if len(prefix) > required:
            raise ValueError("prefix has more blocks than the request needs")
        suffix = self._take(required - len(prefix))
        for page in prefix:
            self._refs[page] += 1
        self._owned[request_id] = prefix + suffix
        return list(self._owned[request_id])

    def attach(self, request_id: str, pages) -> list[int]:
        """Give a request a table made only of pages other holders retain."""
        if request_id in self._owned:
            raise ValueError(f"request already owns blocks: {request_id}")
        pages = [int(p) for p in pages]
        self._check_live(pages, "attached")
        for page in pages:
            self._refs[page] += 1
        self._owned[request_id] = pages
        return list(pages)

    def fork(self, request_id: str, new_request: str, token_count: int):
        """Give ``new_request`` the first ``token_count`` tokens of a request.

        Whole pages are shared; a partly written last page is copied, since both
        requests write on behind it.  The new table ends with that page:
        ``extend`` gives it more.  Returns (the new table, page copies).
        """
        if new_request in self._owned:
            raise ValueError(f"request already owns blocks: {new_request}")
        table = self._owned[request_id]
        if not 0 <= token_count <= len(table) * self.block_size:
            raise ValueError("fork passes the request's pages")
        whole, rest = divmod(token_count, self.block_size)
        copy = self._take(1 if rest else 0)
        for page in table[:whole]:
            self._refs[page] += 1
        self._owned[new_request] = table[:whole] + copy
        return list(self._owned[new_request]), [(table[whole], page) for page in copy]

    def extend(self, request_id: str, token_count: int) -> list[int]:
        """Give a request the private pages that ``token_count`` tokens need beyond its table, if any.

        Returns its table.  Where the pages run out, nothing has changed.
        """
        table = self._owned[request_id]
        table += self._take(max(0, self.blocks_required(token_count) - len(table)))
        return list(table)

    def truncate(self, request_id: str, token_count: int) -> list[int]:
        """Give back the pages of a request behind its first ``token_count`` tokens (after an eviction).

        Returns its table.  Where that now ends inside a page that others hold
        too, ``make_writable`` comes before the next token's write.
        """
        table = self._owned[request_id]
        if not 0 <= token_count <= len(table) * self.block_size:
            raise ValueError("truncation passes the request's pages")
        for page in reversed(table[self.blocks_required(token_count):]):
            self._release(page)
        del table[self.blocks_required(token_count):]
        return list(table)

    def make_writable(self, request_id: str, index: int):
        """Before writing into page ``index`` of a table: a page that others hold too is replaced by a copy.

        Returns (the page to write, page copies).
        """
        table = self._owned[request_id]
        if not 0 <= index < len(table):
            raise IndexError("page index out of range")
        page = table[index]
        if self._refs[page] == 1:
            return page, []
        (copy,) = self._take(1)
        self._release(page)
        table[index] = copy
        return copy, [(page, copy)]

    def compact(self):
        """Move live pages down into free lower ones, and renumber every table.

        Returns the moves, sources rising; no page is both source and
        destination.  Pages pinned from outside stay, since whoever pinned them
        goes by their number.  Until the moves have run on the device, and the
        device's block tables have been renumbered, nothing may be written.
        """
        held = [0] * self.num_blocks
        for table in self._owned.values():
            for page in table:
                held[page] += 1
        movable = [p for p in range(self.num_blocks - 1, -1, -1) if self._refs[p] and self._refs[p] == held[p]]
        moves = [(src, dst) for src, dst in zip(movable, sorted(self._free)) if dst < src]
        number = dict(moves)
        for src, dst in moves:
            self._refs[dst], self._refs[src] = self._refs[src], 0
        for table in self._owned.values():
            table[:] = [number.get(page, page) for page in table]
        self._free = [p for p in range(self.num_blocks - 1, -1, -1) if not self._refs[p]]  # the lowest goes out first
        return moves[::-1]

    def pin(self, pages) -> None:
        """Hold one external reference (e.g. a prefix-cache entry)."""
        pages = list(pages)
        self._check_live(pages, "pinned")
        for page in pages:
            self._refs[page] += 1

    def unpin(self, pages) -> None:
        for page in pages:
            self._release(page)

    def free(self, request_id: str) -> None:
        for page in self._owned.pop(request_id):
            self._release(page)

    def _release(self, page: int) -> None:
        if self._refs[page] <= 0:
            raise ValueError(f"double free of block {page}")
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def table(self, request_id: str) -> list[int]:
        return list(self._owned[request_id])
