"""The books of a paged cache whose rows share blocks, restated with lists.  The reference has no shared blocks; its policy of
lowest ids first and sorted releases is ``src/decode_state.py:72-84``."""

from __future__ import annotations

from dataclasses import dataclass, field


@dataclass
class Books:
    """Rows of block ids with their lengths, the ascending free ids, and the holders of a block beyond its first."""

    block: int
    capacity: int
    rows: list[list[int]]
    lengths: list[int]
    free: list[int]
    references: dict[int, int] = field(default_factory=dict)

    def fork(self, pairs: list[tuple[int, int]]) -> list[tuple[int, int]]:
        """The pages to be copied, (-1, -1) where a fork has none."""
        pages = []
        for source, target in pairs:
            if source < 0:
                pages.append((-1, -1))
                continue
            length = self.lengths[source]
            full = length // self.block
            shared = self.rows[source][:full]
            for block in shared:
                self.references[block] = self.references.get(block, 0) + 1
            row = list(shared)
            page = (-1, -1)
            if length % self.block:
                row.append(self.free.pop(0))
                page = (self.rows[source][full], row[-1])
            pages.append(page)
            self.rows[target], self.lengths[target] = row, length
        return pages

    def release(self, rows: list[int]) -> None:
        for row in rows:
            for block in self.rows[row]:
                if self.references.get(block, 0) > 0:
                    self.references[block] -= 1
                else:
                    self.free.append(block)
            self.rows[row], self.lengths[row] = [], 0
        self.free.sort()

    def compact(self, max_moves: int) -> list[tuple[int, int]]:
        pages = []
        free = list(self.free)
        for source in sorted({b for row in self.rows for b in row}, reverse=True):
            if len(pages) == max_moves or len(pages) == len(self.free) or self.free[len(pages)] > source:
                break
            pages.append((source, self.free[len(pages)]))
        place = dict(pages)
        self.rows = [[place.get(b, b) for b in row] for row in self.rows]
        self.references = {place.get(b, b): n for b, n in self.references.items()}
        self.free = sorted(free[len(pages) :] + [source for source, _ in pages])
        return pages
