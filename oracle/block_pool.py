"""The block pool in plain Python: every block of a sequence by its number, the lowest free block first."""

from __future__ import annotations

from collections import deque


class Pool:
    def __init__(self, num_seqs: int, max_blocks: int, num_blocks: int, block: int):
        self.rows = [[] for _ in range(num_seqs)]
        self.lengths = [0] * num_seqs
        self.num_blocks, self.width, self.block = num_blocks, max_blocks, block
        self.refused = False
        self.copies: list = []  # of the last fork: (source block, target block, parent, child, rows)
        self.moves: dict = {}   # of the last compaction: block -> place

    def references(self) -> list[int]:
        counts = [0] * self.num_blocks
        for row in self.rows:
            for b in row:
                counts[b] += 1
        return counts

    def table(self) -> list[list[int]]:
        return [row + [-1] * (self.width - len(row)) for row in self.rows]

    def free(self) -> deque[int]:
        return deque(b for b, n in enumerate(self.references()) if n == 0)

    def advance(self, tokens: list[int]) -> None:
        references = self.references()
        for s, t in enumerate(tokens):
            row, (now, within) = self.rows[s], divmod(self.lengths[s], self.block)
            j, inside = divmod(self.lengths[s] + t, self.block)
            if t < 0 <= j < len(row) and inside and references[row[j]] > 1:
                self.refused = True  # back into a shared block: the length stays
                continue
            if t > 0 and not within and now < len(row) and references[row[now]] > 1:
                del row[now:]  # held from a longer length and shared: the next rows go into blocks of its own
            self.refused |= not 0 <= self.lengths[s] + t <= self.width * self.block
            self.lengths[s] = max(0, self.lengths[s] + t)
        free = self.free()
        for s, row in enumerate(self.rows):
            need = min(self.width, -(-self.lengths[s] // self.block))
            while len(row) < need:
                if not free:
                    self.refused = True
                    break
                row.append(free.popleft())

    def release(self, sequences: list[int]) -> None:
        for s in sequences:
            if 0 <= s < len(self.rows):
                self.rows[s], self.lengths[s] = [], 0
            else:
                self.refused = True

    def fork(self, parents: list[int], children: list[int]) -> None:
        seqs = range(len(self.rows))
        pairs, named = [], {c for p, c in zip(parents, children) if p in seqs and c in seqs and p != c}
        taken: set = set()
        for p, c in zip(parents, children):
            if p not in seqs or c not in seqs:
                self.refused = True
            elif p != c:
                first = c not in taken
                taken.add(c)
                good = first and p not in named and 0 <= self.lengths[p] <= len(self.rows[p]) * self.block
                self.refused |= not good
                if good:
                    pairs.append((p, c))
        for _, c in pairs:
            self.rows[c], self.lengths[c] = [], 0
        free, self.copies = self.free(), []
        for p, c in pairs:
            shared, rows = divmod(self.lengths[p], self.block)
            if rows and not free:
                self.refused = True
                continue
            self.rows[c], self.lengths[c] = self.rows[p][:shared], self.lengths[p]
            if rows:
                self.rows[c].append(free.popleft())
                self.copies.append((self.rows[p][shared], self.rows[c][-1], p, c, rows))

    def compact(self) -> int:
        counts = self.references()
        live = sum(n > 0 for n in counts)
        holes = [b for b in range(live) if counts[b] == 0]
        movers = [b for b in range(live, self.num_blocks) if counts[b] > 0]
        self.moves = dict(zip(movers, holes))
        self.rows = [[self.moves.get(b, b) for b in row] for row in self.rows]
        return live
