"""Which sequences of a step hold pages together.

Slots that were forked from one another name the same pages at the beginning of their page tables. The reference keeps
a cache a sequence (crates/backends/backend_common/src/kv_cache.rs:270-273) and shares nothing.
"""
from dataclasses import dataclass, field
from functools import cached_property
from typing import List, Tuple

import numpy as np

from .slots import PAGE_TOKENS

MAX_LEVELS = 8          # stretches of shared pages that are told apart along one sequence; what is shared beyond counts as its own


@dataclass
class SharedPages:
    """order: the step's sequences, those that share pages side by side. nodes: (first, count, page, end): the sequences
    order[first : first + count] all hold the same pages in the places [page, end) of their tables; end -1 (count 1): the rest
    of the sequence's pages. Every page of a sequence lies in exactly one of the nodes that it is in."""
    order: np.ndarray
    nodes: List[Tuple[int, int, int, int]]
    _filled: object = field(default=None, repr=False, compare=False)

    def filled_up(self, sequences):
        """The same of a step that is filled up to so many sequences: each of the further ones by itself."""
        n = len(self.order)
        if sequences == n:
            return self
        if self._filled is None or len(self._filled.order) != sequences:
            more = range(n, sequences)
            self._filled = SharedPages(np.concatenate([self.order, np.array(more, dtype=np.int64)]), self.nodes + [(i, 1, 0, -1) for i in more])
        return self._filled

    @cached_property
    def node_array(self):
        """The nodes as one array [nodes, 4]."""
        return np.ascontiguousarray(np.array(self.nodes, dtype=np.int64).reshape(-1, 4))

    @cached_property
    def pages_saved(self):
        """How many pages fewer are read than if every sequence read its own."""
        return sum((count - 1) * (end - page) for _, count, page, end in self.nodes if count > 1)


def shared_pages(table, held):
    """The SharedPages of sequences with the page tables `table` (int [sequences, pages], by row) that hold `held` positions
    before the step; None where no page is shared. Only pages that are full then are looked at: the others are
    written to, and belong to one sequence."""
    table, full = np.asarray(table), np.asarray(held, dtype=np.int64) // PAGE_TOKENS
    if len(full) < 2:
        return None
    order, nodes = [], []

    def walk(members, page, level):
        # (members hold the same pages up to `page`)
        classes = {}
        for i in members:
            classes.setdefault(int(table[i, page]) if full[i] > page and level < MAX_LEVELS else (i,), []).append(i)
        for same in classes.values():
            if len(same) == 1:
                nodes.append((len(order), 1, page, -1))
                order.append(same[0])
                continue
            rows = table[same, page:int(full[same].min())]
            differs = np.nonzero((rows != rows[0]).any(0))[0]
            end = page + (int(differs[0]) if len(differs) else rows.shape[1])
            nodes.append((len(order), len(same), page, end))
            walk(same, end, level + 1)

    walk(range(len(full)), 0, 0)
    if all(count == 1 for _, count, _, _ in nodes):
        return None
    return SharedPages(np.array(order, dtype=np.int64), nodes)
