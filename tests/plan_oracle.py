"""The cut of a step whose sequences share pages, in NumPy: what csrc/hostcall.cpp's plan has to give, number for number."""
import numpy as np

from herbert_rs_amd.kernels.shared import ITEM_INTS, MASKED_COLUMNS


def _even(first, end, most):
    """Cut first .. end into as few stretches of at most `most` as there can be, alike in length: (first, length)."""
    count = -(-(end - first) // most)
    cuts = [first + (end - first) * i // count for i in range(count + 1)]
    return [(a, b - a) for a, b in zip(cuts[:-1], cuts[1:])]


def plan(starts, context, slots, sharing, group, nkv, columns, workgroups, grid=1):
    """How a step is cut up. starts: the first packed row of each sequence and the last one's end; context: the positions it
    holds after the step; slots: theirs; sharing: a SharedPages. Returns int32 arrays (items [n, 8], order [rows], part_start
    [rows + 1], parts) and the most rows of an item; see csrc/attention_shared.hip.

    A node of the sharing is cut into tiles of as many rows as fit `columns`; a tile's pages are cut into ranges of about as many pages
    each that the workgroups (items x kv heads) come to `workgroups`, whole rounds of the waves that take them in turn. The pages
    that a tile of more than 64 columns sees in part are items of their own."""
    starts, context = np.asarray(starts, dtype=np.int64), np.asarray(context, dtype=np.int64)
    counts = np.diff(starts)
    row_of = np.concatenate([[0], np.cumsum(counts[sharing.order])])            # a sequence's first row in the order
    of_row = np.repeat(sharing.order, counts[sharing.order])                    # whose row it is
    order = starts[of_row] + np.arange(len(of_row)) - row_of[np.repeat(np.arange(len(counts)), counts[sharing.order])]
    tall = max(1, columns // group)
    short = max(1, MASKED_COLUMNS // group) if columns == 128 else tall
    tiles = []                                                                  # row0, rows, sequence, first page, end, first page seen in part
    nodes = np.array(sharing.nodes, dtype=np.int64).reshape(-1, 4)
    alone = (nodes[:, 3] < 0) & (counts[sharing.order[nodes[:, 0]]] == 1)       # a sequence's own pages, one row: all of them at once
    for first, count, page, end in nodes[~alone].tolist():
        a, b, seq = int(row_of[first]), int(row_of[first + count]), int(sharing.order[first])
        for r, n in _even(a, b, tall):
            if end >= 0:
                tiles.append((r, n, seq, page, end, end))
                continue
            # A sequence's own rows: all of them see what lies before the first row's page; a tile ends at the page of its last row.
            whole, page_from = (int(context[seq]) - (b - r)) // 64, page
            if n * group > 64 and whole > page:
                tiles.append((r, n, seq, page, whole, whole))
                page_from = whole
            for u, m in _even(r, r + n, short):
                first_seen, last_seen = int(context[seq]) - (b - u), int(context[seq]) - (b - (u + m)) - 1
                tiles.append((u, m, seq, page_from, last_seen // 64 + 1, first_seen // 64))
    first = nodes[alone, 0]
    seen = (context[sharing.order[first]] - 1) // 64
    of_one = np.stack([row_of[first], np.ones_like(first), sharing.order[first], nodes[alone, 2], seen + 1, seen])
    row0, rows, seq, page, end, whole = np.concatenate([np.array(tiles, dtype=np.int64).reshape(-1, 6).T, of_one], axis=1)
    cols, pages = rows * group, end - page
    turns = np.where(cols <= 32, 4, np.where(cols <= 64, 2, 1)) if columns == 128 else np.ones_like(cols)
    share = max(1, -(-int(pages.sum()) * nkv // workgroups))
    per = -(-share // turns) * turns
    ranges = -(-pages // per)
    per = -(-(-(-pages // ranges)) // turns) * turns
    of = np.repeat(np.arange(len(rows)), ranges)
    nth = np.arange(len(of)) - np.repeat(np.cumsum(ranges) - ranges, ranges)
    items = np.zeros((len(of), ITEM_INTS), dtype=np.int64)
    items[:, 0], items[:, 1], items[:, 2] = row0[of], rows[of], np.asarray(slots, dtype=np.int64)[seq[of]]
    items[:, 3] = page[of] + nth * per[of]
    items[:, 4] = np.minimum(items[:, 3] + per[of], end[of])
    items[:, 6] = items[:, 4] > whole[of]
    items = items[items[:, 4] > items[:, 3]]              # (ranges rounded up may leave the last ones nothing)
    n = items[:, 1]
    items[:, 5] = np.cumsum(n) - n
    # a row's partial results lie side by side, in the order of its pages
    total = int(n.sum())
    row = np.repeat(items[:, 0] - items[:, 5], n) + np.arange(total)
    parts = np.empty(total, dtype=np.int64)
    parts[np.argsort(row, kind="stable")] = np.arange(total)
    part_start = np.concatenate([[0], np.cumsum(np.bincount(row, minlength=len(order)))])
    # the longest items first, those over the same pages side by side
    items = items[np.lexsort((items[:, 0], items[:, 3], items[:, 3] - items[:, 4]))]
    most = int(n.max())
    n_items = -(-len(items) // grid) * grid
    items = np.concatenate([items, np.zeros((n_items - len(items), ITEM_INTS), dtype=np.int64)])
    as32 = lambda x: np.ascontiguousarray(x, dtype=np.int32)
    return as32(items), as32(order), as32(part_start), as32(parts), most
