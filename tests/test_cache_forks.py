"""Slots that share pages: forks, copies on the first write, pages that go back with their last holder."""
import random

import numpy as np
import pytest
import torch

from herbert_rs_amd.cache import Cache, KVNeed, StateNeed, pages_for
from herbert_rs_amd.errors import CacheError

FULL, WINDOW = KVNeed(2, 8, None), KVNeed(2, 8, 70)


def make_cache(window=None, state=False, max_tokens=64 * 12, max_positions=512, slots=None):
    needs = {0: FULL, 1: KVNeed(2, 8, window), 2: FULL}
    if state:
        needs[3] = (StateNeed((4,), torch.float32), StateNeed((3, 2), torch.float32))
    return Cache(needs, max_tokens, max_positions, torch.float32, "cpu", slots)


def write(cache, slot, values):
    """One step of a slot: position p of entry e becomes values[p] + 1000 e in keys and values (as a model's kernels would write them)."""
    before = cache.length(slot)
    cache.reserve_all([(slot, len(values))])
    for e in (0, 1, 2):
        kv = cache.kv_view(e)
        for i, v in enumerate(values):
            page, at = int(kv.page_table[slot, (before + i) // 64]), (before + i) % 64
            kv.k[page, :, at] = v + 1000 * e
            kv.v[page, :, :, at] = v + 1000 * e
    cache.commit(slot, len(values))


def read(cache, slot, entry, first=0):
    kv, out = cache.kv_view(entry), []
    for p in range(first, cache.length(slot)):
        page = int(kv.page_table[slot, p // 64])
        assert (kv.k[page, :, p % 64] == kv.k[page, 0, p % 64, 0]).all()
        assert (kv.v[page, :, :, p % 64] == kv.k[page, 0, p % 64, 0]).all()
        out.append(float(kv.k[page, 0, p % 64, 0]) - 1000 * entry)
    return out


def test_a_fork_holds_the_same_pages_until_somebody_writes():
    c = make_cache()
    a = c.alloc_slot()
    write(c, a, list(range(100)))
    g = c.kv_groups[FULL]
    assert g.pages.held_count == 2 and not c.shares_pages
    b, d = c.fork(a, 2)
    c.check()
    assert g.pages.held_count == 2 and c.shares_pages and c.length(b) == c.length(d) == 100
    assert read(c, b, 2) == list(range(100))
    write(c, b, [7.0])                       # the second page is copied for b
    c.check()
    assert g.pages.held_count == 3
    write(c, a, [8.0, 9.0])                  # and for a: d is left with the first one
    assert g.pages.held_count == 4
    write(c, d, [5.0])                       # its only holder writes in place
    assert g.pages.held_count == 4
    c.check()
    for slot, tail in ((a, [8, 9]), (b, [7]), (d, [5])):
        for e in (0, 1, 2):
            assert read(c, slot, e) == list(range(100)) + tail
    found = c.shared_pages([b, a, d], [c.length(s) for s in (b, a, d)])
    assert found.nodes[0] == (0, 3, 0, 1) and found.pages_saved == 2
    c.free_slot(a)
    c.free_slot(d)
    c.check()
    assert g.pages.held_count == 2 and not c.shares_pages and read(c, b, 0) == list(range(100)) + [7]
    c.free_slot(b)
    c.check()
    assert g.pages.held_count == 0


def test_a_step_of_all_holders_copies_for_all_but_one():
    c = make_cache(max_tokens=64 * 6)
    a = c.alloc_slot()
    write(c, a, list(range(70)))
    slots = [a] + c.fork(a, 3)
    g = c.kv_groups[FULL]
    # two pages held; three copies and no new page: five of the six. With a further page wanted by one of them: all six
    c.reserve_all([(s, 1) for s in slots[:3]] + [(slots[3], 64)])
    assert g.pages.free_count == 0
    for s in slots:
        c.unreserve(s)
        c.check()
    assert g.pages.free_count == 1


def test_a_step_that_needs_more_copies_than_there_are_pages_changes_nothing():
    c = make_cache(max_tokens=64 * 4)
    a = c.alloc_slot()
    write(c, a, list(range(70)))
    slots = [a] + c.fork(a, 3)
    table = [g.table_host.copy() for g in c.kv_groups.values()]
    with pytest.raises(CacheError, match="3 more pages"):
        c.reserve_all([(s, 1) for s in slots])
    c.check()
    assert all((g.table_host == t).all() for g, t in zip(c.kv_groups.values(), table))
    c.reserve_all([(s, 1) for s in slots[:2]])


def test_forks_at_a_page_s_end_copy_nothing():
    c = make_cache()
    a = c.alloc_slot()
    write(c, a, list(range(64)))
    b, = c.fork(a)
    write(c, a, [1.0])
    write(c, b, [2.0])
    g = c.kv_groups[FULL]
    assert g.pages.held_count == 3 and g.further == {int(g.table_host[a][0]): 1}
    assert read(c, a, 0)[-1] == 1 and read(c, b, 0)[-1] == 2


def test_rolling_back_into_shared_pages_and_going_on_leaves_the_others_as_they_are():
    c = make_cache()
    a = c.alloc_slot()
    write(c, a, list(range(130)))
    b, = c.fork(a)
    c.truncate(b, 80)
    c.check()
    write(c, b, [500.0] * 3)
    assert read(c, a, 1) == list(range(130)) and read(c, b, 1) == list(range(80)) + [500] * 3
    c.truncate(a, 128)
    write(c, a, [3.0])
    assert read(c, a, 0) == list(range(128)) + [3] and read(c, b, 0) == list(range(80)) + [500] * 3
    c.check()


def test_windows_give_shared_pages_back_with_their_last_holder():
    c = make_cache(window=70, max_tokens=64 * 16)
    a = c.alloc_slot()
    write(c, a, list(range(100)))
    b, = c.fork(a)
    w = c.kv_groups[WINDOW]
    write(c, a, list(range(100, 200)))
    c.check()
    assert read(c, b, 1, first=31) == list(range(31, 100))
    write(c, b, list(range(300, 400)))
    c.check()
    assert read(c, a, 1, first=131) == list(range(131, 200)) and read(c, b, 1, first=131) == list(range(331, 400))
    assert not w.further and c.kv_groups[FULL].further
    c.free_slot(a)
    c.free_slot(b)
    c.check()
    assert w.pages.held_count == 0


def test_states_are_copied():
    c = make_cache(state=True)
    a = c.alloc_slot()
    write(c, a, [1.0] * 5)
    first, second = c.state_views(3)
    first[a], second[a] = 3.0, 4.0
    b, d = c.fork(a, 2)
    first[a] = 9.0
    for s in (b, d):
        assert (first[s] == 3).all() and (second[s] == 4).all()
    e = c.alloc_slot()
    assert (c.state_views(3)[0][e] == 0).all() and (c.state_views(3)[0][b] == 3).all()
    fresh = c.fork(e, 1)[0]                  # a slot that holds nothing yet
    assert (c.state_views(3)[0][fresh] == 0).all() and c.length(fresh) == 0


def test_what_a_fork_refuses():
    c = make_cache(slots=3)
    a = c.alloc_slot()
    write(c, a, [1.0])
    for count in (0, -1):
        with pytest.raises(CacheError, match="one or more"):
            c.fork(a, count)
    with pytest.raises(CacheError, match="only 2 of 3"):
        c.fork(a, 3)
    with pytest.raises(CacheError, match="not held"):
        c.fork(2)
    c.check()
    assert c.slots.held_count == 1 and not c.shares_pages
    assert c.shared_pages([a], [1]) is None


def test_copies_that_find_no_memory_leave_the_slots_as_they_are(monkeypatch):
    c = make_cache()
    a = c.alloc_slot()
    write(c, a, list(range(70)))
    b, = c.fork(a)
    g = c.kv_groups[FULL]

    def no_memory(*args):
        raise MemoryError
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "index_select", no_memory)
        with pytest.raises(MemoryError):
            c.reserve_all([(a, 1), (b, 1)])
    c.check()
    assert g.pages.held_count == 2
    write(c, b, [5.0])
    assert read(c, a, 0) == list(range(70)) and read(c, b, 0) == list(range(70)) + [5]


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_keep_the_books_and_the_contents(seed):
    rnd = random.Random(seed)
    window = 70 if seed % 2 else None
    c = make_cache(window=window, max_tokens=64 * 40, max_positions=300)
    live = {}
    for step in range(250):
        r = rnd.random()
        if r < 0.12 and len(live) < 12:
            live[c.alloc_slot()] = []
        elif r < 0.3 and live and len(live) < 14:
            s, count = rnd.choice(list(live)), rnd.randint(1, 3)
            if count <= c.slots.free_count:
                for new in c.fork(s, count):
                    live[new] = list(live[s])
        elif r < 0.42 and live:
            s = rnd.choice(list(live))
            c.free_slot(s)
            del live[s]
        elif r < 0.5 and live:
            s = rnd.choice(list(live))
            n = rnd.randint(0, len(live[s]))
            try:
                c.truncate(s, n)
            except CacheError:
                assert window
                continue
            live[s] = live[s][:n]
        elif live:
            chosen = rnd.sample(list(live), rnd.randint(1, min(4, len(live))))
            for s in chosen:
                n = rnd.choice([1, 1, 2, 60, 64, 65])
                if len(live[s]) + n > 300:
                    continue
                values = [float(step * 300 + i) for i in range(n)]
                try:
                    write(c, s, values)
                except CacheError:
                    continue
                live[s] += values
        c.check()
        if step % 10 == 0:
            for s, values in live.items():
                assert c.length(s) == len(values) and read(c, s, 0) == values
                seen_from = max(0, len(values) + 1 - window) if window else 0
                assert read(c, s, 1, seen_from) == values[seen_from:]
            if len(live) > 1:
                slots = list(live)
                found = c.shared_pages(slots, [len(live[s]) for s in slots])
                if found is not None:
                    table = c.kv_groups[FULL].table_host
                    for first, count, page, end in found.nodes:
                        rows = table[[slots[i] for i in found.order[first:first + count]], page:end if end >= 0 else page]
                        assert (rows == rows[0]).all() and (rows >= 0).all()
    for s in list(live):
        c.free_slot(s)
    c.check()
    assert all(g.pages.held_count == 0 and not g.further for g in c.kv_groups.values())
