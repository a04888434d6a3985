"""Which pages sequences share, how a step is cut into items, and what the shared attention refuses (no GPU needed)."""
import json
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from herbert_rs_amd.cache import KVNeed, LayerKV, SharedPages, shared_pages
from herbert_rs_amd.cache.sharing import MAX_LEVELS
from herbert_rs_amd.engine import Model, StepEntry, batch
from herbert_rs_amd.errors import BackendError
from herbert_rs_amd.kernels import lib, shared

from . import figalorn_tiny, plan_oracle
from .shared_util import tables
from .tiny import spec_of


def as_sets(found, table, held):
    """{sequence: [(page, end, the sequences that share it), ...]} with every page of every sequence in exactly one node."""
    got = {}
    for first, count, page, end in found.nodes:
        members = sorted(int(i) for i in found.order[first:first + count])
        for i in members:
            got.setdefault(i, []).append((page, end, tuple(members)))
    for i, nodes in got.items():
        at = 0
        for page, end, members in nodes:
            assert page == at and (end > page or end == -1)
            if end >= 0:
                assert len(members) > 1 and end <= held[i] // 64
                for j in members:
                    assert (table[i, page:end] == table[j, page:end]).all()
            else:
                assert members == (i,)
            at = end
        assert at == -1
    return got


def test_sequences_that_share_pages_are_found():
    # two branches of a common beginning, one of them with a branch of its own, and a sequence that shares nothing
    seqs = [[("a", 3), ("b", 2), (None, 2)], [(None, 4)], [("a", 3), ("c", 1), (None, 1)], [("a", 3), ("b", 2), (None, 1)],
            [("a", 3), ("c", 1), ("d", 2), (None, 1)], [("a", 3), ("c", 1), ("d", 2), (None, 3)]]
    table, _ = tables(seqs, 1)
    held = [64 * (sum(p for _, p in s) - 1) + 5 for s in seqs]
    got = as_sets(shared_pages(table, held), table, held)
    assert sorted(got) == list(range(6))
    assert got[0] == [(0, 3, (0, 2, 3, 4, 5)), (3, 5, (0, 3)), (5, -1, (0,))]
    assert got[5] == [(0, 3, (0, 2, 3, 4, 5)), (3, 4, (2, 4, 5)), (4, 6, (4, 5)), (6, -1, (5,))]
    assert got[1] == [(0, -1, (1,))]
    assert shared_pages(table, held).pages_saved == 4 * 3 + 2 + 2 * 1 + 2


def test_only_full_pages_count_as_shared():
    table, _ = tables([[("a", 2)], [("a", 2)]], 2)
    assert shared_pages(table, [127, 127]).nodes == [(0, 2, 0, 1), (0, 1, 1, -1), (1, 1, 1, -1)]
    assert shared_pages(table, [63, 128]) is None           # the first may still write to its only page
    assert shared_pages(table, [64, 63]) is None
    assert shared_pages(table[:1], [128]) is None
    other, _ = tables([[(None, 2)], [(None, 2)]], 2)
    assert shared_pages(other, [128, 128]) is None


def test_places_that_are_not_held_share_nothing():
    table = np.zeros((3, 4), dtype=np.int32)                # (they all name page 0)
    table[0, 0], table[1, 0], table[2, 0] = 5, 6, 7
    assert shared_pages(table, [70, 10, 90]) is None


def test_chains_of_branches_end_at_a_depth():
    n = MAX_LEVELS + 6                                      # every sequence leaves the chain a page later than the one before
    seqs = [[("chain", i + 1), (None, 1)] for i in range(n)]
    table, _ = tables(seqs, 3)
    held = [64 * (i + 1) + 1 for i in range(n)]
    got = as_sets(shared_pages(table, held), table, held)
    assert max(len(nodes) for nodes in got.values()) == MAX_LEVELS + 1


def random_step(rng):
    branches, levels = int(rng.integers(1, 5)), int(rng.integers(1, 3))
    common, seqs, held, news = int(rng.integers(0, 30)), [], [], []
    for b in range(branches):
        deep = int(rng.integers(1, 12))
        for _ in range(int(rng.integers(1, 40))):
            own = int(rng.integers(1, 9))
            s = [("all", common)] + ([(b, deep)] if levels > 1 else []) + [(None, own)]
            n = int(rng.integers(1, min(64 * own, 90) + 1)) if rng.random() < 0.3 else 1
            seqs.append(s)
            news.append(n)
            held.append(64 * sum(p for _, p in s) - int(rng.integers(0, 64)) - n)
            held[-1] = max(held[-1], 64 * sum(p for _, p in s[:-1]))
    return tables(seqs, int(rng.integers(1 << 30)))[0], held, news


@pytest.mark.parametrize("seed", range(40))
def test_items_cover_what_every_row_sees_once(seed):
    rng = np.random.default_rng(seed)
    table, held, news = random_step(rng)
    found = shared_pages(table, held)
    if found is None:
        return
    starts = np.concatenate([[0], np.cumsum(news)])
    context = [h + n for h, n in zip(held, news)]
    for columns, group, nkv in ((128, 4, 8), (128, 1, 2), (128, 32, 1), (128, 7, 4), (16, 2, 4), (16, 16, 1), (16, 24, 2)):
        items, order, part_start, parts, most = shared.plan(starts, context, np.arange(len(held))[::-1], found, group, nkv, columns, 512)
        assert columns == 16 or not items[items[:, 1] * group > max(64, group), 6].any()        # (only narrow items look at a mask)
        items = items[items[:, 1] > 0]
        assert sorted(order.tolist()) == list(range(starts[-1]))
        assert most == items[:, 1].max() and (most * group <= columns or (most == 1 and columns == 16))
        pieces, owner, listed = {}, {}, set()
        for row0, rows, slot, page, end, list0, masked in items[:, :7].tolist():
            assert rows > 0 and end > page >= 0 and 0 <= row0 and row0 + rows <= len(order)
            firsts = [held[i] + int(order[row0 + r]) - starts[i] for r in range(rows)
                      for i in [int(np.searchsorted(starts, order[row0 + r], side="right")) - 1]]
            assert masked or min(firsts) >= 64 * end - 1            # whoever looks at no mask sees all
            for r in range(rows):
                token = int(order[row0 + r])
                i = int(np.searchsorted(starts, token, side="right")) - 1
                assert (table[i, page:end] == table[len(held) - 1 - slot, page:end]).all() and end <= -(-context[i] // 64)
                pieces.setdefault(token, []).append((page, end))
                assert list0 + r not in listed and parts[list0 + r] not in owner
                listed.add(list0 + r)
                owner[parts[list0 + r]] = token
        assert sorted(owner) == list(range(len(parts)))
        for t, token in enumerate(order.tolist()):
            assert [owner[p] for p in range(part_start[t], part_start[t + 1])] == [token] * (part_start[t + 1] - part_start[t])
            i = int(np.searchsorted(starts, token, side="right")) - 1
            position, at = held[i] + token - starts[i], 0
            for page, end in sorted(pieces[token]):
                assert page == at
                at = end
            assert at >= position // 64 + 1


def test_what_the_shared_attention_refuses():
    kv = LayerKV(torch.zeros(4, 2, 64, 64), torch.zeros(4, 2, 64, 64), torch.zeros(2, 2, dtype=torch.int32), 64, 0)
    meta = batch.pack([StepEntry(0, [0], [0]), StepEntry(1, [0], [0])], [64, 64], "cpu")
    q = torch.zeros(2, 4 * 64)
    with pytest.raises(BackendError, match="share no pages"):
        shared.attention(q, meta, kv, q, 4, 2, 64, 0.125)
    meta.shared = shared_pages(np.array([[1, 2], [1, 3]]), [64, 64])
    with pytest.raises(BackendError, match="on the GPU"):
        shared.attention(q, meta, kv, q, 4, 2, 64, 0.125)
    for bad in ((3, 2, 64), (4, 2, 62), (4, 2, 260), (4, 0, 64)):
        with pytest.raises(BackendError, match="refuses"):
            shared.attention(q, meta, kv, q, *bad, 0.125)
    windowed = LayerKV(kv.k, kv.v, kv.page_table, 64, 128)
    keys_only = LayerKV(kv.k, None, kv.page_table, 64, 0)
    for other in (windowed, keys_only, LayerKV(kv.k.bfloat16(), kv.v.bfloat16(), kv.page_table, 64, 0)):
        with pytest.raises(BackendError, match="refuses"):
            shared.attention(q, meta, other, q, 4, 2, 64, 0.125)
    with pytest.raises(BackendError, match="shared by 2 sequences in a step of 3"):
        shared.plan([0, 1, 2, 3], [65, 65, 65], [0, 1, 2], meta.shared, 2, 2, 128, 512)


def call(**changed):
    args = dict(q=None, k=None, v=None, out=None, dtype=1, po=None, pml=None, items=None, n_items=1, max_rows=1, causal=0, direct=0, order=None, start=None,
                parts=None, n_rows=1, positions=None, seq_of=None, slots=None, table=None, max_pages=1, nq=4, nkv=2, hd=64, scale=0.1, softcap=0.0,
                sinks=None, stream=None)
    args.update(changed)
    lib.call("attention_shared", "hb_attn_shared", *args.values())


@pytest.mark.parametrize("changed, text", [
    ({"nq": 5}, "do not group"), ({"n_rows": 0}, "empty"), ({"n_items": 0}, "empty"), ({"hd": 96}, "32, 64 or 128"), ({"dtype": 7}, "dtype"),
    ({"max_rows": 65}, "exceed 128 columns"), ({"scale": 0.0}, "positive"), ({"softcap": -1.0}, "positive"),
    ({"scale": float("nan")}, "positive"), ({"n_rows": 1 << 30}, "exceed|too many rows"), ({"n_items": 1 << 30}, "too many items"),
    ({"dtype": 0, "hd": 62}, "whole quads"), ({"dtype": 0, "hd": 260}, "up to 256"), ({"dtype": 0, "k": 8}, "16-byte"), ({"q": 2}, "16-byte"), ({"v": 24}, "16-byte"),
    ({"dtype": 0, "n_items": 1 << 30}, "too many items"), ({"dtype": 0, "direct": 1}, "parts of rows"), ({"direct": 1, "causal": 1}, "whole rows"),
    ({"direct": 1, "max_rows": 33}, "whole rows")])
def test_calls_that_the_entry_refuses(changed, text):
    with pytest.raises(BackendError, match=text):
        call(**changed)


def decoding(pages, shared_by, count, static, held=None):
    """A decode step of `count` sequences of which the first `shared_by` hold the same `pages` pages, and `static` after it."""
    table, _ = tables([[("p", pages), (None, 1)] if i < shared_by else [(None, pages + 1)] for i in range(count)], 3)
    held = held or [64 * pages + 5] * count
    return static.update([StepEntry(i, [1], [0]) for i in range(count)], held, shared_pages(table, held))


def test_what_a_recorded_step_is_tied_to_says_whether_sharing_pays():
    """Known before any plan is made: a step that was recorded where nothing is gained is not replayed where something is."""
    needs = [KVNeed(8, 128), KVNeed(8, 128, 256), KVNeed(1, 32), KVNeed(4, 128, values=False)]
    static = batch.StaticDecodeMeta(64, "cpu", 99, shared.worth_over(needs, torch.bfloat16))
    decoding(100, 2, 64, static)
    few = static.shared_shape, static.meta.context_bucket, static.meta.unequal
    assert static.meta.shared is None and few[0] is None
    decoding(100, 64, 64, static)
    assert static.meta.shared is not None and (static.shared_shape, static.meta.context_bucket, static.meta.unequal) != few
    assert static.shared_shape == ((False, True),)                 # (a head of 32: 52 MB saved of 152)
    decoding(900, 64, 64, static)
    assert static.shared_shape == ((True, True),)
    decoding(100, 2, 64, static)
    assert static.shared_shape is None
    # a plan that one kind of heads has made, and does not pay for now, does not keep the other kind from theirs
    static.shared_plans["small heads"] = (None, lambda m: False)
    decoding(100, 64, 64, static)
    assert static.meta.shared is not None and static.shared_shape == ((False, True), ("small heads", None))


@pytest.mark.parametrize("dtype, taken", [(torch.float32, True), (torch.bfloat16, False)])
def test_heads_of_two_maps_share_in_float32_alone(dtype, taken):
    """In bfloat16 the kernel that attends takes the maps from each other as well: what a layer says of itself is what it does."""
    mixer = Model(spec_of(figalorn_tiny.CONFIGS["F"][0])[1]).blocks[0].mixer
    assert mixer.maps == 2 and mixer.chunk is None and mixer.window is None
    nodes = [(0, 64, 0, 1000)] + [(i, 1, 1000, -1) for i in range(64)]
    meta = SimpleNamespace(shared=SharedPages(np.arange(64), nodes), max_new=1, num_seqs=64, num_tokens=64)
    kv = LayerKV(torch.zeros(1, mixer.nkv, 64, mixer.hd, dtype=dtype), torch.zeros(1, mixer.nkv, mixer.hd, 64, dtype=dtype),
                 torch.zeros(1, 1, dtype=torch.int32), 64, 0)
    ctx = SimpleNamespace(meta=meta, rt=SimpleNamespace(dtype=dtype))
    assert shared.pays(meta, kv, mixer.kept_heads, mixer.nkv, mixer.hd, dtype)
    assert mixer._shares(ctx, kv) == taken


def decode_of(count, shared_places, context, shared_by=None):
    """What `pays` looks at, of a decode step of `count` sequences (the first `shared_by` of which share so many pages)."""
    shared_by = shared_by or count
    nodes = [(0, shared_by, 0, shared_places)] + [(i, 1, shared_places if i < shared_by else 0, -1) for i in range(count)]
    return SimpleNamespace(shared=SharedPages(np.arange(count), nodes), max_new=1, num_seqs=count, num_tokens=count,
                           host_context=np.full(count, context))


def cache_of(nkv, hd, dtype):
    return LayerKV(torch.zeros(1, nkv, 64, hd, dtype=dtype), torch.zeros(1, nkv, hd, 64, dtype=dtype), torch.zeros(1, 1, dtype=torch.int32), 64, 0)


@pytest.mark.parametrize("count, pages, taken", [
    # 8 kv heads of 128: a page that one sequence more does not read is 256 KiB; 32 MiB and 6 MiB a sequence are asked for
    (2, 175, False), (2, 176, True), (8, 45, False), (8, 46, True), (20, 31, False), (20, 32, True),
    # ... of 20 sequences at most
    (64, 9, False), (64, 10, True), (128, 4, False), (128, 5, True)])
def test_how_much_has_to_be_saved(count, pages, taken):
    assert shared.pays(decode_of(count, pages, 64 * pages + 9), cache_of(8, 128, torch.bfloat16), 32, 8, 128, torch.bfloat16) == taken
    # (in float32 whatever is shared is worth it)
    assert shared.pays(decode_of(count, 1, 100), cache_of(8, 128, torch.float32), 32, 8, 128, torch.float32)


@pytest.mark.parametrize("dtype, most", [(torch.bfloat16, 8), (torch.float32, 200)])
def test_steps_of_many_tokens_a_sequence_are_prompts(dtype, most):
    kv = cache_of(8, 128, dtype)
    for tokens, taken in ((24 * most, True), (24 * most + 1, False)):
        meta = decode_of(24, 1000, 64 * 1000 + most + 50)
        meta.max_new, meta.num_tokens = most + 50, tokens
        assert shared.pays(meta, kv, 32, 8, 128, dtype) == taken
    meta.max_new, meta.shared = 1, None
    assert not shared.pays(meta, kv, 32, 8, 128, dtype)


@pytest.mark.parametrize("count, context, nkv, hd, taken", [
    (2, 192, 4, 64, False), (2, 193, 4, 64, True), (16, 384, 4, 64, True), (16, 385, 4, 64, False), (17, 200, 4, 64, False), (4, 200, 16, 64, True),
    (5, 200, 16, 64, False), (2, 200, 4, 128, False), (2, 200, 2, 32, True)])
def test_short_contexts_behind_a_kernel_of_their_own_are_read_sequence_by_sequence(count, context, nkv, hd, taken):
    """The steps whose sequences are items of their own, as a filtered attention's decode step takes them; and the attention that prepares
    its rows itself does not."""
    meta, kv = decode_of(count, 1, context), cache_of(nkv, hd, torch.bfloat16)
    assert shared.pays(meta, kv, 4 * nkv, nkv, hd, torch.bfloat16, True) == taken
    assert not shared.pays(meta, kv, 4 * nkv, nkv, hd, torch.bfloat16)
    assert shared.worth_over([KVNeed(nkv, hd)], torch.bfloat16, {(nkv, hd)})(meta) == (False, taken)
    assert shared.worth_over([KVNeed(nkv, hd)], torch.bfloat16)(meta) == (False,)
    if taken:
        meta.host_starts, meta.host_slots = np.arange(count + 1), np.arange(count)
        items, order, part_start, parts, most, direct = shared._planned(meta, 4, nkv, torch.bfloat16, shared.plan)
        assert direct and len(items) == count and most == 1


def test_which_layers_prepare_by_a_kernel_of_their_own():
    from . import mefatar_tiny, vipalorn_tiny
    assert Model(spec_of(mefatar_tiny.CONFIGS["Q"][0])[1]).heads_prepared_alone() == {(4, 64), (2, 64)}
    assert Model(spec_of(figalorn_tiny.CONFIGS["F"][0])[1]).heads_prepared_alone() == set()
    assert Model(spec_of(vipalorn_tiny.CONFIGS["Q"][0])[1]).heads_prepared_alone() == set()


@pytest.mark.parametrize("scale, taken", [(0.125, True), (0.0, False), (-0.125, False)])
def test_scores_with_a_scale_that_is_not_positive_stay_with_the_ordinary_attention(scale, taken):
    """In float32 that one takes any scale, and a configuration may name one."""
    from . import mefatar_tiny
    raw = json.loads(json.dumps(mefatar_tiny.CONFIGS["Q"][0]))
    raw["layers"][1]["mixer"]["left"]["scale"] = scale
    mixer = Model(spec_of(raw)[1]).blocks[1].mixer.sides[0]
    ctx = SimpleNamespace(meta=decode_of(4, 2, 130), rt=SimpleNamespace(dtype=torch.float32))
    assert mixer._shares(ctx, cache_of(mixer.nkv, mixer.hd, torch.float32)) == taken


@pytest.mark.parametrize("seed", range(30))
def test_the_plan_is_that_of_the_formulas(seed):
    """The host's native cut against the same one in NumPy, number for number: random trees, single tokens and several, padding, shapes of graphs."""
    rng = np.random.default_rng(1000 + seed)
    table, held, news = random_step(rng)
    found = shared_pages(table, held)
    if found is None:
        found = SharedPages(np.arange(len(held)), [(i, 1, 0, -1) for i in range(len(held))])
    starts, context = np.concatenate([[0], np.cumsum(news)]), [h + n for h, n in zip(held, news)]
    for columns, group, nkv, workgroups, grid in ((128, 4, 8, 512, 1), (128, 1, 2, 512, 16), (128, 32, 1, 1, 16), (128, 7, 4, 100000, 1), (16, 2, 4, 1024, 16),
                                                  (16, 16, 1, 7, 1), (16, 24, 2, 1024, 1)):
        args = starts.astype(np.int32), np.array(context, dtype=np.int32), rng.permutation(len(held)), found, group, nkv, columns, workgroups, grid
        got, want = shared.plan(*args), plan_oracle.plan(*args)
        assert all(g.dtype == np.int32 and g.shape == w.shape and (g == w).all() for g, w in zip(got[:4], want[:4])) and got[4] == want[4]


@pytest.mark.parametrize("change, text", [
    (dict(nodes=[(0, 3, 0, 2), (0, 1, 2, -1), (1, 1, 2, -1)]), "each in its place"),              # a sequence's own pages are nowhere
    (dict(nodes=[(0, 3, 0, 2), (0, 1, 2, -1), (1, 1, 3, -1), (2, 1, 2, -1)]), "each in its place"),          # a page is left out
    (dict(nodes=[(0, 3, 0, 2), (0, 1, 1, -1), (1, 1, 2, -1), (2, 1, 2, -1)]), "each in its place"),          # or there twice
    (dict(nodes=[(0, 3, 0, 3), (0, 1, 3, -1), (1, 1, 3, -1), (2, 1, 3, -1)]), "each in its place"),          # beyond what is held before the step
    (dict(nodes=[(0, 4, 0, 2), (0, 1, 2, -1), (1, 1, 2, -1), (2, 1, 2, -1)]), "each in its place"),
    (dict(nodes=[(0, 3, 0, 2), (0, 1, 2, -1), (1, 1, 2, -1), (1 << 40, 1, 2, -1)]), "each in its place"),
    (dict(nodes=[(0, 3, -1, 2), (0, 1, 2, -1), (1, 1, 2, -1), (2, 1, 2, -1)]), "each in its place"),
    (dict(order=[0, 1, 1]), "each in its place"), (dict(order=[0, 1, 3]), "each in its place"), (dict(order=[0, 1]), "shared by 2 sequences"),
    (dict(context=[140, 0, 150]), "each in its place"), (dict(starts=[0, 1, 1, 2]), "each in its place")])
def test_pages_that_are_not_those_of_the_step_are_refused(change, text):
    args = dict(starts=[0, 1, 2, 3], context=[140, 131, 150], slots=[5, 3, 4], order=[0, 1, 2],
                nodes=[(0, 3, 0, 2), (0, 1, 2, -1), (1, 1, 2, -1), (2, 1, 2, -1)])

    def cut(starts, context, slots, order, nodes):
        return shared.plan(starts, context, slots, SharedPages(np.array(order), nodes), 4, 8, 128, 512)
    assert len(cut(**args)[0]) >= 4
    with pytest.raises(BackendError, match=text):
        cut(**dict(args, **change))


def test_the_native_plan_takes_integers_of_64_bits_alone():
    good = [np.array([0, 1]), np.array([5]), np.array([0]), np.array([0]), np.array([[0, 1, 0, -1]])]
    numbers = (4, 8, 128, 64, 512, 1, 0)
    assert lib.host().plan(*good, *numbers)[1] == 1
    for i in range(5):
        for bad in (good[i].astype(np.int32), good[i].astype(np.float64), [0, 1], None):
            with pytest.raises(TypeError):
                lib.host().plan(*good[:i], bad, *good[i + 1:], *numbers)
    with pytest.raises(TypeError):
        lib.host().plan(*good, *numbers[:-1])
    for i in range(6):
        assert lib.host().plan(*good, *(n if j != i else 0 for j, n in enumerate(numbers))) is None
