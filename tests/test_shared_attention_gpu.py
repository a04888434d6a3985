"""The attention over pages that several sequences share, against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from herbert_rs_amd.cache import LayerKV
from herbert_rs_amd.errors import BackendError, NeedsEagerStep
from herbert_rs_amd.kernels import mfma, shared

from .conftest import observe
from .shared_util import bound, inputs, reference, step, tables

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda", torch.cuda.current_device())


def compare(got, want, dtype, hd, keys, label):
    out, weight, size = want
    got = got.cpu().double().view(out.shape)
    allowed = bound(out, weight, size, dtype, hd, keys)
    assert torch.isfinite(got).all()
    share = ((got - out).abs() / allowed).max().item()
    observe(f"shared attention {label} of its bound", share)
    assert share <= 1.0, f"{share} of what is allowed"


def run(seqs, held, news, nq, nkv, hd, dtype, seed=0, sinks=None, softcap=None, check=True):
    table, pages = tables(seqs, seed)
    meta = step(table, held, news, dev())
    assert meta.shared is not None
    q, kv = inputs(table, pages, sum(news), nq, nkv, hd, dtype, seed, dev())
    out = torch.full_like(q, float("nan"))
    want = reference(q, kv, table, held, news, nq, nkv, hd, hd ** -0.5, sinks, softcap) if check else None
    for whole_rows in ((True, False) if dtype == BF and max(news) == 1 else (False,)):       # (short contexts have another form)
        limit = shared.BY_ITSELF_PAGES
        shared.BY_ITSELF_PAGES = 1 << 20 if whole_rows else 0
        try:
            meta.derived.clear()
            shared.attention(q, meta, kv, out.fill_(float("nan")), nq, nkv, hd, hd ** -0.5, sinks=sinks, softcap=softcap)
        finally:
            shared.BY_ITSELF_PAGES = limit
        assert next(v for k, v in meta.derived.items() if k[0] == "shared_plan").direct == (whole_rows and len(held) * nkv <= 512)
        if check:
            compare(out, want, dtype, hd, max(h + n for h, n in zip(held, news)), "bf16" if dtype == torch.bfloat16 else "f32")
    return q, meta, kv, out, table


def plain_samples(count, pages, own=1):
    return [[("p", pages), (None, own)] for _ in range(count)]


BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nq, nkv, hd", [(4, 2, 64), (8, 2, 128), (3, 3, 32), (5, 1, 64), (32, 1, 128), (14, 2, 64), (6, 2, 128)])
def test_samples_of_one_prompt(nq, nkv, hd, dtype):
    for count, pages, extra in ((2, 1, 0), (3, 2, 63), (9, 5, 17)):
        held = [64 * pages + (extra + 5 * i) % 64 for i in range(count)]
        run(plain_samples(count, pages), held, [1] * count, nq, nkv, hd, dtype, seed=count)


@pytest.mark.parametrize("nq, nkv, hd, dtype", [(2, 2, 80, F32), (4, 1, 256, F32), (40, 2, 12, F32), (2, 1, 200, F32)])
def test_float32_heads_of_other_sizes(nq, nkv, hd, dtype):
    run(plain_samples(5, 3), [192, 193, 200, 255, 240], [1] * 5, nq, nkv, hd, dtype)


@pytest.mark.parametrize("count", [8, 9, 16, 17, 24, 32, 33, 40, 70])
def test_every_number_of_column_tiles(count):
    """A group of four: 8 sequences fill a tile of 32 columns, 32 a workgroup."""
    held = [64 * 7 + (11 * i) % 64 for i in range(count)]
    run(plain_samples(count, 7), held, [1] * count, 4, 1, 64, BF, seed=count)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_trees_and_sequences_that_share_nothing(dtype):
    seqs = [[("a", 3), ("b", 4), (None, 2)], [(None, 4)], [("a", 3), ("c", 1), (None, 1)], [("a", 3), ("b", 4), (None, 1)],
            [("a", 3), ("c", 1), ("d", 6), (None, 1)], [("a", 3), ("c", 1), ("d", 6), (None, 5)], [(None, 1)], [("e", 2), (None, 1)],
            [("e", 2), (None, 1)]]
    held = [64 * (sum(p for _, p in s) - 1) + (7 * i) % 64 for i, s in enumerate(seqs)]
    held[6] = 0                                                     # a sequence's very first token
    run(seqs, held, [1] * len(seqs), 8, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nq, nkv, hd", [(4, 2, 64), (8, 1, 128), (5, 5, 32)])
def test_several_tokens_a_sequence(nq, nkv, hd, dtype):
    """Continuations of unequal lengths, causal among themselves, over page borders, one of a single token."""
    news = [1, 40, 64, 65, 7, 130]
    seqs = [[("p", 3), (None, 4)] for _ in news]
    held = [192, 192 + 50, 192, 192 + 63, 192 + 60, 192 + 1]
    run(seqs, held, news, nq, nkv, hd, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sinks_and_capped_scores(dtype):
    sinks = torch.tensor([0.0, 3.0, -float("inf"), 12.0], device=dev())
    held = [130, 150, 191]
    for s, cap in ((sinks, None), (None, 3.0), (sinks, 5.0)):
        run(plain_samples(3, 2), held, [1, 1, 1], 4, 2, 64, dtype, sinks=s, softcap=cap)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_long_prompt_in_many_ranges(dtype):
    pages = 150 if dtype == BF else 40
    run(plain_samples(3, pages, 3), [64 * pages + 70, 64 * pages + 3, 64 * pages + 191], [1, 1, 1], 2, 1, 64, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news", [[1, 1, 1], [3, 20, 1]])
def test_what_lies_in_places_that_no_token_sees_does_not_matter(dtype, news):
    """Not-finite keys and values behind a sequence's end, in pages of nobody, and in a place that only later tokens see."""
    nq, nkv, hd = 4, 2, 64
    table, pages = tables(plain_samples(3, 2), 4)
    held = [128 + 9, 128, 128 + 40]
    meta = step(table, held, news, dev())
    q, kv = inputs(table, pages, sum(news), nq, nkv, hd, dtype, 4, dev())
    want = reference(q, kv, table, held, news, nq, nkv, hd, 0.125)
    for i in range(3):
        end = held[i] + news[i] - 128
        kv.k[table[i, 2], :, end:] = float("nan")
        kv.v[table[i, 2], :, :, end:] = float("inf")
    unused = [p for p in range(pages) if p not in set(table.ravel().tolist())]
    kv.k[unused], kv.v[unused] = float("nan"), float("nan")
    out = torch.empty_like(q)
    shared.attention(q, meta, kv, out, nq, nkv, hd, 0.125)
    compare(out, want, dtype, hd, 200, "hidden")
    if max(news) > 1:
        # the second sequence's 11th token: its value is infinite for it and the tokens behind it, for nobody else
        kv.v[table[1, 2], 0, 5, 10] = float("inf")
        kv.v[table[1, 2], 1, 7, 10] = float("nan")
        shared.attention(q, meta, kv, out, nq, nkv, hd, 0.125)
        got, first = out.cpu().double().view(-1, nq, hd), news[0]
        spoiled = torch.zeros_like(got, dtype=torch.bool)
        spoiled[first + 10:first + 20, 0:2, 5] = True
        spoiled[first + 10:first + 20, 2:4, 7] = True
        assert not torch.isfinite(got[spoiled]).any()
        clean = torch.where(spoiled, want[0], got)
        compare(clean, want, dtype, hd, 200, "hidden")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_value_without_a_size_in_a_shared_page_reaches_everybody(dtype):
    q, meta, kv, out, table = run(plain_samples(4, 2), [128, 129, 140, 150], [1] * 4, 2, 1, 64, dtype)
    kv.v[table[0, 0], 0, 3, 17] = float("nan")
    shared.attention(q, meta, kv, out, 2, 1, 64, 0.125)
    bad = ~torch.isfinite(out.view(4, 2, 64))
    assert bad[:, :, 3].all() and bad.sum() == 8


def test_scores_far_apart_and_equal():
    """Scores of hundreds (one key holds all the weight, in a shared page or in a sequence's own) and scores that are all alike."""
    nq, nkv, hd = 4, 1, 64
    for dtype in (BF, F32):
        table, pages = tables(plain_samples(6, 4), 5)
        held = [256 + i for i in range(6)]
        meta = step(table, held, [1] * 6, dev())
        q, kv = inputs(table, pages, 6, nq, nkv, hd, dtype, 5, dev(), q_scale=0.01)
        kv.k[table[0, 1], 0, 30] = 40.0
        q[0::2] = 4.0
        kv.k[table[5, 4], 0, 5] = 60.0                      # the last sequence's own newest key
        q[5] = 5.0
        q[3] = 0.0
        out = torch.empty_like(q)
        shared.attention(q, meta, kv, out, nq, nkv, hd, 0.125)
        # (scores of up to 2,560: in float32 their exponents are off by that times 2^-24 times a few)
        out64, weight, size = reference(q, kv, table, held, [1] * 6, nq, nkv, hd, 0.125)
        allowed = bound(out64, weight, size, dtype, hd, 261) + 4 * 2.0 ** -24 * size[..., None] * weight
        assert ((out.cpu().double().view(out64.shape) - out64).abs() <= allowed).all()


def test_the_result_does_not_hang_on_the_stream_or_the_call():
    q, meta, kv, out, _ = run(plain_samples(20, 9), [64 * 9 + i for i in range(20)], [1] * 20, 8, 2, 128, BF)
    again = torch.empty_like(q)
    side, scratch = torch.cuda.Stream(), mfma.Scratch()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            shared.attention(q, meta, kv, again, 8, 2, 128, 128 ** -0.5, scratch=scratch)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, out)


def test_a_captured_call_replays_alike():
    q, meta, kv, out, _ = run(plain_samples(12, 6), [64 * 6 + i for i in range(12)], [1] * 12, 8, 2, 64, BF)
    again, scratch = torch.empty_like(q), mfma.Scratch()
    shared.attention(q, meta, kv, again, 8, 2, 64, 0.125, scratch=scratch)      # (its scratch is made here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared.attention(q, meta, kv, again, 8, 2, 64, 0.125, scratch=scratch)
    for i in range(4):
        again.fill_(float("nan"))
        if i % 2:
            q.copy_(torch.randn_like(q.float()).to(q.dtype))
            shared.attention(q, meta, kv, out, 8, 2, 64, 0.125)
            torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_value_without_a_size_is_not_lost_behind_a_weight_of_nothing(dtype):
    """One key holds all the weight (its score is hundreds above the others): 0 x inf in another page is NaN, as in the formula's own arithmetic."""
    q, meta, kv, out, table = run(plain_samples(4, 5), [5 * 64 + 9] * 4, [1] * 4, 2, 1, 64, dtype)
    q.fill_(4.0)
    kv.k[:] = 0.0
    kv.k[table[:, 5], 0, 3] = 40.0                       # score 1,280
    kv.v[table[0, 0], 0, 7, 11] = float("inf")
    shared.attention(q, meta, kv, out, 2, 1, 64, 0.125)
    bad = ~torch.isfinite(out.view(4, 2, 64))
    assert bad[:, :, 7].all() and bad.sum() == 8


def test_a_call_without_scratch_is_its_own_on_every_stream():
    """Two streams at a time, no scratch given: their partial results do not meet."""
    case = (plain_samples(20, 9), [64 * 9 + i for i in range(20)], [1] * 20, 8, 2, 128, BF)
    made = [run(*case), run(plain_samples(20, 5), [64 * 5 + 3 * i for i in range(20)], [1] * 20, 8, 2, 128, BF)]
    want = [m[3].clone() for m in made]
    outs = [[torch.empty_like(m[3]) for _ in range(12)] for m in made]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(12):
        for (q, meta, kv, _, _), side, out in zip(made, sides, outs):
            with torch.cuda.stream(side):
                shared.attention(q, meta, kv, out[i], 8, 2, 128, 128 ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for out, w in zip(outs, want) for o in out)


def test_a_plan_follows_what_is_shared_and_is_not_made_while_recording():
    seqs, held = plain_samples(6, 4), [64 * 4 + i for i in range(6)]
    q, meta, kv, out, table = run(seqs, held, [1] * 6, 4, 2, 64, BF)
    from herbert_rs_amd.cache import SharedPages
    nodes = meta.shared.nodes
    assert nodes[0][1] == 6
    # the same step with the first three pages shared alone: other sums, the same result within the rounding of the outputs
    first = [(0, 6, 0, 3)] + [(i, 1, 3, -1) for i in range(6)]
    meta.shared = SharedPages(meta.shared.order, first)
    again = torch.empty_like(out)
    shared.attention(q, meta, kv, again, 4, 2, 64, 0.125)
    assert len([v for k, v in meta.derived.items() if k[0] == "shared_plan"]) == 1
    assert next(v for k, v in meta.derived.items() if k[0] == "shared_plan").sharing is meta.shared
    compare(again, reference(q, kv, table, held, [1] * 6, 4, 2, 64, 0.125), BF, 64, max(held) + 1, "another cut")
    fresh = step(table, held, [1] * 6, dev())
    scratch = mfma.Scratch()
    shared.attention(q, meta, kv, again, 4, 2, 64, 0.125, scratch=scratch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            with pytest.raises(NeedsEagerStep, match="plan"):
                shared.attention(q, fresh, kv, again, 4, 2, 64, 0.125, scratch=scratch)
            again.zero_()
        finally:
            graph.capture_end()
    torch.cuda.synchronize()


def test_calls_refused_before_a_launch(monkeypatch):
    q, meta, kv, out, table = run(plain_samples(3, 2), [128 + 9, 128, 128 + 40], [1] * 3, 4, 2, 64, BF)
    with pytest.raises(BackendError, match="does not fit a table of 2"):
        shared.attention(q, meta, LayerKV(kv.k, kv.v, kv.page_table[:, :2].contiguous(), 64, 0), out, 4, 2, 64, 0.125)
    with pytest.raises(BackendError, match="contiguous"):
        shared.attention(q, meta, LayerKV(kv.k.transpose(2, 3), kv.v, kv.page_table, 64, 0), out, 4, 2, 64, 0.125)
    with pytest.raises(BackendError, match="out must be"):
        shared.attention(q, meta, kv, out.float(), 4, 2, 64, 0.125)
    with pytest.raises(BackendError, match="sinks must"):
        shared.attention(q, meta, kv, out, 4, 2, 64, 0.125, sinks=torch.zeros(3, device="cuda"))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 5)
    with pytest.raises(BackendError, match="tensors lie on GPUs .0., the current one is 5"):
        shared.attention(q, meta, kv, out, 4, 2, 64, 0.125)


def chains(weight, q, kv, table, held, news, nq, nkv, hd):
    """What float32 results may be off by, counted along the kernel's own chains as a walk of independent roundings, each evenly within u = 2^-24 (half
    a step) of its value, whose square root of the sum of squares is taken six times.
    A score is four sums side by side of n = 16 ceil(hd / 64) products each: a sum of random signs is as large as the root of the sum of its products'
    squares, r, at most, so 6 sqrt(n) u r / sqrt(3); the sums of sums, the scale, the difference from the reference, the exponential and the
    factors of a page and of an item are eight further roundings of u (1 + 2 |score|). A weight is off by as much of itself, numerator and
    denominator: twice that. The products with values: chains of 32, a sum and a rescaling a page and an item (no more than pages), numerator and
    denominator: 2 x 6 sqrt(34 + 4 pages) u / sqrt(3)."""
    out = torch.empty_like(weight[..., 0])
    k, q, row = kv.k.cpu().double(), q.cpu().double().view(-1, nq, hd), 0
    for i, (before, n) in enumerate(zip(held, news)):
        keys = k[torch.from_numpy(table[i, :-(-(before + n) // 64)].astype(np.int64))].permute(1, 0, 2, 3).reshape(nkv, -1, hd)
        pages = (before + n) // 64 + 1
        for t in range(row, row + n):
            for h in range(nq):
                seen = keys[h // (nq // nkv), :before + t - row + 1]
                r = (seen.square() @ q[t, h].square()).max().sqrt() * hd ** -0.5
                top = (seen @ q[t, h]).abs().max() * hd ** -0.5
                out[t, h] = 2 * (6 * (16 * -(-hd // 64) / 3) ** 0.5 * r + 8 * (1 + 2 * top)) + 2 * 6 * ((34 + 4 * pages) / 3) ** 0.5
        row += n
    return 2.0 ** -24 * out[..., None] * weight + 1e-30


@pytest.mark.parametrize("seqs, held, news, nq, nkv, hd", [
    (plain_samples(9, 5), [64 * 5 + 5 * i for i in range(9)], [1] * 9, 8, 2, 128),
    (plain_samples(5, 40, 2), [64 * 40 + 9 + i for i in range(5)], [1] * 5, 4, 2, 64),
    (plain_samples(4, 3, 2), [192, 200, 230, 192], [40, 7, 64, 1], 4, 2, 80),
    (plain_samples(3, 2), [130, 150, 190], [1] * 3, 2, 1, 256)])
def test_float32_results_lie_within_the_roundings_of_their_chains(seqs, held, news, nq, nkv, hd):
    q, meta, kv, out, table = run(seqs, held, news, nq, nkv, hd, F32, seed=7)
    want, weight, _ = reference(q, kv, table, held, news, nq, nkv, hd, hd ** -0.5)
    allowed = chains(weight, q, kv, table, held, news, nq, nkv, hd)
    share = ((out.cpu().double().view(want.shape) - want).abs() / allowed).max().item()
    observe("shared attention f32 of its chains' roundings", share)
    assert share <= 1.0
