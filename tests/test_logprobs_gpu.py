"""Log probabilities of given tokens, entropy and top alternatives, against the formulas in 64 bits."""
import math

import pytest
import torch

from herbert_rs_amd.errors import BackendError
from herbert_rs_amd.kernels import ops

from .conftest import observe

pytestmark = pytest.mark.gpu


def results(logits, tokens, top, scratch=None):
    R, dev = logits.shape[0], logits.device
    chosen, entropy = torch.empty(R, device=dev), torch.empty(R, device=dev)
    ids = torch.empty((R, top), dtype=torch.int32, device=dev) if top else None
    best = torch.empty((R, top), device=dev) if top else None
    ops.token_logprobs(logits, tokens, chosen, entropy, ids, best, scratch)
    return chosen, entropy, ids, best


def check(logits, tokens, top, scratch=None):
    chosen, entropy, ids, best = results(logits, tokens, top, scratch)
    x = logits.double()
    V = x.shape[1]
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = logp.exp()
    want_entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    want = logp.gather(1, tokens.long()[:, None])[:, 0]
    top_x = x.amax(-1)
    # A log probability: the difference from the largest logit (half a step of it), log S (S a sum of exponentials, each off by a few steps,
    # over a tree of 16 + 8 + 6 and then at most 40 + 8 levels of roundings: 100 x 2^-24 of it) and their difference.
    def allowed(value, raw):
        return 2.0 ** -24 * ((raw - top_x).abs() + value.abs() + 100 + math.log(V)) + 1e-12
    at = x.gather(1, tokens.long()[:, None])[:, 0]
    finite = torch.isfinite(want)
    assert torch.equal(chosen.double()[~finite], want[~finite])
    share = ((chosen.double() - want).abs() / allowed(want, at))[finite]
    # the entropy: the same of log S, and a mean of x - m with weights that are off by as much
    mean = torch.where(p > 0, p * (x - top_x[:, None]).clamp(min=-1e30), torch.zeros_like(p)).sum(-1).abs()
    off = (entropy.double() - want_entropy).abs() / (2.0 ** -24 * (200 * mean + 100 + math.log(V) + want_entropy) + 1e-12)
    worst = max(off.max().item(), share.max().item() if finite.any() else 0.0)
    observe("log probabilities of their bound", worst)
    assert worst <= 1.0
    if top:
        order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :top]
        assert torch.equal(ids.long(), order)
        want_best = logp.gather(1, order)
        seen = torch.isfinite(want_best)
        assert torch.equal(best.double()[~seen], want_best[~seen])
        raw = x.gather(1, order)
        limit = 2.0 ** -24 * ((raw - top_x[:, None]).abs() + want_best.abs() + 100 + math.log(V)) + 1e-12
        assert ((best.double() - want_best).abs()[seen] <= limit[seen]).all()


def random_logits(R, V, seed, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((R, V), generator=gen, device="cuda") * scale
    tokens = torch.randint(0, V, (R,), generator=gen, device="cuda", dtype=torch.int32)
    return logits, tokens


@pytest.mark.parametrize("V", [1, 2, 3, 63, 255, 257, 4095, 4096, 4097, 4099, 8192, 12290, 151936])
@pytest.mark.parametrize("R", [1, 3])
def test_vocabularies_of_every_kind(R, V):
    logits, tokens = random_logits(R, V, V)
    for top in (0, 1, 5, 64):
        if top <= V:
            check(logits, tokens, top)


@pytest.mark.parametrize("R, V, top", [(257, 5000, 20), (65, 32771, 33), (1000, 777, 3)])
def test_many_rows(R, V, top):
    logits, tokens = random_logits(R, V, R)
    check(logits, tokens, top, ops.logprob_scratch(R + 3, V, top, logits.device))


@pytest.mark.parametrize("V", [700, 4096, 20000])
def test_equal_logits_go_by_the_lower_id(V):
    for logits in (torch.zeros(2, V, device="cuda"), torch.randint(-3, 4, (2, V), device="cuda").float(),
                   torch.randint(-1, 1, (2, V), device="cuda").float() * 0.0):         # (zeros of both signs are equal)
        check(logits, torch.tensor([0, V - 1], dtype=torch.int32, device="cuda"), 64)


@pytest.mark.parametrize("V", [700, 4096, 20000])
def test_sorted_rows(V):
    """The largest logits side by side, in one thread's hands or one chunk's, rising and falling."""
    rising = torch.arange(V, device="cuda").float() / 50
    logits = torch.stack([rising, rising.flip(0), torch.where(rising % 1 < 0.3, rising, -rising)]).contiguous()
    for top in (1, 17, 64):
        check(logits, torch.tensor([V - 1, 0, 5], dtype=torch.int32, device="cuda"), top)


@pytest.mark.parametrize("V, top", [(1121, 64), (4096, 33), (4096, 64), (40000, 64), (151936, 64)])
def test_more_candidates_than_are_ranked(V, top):
    """Rows in which one bound from the largest of a few threads' logits leaves hundreds of candidates, or more than are listed: many equal
    ones, zeros of both signs, a few finite ones among banned ones, neighbours that differ in the last bit, and all of it below zero."""
    logits, tokens = random_logits(8, V, V + top)
    at = torch.arange(V, device="cuda")
    logits[1] = torch.where(at % 7 < 6, 1.0, logits[1])
    logits[2] = torch.where(at % 3 == 0, -0.0, torch.where(at % 3 == 1, 0.0, -logits[2].abs() - 1))
    logits[3] = torch.where((at // 4) % 256 < 4, logits[3], -float("inf"))
    logits[3, 0] = 0.0
    logits[4] = (torch.full((V,), 1.0, device="cuda").view(torch.int32) + (at * 48271 % 8191).int()).view(torch.float32)
    logits[5] = -(torch.full((V,), 3.0, device="cuda").view(torch.int32) + (at * 48271 % 8191).int()).view(torch.float32)
    logits[6] = torch.where((at // 4) % 256 < 200, 5.0 + logits[6].abs(), -90.0)
    logits[7] = torch.where(at < top // 2, 0.0, -float("inf"))
    check(logits, tokens, top)


def test_the_largest_logits_all_with_the_same_threads():
    """A thread of the first kernel holds 16 logits of a chunk: four threads that hold the 64 largest of their chunk, and a row in which
    a few threads hold so many that the list of candidates does not hold them."""
    V = 4096
    logits, tokens = random_logits(4, 3 * V, 9, 0.1)
    for t in range(4):
        for j in range(4):
            at = (j * 256 + t) * 4
            logits[0, V + at:V + at + 4] += 50 + j
    for t in range(256):
        for j in range(4):
            logits[1, (j * 256 + t) * 4:(j * 256 + t) * 4 + 4] = 50.0 + (t // 4) * 1e-3 + j
    logits[2, ::16] += 10
    check(logits, tokens, 64)


@pytest.mark.parametrize("V", [300, 9000])
def test_banned_tokens(V):
    logits, tokens = random_logits(5, V, 3)
    logits[0, :] = -math.inf
    logits[0, 77] = 1.5                       # one token is left
    logits[1, ::2] = -math.inf
    logits[2, 5:] = -math.inf                 # fewer than are asked for
    logits[3, :V - 3] = torch.finfo(torch.float32).min
    tokens[0], tokens[1], tokens[2], tokens[3] = 77, 4, 100, V - 1
    check(logits, tokens, 20)


def test_far_apart_and_large_logits():
    logits, tokens = random_logits(4, 6000, 4)
    logits[0] *= 1e6
    logits[1] += 1e30
    logits[2] *= 1e-30
    logits[3, 100] = 3e38
    logits[3, 200] = -3e38
    tokens[3] = 100
    check(logits[:1].contiguous(), tokens[:1], 8)
    check(logits[2:].contiguous(), tokens[2:], 8)
    chosen, entropy, _, _ = results(logits[1:2].contiguous(), tokens[1:2], 0)           # (all of them are 1e30)
    assert abs(chosen.item() + math.log(6000)) < 1e-5 and abs(entropy.item() - math.log(6000)) < 1e-5


@pytest.mark.parametrize("V", [500, 10000])
def test_rows_that_are_no_distribution_and_tokens_that_are_none(V):
    logits, tokens = random_logits(6, V, 5)
    logits[0, 3] = math.nan
    logits[1, V - 1] = math.inf
    logits[2, :] = -math.inf
    logits[3, :] = math.nan
    tokens[4], tokens[5] = -1, V
    for top in (0, 6):
        chosen, entropy, ids, best = results(logits, tokens, top)
        assert torch.isnan(chosen).all()
        assert torch.isnan(entropy[:4]).all() and torch.isfinite(entropy[4:]).all()
        if top:
            assert (ids[:4] == -1).all() and torch.isnan(best[:4]).all() and torch.isfinite(best[4:]).all() and (ids[4:] >= 0).all()


def test_scratch_that_is_too_small_and_shapes_that_do_not_fit():
    logits, tokens = random_logits(4, 9000, 6)
    with pytest.raises(BackendError, match="too small"):
        results(logits, tokens, 5, ops.logprob_scratch(3, 9000, 5, logits.device))
    with pytest.raises(BackendError, match="too small"):
        results(logits, tokens, 5, ops.logprob_scratch(4, 9000, 4, logits.device))
    with pytest.raises(BackendError, match="alternatives"):
        results(logits, tokens, 65)
    with pytest.raises(BackendError, match="tokens"):
        results(logits, tokens.long(), 0)
    with pytest.raises(BackendError, match="contiguous"):
        results(logits[:, ::2], tokens, 0)
    with pytest.raises(BackendError, match="together"):
        ops.token_logprobs(logits, tokens, torch.empty(4, device="cuda"), torch.empty(4, device="cuda"), ids=torch.empty(4, 2, dtype=torch.int32, device="cuda"))


def test_tensors_of_another_gpu_than_the_current_one_are_refused(monkeypatch):
    logits, tokens = random_logits(2, 300, 6)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 3)
    with pytest.raises(BackendError, match="tensors lie on GPUs .0., the current one is 3"):
        ops.token_logprobs(logits, tokens, torch.empty(2, device="cuda:0"), torch.empty(2, device="cuda:0"))


def test_a_captured_call_replays_alike():
    logits, tokens = random_logits(7, 30000, 7)
    scratch = ops.logprob_scratch(7, 30000, 5, logits.device)
    R = 7
    chosen, entropy = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    ids, best = torch.empty((R, 5), dtype=torch.int32, device="cuda"), torch.empty((R, 5), device="cuda")
    ops.token_logprobs(logits, tokens, chosen, entropy, ids, best, scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(logits, tokens, chosen, entropy, ids, best, scratch)
    for i in range(4):
        logits.copy_(torch.randn_like(logits) * (i + 1))
        want = results(logits, tokens, 5)
        torch.cuda.synchronize()
        graph.replay()
        for got, w in zip((chosen, entropy, ids, best), want):
            assert torch.equal(got, w)
