"""Several answers to a prompt through the generation loop, with a stand-in engine (no GPU needed)."""
import pytest
import torch

from herbert_rs_amd.cache import FreeList
from herbert_rs_amd.engine.generate import GenerationResult, Generator, plan_batches
from herbert_rs_amd.errors import RequestError
from herbert_rs_amd.sampling import SamplingParams

from .test_cache_and_loop import FakeEngine


class ForkingEngine(FakeEngine):
    """Logits that favour the token after the last one; a request's chooser adds its own number."""

    def __init__(self, n_pages=64, fail_at=None):
        super().__init__(n_pages)
        self.forks, self.fail_at = [], fail_at

    def step(self, entries):
        if self.fail_at is not None and len(self.steps) == self.fail_at:
            raise RuntimeError("failed")
        rows = super().step(entries)
        return None if rows is None else torch.from_numpy(rows)

    def fork(self, slot, count):
        new = [self.alloc_slot() for _ in range(count)]
        for s in new:
            self.cache.lengths[s] = self.cache.lengths[slot]
        self.forks.append((slot, new))
        return new


class OffsetChooser:
    """Request i's tokens are i further on each time: answers to one prompt differ."""

    def __init__(self, params, n, vocab, device):
        self.n, self.calls = n, []

    def choose(self, logits, order):
        self.calls.append(list(order))
        assert len(logits) == len(order)
        return [(int(r.argmax()) + i) % 50 for i, r in zip(order, logits)]


def run(prompts, samples, engine=None, max_batch=8, chunk=None, **kw):
    engine = engine or ForkingEngine()
    gen = Generator(engine, max_batch=max_batch, make_chooser=OffsetChooser, prefill_chunk=chunk)
    params = SamplingParams(temperature=0.0, samples=samples, ignore_eos=True, repeat_check=False, **kw)
    return engine, gen, gen.generate(prompts, params)


def want(prompt, i, n):
    out, last = [], prompt[-1]
    for _ in range(n):
        last = (last + 1 + i) % 50
        out.append(last)
    return out


@pytest.mark.parametrize("chunk", [None, 2])
@pytest.mark.parametrize("max_batch", [8, 2, 5])
def test_answers_come_prompt_by_prompt_and_the_prompt_goes_through_once(max_batch, chunk):
    prompts = [[5, 6, 7], [20], [30, 31, 32, 33, 34]]
    engine, gen, results = run(prompts, 3, max_batch=max_batch, chunk=chunk, max_tokens=4)
    assert [r.tokens for r in results] == [want(prompts[i // 3], i, 4) for i in range(9)]
    assert [r.prompt_tokens for r in results] == [len(prompts[i // 3]) for i in range(9)]
    assert engine.cache.slots.held_count == 0
    batches = plan_batches([3, 1, 5], 4, max_batch, 64 * 64, 40, 3)
    leaders = sum(len({i // 3 for i in b}) for b in batches)
    fed = sum(n for step in engine.steps for _, n in step)
    assert fed == sum(len(prompts[p]) for b in batches for p in {i // 3 for i in b}) + 9 * 3
    assert sum(len(new) for _, new in engine.forks) == 9 - leaders
    assert gen.stats.generated_tokens == 36


def test_one_answer_forks_nothing():
    engine, _, results = run([[5], [6]], 1, max_tokens=3)
    assert engine.forks == [] and [r.tokens for r in results] == [want([5], 0, 3), want([6], 1, 3)]


@pytest.mark.parametrize("fail_at", [0, 1, 2])
def test_slots_come_back_when_a_step_fails(fail_at):
    engine = ForkingEngine(fail_at=fail_at)
    with pytest.raises(RuntimeError):
        run([[5], [7]], 3, engine=engine, max_tokens=4)
    assert engine.cache.slots.held_count == 0


def test_slots_come_back_when_a_fork_fails():
    engine = ForkingEngine()

    def fork(slot, count):
        raise RequestError("no slots")
    engine.fork = fork
    with pytest.raises(RequestError):
        run([[5]], 3, engine=engine, max_tokens=4)
    assert engine.cache.slots.held_count == 0


def test_batches_count_a_shared_prompt_once():
    # a prompt of 130 tokens and 20 new ones: three pages; every further answer one (the prompt's last page is its own)
    assert plan_batches([130], 20, 64, 64 * 6, 512, 4) == [[0, 1, 2, 3]]
    assert plan_batches([130], 20, 64, 64 * 5, 512, 4) == [[0, 1, 2], [3]]
    assert plan_batches([130], 20, 64, 64 * 3, 512, 2) == [[0], [1]]
    assert plan_batches([128], 64, 64, 64 * 4, 512, 2) == [[0, 1]]
    assert plan_batches([130, 10], 20, 64, 64 * 7, 512, 3) == [[0, 1, 2, 3, 4], [5]]
    assert plan_batches([10, 10], 20, 3, 64 * 64, 512, 2) == [[0, 1, 2], [3]]


def test_parameters_are_checked():
    for bad in (dict(samples=0), dict(logprobs=-1), dict(logprobs=65)):
        with pytest.raises(RequestError):
            SamplingParams(**bad).validate()
    SamplingParams(samples=3, logprobs=0).validate()
    gen = Generator(ForkingEngine(), make_chooser=OffsetChooser)
    with pytest.raises(RequestError, match="one answer"):
        gen.extend(0, [1], SamplingParams(samples=2), OffsetChooser(None, 1, 50, "cpu"))


def test_the_books_of_free_slots_hold():
    slots = FreeList(4, "slot")
    engine = ForkingEngine()
    engine.cache.slots = slots
    run([[5]], 4, engine=engine, max_tokens=2)
    slots.check()
    assert slots.held_count == 0


@pytest.mark.parametrize("chunk", [None, 2])
@pytest.mark.parametrize("slots, held", [(2, 0), (1, 0), (4, 2)])
def test_answers_run_in_as_many_batches_as_there_are_slots_for(slots, held, chunk):
    """More answers than free slots; a prompt of as many positions as the model has, whose further answers need no page of their own."""
    engine = ForkingEngine()
    engine.cache.slots = FreeList(slots, "slot")
    mine = [engine.alloc_slot() for _ in range(held)]
    prompts = [[5, 6, 7], [20]]
    _, gen, results = run(prompts, 5, engine=engine, chunk=chunk, max_tokens=4)
    assert [r.tokens for r in results] == [want(prompts[i // 5], i, 4) for i in range(10)]
    assert gen.stats.batches == 10 // (slots - held)
    assert engine.cache.slots.held_count == held
    engine.spec.max_positions = 64
    full = [3] * 64
    _, _, results = run([full], 5, engine=engine, chunk=chunk, max_tokens=4)
    assert [(r.tokens, r.stop_reason) for r in results] == [(want(full, i, 1), "length") for i in range(5)]
    for s in mine:
        engine.free_slot(s)
    assert engine.cache.slots.held_count == 0


class Loaded:
    """What `load` gave: how many tokens it was to hold, and which calls it got."""

    def __init__(self):
        self.room, self.asked = [], []

    def __call__(self, model, dtype="bfloat16", cache_tokens=None, max_slots=None):
        self.room.append(cache_tokens)
        return self

    def generate(self, prompts, params, **kw):
        self.asked.append(params.samples)
        return [GenerationResult([1], "length", len(p)) for p in prompts for _ in range(params.samples)]

    def score(self, prompt, continuations, top):
        return [[] for _ in continuations]


def test_caches_are_as_large_as_what_runs_at_once(monkeypatch):
    """A thousand answers in batches of 64 need the room of 64."""
    from herbert_rs_amd import api
    loaded = Loaded()
    monkeypatch.setattr(api, "load", loaded)
    for prompts, samples, max_batch in (([[1] * 200], 1000, 64), ([[1] * 200], 64, 64), ([[1] * 200] * 30, 7, 64), ([[1] * 200] * 300, 3, 16)):
        out = api.generate("folder", prompts, max_tokens=100, samples=samples, max_batch=max_batch)
        assert len(out) == len(prompts) and all(len(a) == samples for a in out)
        room = loaded.room[-1]
        biggest = max(batch_pages(b, [200] * len(prompts), 100, samples)
                      for b in plan_batches([200] * len(prompts), 100, max_batch, 64 * 10 ** 6, 4096, samples))
        assert 64 * biggest <= room <= 64 * (biggest + 4 * max_batch)
    for n in (10, 512, 20000):
        api.score("folder", [1] * 200, [[5] * 30] * n)
        assert loaded.room[-1] <= 200 + 128 + 192 * min(n, 512)


def batch_pages(members, lengths, max_new, samples):
    """Pages that a batch holds at its end: a prompt's whole pages once."""
    total = 0
    for p in {i // samples for i in members}:
        whole, count = -(-(lengths[p] + max_new) // 64), sum(i // samples == p for i in members)
        total += whole + (count - 1) * (whole - lengths[p] // 64)
    return total


def test_wrong_parameters_are_refused_before_a_model_is_loaded(monkeypatch):
    from herbert_rs_amd import api
    loaded = Loaded()
    monkeypatch.setattr(api, "load", loaded)
    for bad in (dict(samples=0), dict(samples=-3), dict(temperature=-1.0)):
        with pytest.raises(RequestError):
            api.generate("folder", [[1, 2]], **bad)
    assert loaded.room == []


def test_the_command_line_asks_for_the_room_of_what_runs_at_once(monkeypatch, tmp_path):
    from herbert_rs_amd import api, cli
    from .tiny import make_folder
    folder, asked = make_folder(tmp_path, "A"), []

    def load(model, dtype, cache_tokens):
        asked.append(cache_tokens)
        raise RequestError("far enough")
    monkeypatch.setattr(api, "load", load)
    for samples in (1, 3, 64, 1000):
        assert cli.main(["--model", folder, "--prompt", "5,17,3", "--max-tokens", "40", "--samples", str(samples)]) == 1
    assert asked == [3 + 105, 3 + 105 + 2 * 232, 3 + 105 + 63 * 232, 3 + 105 + 63 * 232]
