"""The generation loop above the step function.

Requests are served in batches, one after another: the prompts of a batch in
one step, then one token for every sequence that still runs. A sequence ends
on its end-of-sequence token (kept in the output, as the reference keeps it:
crates/cli/src/main.rs:1272,1357-1359), on a stop token, after max_tokens
tokens, on a repetition loop (crates/core/src/decode_utils.rs:14-33), when
the caller's `on_token` says so (stop strings are the caller's, since text is:
crates/cli/src/main.rs:1328-1332,1360) or at the model's last position; it
gives its slot back at once and the others go on. Before every decode step
the caller's interrupt flag is looked at (crates/cli/src/main.rs:1242-1245):
when it is set, every running sequence ends with what it has and every slot
is given back.

Where engine and sampler allow it, decode steps are put on the GPU's stream
one ahead of the host (`_decode_ahead`): a step takes its tokens from where
the sampler left them on the GPU, and the host reads them, applies the stop
rules and calls `on_token` while the next step already runs. The tokens and
stop reasons are those of the step-by-step loop.

Several answers to a prompt (`SamplingParams.samples`, not in the reference) are requests of their own with generator streams of their own,
but the prompt goes through the model once: the first answer's slot is forked for the others (`Engine.fork`), whose steps
then read the prompt's keys and values together. With `SamplingParams.logprobs` every token comes with what its logits said of it.

`max_tokens` here counts every generated token, the one the prompt's step
gives included: the reference's chat and server loops (`for _ in
1..max_tokens` after the first token, crates/cli/src/chat.rs:231). Its
single-shot command line runs `for _step in 0..max_tokens` decode steps after
the first token (crates/cli/src/main.rs:1040,1241), one token more; the
command line here asks this loop for max_tokens + 1 to give what that gives.
"""
import time
from dataclasses import dataclass, field
from typing import List, Optional

import torch

from ..cache import PAGE_TOKENS
from ..errors import BackendError, RequestError
from ..sampling import (EOS, INTERRUPTED, LENGTH, MAX_TOKENS, REPETITION_LOOP, STOP_TOKEN,
                        SamplingParams, detect_repetition_loop)
from .batch import StepEntry


@dataclass
class GenerationResult:
    tokens: List[int]
    stop_reason: str
    prompt_tokens: int
    logprobs: Optional[List] = None      # a sampling.logprobs.TokenLogprob a token, where they were asked for


@dataclass
class GenerationStats:
    prompt_tokens: int = 0
    generated_tokens: int = 0
    prefill_seconds: float = 0.0
    decode_seconds: float = 0.0
    decode_steps: int = 0
    batches: int = 0


def _rounded(n):
    return (n + PAGE_TOKENS - 1) // PAGE_TOKENS * PAGE_TOKENS


def plan_batches(prompt_lengths, max_new, max_batch, capacity_tokens, max_positions, samples=1):
    """Lists of request indices, in order, each list one batch that fits the cache. Request i is an answer to prompt i // samples (of
    which prompt_lengths has one length each); answers to one prompt share its whole pages within a batch."""
    batches, current, used = [], [], 0
    for p, n in enumerate(prompt_lengths):
        if n <= 0:
            raise RequestError(f"request {p} has an empty prompt")
        if n > max_positions:
            raise RequestError(f"request {p}: prompt of {n} tokens exceeds "
                               f"max_position_embeddings ({max_positions})")
        whole = _rounded(min(n + max_new, max_positions))
        if whole > capacity_tokens:
            raise RequestError(f"request {p} needs room for {whole} tokens but the cache holds "
                               f"{capacity_tokens}")
        own = whole - n // PAGE_TOKENS * PAGE_TOKENS       # beside an answer in the same batch: the prompt's last page is copied
        for i in range(p * samples, (p + 1) * samples):
            need = own if current and current[-1] // samples == p else whole
            if current and (len(current) >= max_batch or used + need > capacity_tokens):
                batches.append(current)
                current, used, need = [], 0, whole
            current.append(i)
            used += need
    if current:
        batches.append(current)
    return batches


def stop_reason(generated, params, eos_id):
    """Why a sequence ends after its newest token, or None."""
    tok = generated[-1]
    if not params.ignore_eos and eos_id is not None and tok == eos_id:
        return EOS
    if tok in params.stop_ids:
        return STOP_TOKEN
    if len(generated) >= params.max_tokens:
        return MAX_TOKENS
    if params.repeat_check and detect_repetition_loop(generated) is not None:
        return REPETITION_LOOP
    return None


class Generator:
    """Runs requests through an engine. `make_chooser(params, n, vocab, device)` builds the object
    whose `choose(logits, sequence_indices)` picks tokens (the GPU sampler by default)."""

    def __init__(self, engine, max_batch=64, make_chooser=None, prefill_chunk=None, run_ahead=True):
        self.engine = engine
        self.max_batch = int(max_batch)
        # decode steps are put on the GPU's stream one ahead of the host where engine and chooser can
        self.run_ahead = bool(run_ahead)
        # prompts longer than this many tokens are fed in pieces of that size, one step a piece
        # (the reference's prefill_chunk_size: crates/cli/src/main.rs:400-408)
        self.prefill_chunk = int(prefill_chunk) if prefill_chunk else None
        if self.prefill_chunk is not None and self.prefill_chunk <= 0:
            raise RequestError("prefill_chunk must be > 0")
        if make_chooser is None:
            from ..sampling.sampler import Sampler
            make_chooser = Sampler
        self.make_chooser = make_chooser
        self.stats = GenerationStats()
        # the loop is done with a decode step's logits before its next step: it takes the engine's
        # own rows where the engine would otherwise hand out a copy
        self._views = {"keep_logits": False} if getattr(engine, "hands_out_copies", False) else {}

    def generate(self, prompts, params=None, on_token=None, interrupt=None):
        """One GenerationResult per prompt (a list of token ids), in the prompts' order; with params.samples > 1 that many for every
        prompt, one after the other: request i is then an answer to prompt i // samples.
        on_token(request index, token) is called for every generated token; if it returns a
        string, the sequence ends there with that stop reason (the token is kept). It must not
        use the engine: the step after the token's may already be on the GPU. `interrupt()`
        is asked before every decode step and before every batch: once it is true, running
        sequences end with reason "interrupted" and requests not yet started return no tokens."""
        params = params or SamplingParams()
        params.validate()
        eng = self.engine
        spec = eng.spec
        capacity = eng.cache.n_pages * PAGE_TOKENS
        # (further answers to a prompt may need no page of their own, but every one a slot)
        at_once = min(self.max_batch, max(1, eng.cache.slots.free_count))
        batches = plan_batches([len(p) for p in prompts], params.max_tokens, at_once, capacity,
                               spec.max_positions, params.samples)
        prompts = [p for p in prompts for _ in range(params.samples)]
        chooser = self.make_chooser(params, len(prompts), spec.vocab_size, eng.device)
        results = [None] * len(prompts)
        self.stats = GenerationStats()
        for members in batches:
            if interrupt is not None and interrupt():
                for i in members:
                    results[i] = GenerationResult([], INTERRUPTED, len(prompts[i]), None if params.logprobs is None else [])
                continue
            self._run_batch(members, prompts, params, chooser, results, on_token, interrupt)
            self.stats.batches += 1
        return results

    def _choose(self, chooser, logits, order, logprobs):
        """Tokens of the rows of a step's logits, and what the logits said of them (None: not asked for)."""
        if logprobs is None:
            return chooser.choose(logits, order), None
        if getattr(chooser, "changes_logits", False):
            said = logits.clone()           # (as the model gave them)
            tokens = chooser.choose(logits, order)
            return tokens, logprobs.of(said, tokens)
        tokens = chooser.choose(logits, order)
        return tokens, logprobs.of(logits, tokens)

    def _prompts(self, live, prompts, slots, chooser, leader, logprobs):
        """The prompts of a batch through the engine; the first token of each sequence, in the
        order of `live`, and what the logits said of them. Whole in one step, or, with a prefill chunk, in steps that carry the
        next piece of every prompt that still has one: a sequence's token is chosen in the step
        that brings its last piece. leader[i]: the request whose slot the prompt of request i goes through; the others' slots are
        forked from it."""
        eng, chunk = self.engine, self.prefill_chunk
        leading = [i for i in live if leader[i] == i]
        following = {i: [j for j in live if leader[j] == i] for i in leading}         # (with itself, first)

        def ended(leaders, logits):
            order = [j for i in leaders for j in following[i]]
            if len(order) > len(leaders):
                rows = [r for r, i in enumerate(leaders) for _ in following[i]]
                logits = logits[torch.tensor(rows, dtype=torch.long, device=logits.device)]
                for i in leaders:
                    others = following[i][1:]
                    if others:
                        slots.update(zip(others, eng.fork(slots[i], len(others))))
            tokens, said = self._choose(chooser, logits, order, logprobs)
            first.update(zip(order, zip(tokens, said if said is not None else [None] * len(order))))

        first = {}
        if chunk is None or all(len(prompts[i]) <= chunk for i in leading):
            entries = [StepEntry(slots[i], list(prompts[i]), [len(prompts[i]) - 1]) for i in leading]
            ended(leading, eng.step(entries))
        else:
            fed = {i: 0 for i in leading}
            while len(first) < len(live):
                entries, ending = [], []
                for i in leading:
                    left = len(prompts[i]) - fed[i]
                    if left <= 0:
                        continue
                    n = min(chunk, left)
                    entries.append(StepEntry(slots[i], list(prompts[i][fed[i]:fed[i] + n]), [n - 1] if n == left else []))
                    if n == left:
                        ending.append(i)
                    fed[i] += n
                logits = eng.step(entries)
                if ending:
                    ended(ending, logits)
        return [first[i][0] for i in live], None if logprobs is None else [first[i][1] for i in live]

    def _decode_ahead(self, live, slots, generated, params, chooser, take, kept=(), logprobs=None):
        """Decoding with the host one step behind the GPU. The tokens that a step chooses stay on
        the GPU, and the next step is put on the stream with them at once, before the host has
        seen them; the host reads a step's tokens while the next one runs, so the GPU does not
        wait for the host's share of a step. A sequence whose newest token turns out to end it
        (end of sequence, a stop token, the caller's word) has then already been through one step
        more: that step's work on it is thrown away, its slot is given back as always, and every
        other sequence's tokens are what they would have been. Sequences that end for a reason the
        host knows beforehand (max_tokens, the model's last position) are not taken ahead.
        The step thrown away has also taken a draw from the sequence's generator stream: for a
        sequence whose slot the caller keeps (`kept`: its chooser goes on into the next turn) the
        streams are saved before every step that runs ahead (`chooser.save_streams`) and the
        sequence's is put back when it ends, so that a seeded conversation draws what the
        step-by-step loop draws, one draw a token."""
        eng = self.engine
        saves = bool(kept) and hasattr(chooser, "save_streams")

        def launch(order, device_tokens):
            entries = [StepEntry(slots[i], [generated[i][-1]] if device_tokens is None else [0], [0])
                       for i in order]
            logits = eng.step(entries, tokens_on_device=device_tokens, **self._views)
            self.stats.decode_steps += 1
            pending = chooser.choose_ahead(logits, order)
            said = logprobs.launch(logits, pending.device) if logprobs is not None else None
            return pending, said, {i: eng.cache.length(slots[i]) for i in order}

        if not live:
            return
        order = list(live)
        pending, said, held = launch(order, None)
        while True:
            # the step after the one in flight, for the sequences that its token cannot end by count
            ahead = [i for i in order if i in slots and len(generated[i]) + 2 <= params.max_tokens
                     and eng.cache.length(slots[i]) < eng.spec.max_positions]
            following = saved = None
            if ahead:
                rows = [order.index(i) for i in ahead]
                if saves:
                    saved = chooser.save_streams()
                following = launch(ahead, chooser.rows_of(pending, rows))
            tokens = chooser.read(pending)
            take(order, tokens, held, logprobs.read(said, tokens) if logprobs is not None else None)
            if saved is not None:
                for i in ahead:
                    if i not in slots and i in kept:        # it ended on this token: the draw after it never was
                        chooser.restore_stream(i, saved)
            if not live or following is None:
                break
            order, (pending, said, held) = ahead, following

    def extend(self, slot, tokens, params, chooser, on_token=None, interrupt=None):
        """One more turn of a sequence whose slot the caller keeps (the reference's
        continue_prefill and decode on a kept KvHandle, crates/cli/src/chat.rs:1060-1075,
        164-352): `tokens` go on from what the slot holds (nothing, for a first turn), then
        tokens are generated as in `generate`. The slot is not given back; when this returns it
        holds everything up to the newest generated token, which itself has not been through
        the model: the next turn's tokens begin with it. `chooser` is the caller's too (its
        generator streams go on from turn to turn); sequence index 0 is used. Returns one
        GenerationResult."""
        params.validate()
        if params.samples != 1:
            raise RequestError("a turn has one answer")
        if not tokens:
            raise RequestError("a turn needs at least one token")
        eng = self.engine
        room = eng.spec.max_positions - eng.cache.length(slot)
        if len(tokens) > room:
            raise RequestError(f"a turn of {len(tokens)} tokens does not fit: the sequence holds "
                               f"{eng.cache.length(slot)} of max_position_embeddings ({eng.spec.max_positions})")
        results = [None]
        self.stats = GenerationStats()
        self._run_batch([0], [list(tokens)], params, chooser, results, on_token, interrupt, kept={0: slot})
        self.stats.batches += 1
        return results[0]

    def _run_batch(self, members, prompts, params, chooser, results, on_token, interrupt=None, kept=None):
        """`kept`: request index -> a slot of the caller's (see `extend`) instead of one taken
        here and given back at the end."""
        eng = self.engine
        eos = eng.spec.eos_token_id
        kept = kept or {}
        # answers to one prompt that stand side by side: the first one's slot takes the prompt, the others are forked from it
        leader = {}
        for at, i in enumerate(members):
            same = params.samples > 1 and at > 0 and members[at - 1] // params.samples == i // params.samples
            leader[i] = leader[members[at - 1]] if same else i
        logprobs = None
        if params.logprobs is not None:
            from ..sampling.logprobs import LogprobReader
            logprobs = LogprobReader(params.logprobs, eng.spec.vocab_size, eng.device)
        slots = {}
        before = {i: eng.cache.length(kept[i]) for i in kept}
        generated = {i: [] for i in members}
        said_of = {i: None if logprobs is None else [] for i in members}
        live = list(members)

        def finish(i, reason):
            results[i] = GenerationResult(generated[i], reason, len(prompts[i]), said_of[i])
            slot = slots.pop(i)
            if i in kept:
                # a step that ran ahead of the host has taken the newest token in already
                eng.truncate(slot, before[i] + len(prompts[i]) + len(generated[i]) - 1)
            else:
                eng.free_slot(slot)
            live.remove(i)

        try:
            for i in members:
                if leader[i] == i:
                    slots[i] = kept[i] if i in kept else eng.alloc_slot()
            t0 = time.perf_counter()
            tokens, said = self._prompts(live, prompts, slots, chooser, leader, logprobs)
            self.stats.prefill_seconds += time.perf_counter() - t0
            self.stats.prompt_tokens += sum(len(prompts[i]) for i in live if leader[i] == i)
            t0 = time.perf_counter()

            def take(order, tokens, held=None, said=None):
                """The newest tokens of the sequences `order` (those that have ended since are
                skipped). `held`: the positions each sequence held when the step that chose these
                tokens had been put on the stream, if a later step has been since."""
                for at, (i, tok) in enumerate(zip(order, tokens)):
                    if i not in slots:
                        continue
                    if not 0 <= int(tok) < eng.spec.vocab_size:
                        # (the chooser's answer for a row of logits without a finite value: what a
                        # token id out of range, fed from the GPU where no host check sees it, leaves)
                        raise BackendError(f"request {i}: no token could be chosen (got {int(tok)}): its logits "
                                           "hold no finite value")
                    generated[i].append(int(tok))
                    if said is not None:
                        said_of[i].append(said[at])
                    self.stats.generated_tokens += 1
                    answer = on_token(i, int(tok)) if on_token is not None else None
                    reason = stop_reason(generated[i], params, eos)
                    if reason is None and isinstance(answer, str):
                        reason = answer
                    length = eng.cache.length(slots[i]) if held is None else held[i]
                    if reason is None and length >= eng.spec.max_positions:
                        reason = LENGTH
                    if reason is not None:
                        finish(i, reason)
                if live and interrupt is not None and interrupt():
                    for i in list(live):
                        finish(i, INTERRUPTED)

            take(list(live), tokens, None, said)
            # (a kept slot is rolled back by the one step that ran ahead: only where the cache can)
            if self.run_ahead and getattr(chooser, "can_run_ahead", False) and \
                    getattr(eng, "accepts_device_tokens", False) and \
                    (not kept or getattr(eng.cache, "rolls_back_freely", False)):
                self._decode_ahead(live, slots, generated, params, chooser, take, kept, logprobs)
            else:
                while live:
                    order = list(live)
                    logits = eng.step([StepEntry(slots[i], [generated[i][-1]], [0]) for i in order], **self._views)
                    self.stats.decode_steps += 1
                    tokens, said = self._choose(chooser, logits, order, logprobs)
                    take(order, tokens, None, said)
            self.stats.decode_seconds += time.perf_counter() - t0
        finally:
            for i in list(slots):
                slot = slots.pop(i)
                if i not in kept:
                    eng.free_slot(slot)
