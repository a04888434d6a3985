"""What the logits of a step say of given tokens, on its way from the GPU to the host.

The reference reports no probabilities: its sampler works them out on the host and drops them
(crates/core/src/sampler.rs:72-145).
"""
from dataclasses import dataclass
from typing import List, Tuple

import torch

from ..kernels import ops


@dataclass
class TokenLogprob:
    """A token's natural log probability under the softmax of its logits (temperature 1, nothing cut), that softmax's entropy, and its most
    probable tokens with theirs, the most probable first and the lower id first among equals. Logits that are no distribution (NaN,
    +inf, nothing above -inf) give NaN and ids of -1."""
    token: int
    logprob: float
    entropy: float
    top: List[Tuple[int, float]]


class PendingLogprobs:
    def __init__(self, tokens, host, event):
        self.tokens, self.host, self.event = tokens, host, event


class LogprobReader:
    """Log probabilities of steps' tokens with `top` alternatives each, put on the stream (`launch`) and read later (`read`). It
    keeps its memory; what was launched four launches ago has to be read before the next one."""

    RING = 4

    def __init__(self, top, vocab_size, device):
        self.top = min(int(top), vocab_size)
        self.vocab_size, self.device = vocab_size, device
        self._scratch = self._rows = None
        self._host, self._next = [], 0

    def _room(self, rows):
        if self._rows is None or self._rows < rows:
            self._rows = max(rows, 2 * (self._rows or 0))
            # (a row: log probability, entropy, the alternatives' ids and their log probabilities; the ids as the bits they are)
            self._scratch = ops.logprob_scratch(self._rows, self.vocab_size, self.top, self.device)
            self._out = torch.empty((2 + 2 * self.top) * self._rows, dtype=torch.float32, device=self.device)
            pinned = self.device.type == "cuda"
            self._host = [torch.empty(self._out.numel(), dtype=torch.float32, pin_memory=pinned) for _ in range(self.RING)]

    def launch(self, logits, tokens):
        """logits f32 [rows, vocabulary] and tokens int32 [rows] on the GPU."""
        rows, n = logits.shape[0], self.top
        self._room(rows)
        out = self._out[:(2 + 2 * n) * rows]
        ids = best = None
        if n:
            ids, best = out[2 * rows:(2 + n) * rows].view(torch.int32).view(rows, n), out[(2 + n) * rows:].view(rows, n)
        ops.token_logprobs(logits, tokens, out[:rows], out[rows:2 * rows], ids, best, self._scratch)
        host = self._host[self._next % self.RING][:out.numel()]
        self._next += 1
        host.copy_(out, non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        return PendingLogprobs(rows, host, event)

    def read(self, pending, tokens):
        """A TokenLogprob a row of a `launch`, once it has arrived; tokens: the same ones, as a list."""
        pending.event.synchronize()
        rows, n, host = pending.tokens, self.top, pending.host
        chosen, entropy = host[:rows].tolist(), host[rows:2 * rows].tolist()
        if not n:
            return [TokenLogprob(int(t), c, e, []) for t, c, e in zip(tokens, chosen, entropy)]
        ids = host[2 * rows:(2 + n) * rows].view(torch.int32).view(rows, n).tolist()
        best = host[(2 + n) * rows:].view(rows, n).tolist()
        return [TokenLogprob(int(t), c, e, list(zip(i, b))) for t, c, e, i, b in zip(tokens, chosen, entropy, ids, best)]

    def of(self, logits, tokens):
        """The same at once, for a list of tokens."""
        on_device = torch.tensor(list(tokens), dtype=torch.int32).to(self.device)
        return self.read(self.launch(logits, on_device), tokens)
