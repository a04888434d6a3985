"""Host side of the attention over pages that several sequences of a step share: how a step is cut into items, operand
checks, the launch (csrc/attention_shared.hip).

The reference attends over every sequence's cache by itself
(crates/backends/backend_common/src/attention_common.rs:20-124)."""
import ctypes
from functools import lru_cache

import numpy as np
import torch

from ..cache import SharedPages
from ..errors import BackendError
from ..hosted import send, send_into
from . import lib, mfma, ops
from .ops import _stream

_P, _I, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
lib.register_signatures("attention_shared", {
    "hb_attn_shared": [_P, _P, _P, _P, _I, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _F, _F, _P, _P],
})

ITEM_INTS = 8
COLUMNS = {torch.bfloat16: 128, torch.float32: 16}      # (row, head) pairs of a kv head that an item holds at most
F32_MOST_DIM = 256
# Workgroups that a step is cut into: as many as the GPU holds at a time, two a CU in bfloat16, four in float32. Measured with 256, 384 and 512 in
# bfloat16, one call after another over the same pages (caches warm; with cold ones 97 and 38 us of the first two at 512): 128 answers to 32,768 tokens 110, 95
# and 89 us, 64 to 8,192 37, 33 and 33 us, 12 continuations of a text of 2,000 tokens 46, 44 and 46 us.
WORKGROUPS = {torch.bfloat16: 512, torch.float32: 1024}
OPERANDS = ("q", "out", "key pages", "value pages", "page_table", "positions", "seq_of", "slots", "sinks")
MASKED_COLUMNS = 64             # of an item in whose pages are places that some of its rows see and others do not: the wide ones ask no mask
# Pages of the longest sequence up to which every sequence is an item of its own, whose pages four waves of one CU read (at 40 bytes a nanosecond), and nothing
# is joined. Caches warm, 2, 8 and 64 sequences of 4, 8 and 8 kv heads of 128: of 4 pages 8.0, 8.1, 12.0 us by themselves, 10.1, 11.3, 15.3 joined; of 6 9.2, 9.4, 15.5 and 11.0, 11.8,
# 15.9; of 8 10.5, 10.8, 18.5 and 10.9, 11.8, 16.6.
BY_ITSELF_PAGES = 6
# The attention of one sequence after another also normalizes, rotates and writes what the projection gave; before the shared one that is a kernel of its
# own. Bytes that need not be read again from which the shared one ends sooner all the same, in a model's decode steps (36 layers of 32 heads of
# 128 over 8; microseconds a layer, shared less separate): 2 answers to 8,192 and 16,384 tokens (34, 67 MB) +2.1, -3.8; 4 to 2,048 and
# 4,096 (25, 50 MB) +1.0, -0.8; 8 to 1,024 and 2,048 (29, 59 MB) +4.3, +0.8; 16 to 1,024, 2,048 and 2,560 (63, 126, 157 MB) +6.1, +0.5, -2.4; 32
# to 1,024 and 2,048 (130, 260 MB) +4.3, -5.2; 48 to 1,024 (197 MB) -6; 64 to 256, 512 and 1,024 (66, 132, 264 MB) +5.6, +1.0, -9.7; 96 to 512 (199 MB) -2.4; 128 to 256
# and 512 (133, 266 MB) +5.9, -6.9.
SAVED_BYTES = 32 << 20
SAVED_BYTES_EACH = 6 << 20      # and these for each sequence, of SAVED_SEQUENCES at most
SAVED_SEQUENCES = 20
# Where a kernel of its own norms, rotates and writes in any case (a filter along time, a cache that another entry fills, part of a head rotated), a step
# whose sequences are items of their own ends sooner than by the attention of one sequence after another at heads of up to so many entries, so
# many sequences x kv heads, and from the page behind so many on. A model's decode steps, microseconds that whole rows save of 710 to 900, 12 filtered
# layers, prompts of 70, 134, 198 and 326 tokens: 16 heads of 64 over 4, 2 sequences 5, 1, 6, 10, 8 sequences 9, 3, 8, 18, 16 sequences 5, 2, 8, 18, 32 sequences
# 0, -1, 1, 0; over 16, 2 sequences 1, -1, 4, 11, 8 sequences 6, 1, 6, -2; 16 heads of 32 over 2, 2 sequences 2, 0, 4, 20, 8 sequences 4, 4, 10, 28, 16 sequences 0,
# 3, 5, 24; 8 over 8, 2 sequences 0, -5, 1, 18, 8 sequences -5, -6, 0, 18. Heads of 128 by themselves: 2 sequences of 4 kv heads 5.6, 6.4, 7.7, 7.1 us separate,
# 6.0, 6.9, 7.7, 9.0 as whole rows.
ALONE_DIM = 64
ALONE_PAIRS = 64
ALONE_PAGES = 3
# New tokens a sequence, on the mean, up to which a step is taken: beyond, its own columns fill the products. Microseconds shared / separate. bfloat16, 32 heads
# of 128 over 8: 24 sequences of 4, 8, 12, 16 and 40 tokens behind 2,000 29/33, 30/33, 33/33, 39/34, 62/68, of 200 297/196; 64 behind 1,000 28/42, 33/43, 44/45, 50/47,
# 114/80; behind 4,000, where more is saved, 24 sequences 27/59, 35/58, 40/59, 50/61, 88/122. float32, 16 sequences of 16, 40, 80 and 200 tokens: 16 heads of 128
# over 8 behind 256 27/22, 49/48, 91/83, 239/216, behind 2,000 87/100, 198/227, 378/364, 947/921; 32 over 8 behind 2,000 159/146, 378/358, 741/700, 1,875/1,760; 8 of 64 over 2
# behind 256 12/15, 17/19, 27/25, 58/60, behind 2,000 28/65, 54/87, 97/115, 235/262; 8 sequences of 1, 8 and 40, 8 of 256 over 4, behind 2,000 18/527, 53/532, 151/529.
MANY_TOKENS = {torch.bfloat16: 8, torch.float32: 200}


def supported(kv, nq, nkv, hd, dtype):
    """True if the shared attention takes such heads and such a cache."""
    if kv.v is None or kv.window or kv.page_size != 64 or kv.k.dtype != dtype or nkv <= 0 or nq % nkv:
        return False
    if dtype == torch.bfloat16:
        return hd in mfma.ATTENTION_HEAD_DIMS and nq // nkv <= 32
    return dtype == torch.float32 and hd % 4 == 0 and 0 < hd <= F32_MOST_DIM


def plan(starts, context, slots, sharing, group, nkv, columns, workgroups, grid=1):
    """How a step is cut up. starts: the first packed row of each sequence and the last one's end; context: the positions it
    holds after the step; slots: theirs; sharing: a SharedPages. Returns int32 arrays (items [n, 8], order [rows], part_start
    [rows + 1], parts) and the most rows of an item; see csrc/attention_shared.hip.

    A node of the sharing is cut into tiles of as many rows as fit `columns`; a tile's pages are cut into ranges of about as many pages
    each that the workgroups (items x kv heads) come to `workgroups`, whole rounds of the waves that take them in turn. The pages
    that a tile of more than 64 columns sees in part are items of their own.

    Cut natively (csrc/hostcall.cpp): steps of many sequences begin a page nearly every time, and models whose steps wait for the host waited for
    NumPy. 128 forks of 2,000 tokens, one layer 560 us a step, now 450 (410 with every sequence reading its own pages), four layers 562, now 503 (755)."""
    numbers, n_items, _, most = _cut(starts, context, slots, sharing, group, nkv, columns, workgroups, grid)
    rows = int(starts[-1])
    at = np.cumsum([ITEM_INTS * n_items, rows, rows + 1])
    return numbers[:at[0]].reshape(n_items, ITEM_INTS), numbers[at[0]:at[1]], numbers[at[1]:at[2]], numbers[at[2]:], most


def _cut(starts, context, slots, sharing, group, nkv, columns, workgroups, grid, room=0):
    """What `plan` gives, one behind the other, the items in the room of `room` at least; how many items and parts, the most rows of an item."""
    if len(sharing.order) != len(starts) - 1:
        raise BackendError(f"shared attention: pages shared by {len(sharing.order)} sequences in a step of {len(starts) - 1}")
    as64 = lambda x: np.ascontiguousarray(x, dtype=np.int64)
    made = lib.host().plan(as64(starts), as64(context), as64(slots), as64(sharing.order), sharing.node_array, group, nkv, columns, MASKED_COLUMNS,
                           workgroups, grid, room)
    if made is None:
        raise BackendError("shared attention: the pages that are said to be shared are not those of this step's sequences, each in its place")
    return (np.frombuffer(made[0], dtype=np.int32), *made[1:])


def _by_itself(meta, nkv, dtype):
    """True for steps of short contexts, which end sooner without a second kernel: every sequence is an item, whose result is the row's."""
    return (dtype == torch.bfloat16 and meta.max_new == 1 and meta.num_seqs * nkv <= WORKGROUPS[dtype]
            and int(meta.host_context.max()) <= 64 * BY_ITSELF_PAGES)


@lru_cache(maxsize=64)
def _all_alone(n):
    return SharedPages(np.arange(n), [(i, 1, 0, -1) for i in range(n)])


def _planned(meta, group, nkv, dtype, cut, *grid_and_room):
    """(What `cut`, that is `plan` or `_cut`, gives of a step, whether every row is one item's.)"""
    sharing, workgroups, direct = meta.shared, WORKGROUPS[dtype], _by_itself(meta, nkv, dtype)
    if direct:
        sharing, workgroups = _all_alone(len(sharing.order)), 1
    return (*cut(meta.host_starts, meta.host_context, meta.host_slots, sharing, group, nkv, COLUMNS[dtype], workgroups, *grid_and_room), direct)


class Plan:
    """A plan on the GPU: of meta.shared as it is now."""

    def __init__(self, meta, group, nkv, dtype):
        numbers, self.n_items, self.n_parts, self.max_rows, self.direct = _planned(meta, group, nkv, dtype, _cut, 1)
        at = np.cumsum([ITEM_INTS * self.n_items, meta.num_tokens, meta.num_tokens + 1])
        b = send(numbers, meta.positions.device)
        self.items, self.order, self.part_start, self.parts = b[:at[0]], b[at[0]:at[1]], b[at[1]:at[2]], b[at[2]:]
        self.sharing = meta.shared


class StaticPlan:
    """The plans of decode steps of one batch size, in buffers that stay where they are while they are large enough: a recorded
    graph reads them. `shape` is what such a graph is tied to: which buffers, how many workgroups (in steps of GRID), how much room
    for partial results (powers of two), and whether there are any."""
    GRID = 16

    def __init__(self, group, nkv, dtype, rows, device):
        self.group, self.nkv, self.dtype, self.rows, self.device = group, nkv, dtype, rows, device
        self.direct = False
        self.made = 0               # buffers so far: those that were outgrown are kept, a graph may hold their addresses
        self._outgrown = []
        self._buffer, self._rooms, self._filled_for = None, (0, 0), None
        self.n_items = self.n_parts = 0

    @property
    def shape(self):
        return self.made, self.n_items, self.n_parts, self.direct

    @property
    def max_rows(self):
        return 1 if self.direct else max(1, COLUMNS[self.dtype] // self.group)

    def refill(self, meta):
        """Work the step's plan out and send it, unless it is that of the step before (it changes where a sequence begins a page)."""
        filled_for = (meta.shared, meta.host_slots.tobytes(), ((meta.host_context - 1) // 64).tobytes())
        before = self._filled_for
        if before is not None and before[0] is meta.shared and before[1:] == filled_for[1:]:
            return
        numbers, self.n_items, n_parts, _, self.direct = _planned(meta, self.group, self.nkv, self.dtype, _cut, self.GRID, self._rooms[0])
        self.n_parts = 1 << (n_parts - 1).bit_length()
        if self.n_items > self._rooms[0] or n_parts > self._rooms[1]:
            if self._buffer is not None:
                self._outgrown.append(self._buffer)
            self._rooms = (2 * self.n_items, 2 * n_parts)
            at = np.cumsum([ITEM_INTS * self._rooms[0], self.rows, self.rows + 1, self._rooms[1]])
            b = self._buffer = torch.zeros(at[3], dtype=torch.int32, device=self.device)
            self.items, self.order, self.part_start, self.parts = b[:at[0]], b[at[0]:at[1]], b[at[1]:at[2]], b[at[2]:]
            self.made += 1
            numbers = _planned(meta, self.group, self.nkv, self.dtype, _cut, self.GRID, self._rooms[0])[0]
        send_into(numbers, self._buffer[:len(numbers)])
        self._filled_for = filled_for


def _saved(meta, nkv, hd, dtype):
    return meta.shared.pages_saved * nkv * 64 * hd * 2 * (4 if dtype == torch.float32 else 2)


def pays(meta, kv, nq, nkv, hd, dtype, alone=False):
    """True where the shared attention takes this step over this cache and ends sooner than the attention that reads every sequence's pages
    by itself: by the bytes of keys and values that are not read again, or, where queries, keys and values are prepared by a kernel of their own
    in any case (alone), in steps of four to six pages."""
    return meta.shared is not None and supported(kv, nq, nkv, hd, dtype) and _ends_sooner(meta, nkv, hd, dtype, alone)


def _ends_sooner(meta, nkv, hd, dtype, alone=False):
    if meta.shared is None:
        return False
    if meta.max_new > 1 and meta.num_tokens > MANY_TOKENS[dtype] * meta.num_seqs:
        return False
    if dtype == torch.float32:          # (8 sequences of 128 tokens: 11 us shared, 17 separate; of 2,048: 17 and 103)
        return True
    if alone and hd <= ALONE_DIM and meta.num_seqs * nkv <= ALONE_PAIRS and _by_itself(meta, nkv, dtype):
        return int(meta.host_context.max()) > 64 * ALONE_PAGES
    return _saved(meta, nkv, hd, dtype) >= SAVED_BYTES + SAVED_BYTES_EACH * min(meta.num_seqs, SAVED_SEQUENCES)


def worth_over(needs, dtype, alone=()):
    """A function of a step's BatchMeta: of each kind of cache among `needs` (KVNeeds) whose pages may be read together, whether that pays.
    alone: (kv heads, head size) of those that are read where a kernel of its own prepares (see pays). A recorded step is tied to its
    answers: they are known before any layer has asked for a plan."""
    kinds = sorted({(n.kv_heads, n.head_dim) for n in needs if n.values and not n.window})
    kinds = [(*k, False) for k in kinds] + [(*k, True) for k in kinds if k in set(alone)]
    return lambda meta: tuple(_ends_sooner(meta, nkv, hd, dtype, by_itself) for nkv, hd, by_itself in kinds)


def _plan_of(meta, nq, nkv, hd, dtype, alone):
    key = ("shared_plan", nq // nkv, nkv, hd, dtype, alone)
    if meta.static is not None:
        found = meta.static.shared_plan(key, lambda rows, device: StaticPlan(nq // nkv, nkv, dtype, rows, device),
                                        lambda m: _ends_sooner(m, nkv, hd, dtype, alone))
        if found is None:
            raise BackendError("shared attention: it does not pay for this step (see pays)")
        return found
    found = meta.derived.get(key)          # every layer's attention asks: worked out once a step
    if found is None or found.sharing is not meta.shared:
        mfma._not_while_recording("the plan of a step's shared pages")
        found = meta.derived[key] = Plan(meta, nq // nkv, nkv, dtype)
    return found


def attention(q, meta, kv, out, nq, nkv, hd, scale, sinks=None, softcap=None, scratch=None, alone=False):
    """Causal attention of the step's tokens over their slots' pages, a page that several sequences share read once for all of
    them. q, out [T, nq hd] in the cache's dtype, bfloat16 (heads of 32, 64 or 128) or float32 (up to 256, a multiple of 4); meta.shared: a cache.SharedPages of
    the step's sequences. sinks f32 [nq]: the softmax's denominator of head h also holds exp(sinks[h]). softcap: a scaled score s
    becomes softcap tanh(s / softcap). scratch: a mfma.Scratch whose memory the partial results take, for one call (or recorded graph) at a
    time; None: memory of this call's own. alone: as it was told `pays`. meta is used on the stream that it was packed on."""
    T = q.shape[0]
    if meta.shared is None:
        raise BackendError("shared attention: the sequences of this step share no pages")
    if not supported(kv, nq, nkv, hd, q.dtype):
        raise BackendError(f"shared attention refuses {nq}/{nkv} heads of {hd} in {q.dtype} over this cache")
    keys, values, table = kv.k, kv.v, kv.page_table
    pages, dtype, i32 = keys.shape[0], keys.dtype, torch.int32
    further = () if sinks is None else (sinks, torch.float32, (nq,))
    ops._check_all("shared attention", OPERANDS, q, dtype, (T, nq * hd), out, dtype, (T, nq * hd), keys, None, (pages, nkv, 64, hd),
                   values, dtype, (pages, nkv, hd, 64), table, i32, (None, None), meta.positions, i32, (T,), meta.seq_of, i32, (T,),
                   meta.slots, i32, (meta.num_seqs,), *further)
    if meta.max_context > 64 * table.shape[1]:
        raise BackendError(f"shared attention: a context of {meta.max_context} tokens does not fit a table of {table.shape[1]} pages")
    p = _plan_of(meta, nq, nkv, hd, q.dtype, alone)
    if p.direct:
        po = pml = None
    elif scratch is None:
        po, pml = (torch.empty(p.n_parts * nq * n, dtype=torch.float32, device=q.device) for n in (hd, 2))
    else:
        po, pml = mfma._partial_buffers(scratch, q.device, p.n_parts * nq, 1, hd)
    lib.call("attention_shared", "hb_attn_shared", q, keys, values, out, ops.dtype_code(q), po, pml, p.items, p.n_items, p.max_rows,
             1 if meta.max_new > 1 else 0, 1 if p.direct else 0, p.order, p.part_start, p.parts, T, meta.positions, meta.seq_of, meta.slots, table, table.shape[1],
             nq, nkv, hd, float(scale), float(softcap or 0.0), sinks, _stream())
