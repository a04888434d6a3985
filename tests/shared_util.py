"""Steps whose sequences share pages, for the tests of the shared attention: page tables, inputs and the formula in 64 bits."""
import numpy as np
import torch

from herbert_rs_amd.cache import LayerKV, shared_pages
from herbert_rs_amd.engine import StepEntry, batch

PAGE = 64


def tables(sequences, seed, spare=3):
    """sequences: for each a list of (name, pages) stretches in order, a stretch of one name being the same pages wherever it is
    named (None: the sequence's own). Returns the page table [sequences, most pages] and how many pages there are; page
    numbers lie anywhere, and places that are not held name page 0."""
    known, count, rows = {}, 0, []
    for stretches in sequences:
        row = []
        for name, pages in stretches:
            for p in range(pages):
                key = None if name is None else (name, p)
                if key is None or key not in known:
                    if key is not None:
                        known[key] = count
                    row.append(count)
                    count += 1
                else:
                    row.append(known[key])
        rows.append(row)
    place = np.random.default_rng(seed).permutation(count + spare)
    table = np.zeros((len(rows), max(map(len, rows))), dtype=np.int32)
    for i, row in enumerate(rows):
        table[i, :len(row)] = place[row]
    return table, count + spare


def step(table, held, news, device):
    """The metadata of a step in which sequence i brings news[i] tokens behind held[i] positions."""
    meta = batch.pack([StepEntry(i, [0] * n, [n - 1]) for i, n in enumerate(news)], list(held), device)
    meta.shared = shared_pages(table, held)
    return meta


def inputs(table, pages, tokens, nq, nkv, hd, dtype, seed, device, q_scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    k = torch.randn((pages, nkv, PAGE, hd), generator=gen).to(dtype)
    v = torch.randn((pages, nkv, hd, PAGE), generator=gen).to(dtype)
    q = (torch.randn((tokens, nq * hd), generator=gen) * q_scale).to(dtype)
    kv = LayerKV(k.to(device), v.to(device), torch.from_numpy(table).to(device), PAGE, 0)
    return q.to(device), kv


def reference(q, kv, table, held, news, nq, nkv, hd, scale, sinks=None, softcap=None):
    """(out, weight): the formula in 64 bits on the CPU, [tokens, nq, hd]; weight = sum p |v| / denominator, what errors are
    measured against, and the largest sum of |q k| scale of a token and head [tokens, nq]."""
    k, v, q = kv.k.cpu().double(), kv.v.cpu().double(), q.cpu().double().view(-1, nq, hd)
    out, weight = torch.empty_like(q), torch.empty_like(q)
    size = torch.empty(q.shape[:2], dtype=torch.float64)
    row, group = 0, nq // nkv
    for i, (before, n) in enumerate(zip(held, news)):
        pages = torch.from_numpy(table[i, :-(-(before + n) // PAGE)].astype(np.int64))
        keys = k[pages].permute(1, 0, 2, 3).reshape(nkv, -1, hd)
        values = v[pages].permute(1, 0, 3, 2).reshape(nkv, -1, hd)
        for t in range(n):
            seen = before + t + 1
            for h in range(nq):
                kk, vv = keys[h // group, :seen], values[h // group, :seen]
                s = (kk @ q[row + t, h]) * scale
                size[row + t, h] = (kk.abs() @ q[row + t, h].abs()).max() * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if sinks is not None:
                    s = torch.cat([s, sinks[h].cpu().double()[None]])
                p = torch.softmax(s, 0)[:seen]
                out[row + t, h] = p @ vv
                weight[row + t, h] = p @ vv.abs()
        row += n
    return out, weight, size


def bound(out, weight, size, dtype, hd, keys):
    """How far a result may be off. bfloat16: every weight is rounded before its product (half a step, 2^-8 of it) and the
    output once more; scores, exponentials and sums in float32 are 1e-4 of the weights at most (a score of 50 is off by 50 x 2^-24 in
    an exponent, sums of 128 products by 128 x 2^-24 of their size). float32: a score is a chain of hd sums (hd x 2^-24 of the sum of its
    products' sizes, which its weight is off by), as many sums of weights as there are keys, a few roundings more."""
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * (weight + out.abs()) * (1 + 2.0 ** -7) + 1e-4 * weight + 1e-30
    return 2.0 ** -24 * (2 * (hd + 8) * size[..., None] + 2 * keys + 64) * weight + 1e-30
