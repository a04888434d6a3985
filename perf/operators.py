"""Two operators for many answers to one prompt, and what they are timed on.

  attention  the attention of a step whose sequences share the beginning of their contexts (samples of one
             prompt, answers that are scored, questions behind one document): the pages that several sequences
             hold together are read once for all of them. Queries [tokens, heads x dim], a paged cache (keys
             [pages, kv heads, 64, dim], values [pages, kv heads, dim, 64]) whose page table names a shared page in
             every row that holds it. Token t of a sequence at position p sees the keys 0 .. p of its own context:
               s_j = q . k_j / sqrt(dim)  (softcap: s_j = cap tanh(s_j / cap)),
               out = sum_j e^(s_j) v_j / (sum_j e^(s_j) + e^(sink of the head, if it has one))
  logprobs   what a step's logits say of given tokens: a row's
               log p(token) = x_token - log sum e^x,  entropy = log sum e^x - sum p x,
             and its `top` largest entries, largest first, the lower id first among equals, with their log p

With `own` false both are elementary torch operations in float32, a sequence after another.
"""
import math

import torch

own = False

PAGE = 64


# ---------------------------------------------------------------- the cases
def attention(name, batch, heads, kv_heads, dim, prompt, own_tokens, branches=1, branch=0, spread=0.0, new=1, sinks=False,
              softcap=0.0, dtype="bfloat16"):
    """`batch` sequences that share the first `prompt` tokens, in `branches` equal parts each of which shares `branch`
    tokens more; `own_tokens` of a sequence's own at most (down to 1 - spread of that), the last `new` of which are this
    step's (as many at most, likewise)."""
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "prompt": prompt,
            "own": own_tokens, "branches": branches, "branch": branch, "spread": spread, "new": new, "sinks": sinks,
            "softcap": softcap, "dtype": dtype}


def logprobs(name, rows, vocab, top, banned=0.0, steps=0):
    """`banned`: the share of the vocabulary at -inf in every second row. `steps` > 0: logits are whole multiples of
    1 / steps, so that many are equal."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "banned": banned, "steps": steps}


def listed():
    return [
        # two answers to a short prompt on a small model: nothing but latency
        attention("two_answers_small", 2, 8, 4, 128, 200, 30),
        # eight samples of one prompt in the middle of their generation, heads of the 8B shape
        attention("samples_8b_batch8", 8, 32, 8, 128, 4096, 300, spread=0.3),
        # 64 samples of a long prompt, as a vote over many answers draws them
        attention("samples_8b_batch64", 64, 32, 8, 128, 8192, 512, spread=0.9),
        # 128 short answers to questions about one long document: the largest
        attention("document_8b_batch128", 128, 32, 8, 128, 32768, 160, spread=0.6),
        # six questions behind one system prompt, eight samples each, heads of the 1.7B shape
        attention("questions_1.7b", 48, 16, 8, 128, 1024, 333, branches=6, branch=700, spread=0.5),
        # given continuations of unequal lengths that are scored in one step
        attention("continuations_8b", 24, 32, 8, 128, 2000, 40, spread=0.9, new=40),
        # the all-float32 mode: five samples, heads with sinks
        attention("float32_samples", 5, 16, 8, 128, 1500, 77, spread=0.5, sinks=True, dtype="float32"),
        # one greedy sequence's newest token with five alternatives
        logprobs("one_row", 1, 151936, 5),
        # the newest tokens of a batch of samples
        logprobs("samples_64", 64, 151936, 20),
        # the same where a grammar bans most of the vocabulary, and where logits are coarse and often equal
        logprobs("banned_and_equal", 37, 32771, 8, banned=0.95, steps=16),
        # every position of a long text that is scored
        logprobs("scored_text", 2048, 151936, 0),
    ]


def draw(rng):
    """Either operator over its whole range; no case costs more than the largest listed one."""
    def spread_over(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    if rng.random() < 0.4:
        vocab = spread_over(300, 160000)
        top = rng.choice((0, 1, 2, 5, 10, 20, 33, 64))
        rows = spread_over(1, max(2, min(2048, (40 if top else 300) * 1000000 // vocab)))
        return {"op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "banned": rng.choice((0.0, 0.0, 0.5, 0.9)),
                "steps": rng.choice((0, 0, 8, 64))}
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 5, 8))
    branches = rng.choice((1, 1, 1, 2, 3, 5))
    batch = branches * max(2, spread_over(2, (160 if dtype == "bfloat16" else 24)) // branches)
    new = rng.choice((1, 1, 1, 1, 7, 30))
    prompt = rng.choice((0, 1, 1, 1)) * spread_over(64, 30000 if dtype == "bfloat16" else 3000) if branches > 1 else \
        spread_over(64, 30000 if dtype == "bfloat16" else 3000)
    branch = spread_over(64, 2000) if branches > 1 else 0
    own_tokens = new + spread_over(1, 1200)
    while batch * new * (prompt + branch + own_tokens) * heads > 128 * 32928 * 32 and batch > 2 * branches:
        batch -= branches
    prompt = min(prompt, 128 * 32928 * 32 // (batch * new * heads))
    return {"op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128)),
            "prompt": prompt, "own": own_tokens, "branches": branches, "branch": branch, "spread": rng.choice((0.0, 0.3, 0.9)),
            "new": new, "sinks": rng.random() < 0.25, "softcap": rng.choice((0.0, 0.0, 0.0, 30.0)), "dtype": dtype}


def down_from(most, spread, i):
    """A number from `most` down to (1 - spread) of it, at least one: the i-th of a fixed sequence without a pattern."""
    return max(1, int(round(most * (1.0 - spread * ((i * 0.6180339887) % 1.0)))))


def lengths(c):
    """Of every sequence: (pages it shares with all, pages it shares with its branch, positions it holds after the step,
    new tokens). A prompt that ends within a page shares its whole pages, the rest is copied to every sequence."""
    common = c["prompt"] // PAGE
    upto = (c["prompt"] + c["branch"]) // PAGE if c["branches"] > 1 else common
    at_least = c["prompt"] + (c["branch"] if c["branches"] > 1 else 0)
    out = []
    for i in range(c["batch"]):
        new = down_from(c["new"], c["spread"], i + 1)
        out.append((common, upto, at_least + max(new, down_from(c["own"], c["spread"], i)), new))
    return out


def page_rows(c):
    """The logical pages of the sequences, [[page, ...], ...], numbered from 0 without gaps, and how many there are."""
    rows, count, shared = [], 0, {}
    for i, (common, upto, held, _) in enumerate(lengths(c)):
        part = i * c["branches"] // c["batch"]
        row = []
        for p in range(-(-held // PAGE)):
            key = ("all", p) if p < common else (part, p) if p < upto else None
            if key is None or key not in shared:
                if key is not None:
                    shared[key] = count
                row.append(count)
                count += 1
            else:
                row.append(shared[key])
        rows.append(row)
    return rows, count


# ---------------------------------------------------------------- inputs
def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 31) + 17)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return prepare_attention(c, gen, rand) if c["op"] == "attention" else prepare_logprobs(c, gen, rand)


def prepare_attention(c, gen, rand):
    dtype = torch.float32 if c["dtype"] == "float32" else torch.bfloat16
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    rows, count = page_rows(c)
    place = torch.randperm(count, generator=gen, device="cuda").cpu()        # pages lie anywhere in the pool
    table = torch.zeros((len(rows), max(len(r) for r in rows)), dtype=torch.int32)
    for i, row in enumerate(rows):
        table[i, :len(row)] = place[torch.tensor(row)].to(torch.int32)
    news = [n for _, _, _, n in lengths(c)]
    state = {"case": c, "held": [h for _, _, h, _ in lengths(c)], "news": news, "table": table.cuda(),
             # normed and rotated keys and queries have entries around one; a trained head's scores spread wider than 1
             "q": (rand(sum(news), H * D) * 2.0).to(dtype), "k": rand(count, G, PAGE, D).to(dtype),
             "v": rand(count, G, D, PAGE).to(dtype), "sinks": rand(H) * 2.0 if c["sinks"] else None}
    if own:
        # what a program has beside its cache: the step's metadata, made once for all layers, and memory that it keeps
        from herbert_rs_amd.cache import LayerKV, shared_pages
        from herbert_rs_amd.engine import StepEntry, batch
        from herbert_rs_amd.kernels import mfma
        before = [h - n for h, n in zip(state["held"], news)]
        entries = [StepEntry(i, [0] * n, [n - 1]) for i, n in enumerate(news)]
        meta = batch.pack(entries, before, state["table"].device)
        meta.shared = shared_pages(table.numpy(), before)
        state.update(meta=meta, kv=LayerKV(state["k"], state["v"], state["table"], PAGE, 0), scratch=mfma.Scratch(),
                     out=torch.empty_like(state["q"]))
    return state


def prepare_logprobs(c, gen, rand):
    R, V = c["rows"], c["vocab"]
    logits = rand(R, V) * 2.5
    if c["steps"]:
        logits = torch.round(logits * c["steps"]) / c["steps"]
    if c["banned"]:
        banned = torch.rand((R, V), generator=gen, device="cuda") < c["banned"]
        banned[::2] = False
        logits.masked_fill_(banned, -math.inf)
        del banned
    # tokens drawn by the logits' own distribution, as sampling draws them
    noise = torch.rand((R, V), generator=gen, device="cuda").clamp_(1e-12).log_().neg_().log_().neg_()
    tokens = (logits + noise).argmax(-1).to(torch.int32)
    del noise
    state = {"case": c, "logits": logits, "tokens": tokens}
    if own:
        from herbert_rs_amd.kernels import ops
        top, dev = c["top"], logits.device
        state.update(scratch=ops.logprob_scratch(R, V, top, dev), chosen=torch.empty(R, dtype=torch.float32, device=dev),
                     entropy=torch.empty(R, dtype=torch.float32, device=dev))
        if top:
            state.update(ids=torch.empty((R, top), dtype=torch.int32, device=dev),
                         best=torch.empty((R, top), dtype=torch.float32, device=dev))
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if not own:
        return plain_attention(state) if c["op"] == "attention" else plain_logprobs(state)
    if c["op"] == "attention":
        from herbert_rs_amd.kernels import shared
        shared.attention(state["q"], state["meta"], state["kv"], state["out"], c["heads"], c["kv_heads"], c["dim"],
                         c["dim"] ** -0.5, sinks=state["sinks"], softcap=c["softcap"] or None, scratch=state["scratch"])
        return state["out"]
    from herbert_rs_amd.kernels import ops
    ops.token_logprobs(state["logits"], state["tokens"], state["chosen"], state["entropy"], state.get("ids"), state.get("best"),
                       scratch=state["scratch"])
    return tuple(state[k] for k in ("chosen", "entropy", "ids", "best") if k in state)


def plain_attention(state):
    c = state["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    outs, row = [], 0
    for i, (held, new) in enumerate(zip(state["held"], state["news"])):
        pages = state["table"][i, :-(-held // PAGE)].long()
        k = state["k"][pages].float().permute(1, 0, 2, 3).reshape(G, -1, D)[:, :held]
        v = state["v"][pages].float().permute(1, 0, 3, 2).reshape(G, -1, D)[:, :held]
        q = state["q"][row:row + new].float().view(new, G, H // G, D).permute(1, 0, 2, 3).reshape(G, -1, D)
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) * D ** -0.5
        if c["softcap"]:
            s = torch.tanh(s / c["softcap"]) * c["softcap"]
        if new > 1:
            behind = torch.arange(held, device=s.device) > torch.arange(held - new, held, device=s.device)[:, None]
            s = s.masked_fill(behind.repeat_interleave(H // G, 0), -math.inf)
        top = s.amax(-1, keepdim=True)
        sink = None
        if state["sinks"] is not None:
            sink = state["sinks"].view(G, 1, H // G).expand(G, new, H // G).reshape(G, -1, 1)
            top = torch.maximum(top, sink)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        if sink is not None:
            total = total + torch.exp(sink - top)
        o = torch.matmul(e, v) / total
        outs.append(o.view(G, new, H // G, D).permute(1, 0, 2, 3).reshape(new, H * D))
        row += new
    return torch.cat(outs).to(state["q"].dtype)


def plain_logprobs(state):
    x, top = state["logits"], state["case"]["top"]
    shifted = x - x.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    chosen = shifted.gather(1, state["tokens"].long()[:, None]) - log_total
    entropy = log_total - torch.where(e > 0, e * shifted, torch.zeros_like(e)).sum(-1, keepdim=True) / total
    if not top:
        return chosen[:, 0], entropy[:, 0]
    values, ids = torch.sort(shifted, dim=-1, descending=True, stable=True)
    return chosen[:, 0], entropy[:, 0], ids[:, :top].to(torch.int32), (values[:, :top] - log_total).contiguous()


# ---------------------------------------------------------------- what a pass cannot do without
def work(c):
    if c["op"] == "logprobs":
        R, V = c["rows"], c["vocab"]
        # a difference, an exponential, a product and two sums an entry
        return {"bytes": R * (4 * V + 12 + 8 * c["top"]), "flops": 5 * R * V}
    size = 4 if c["dtype"] == "float32" else 2
    per = lengths(c)
    # every position that is held by somebody: shared pages whole and once, a sequence's own up to its end
    kept = per[0][0] * PAGE + c["branches"] * (per[0][1] - per[0][0]) * PAGE + sum(h - u * PAGE for _, u, h, _ in per)
    tokens = sum(n for _, _, _, n in per)
    seen = sum(n * (h - n) + n * (n + 1) // 2 for _, _, h, n in per)
    return {"bytes": size * (2 * kept * c["kv_heads"] * c["dim"] + 2 * tokens * c["heads"] * c["dim"]),
            "flops": 4 * seen * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- in 64 bits
def exact(c, seed):
    state = prepare(c, seed)
    return exact_attention(c, state) if c["op"] == "attention" else exact_logprobs(c, state)


def exact_attention(c, state):
    """By kv heads, every token by itself over its sequence's keys, softmax by the definition."""
    H, G, D, group = c["heads"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    q = state["q"].double().view(-1, H, D)
    out = torch.empty_like(q)
    for g in range(G):
        keys = state["k"][:, g].double()                        # [pages, 64, D]
        values = state["v"][:, g].double().transpose(1, 2).contiguous()
        row = 0
        for i, (held, new) in enumerate(zip(state["held"], state["news"])):
            pages = state["table"][i, :-(-held // PAGE)].long()
            k, v = keys[pages].flatten(0, 1), values[pages].flatten(0, 1)
            for t in range(new):
                n = held - new + t + 1
                mine = q[row + t, g * group:(g + 1) * group]
                scores = (k[:n] @ mine.t().contiguous()).t() / math.sqrt(D)
                if c["softcap"]:
                    scores = c["softcap"] * torch.tanh(scores / c["softcap"])
                if state["sinks"] is not None:
                    scores = torch.cat([scores, state["sinks"][g * group:(g + 1) * group].double()[:, None]], 1)
                weights = torch.softmax(scores, -1)[:, :n].contiguous()
                out[row + t, g * group:(g + 1) * group] = weights @ v[:n]
            row += new
    return out.view(-1, H * D)


def exact_logprobs(c, state):
    chosen, entropy, ids, best = [], [], [], []
    for r in range(0, c["rows"], 64):                           # a few rows at a time
        x = state["logits"][r:r + 64].double()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        chosen.append(logp.gather(1, state["tokens"][r:r + 64].long()[:, None])[:, 0])
        p = torch.exp(logp)
        entropy.append(-torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1))
        if c["top"]:
            at = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :c["top"]]
            ids.append(at.to(torch.int32))
            best.append(logp.gather(1, at))
    if not c["top"]:
        return torch.cat(chosen), torch.cat(entropy)
    return torch.cat(chosen), torch.cat(entropy), torch.cat(ids), torch.cat(best)
