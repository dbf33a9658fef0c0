"""The operators of one decode step and of scoring its answers, as measured cases.

Four operators: the root-mean-square norm with the residual's addition and an 8-bit output
("rmsnorm"), writing new keys and values into a paged 8-bit cache ("append"), attention over that
cache ("attention"), and the log probabilities of given tokens with entropy and the largest
alternatives ("logprobs") with their gradient ("logprobs_grad").

`run` computes an operator from elementary torch operations in 32 bits, or, where `own` is true,
by the call a user makes of `newt_b200.ops`.  `exact` computes the same in 64 bits, from the
definition.  Outputs held in 8 bits are returned as float8 tensors beside their scales; `exact`
gives for them the values before the rounding to 8 bits, as it does for the 16-bit ones.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one token of each of eight sequences between two layers: the call is all latency
        dict(name="rmsnorm 8x4096 bf16 row", op="rmsnorm", rows=8, n=4096, dtype="bf16",
             residual=True, out="e4m3", group=0),
        # a prompt's tokens, a scale for every 128 columns, one row short of a round number
        dict(name="rmsnorm 8191x4096 fp16 g128", op="rmsnorm", rows=8191, n=4096, dtype="fp16",
             residual=True, out="e4m3", group=128),
        # a decode step of 64 sequences: one new token each, somewhere in its page
        dict(name="append 64x1 d64 fp16", op="append", batch=64, most=1, start=4000, heads=8, d=64,
             page=16, dtype="fp16"),
        # four prompts of different lengths, two of them behind what the cache holds already
        dict(name="append 4x4001 d128 bf16", op="append", batch=4, most=4001, start=100, heads=8,
             d=128, page=64, dtype="bf16"),
        # one short conversation: latency again
        dict(name="attention 1x333 bf16", op="attention", batch=1, longest=333, ragged=False, nq=1,
             heads=32, kv_heads=8, d=128, page=64, window=0, sinks=0, dtype="bf16"),
        # one long document in small pages, multi-query heads: few rows, the long axis is split
        dict(name="attention 1x131001 bf16 p16", op="attention", batch=1, longest=131001,
             ragged=False, nq=1, heads=32, kv_heads=4, d=128, page=16, window=0, sinks=0,
             dtype="bf16"),
        # a full server: 64 sequences of different lengths
        dict(name="attention 64x8192 bf16", op="attention", batch=64, longest=8192, ragged=True,
             nq=1, heads=32, kv_heads=8, d=128, page=64, window=0, sinks=0, dtype="bf16"),
        # a window with its first tokens kept, four drafted tokens checked at once
        dict(name="attention 32x16384 w2048 fp16", op="attention", batch=32, longest=16384,
             ragged=True, nq=4, heads=16, kv_heads=8, d=64, page=32, window=2048, sinks=4,
             dtype="fp16"),
        # what a decode step answers with: the tokens taken, and twenty alternatives
        dict(name="logprobs 16x129001 fp32 top20", op="logprobs", rows=16, vocab=129001,
             dtype="fp32", top=20, inv_t=1.0),
        # scoring sampled answers for training: many rows, an odd vocabulary, no alternatives
        dict(name="logprobs 4096x50021 bf16", op="logprobs", rows=4096, vocab=50021, dtype="bf16",
             top=0, inv_t=1.25),
        # the gradient of that score, a short answer and a batch of them
        dict(name="logprobs_grad 65x32000 fp32", op="logprobs_grad", rows=65, vocab=32000,
             dtype="fp32", inv_t=1.0),
        dict(name="logprobs_grad 4096x50021 bf16", op="logprobs_grad", rows=4096, vocab=50021,
             dtype="bf16", inv_t=1.25),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rmsnorm", "append", "attention", "attention", "logprobs", "logprobs_grad"])
    if op == "rmsnorm":
        n = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            n = (n + 7) // 8 * 8
        rows = min(_log(rng, 1, 8192), (1 << 25) // n)
        return dict(op=op, rows=rows, n=n, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    residual=rng.random() < 0.7, out=rng.choice(["e4m3", "e4m3", "same"]),
                    group=rng.choice([0, 32, 64, 128]))
    if op == "append":
        batch = _log(rng, 1, 128)
        return dict(op=op, batch=batch, most=_log(rng, 1, max(2, 16000 // batch)),
                    start=_log(rng, 1, 4000), heads=rng.choice([1, 2, 4, 8]),
                    d=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "fp16"]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        group, nq = rng.choice([1, 2, 4, 7, 8]), rng.choice([1, 1, 1, 2, 3, 4, 8])
        most = (64 * 8192 * 8) // (batch * kv_heads * max(1, group * nq // 8))
        longest = min(_log(rng, 1, 131072), most)
        windowed = rng.random() < 0.5
        return dict(op=op, batch=batch, longest=longest, ragged=rng.random() < 0.7,
                    nq=min(longest, nq), heads=kv_heads * group, kv_heads=kv_heads,
                    d=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                    window=_log(rng, 1, max(2, longest)) if windowed else 0,
                    sinks=rng.choice([0, 1, 4, 130]) if windowed else 0,
                    dtype=rng.choice(["bf16", "fp16"]))
    vocab = _log(rng, 1000, 160000)
    rows = min(_log(rng, 1, 4096), 200_000_000 // vocab)
    case = dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                inv_t=rng.choice([1.0, 0.5, 1.25]))
    if case["dtype"] == "fp32":
        case["rows"] = max(1, rows // 2)
    if op == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, 32])
    return case


# ---- inputs ------------------------------------------------------------------------------------

def _spread(low, high, count):
    """`count` whole numbers from `high` down towards `low`, evenly."""
    return [high - (high - low) * i // count for i in range(count)]


def _lengths(case):
    """Tokens of each sequence in the cache, the new ones among them."""
    low = max(case["nq"], case["longest"] // 2) if case["ragged"] else case["longest"]
    return _spread(low, case["longest"], case["batch"])


def _new_tokens(case):
    """How many tokens each sequence brings to the cache."""
    return _spread(max(1, case["most"] // 2), case["most"], case["batch"])


def _paged(lengths, page, rng, total=None):
    """A table of pages, in no order, and how many pages there are; entries behind a sequence's
    last page are -1."""
    counts = [(n + page - 1) // page for n in lengths]
    total = total or sum(counts) + 3
    ids = rng.permutation(total)
    table = np.full((len(lengths), max(max(counts), 1)), -1, np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    return torch.from_numpy(table).to(DEVICE), total


def _cache(pages, heads, page, d, gen):
    """Pages as they are after use: values of about unit size over scales that differ by page."""
    k, v = ((torch.randn(pages, heads, page, d, generator=gen, device=DEVICE, dtype=torch.bfloat16)
             * 100).clamp_(-F8_MAX, F8_MAX).to(F8) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-8, -5, (pages, heads), generator=gen,
                                       device=DEVICE).float()) for _ in range(2))
    return k, v, ks, vs


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))
    op, dtype = case["op"], TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * scale).to(dtype)

    state = dict(case)
    if op == "rmsnorm":
        rows, n = case["rows"], case["n"]
        state["x"] = normal(rows, n)
        state["r"] = normal(rows, n, scale=3.0) if case["residual"] else None
        state["w"] = (1 + 0.1 * torch.randn(n, generator=gen, device=DEVICE)).to(dtype)
        return state
    if op == "append":
        batch, most = case["batch"], case["most"]
        new = rng.permutation(_new_tokens(case))
        start = rng.randint(0, case["start"] + 1, batch)
        start[rng.rand(batch) < 0.25] = 0
        room = batch * ((case["start"] + most + case["page"] - 1) // case["page"])
        state["table"], pages = _paged([int(a + b) for a, b in zip(start, new)], case["page"], rng,
                                       total=room)
        state["cache"] = _cache(pages, case["heads"], case["page"], case["d"], gen)
        state["starts"] = torch.from_numpy(start.astype(np.int32)).to(DEVICE)
        offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        state["offsets"] = torch.from_numpy(offsets).to(DEVICE)
        total = int(offsets[-1]) + 2            # two rows of padding behind the last sequence
        state["k"] = normal(total, case["heads"], case["d"], scale=1.5)
        state["v"] = normal(total, case["heads"], case["d"])
        return state
    if op == "attention":
        lengths = rng.permutation(_lengths(case)).tolist()
        state["table"], pages = _paged(lengths, case["page"], rng)
        state["cache"] = _cache(pages, case["kv_heads"], case["page"], case["d"], gen)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        state["q"] = normal(case["batch"], case["nq"], case["heads"], case["d"], scale=2.0)
        return state
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device=DEVICE).mul_(2.5).to(dtype)
    x[:, vocab - vocab // 400:] = float("-inf")   # columns that only pad the vocabulary
    state["x"] = x
    tokens = torch.randint(0, vocab - vocab // 400, (rows,), generator=gen, device=DEVICE)
    if op == "logprobs_grad" or case["top"] == 0:   # training: a prompt's tokens have no score
        tokens[torch.rand(rows, generator=gen, device=DEVICE) < 0.1] = -100
    state["tokens"] = tokens
    if op == "logprobs_grad":
        z = x.float() * case["inv_t"]
        lse = torch.logsumexp(z, 1)
        p = torch.exp(z - lse[:, None])
        state["lse"] = lse
        state["entropy"] = lse - (p * z.clamp(min=-1e30)).sum(1)
        state["g"] = normal(rows, dtype=torch.float32)
        state["g_entropy"] = normal(rows, scale=0.01, dtype=torch.float32)
    return state


# ---- one pass ----------------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"rmsnorm": _rmsnorm, "append": _append, "attention": _attention, "logprobs": _logprobs,
            "logprobs_grad": _logprobs_grad}[state["op"]](state)


def _own(state):
    from newt_b200 import ops

    op = state["op"]
    if op == "rmsnorm":
        out, scales, h = ops.rmsnorm(state["x"], state["w"], residual=state["r"], eps=EPS,
                                     out_dtype=F8 if state["out"] == "e4m3" else None,
                                     group=state["group"] if state["out"] == "e4m3" else 0)
        return {"out": out, "scales": scales, "residual": h}
    if op == "append":
        cache = ops.KVCache(*state["cache"])
        ops.kv_append(cache, state["k"], state["v"], state["table"], state["starts"],
                      state["offsets"], state["most"])
        return list(cache)
    if op == "attention":
        return ops.kv_attention(state["q"], ops.KVCache(*state["cache"]), state["table"],
                                state["lengths"], window=state["window"], sinks=state["sinks"])
    if op == "logprobs":
        got = ops.token_logprobs(state["x"], state["tokens"], top=state["top"],
                                 inv_temperature=state["inv_t"])
        return {"logprob": got.logprob, "entropy": got.entropy, "lse": got.lse,
                "top": got.top_logprob, "index": got.top_index}
    return ops.token_logprobs_backward(state["x"], state["tokens"], state["lse"], state["entropy"],
                                       state["g"], state["g_entropy"],
                                       inv_temperature=state["inv_t"])


def _rmsnorm(state):
    x, n = state["x"], state["n"]
    h = x.float()
    if state["r"] is not None:
        h = h + state["r"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * state["w"].float()
    residual = h.to(x.dtype) if state["r"] is not None else None
    if state["out"] != "e4m3":
        return {"out": y.to(x.dtype), "scales": None, "residual": residual}
    group = state["group"] or n
    groups = (n + group - 1) // group
    wide = torch.zeros(x.shape[0], groups * group, device=x.device)
    wide[:, :n] = y
    wide = wide.view(-1, groups, group)
    amax = wide.abs().amax(2)
    scales = torch.where(amax > 0, amax / F8_MAX, 1.0)
    q = (wide / scales[:, :, None]).clamp(-F8_MAX, F8_MAX).view(-1, groups * group)[:, :n].to(F8)
    return {"out": q, "scales": scales, "residual": residual}


def _power(amax):
    """The smallest power of two s, 2^-60 <= s <= 2^60, with amax <= 448 s."""
    m, e = torch.frexp(amax.float())              # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-60, 60)
    return torch.exp2(torch.where(amax > 0, e, torch.full_like(e, -60)).float())


def _append(state):
    table, starts, offsets = state["table"].long(), state["starts"].long(), state["offsets"].long()
    k_cache, v_cache, k_scales, v_scales = state["cache"]
    page, pages = state["page"], k_cache.shape[0]
    new = offsets[1:] - offsets[:-1]
    slots = torch.arange((state["most"] + page - 2) // page + 1, device=table.device)
    at = (starts // page)[:, None] + slots                        # which page of the sequence
    inside = at * page < (starts + new)[:, None]
    ids = torch.where(inside, table.gather(1, at.clamp(max=table.shape[1] - 1)), -1)
    position = at[:, :, None] * page + torch.arange(page, device=table.device)
    row = position - starts[:, None, None]                        # of the new tokens; < 0: old
    is_new = (row >= 0) & (row < new[:, None, None]) & (ids >= 0)[:, :, None]
    is_old = (row < 0) & (ids >= 0)[:, :, None]
    source = (row + offsets[:-1, None, None]).clamp(0, state["k"].shape[0] - 1)
    begins = (at * page >= starts[:, None])[:, :, None]
    safe = ids.clamp(0, pages - 1)
    used = ids.flatten() >= 0
    for x, cache, scales in ((state["k"], k_cache, k_scales), (state["v"], v_cache, v_scales)):
        fresh = x[source].float()                                 # [batch, slot, token, head, d]
        there = cache.view(torch.uint8)[safe].view(F8).float().transpose(2, 3)
        before = scales[safe]
        need = _power((fresh.abs() * is_new[..., None, None]).amax((2, 4)))
        after = torch.where(begins, need, torch.maximum(before, need))
        shrunk = there * (before / after)[:, :, None, :, None]
        value = torch.where(is_new[..., None, None], fresh / after[:, :, None, :, None], shrunk)
        value = value.clamp(-F8_MAX, F8_MAX).to(F8).view(torch.uint8)
        kept = cache.view(torch.uint8)[safe].transpose(2, 3)
        value = torch.where((is_new | is_old)[..., None, None], value, kept).transpose(2, 3)
        cache.view(torch.uint8)[ids.flatten()[used]] = value.flatten(0, 1)[used]
        scales[ids.flatten()[used]] = after.flatten(0, 1)[used]
    return list(state["cache"])


def _visible(lengths, nq, longest, window, sinks):
    """[batch, nq, longest]: which tokens of the cache a query token sees."""
    j = torch.arange(longest, device=lengths.device)
    at = lengths[:, None] - nq + torch.arange(nq, device=lengths.device)
    seen = j <= at[:, :, None]
    if window:
        seen = seen & ((j > at[:, :, None] - window) | (j < sinks))
    return seen


def _attention(state):
    q, table = state["q"], state["table"].long()
    k_cache, v_cache, k_scales, v_scales = state["cache"]
    batch, nq, heads, d = q.shape
    kv_heads, page = k_cache.shape[1], k_cache.shape[2]
    longest = table.shape[1] * page
    safe = table.clamp(min=0)

    def tokens(cache, scales):                                    # [batch, kv_heads, longest, d]
        got = cache.view(torch.uint8)[safe].view(F8).float() * scales[safe][..., None, None]
        return got.transpose(1, 2).reshape(batch, kv_heads, longest, d)

    qs = q.float().view(batch, nq, kv_heads, -1, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = (qs @ tokens(k_cache, k_scales).transpose(2, 3)) / math.sqrt(d)
    seen = _visible(state["lengths"].long(), nq, longest, state["window"], state["sinks"])
    seen = seen[:, None, :, None, :].expand(-1, kv_heads, -1, heads // kv_heads, -1).flatten(2, 3)
    s = torch.where(seen, s, -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(3, keepdim=True)
    o = (e @ tokens(v_cache, v_scales)) / torch.where(total > 0, total, 1.0)
    o = o.view(batch, kv_heads, nq, -1, d).permute(0, 2, 1, 3, 4).reshape(batch, nq, heads, d)
    return o.to(q.dtype)


def _logprobs(state):
    x, tokens, top, vocab = state["x"], state["tokens"], state["top"], state["vocab"]
    z = x.float() * state["inv_t"]
    most = z.amax(1, keepdim=True)
    shifted = z - most
    e = torch.exp(shifted)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (e * shifted.clamp(min=-1e30)).sum(1) / total
    lse = most[:, 0] + log_total
    given = shifted.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0] - log_total
    logprob = torch.where(tokens < 0, 0.0, given)
    if top == 0:
        return {"logprob": logprob, "entropy": entropy, "lse": lse, "top": None, "index": None}
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    return {"logprob": logprob, "entropy": entropy, "lse": lse,
            "top": shifted.gather(1, order) - log_total[:, None], "index": order}


def _logprobs_grad(state):
    x, tokens = state["x"], state["tokens"]
    log_p = x.float() * state["inv_t"] - state["lse"][:, None]
    p = torch.exp(log_p)
    g = torch.where(tokens < 0, 0.0, state["g"])
    dx = -p * (g[:, None] + state["g_entropy"][:, None]
               * (log_p.clamp(min=-1e30) + state["entropy"][:, None]))
    dx.scatter_add_(1, tokens.clamp(min=0)[:, None], g[:, None])
    return (dx * state["inv_t"]).to(x.dtype)


# ---- the work of a pass ------------------------------------------------------------------------

def _seen_tokens(case, lengths):
    """How many tokens of the cache the query tokens of each sequence see together."""
    seen = []
    for n in lengths:
        first = max(n - case["nq"] - case["window"] + 1, 0) if case["window"] else 0
        seen.append(n - first + min(case["sinks"], first))
    return seen


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op == "rmsnorm":
        n = case["rows"] * case["n"]
        out = 1 if case["out"] == "e4m3" else size
        moved = n * (size + out + (2 * size if case["residual"] else 0)) + case["n"] * size
        return {"bytes": moved, "flops": 6 * n}
    if op == "append":
        n = 2 * sum(_new_tokens(case)) * case["heads"] * case["d"]
        return {"bytes": n * (size + 1), "flops": 3 * n}
    if op == "attention":
        seen = sum(_seen_tokens(case, _lengths(case)))
        rows = case["nq"] * case["heads"]
        return {"bytes": 2 * seen * case["kv_heads"] * case["d"]
                + 2 * size * case["batch"] * rows * case["d"],
                "flops": 4 * seen * rows * case["d"]}
    n = case["rows"] * case["vocab"]
    if op == "logprobs":
        return {"bytes": n * size + case["rows"] * (20 + 12 * case["top"]), "flops": 5 * n}
    return {"bytes": 2 * n * size + case["rows"] * 24, "flops": 6 * n}


# ---- 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "rmsnorm":
        total = state["x"].double()
        if state["r"] is not None:
            total = total + state["r"].double()
        root = ((total ** 2).sum(1) / case["n"] + EPS).sqrt()
        y = state["w"].double() * (total / root[:, None])
        kept = total if state["r"] is not None else None
        if case["out"] != "e4m3":
            return {"out": y, "scales": None, "residual": kept}
        scales = []
        for part in y.split(case["group"] or case["n"], 1):
            most = part.abs().max(1)[0]
            scales.append(torch.where(most > 0, most / F8_MAX, torch.ones_like(most)))
        scales = torch.stack(scales, 1)
        width = case["group"] or case["n"]
        return {"out": y / scales.repeat_interleave(width, 1)[:, :case["n"]], "scales": scales,
                "residual": kept}
    if op == "append":
        return _exact_append(case, state)
    if op == "attention":
        return _exact_attention(case, state)
    z = state["x"].double() * case["inv_t"]
    lse = torch.logsumexp(z, 1)
    log_p = z - lse[:, None]
    p = log_p.exp()
    tokens = state["tokens"]
    scored = tokens >= 0
    if op == "logprobs":
        entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)
        own_log = torch.where(scored, log_p[torch.arange(len(tokens), device=p.device),
                                            tokens.clamp(min=0)], torch.zeros_like(lse))
        top = index = None
        if case["top"]:
            # the largest k, ties to the lowest index
            rank = torch.argsort(state["x"].double(), dim=1, descending=True, stable=True)
            index = rank[:, :case["top"]]
            top = log_p.gather(1, index)
        return {"logprob": own_log, "entropy": entropy, "lse": lse, "top": top, "index": index}
    hit = torch.zeros_like(p)
    hit[scored, tokens[scored]] = 1.0
    d_log = torch.where(scored, state["g"].double(), torch.zeros_like(lse))[:, None]
    d_entropy = state["g_entropy"].double()[:, None]
    surprise = torch.where(p > 0, log_p, torch.zeros_like(p)) + state["entropy"].double()[:, None]
    return case["inv_t"] * (d_log * (hit - p) - d_entropy * p * surprise)


def _exact_append(case, state):
    page = case["page"]
    table, starts, offsets = (state[key].cpu().numpy() for key in ("table", "starts", "offsets"))
    got = []
    for x, cache, scales in ((state["k"], state["cache"][0], state["cache"][2]),
                             (state["v"], state["cache"][1], state["cache"][3])):
        x = x.double().cpu()
        cache, scales = cache.cpu().to(torch.float64), scales.double().cpu()
        for b in range(case["batch"]):
            begin, end = int(starts[b]), int(starts[b]) + int(offsets[b + 1] - offsets[b])
            for slot in range(begin // page, (end + page - 1) // page):
                low, high = max(begin, slot * page), min(end, (slot + 1) * page)
                where, first = int(table[b, slot]), low - slot * page
                rows = x[offsets[b] + low - begin:offsets[b] + high - begin].transpose(0, 1)
                most = rows.abs().amax((1, 2))
                need = torch.exp2(torch.log2(most.clamp(min=1e-30) / F8_MAX).ceil()
                                  .clamp(-60, 60))
                if first > 0:
                    before = scales[where]
                    need = torch.maximum(need, before)
                    cache[where, :, :first] *= (before / need)[:, None, None]
                cache[where, :, first:first + high - low] = rows / need[:, None, None]
                scales[where] = need
        got.append((cache, scales))
    return [got[0][0], got[1][0], got[0][1], got[1][1]]


def _exact_attention(case, state):
    q = state["q"].double()
    batch, nq, heads, d = q.shape
    out = torch.zeros_like(q)
    group = heads // case["kv_heads"]
    table, lengths = state["table"].long(), state["lengths"].tolist()
    for b, length in enumerate(lengths):
        ids = table[b, :(length + case["page"] - 1) // case["page"]]
        kv = []
        for cache, scales in ((state["cache"][0], state["cache"][2]),
                              (state["cache"][1], state["cache"][3])):
            part = cache.view(torch.uint8)[ids].view(F8).to(torch.float64)
            part = part * scales[ids].double()[:, :, None, None]
            part = part.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, d)[:, :length]
            kv.append(part.repeat_interleave(group, 0))
        for i in range(nq):
            at = length - nq + i
            j = torch.arange(length, device=q.device)
            hidden = j > at
            if case["window"]:
                hidden |= (j <= at - case["window"]) & (j >= case["sinks"])
            score = torch.einsum("hd,hjd->hj", q[b, i], kv[0]) * d ** -0.5
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), 1)
            if at >= 0:
                out[b, i] = torch.einsum("hj,hjd->hd", weight, kv[1])
    return out
