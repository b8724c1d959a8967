"""Measured cases of the serving attentions: sliding window with sinks, and a batch that shares a prefix.

``run`` computes a case in plain torch operations (32 bits) or, with ``own`` set, through the framework's operators;
``exact`` computes it in 64 bits from the definition.  Queries are ``[B, Hq, Sq, D]``, caches ``[B, Hkv, Skv, D]``
(shared prefix ``[Hkv, P, D]``); query i of sequence b stands at position ``len_b - Sq + i`` of its own keys.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _window(name, batch, heads, kv_heads, queries, cache, dim, window, sinks, dtype, slack, token_major):
    return {"name": name, "op": "window", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries, "cache": cache, "prefix": 0,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "slack": slack, "token_major": token_major}


def _prefix(name, batch, heads, kv_heads, queries, cache, prefix, dim, dtype, slack, token_major):
    return {"name": name, "op": "prefix", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries, "cache": cache, "prefix": prefix,
            "dim": dim, "window": 0, "sinks": 0, "dtype": dtype, "slack": slack, "token_major": token_major}


def listed():
    return [
        # one user, one token at a time: the latency of a decode step
        _window("window decode, 1 sequence", 1, 32, 8, 1, 8192, 128, 2048, 4, "bf16", 0, False),
        # a server's decode step: many sequences, each at another length of its cache
        _window("window decode, 64 sequences", 64, 32, 8, 1, 4096, 128, 2048, 4, "bf16", 3500, False),
        # a draft of a few tokens is verified, one key head per query head, half-size heads
        _window("window verify, 5 tokens", 12, 16, 16, 5, 2047, 64, 500, 16, "f16", 900, False),
        # prompts of the benchmark's attention shape, token-major projections seen as [B, H, S, D]
        _window("window prefill, 8 x 2048", 8, 16, 16, 2048, 2048, 128, 512, 4, "bf16", 0, True),
        # one long prompt, shared key heads
        _window("window prefill, 1 x 8192", 1, 32, 8, 8192, 8192, 128, 2048, 4, "bf16", 0, True),
        # a chunk of a prompt behind a filled cache, ragged, odd sizes
        _window("window chunk, 777 of 4099", 3, 12, 4, 777, 4099, 64, 1000, 1, "f16", 1500, False),
        # few users behind a system prompt
        _prefix("prefix decode, 4 sequences", 4, 32, 8, 1, 512, 4096, 128, "bf16", 300, False),
        # a busy server behind a long system prompt
        _prefix("prefix decode, 64 sequences", 64, 32, 8, 1, 512, 16384, 128, "bf16", 400, False),
        # very many samples of one document
        _prefix("prefix decode, 256 sequences", 256, 32, 8, 1, 256, 32768, 128, "bf16", 200, False),
        # drafts of three tokens, odd sizes, half-size heads
        _prefix("prefix verify, 13 x 3 tokens", 13, 14, 2, 3, 333, 5003, 64, "f16", 200, False),
        # questions of a thousand tokens on one document
        _prefix("prefix prefill, 4 x 1024", 4, 16, 16, 1024, 1024, 4096, 128, "bf16", 0, True),
    ]


def _plain_pairs(case):
    return case["batch"] * case["heads"] * case["queries"] * (case["prefix"] + case["cache"])


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = max(_plain_pairs(c) * c["dim"] for c in listed())
    most = max(work(c)["flops"] for c in listed())
    while True:
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
        queries = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 8192)])
        case = {"op": rng.choice(["window", "prefix"]), "heads": heads, "kv_heads": kv_heads, "queries": queries, "dim": rng.choice([64, 128]),
                "dtype": rng.choice(["bf16", "f16"]), "token_major": rng.random() < 0.5}
        case["batch"] = _log(rng, 1, 256)
        case["cache"] = queries + _log(rng, 1, 8192) - 1
        case["slack"] = rng.choice([0, rng.randint(0, case["cache"] - 1)])
        case["prefix"] = _log(rng, 16, 32768) if case["op"] == "prefix" else 0
        case["window"] = _log(rng, 16, 4096) if case["op"] == "window" else 0
        case["sinks"] = rng.choice([0, 1, 4, 16, 130]) if case["op"] == "window" else 0
        small = case["batch"] * (case["kv_heads"] * case["cache"] + heads * queries) * case["dim"] < 1 << 29
        if heads <= 64 and small and _plain_pairs(case) * case["dim"] <= top and work(case)["flops"] <= most:
            return case


def _lengths(case):
    """Keys in use per sequence: spread over the last ``slack`` places of the cache."""
    return [case["cache"] - (b * 7919) % (case["slack"] + 1) for b in range(case["batch"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def rows(batch, heads, length):
        # projections come out token-major, [B, S, H, D]; the attention sees them as [B, H, S, D]
        shape = (batch, length, heads, case["dim"]) if case["token_major"] else (batch, heads, length, case["dim"])
        t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
        return t.transpose(1, 2) if case["token_major"] else t

    state = {"case": case, "q": rows(case["batch"], case["heads"], case["queries"])}
    state["k"], state["v"] = (rows(case["batch"], case["kv_heads"], case["cache"]) for _ in range(2))
    if case["op"] == "prefix":
        state["pk"], state["pv"] = (torch.randn((case["kv_heads"], case["prefix"], case["dim"]), generator=gen, device="cuda").to(dtype) for _ in range(2))
    state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["slack"] else None
    return state


def run(state):
    case, q, k, v, lengths = state["case"], state["q"], state["k"], state["v"], state["lengths"]
    if own:
        import conductor

        if case["op"] == "window":
            return conductor.ops.window_attention(q, k, v, case["window"], case["sinks"], lengths=lengths)
        return conductor.ops.prefix_attention(q, state["pk"], state["pv"], k, v, lengths=lengths)
    batch, heads, queries, dim = q.shape
    kv_heads, cache = k.shape[1], k.shape[2]
    group = heads // kv_heads
    qf = q.float().reshape(batch, kv_heads, group * queries, dim) * (1.0 / math.sqrt(dim))
    length = torch.full((batch,), cache, device=q.device) if lengths is None else lengths
    place = length.view(batch, 1, 1) - queries + torch.arange(queries, device=q.device).view(1, queries, 1)
    key = torch.arange(cache, device=q.device).view(1, 1, cache)
    seen = key <= place
    if case["op"] == "window":
        seen = seen & ((key > place - case["window"]) | (key < case["sinks"]))
    scores = (qf @ k.float().transpose(-1, -2)).view(batch, kv_heads, group, queries, cache)
    scores = scores.masked_fill(~seen.view(batch, 1, 1, queries, cache), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if case["op"] == "prefix":
        # the prefix is one matrix product for the rows of all sequences
        shared = qf.view(batch, kv_heads, group * queries, dim).transpose(0, 1).reshape(kv_heads, batch * group * queries, dim)
        first = (shared @ state["pk"].float().transpose(-1, -2)).view(kv_heads, batch, group, queries, -1)
        top = torch.maximum(top, first.amax(-1, keepdim=True).transpose(0, 1))
    top = top.masked_fill(top == float("-inf"), 0.0)
    weight = (scores - top).exp_()
    del scores
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(batch, kv_heads, group * queries, cache) @ v.float()).view(batch, kv_heads, group, queries, dim)
    if case["op"] == "prefix":
        first = (first - top.transpose(0, 1)).exp_()
        total = total + first.sum(-1, keepdim=True).transpose(0, 1)
        more = first.view(kv_heads, batch * group * queries, -1) @ state["pv"].float()
        out = out + more.view(kv_heads, batch, group, queries, dim).transpose(0, 1)
    out = out / total.masked_fill(total == 0, 1.0)
    out = out * (place >= 0).view(batch, 1, 1, queries, 1)
    return out.reshape(batch, heads, queries, dim).to(q.dtype)


def exact(case, seed):
    """Row by row from the definition, in 64 bits: only the keys that some query of a sequence sees."""
    state = prepare(case, seed)
    q, k, v = state["q"], state["k"], state["v"]
    heads, kv_heads, queries, dim = case["heads"], case["kv_heads"], case["queries"], case["dim"]
    group = heads // kv_heads
    out = torch.zeros((case["batch"], heads, queries, dim), dtype=torch.float64, device=q.device)
    for b, length in enumerate(_lengths(case)):
        row = torch.arange(length - queries, length, device=q.device)[:, None]
        col = torch.arange(length, device=q.device)[None, :]
        hidden = col > row
        if case["op"] == "window":
            hidden |= (col <= row - case["window"]) & (col >= case["sinks"])
        if case["prefix"]:
            hidden = torch.cat([(row < 0).expand(queries, case["prefix"]), hidden], 1)
        empty = hidden.all(1)
        for h in range(kv_heads):
            keys, values = k[b, h, :length].double(), v[b, h, :length].double()
            if case["prefix"]:
                keys, values = torch.cat([state["pk"][h].double(), keys]), torch.cat([state["pv"][h].double(), values])
            for g in range(h * group, (h + 1) * group):
                logit = torch.einsum("id,jd->ij", q[b, g].double(), keys) / math.sqrt(dim)
                logit[hidden] = -math.inf
                logit[empty] = 0.0
                prob = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True))
                prob[empty] = 0.0
                out[b, g] = torch.einsum("ij,jd->id", prob, values)
    return out


def work(case):
    """Every query, every key and value that some row sees, and every output once; two products per visible pair."""
    queries, dim = case["queries"], case["dim"]
    keys = pairs = 0
    for length in _lengths(case):
        if case["op"] == "prefix":
            rows = min(queries, length)
            keys += length
            pairs += rows * case["prefix"] + rows * length - rows * (rows - 1) // 2
            continue
        first = max(length - queries, 0)
        start = max(0, first - case["window"] + 1)
        keys += length - start + min(case["sinks"], start)
        # row at position p sees min(p + 1, window) keys of its window and the sinks in front of it
        w, s = case["window"], case["sinks"]
        full = sum_to(length) - sum_to(first)
        beyond = sum_to(max(length - w, 0)) - sum_to(max(first - w, 0))           # keys in front of the windows
        kept = sum_capped(max(length - w, 0), s) - sum_capped(max(first - w, 0), s)  # of these, the sinks
        pairs += full - beyond + kept
    moved = case["kv_heads"] * (keys + case["prefix"]) + case["batch"] * case["heads"] * queries
    return {"bytes": 2 * dim * 2 * moved, "flops": 4 * dim * case["heads"] * pairs}


def sum_to(n):
    """1 + 2 + ... + n."""
    return n * (n + 1) // 2


def sum_capped(n, cap):
    """min(1, cap) + min(2, cap) + ... + min(n, cap)."""
    return sum_to(min(n, cap)) + max(n - cap, 0) * cap
