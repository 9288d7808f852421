"""Attention beyond the causal prompt, and the cache that it reads, as cases to
time and to compare: attention to states of another length (``cross_attention``
and its gradients), attention of a batch that shares a long prefix
(``prefix_attention``, ``prefix_attention_decode``), and a cache that is cut to
the rows which attention has weighed most (``window_attention_weights``,
``window_attention_decode`` with ``weights``, ``cache_evict``).

    own                 False: run() computes the plain form; True: it calls the library
    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, made from the seed alone
    run(state)          one pass, and its outputs
    exact(case, seed)   the same outputs in 64 bits
    work(case)          bytes and floating-point operations a pass cannot do without

Kinds of case, by "op":

    "cross"          out and the rows' log-sum-exp; every query sees every key of its sequence
    "cross_train"    out, then dq, dk, dv
    "prefix"         queries that see a prefix common to the batch and, causally, their own sequence
    "prefix_token"   one token a sequence: a common prefix and an own cache, which takes the token
    "weights"        what each key has received, summed over the queries of a prompt or a chunk
    "weights_token"  one token a sequence against a cache that counts what its rows receive
    "evict"          the rows of a cache that stay, and the smaller cache that holds them
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}
# The plain forms hold the scores of at most so many (query, key) pairs over all heads.
_MOST_SCORES = 1 << 30


def _cross(name, op, batch, heads, kv_heads, lq, lk, dim, dtype, ragged):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "lq": lq, "lk": lk,
            "dim": dim, "dtype": dtype, "ragged": ragged}


def _prefix(name, op, batch, heads, kv_heads, prefix, lq, lk, dim, dtype, ragged):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "prefix": prefix,
            "lq": lq, "lk": lk, "dim": dim, "dtype": dtype, "ragged": ragged}


def _weights(name, batch, heads, kv_heads, lq, lk, dim, window, sinks, dtype):
    return {"name": name, "op": "weights", "batch": batch, "heads": heads, "kv_heads": kv_heads, "lq": lq, "lk": lk,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype}


def _weights_token(name, batch, heads, kv_heads, capacity, longest, dim, window, sinks, dtype):
    return {"name": name, "op": "weights_token", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "capacity": capacity, "longest": longest, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype}


def _evict(name, batch, kv_heads, capacity, keep, recent, sinks, dim, dtype, ragged):
    return {"name": name, "op": "evict", "batch": batch, "kv_heads": kv_heads, "capacity": capacity, "keep": keep,
            "recent": recent, "sinks": sinks, "dim": dim, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # a decoder's prompts over long states, four query heads a key head: the largest product
        _cross("cross_prompt_bf16", "cross", 4, 32, 8, 2048, 4096, 128, "bf16", False),
        # one token of each of 16 sequences over 1500 states
        _cross("cross_token_f16", "cross", 16, 16, 16, 1, 1500, 64, "f16", False),
        # training: targets of ordinary length over states of an odd one; a small padded batch, head dim 80
        _cross("cross_train_bf16", "cross_train", 4, 16, 16, 1024, 1500, 64, "bf16", False),
        _cross("cross_train_ragged_f16", "cross_train", 3, 6, 3, 333, 1000, 80, "f16", True),
        # 64 answers to one long text, token by token
        _prefix("prefix_token_bf16", "prefix_token", 64, 32, 8, 8192, 1, 1024, 128, "bf16", True),
        # four short answers to a short text, where the launches count
        _prefix("prefix_token_few_f16", "prefix_token", 4, 8, 8, 1000, 1, 200, 64, "f16", True),
        # 8 questions of odd lengths behind one text
        _prefix("prefix_questions_bf16", "prefix", 8, 32, 8, 4096, 200, 200, 128, "bf16", True),
        # what a prompt's tokens have received; what a chunk adds to a windowed sequence of odd length
        _weights("weights_prompt_bf16", 1, 32, 8, 4096, 4096, 128, 0, 0, "bf16"),
        _weights("weights_chunk_f16", 2, 8, 4, 100, 3001, 80, 1000, 4, "f16"),
        # a decode step of 32 sequences that counts
        _weights_token("weights_token_bf16", 32, 32, 8, 4096, 4096, 128, 0, 0, "bf16"),
        # prompts of a batch cut to a quarter; one short odd cache
        _evict("evict_bf16", 16, 8, 8192, 2048, 256, 4, 128, "bf16", True),
        _evict("evict_small_f16", 1, 8, 600, 250, 32, 4, 64, "f16", False),
    ]


def _log_size(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    op = rng.choice(["cross", "cross", "cross_train", "cross_train", "prefix", "prefix_token", "prefix_token",
                     "weights", "weights_token", "evict", "evict"])
    dtype = rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 80, 96, 128, 128])
    if op in ("cross", "cross_train"):
        token = op == "cross" and rng.random() < 0.4
        batch = _log_size(rng, 1, 64) if token else rng.choice([1, 1, 2, 3, 6])
        lq = _log_size(rng, 1, 4) if token else _log_size(rng, 5, 4096)
        return _cross("", op, batch, heads, kv_heads, lq, _log_size(rng, 16, 8192), dim, dtype, rng.random() < 0.5)
    if op == "prefix":
        lq = _log_size(rng, 1, 1024)
        lk = lq if rng.random() < 0.5 else lq + _log_size(rng, 1, 1024)
        return _prefix("", op, _log_size(rng, 2, 64), heads, kv_heads, _log_size(rng, 16, 8192), lq, lk, dim, dtype,
                       lk == lq and rng.random() < 0.5)
    if op == "prefix_token":
        return _prefix("", op, _log_size(rng, 1, 128), heads, kv_heads, _log_size(rng, 16, 16384), 1,
                       _log_size(rng, 16, 2048), dim, dtype, True)
    if op == "evict":
        capacity = _log_size(rng, 64, 16384)
        keep = _log_size(rng, 16, capacity)
        sinks = rng.choice([0, 1, 4])
        return _evict("", _log_size(rng, 1, 32), kv_heads, capacity, keep, rng.randint(0, keep - sinks) // 2, sinks,
                      dim, dtype, rng.random() < 0.5)
    window, sinks = rng.choice([0, 0, _log_size(rng, 16, 4096)]), rng.choice([0, 0, 1, 4, 100])
    if op == "weights_token":
        capacity = _log_size(rng, 128, 8192)
        return _weights_token("", _log_size(rng, 1, 64), heads, kv_heads, capacity, _log_size(rng, 16, 16384), dim,
                              window, sinks, dtype)
    lk = _log_size(rng, 16, 8192)
    lq = min(lk, _log_size(rng, 1, 512)) if rng.random() < 0.4 else lk
    return _weights("", rng.choice([1, 1, 2, 3]), heads, kv_heads, lq, lk, dim, window, sinks, dtype)


def _scores(case):
    keys = case["lk"] + case.get("prefix", 0) if "lk" in case else 0
    return case["batch"] * case.get("heads", 0) * case.get("lq", 1) * keys


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        case = _drawn(rng)
        del case["name"]
        w = work(case)
        if _scores(case) <= _MOST_SCORES and all(w[x] <= max(m[x] for m in most) for x in w):
            return case


# ---------------------------------------------------------------------------
# lengths of a case's sequences
# ---------------------------------------------------------------------------
def _spread(longest, batch, ragged):
    """All different in a padded batch, down to half of the longest."""
    return [longest - (i * longest) // (2 * batch) if ragged else longest for i in range(batch)]


def _lengths(case):
    """(queries, keys) of each sequence; of a cache the tokens that it was given."""
    b = case["batch"]
    if case["op"] == "weights_token":
        return [1] * b, [1 + (case["longest"] - 1) * (i + 1) // b for i in range(b)]
    if case["op"] == "prefix_token":
        return [1] * b, [1 + (case["lk"] - 1) * (i + 1) // b for i in range(b)]
    if case["op"] == "evict":
        return [0] * b, _spread(case["capacity"], b, case["ragged"])
    if case["op"] == "weights":
        return [case["lq"]] * b, [case["lk"]] * b
    queries, keys = _spread(case["lq"], b, case["ragged"]), _spread(case["lk"], b, case["ragged"])
    return (queries, queries) if case["op"] == "prefix" and case["ragged"] else (queries, keys)


def _window_of(case):
    window = case["window"] or 1 << 40
    return min(window, case["capacity"] - case["sinks"]) if case["op"] == "weights_token" else window


def _pairs(case):
    """(query, key) pairs that see each other, over the batch, for one head."""
    queries, keys = _lengths(case)
    if case["op"].startswith("cross"):
        return sum(x * y for x, y in zip(queries, keys))
    total = 0
    for x, y in zip(queries, keys):
        if case["op"].startswith("prefix"):
            total += x * case["prefix"] + x * (y - x) + x * (x + 1) // 2
        else:
            p = torch.arange(y - x, y, dtype=torch.int64)
            near = torch.clamp(p + 1, max=_window_of(case))
            total += int((near + torch.clamp(p + 1 - near, max=case["sinks"])).sum())
    return total


def work(case):
    b, g, d = case["batch"], case["kv_heads"], case["dim"]
    queries, keys = _lengths(case)
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in keys)
        moved = 2 * 2 * kept * g * d * 2 + 2 * kept * g * 4
        return {"bytes": moved + sum(keys) * g * 4 + b * case["keep"] * g * 4, "flops": 2 * sum(keys) * g}
    h, pairs = case["heads"], _pairs(case)
    rows = sum(queries) * h * d * 2
    if case["op"] == "weights_token":
        return {"bytes": 2 * pairs * g * d * 2 + 2 * pairs * g * 4 + 4 * b * g * d * 2 + 2 * rows, "flops": 4 * pairs * h * d}
    if case["op"] == "weights":
        reach = min(sum(keys), b * ((case["window"] or case["lk"]) + case["lq"] + case["sinks"]))
        return {"bytes": rows + reach * g * d * 2 + sum(queries) * h * 4 + b * case["lk"] * g * 4, "flops": 2 * pairs * h * d}
    states = sum(keys) * g * d * 2
    if case["op"] == "cross":
        return {"bytes": 2 * rows + 2 * states + sum(queries) * h * 4, "flops": 4 * pairs * h * d}
    if case["op"] == "cross_train":
        return {"bytes": 4 * rows + 4 * states, "flops": 14 * pairs * h * d}
    common = case["prefix"] * g * d * 2
    new = 4 * b * g * d * 2 if case["op"] == "prefix_token" else 0
    return {"bytes": 2 * rows + 2 * common + 2 * states + new, "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    r = torch.Generator(device="cuda")
    r.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=r, device="cuda").to(_TORCH[case["dtype"]])

    s = dict(case)
    b, g, d, op = case["batch"], case["kv_heads"], case["dim"], case["op"]
    queries, keys = _lengths(case)
    s["k_lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["q_lens"] = torch.tensor(queries, dtype=torch.int32, device="cuda")
    if op == "evict":
        s["k_cache"], s["v_cache"] = (normal(b, case["capacity"], g, d) for _ in range(2))
        # a few rows with most of the weight, and some that no query has weighed
        w = torch.exp(1.5 * torch.randn((b, g, case["capacity"]), generator=r, device="cuda"))
        s["weights"] = torch.where(torch.rand(w.shape, generator=r, device="cuda") < 0.05, 0.0, w)
        return s
    h = case["heads"]
    s["scale"] = 1 / math.sqrt(d)
    if op in ("prefix_token", "weights_token"):
        rows = case["lk"] if op == "prefix_token" else case["capacity"]
        s["q"] = normal(b, h, d)
        s["k_new"], s["v_new"] = normal(b, g, d), normal(b, g, d)
        s["k_cache"], s["v_cache"] = normal(b, rows, g, d), normal(b, rows, g, d)
        if op == "weights_token":
            s["weights"] = 4 * torch.rand((b, g, rows), generator=r, device="cuda")
    else:
        s["q"] = normal(b, case["lq"], h, d)
        s["k"], s["v"] = (normal(b, case["lk"], g, d) for _ in range(2))
    if op.startswith("prefix"):
        s["k_prefix"], s["v_prefix"] = normal(case["prefix"], g, d), normal(case["prefix"], g, d)
    if op == "cross_train":
        s["dout"] = normal(b, case["lq"], h, d)
    if op == "weights":  # the log-sum-exps that attention has returned
        s["lse"] = torch.empty(b, h, case["lq"], device="cuda")
        seen = _seen(case["lk"] - case["lq"] + torch.arange(case["lq"], device="cuda"),
                     torch.arange(case["lk"], device="cuda"), case["window"], case["sinks"])
        for i in range(b):
            for x in range(h):
                y = s["q"][i, :, x].float() @ s["k"][i, :, x * g // h].float().t() * s["scale"]
                s["lse"][i, x] = torch.logsumexp(y.masked_fill(~seen, -math.inf), 1)
    return s


def _seen(q_pos, k_pos, window, sinks):
    """[queries, keys]: whether the query at position q_pos sees the key at k_pos."""
    back = q_pos[:, None] - k_pos[None]
    return (back >= 0) & ((back < (window or 1 << 40)) | (k_pos[None] < sinks))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import welder_typical_chain_amd as w
    op = s["op"]
    if op == "evict":
        k, v, weights, rows, lengths = w.cache_evict(s["k_cache"], s["v_cache"], s["weights"], s["k_lens"], s["keep"],
                                                     recent=s["recent"], sinks=s["sinks"])
        return {"k": k, "v": v, "weights": weights, "rows": rows, "lengths": lengths}
    lens = {"q_lens": s["q_lens"], "k_lens": s["k_lens"]} if s.get("ragged") else {}
    if op in ("cross", "cross_train"):
        out, lse = w.cross_attention(s["q"], s["k"], s["v"], scale=s["scale"], return_lse=True, **lens)
        if op == "cross":
            return {"out": out, "lse": lse}
        dq, dk, dv = w.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, scale=s["scale"], **lens)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if op == "prefix":
        return w.prefix_attention(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], scale=s["scale"], **lens)
    if op == "prefix_token":
        out = w.prefix_attention_decode(s["q"], s["k_prefix"], s["v_prefix"], s["k_cache"], s["v_cache"], s["k_lens"],
                                        k_new=s["k_new"], v_new=s["v_new"], scale=s["scale"])
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    mask = {"window": s["window"] or None, "sinks": s["sinks"], "scale": s["scale"]}
    if op == "weights":
        return w.window_attention_weights(s["q"], s["k"], s["lse"], **mask)
    weights = s["weights"].clone()  # (what came before stays, so that a pass can be made again)
    out = w.window_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["k_lens"], k_new=s["k_new"],
                                    v_new=s["v_new"], weights=weights, **mask)
    return {"out": out, "weights": weights, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _heads_first(x):
    """[b, g, tokens, d] in 32 bits of [b, tokens, g, d]."""
    return x.float().transpose(1, 2).contiguous()


def _grouped(x, g):
    """[b, g, r * tokens, d] in 32 bits of [b, tokens, h, d]: a key head's query heads, one after another."""
    b, n, h, d = x.shape
    return x.float().transpose(1, 2).reshape(b, g, h // g * n, d)


def _rows(x, h):
    """[b, tokens, h, d] of _grouped's order."""
    b, g, n, d = x.shape
    return x.reshape(b, h, n * g // h, d).transpose(1, 2)


def _softmax(y, seen):
    """(weights, log-sum-exp) of the last dimension; rows that see nothing get 0 and -inf."""
    y = torch.where(seen, y, -math.inf)
    top = y.amax(-1, keepdim=True)
    e = torch.exp(y - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), (top + torch.log(total))[..., 0]


def _within(s):
    """[b, 1, 1, lq, lk]: queries and keys that are part of their sequence; and the queries' positions [b, lq]."""
    i, j = (torch.arange(s[x], device="cuda") for x in ("lq", "lk"))
    n, m = s["q_lens"].long()[:, None], s["k_lens"].long()[:, None]
    seen = (i < n)[:, :, None] & (j < m)[:, None]
    return seen[:, None, None], i + m - n


def _plain_cross(s):
    b, lq, h, d = s["q"].shape
    lk, g = s["k"].shape[1:3]
    q, k, v = _grouped(s["q"], g), _heads_first(s["k"]), _heads_first(s["v"])
    seen, _ = _within(s)
    p, lse = _softmax((torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, g, h // g, lq, lk), seen)
    p = p.view(b, g, h // g * lq, lk)
    out = torch.matmul(p, v)
    dtype = s["q"].dtype
    if s["op"] == "cross":
        return {"out": _rows(out, h).to(dtype), "lse": lse.reshape(b, h, lq)}
    dout = _grouped(s["dout"], g)
    dp = torch.matmul(dout, v.transpose(2, 3))
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * s["scale"]
    return {"out": _rows(out, h).to(dtype), "dq": _rows(torch.matmul(ds, k), h).to(dtype),
            "dk": torch.matmul(ds.transpose(2, 3), q).transpose(1, 2).to(dtype),
            "dv": torch.matmul(p.transpose(2, 3), dout).transpose(1, 2).to(dtype)}


def _plain_prefix(s):
    token = s["op"] == "prefix_token"
    if token:
        each, last = torch.arange(s["batch"], device="cuda"), s["k_lens"].long() - 1
        s["k_cache"][each, last] = s["k_new"]
        s["v_cache"][each, last] = s["v_new"]
    q4 = s["q"][:, None] if token else s["q"]
    own_k, own_v = (s["k_cache"], s["v_cache"]) if token else (s["k"], s["v"])
    b, lq, h, d = q4.shape
    lk, g = own_k.shape[1:3]
    n = s["prefix"]
    q = _grouped(q4, g)
    k, v = (torch.cat([_heads_first(x[None]).expand(b, g, n, d), _heads_first(y)], 2)
            for x, y in ((s["k_prefix"], own_k), (s["v_prefix"], own_v)))
    within, pos = _within(s)
    causal = pos[:, None, None, :, None] >= torch.arange(lk, device="cuda")
    query = torch.arange(lq, device="cuda") < s["q_lens"].long()[:, None]
    common = query[:, None, None, :, None].expand(b, 1, 1, lq, n)
    y = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, g, h // g, lq, n + lk)
    p, _ = _softmax(y, torch.cat([common, within & causal], -1))
    out = _rows(torch.matmul(p.view(b, g, h // g * lq, n + lk), v), h).to(q4.dtype)
    return {"out": out[:, 0], "k_cache": own_k, "v_cache": own_v} if token else out


def _plain_weights(s):
    b, lq, h, d = s["q"].shape
    lk, g = s["k"].shape[1:3]
    y = torch.matmul(_grouped(s["q"], g), _heads_first(s["k"]).transpose(2, 3)).view(b, h, lq, lk) * s["scale"]
    seen = _seen(lk - lq + torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda"), s["window"], s["sinks"])
    p = torch.exp(torch.where(seen, y - s["lse"][..., None], -math.inf))
    return p.sum(2).view(b, g, h // g, lk).sum(2)


def _plain_weights_token(s):
    b, h, d = s["q"].shape
    cap, g = s["k_cache"].shape[1:3]
    sinks, rest, last = s["sinks"], cap - s["sinks"], s["k_lens"].long()[:, None] - 1
    # a token's place: the first `sinks` stay, the others take turns in what is left
    new = torch.where(last < sinks, last, sinks + torch.remainder(last - sinks, rest))
    each = torch.arange(b, device="cuda")
    s["k_cache"][each, new[:, 0]] = s["k_new"]
    s["v_cache"][each, new[:, 0]] = s["v_new"]
    row = torch.arange(cap, device="cuda")[None]
    at = torch.where(row < sinks, row, last - torch.remainder(last - row, rest))
    seen = (at <= last) & ((row < sinks) | ((at >= sinks) & (last - at < (s["window"] or 1 << 40))))
    k, v = _heads_first(s["k_cache"]), _heads_first(s["v_cache"])
    q = s["q"].float().view(b, g, h // g, d)
    p, _ = _softmax(torch.matmul(q, k.transpose(2, 3)) * s["scale"], seen[:, None, None])
    out = torch.matmul(p, v).view(b, h, d).to(s["q"].dtype)
    # the newest token's row counts from here on
    weights = torch.where((row == new)[:, None], 0.0, s["weights"]) + p.sum(2)
    return {"out": out, "weights": weights, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_evict(s):
    b, cap, g, d = s["k_cache"].shape
    keep, recent, sinks = s["keep"], s["recent"], s["sinks"]
    n = s["k_lens"].long()[:, None, None]
    row = torch.arange(cap, device="cuda").expand(b, g, cap)
    score = torch.where((row < sinks) | (row >= n - recent), math.inf, s["weights"])
    score = torch.where(row < n, score, -math.inf)
    best = torch.sort(score, dim=2, descending=True, stable=True)[1][:, :, :keep].sort(2)[0]
    fits = best < n  # rows behind a sequence's end come last
    at = best.transpose(1, 2)[..., None].expand(b, keep, g, d)
    k, v = (torch.where(fits.transpose(1, 2)[..., None], torch.gather(s[x], 1, at), 0) for x in ("k_cache", "v_cache"))
    return {"k": k, "v": v, "weights": torch.where(fits, torch.gather(s["weights"], 2, best), 0.0),
            "rows": torch.where(fits, best, -1).int(), "lengths": s["k_lens"].clamp(max=keep)}


def _run_plain(s):
    plain = {"cross": _plain_cross, "cross_train": _plain_cross, "prefix": _plain_prefix,
             "prefix_token": _plain_prefix, "weights": _plain_weights, "weights_token": _plain_weights_token,
             "evict": _plain_evict}
    return plain[s["op"]](s)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions: sequence by sequence and head by head
# ---------------------------------------------------------------------------
def _zeros(*shape):
    return torch.zeros(shape, dtype=torch.float64, device="cuda")


def _exact_cross(s):
    b, lq, h, d = s["q"].shape
    g = s["k"].shape[2]
    out, dq = torch.zeros_like(s["q"], dtype=torch.float64), torch.zeros_like(s["q"], dtype=torch.float64)
    dk, dv = torch.zeros_like(s["k"], dtype=torch.float64), torch.zeros_like(s["k"], dtype=torch.float64)
    lse = torch.full((b, h, lq), -math.inf, dtype=torch.float64, device="cuda")
    for i, (n, m) in enumerate(zip(*_lengths(s))):
        for x in range(h):
            q, k, v = s["q"][i, :n, x].double(), s["k"][i, :m, x * g // h].double(), s["v"][i, :m, x * g // h].double()
            y = torch.mm(q, k.t()) * s["scale"]
            lse[i, x, :n] = torch.logsumexp(y, 1)
            w = torch.exp(y - lse[i, x, :n, None])
            out[i, :n, x] = torch.mm(w, v)
            if s["op"] == "cross_train":
                grad = s["dout"][i, :n, x].double()
                dy = w * (torch.mm(grad, v.t()) - (grad * out[i, :n, x]).sum(1, keepdim=True)) * s["scale"]
                dq[i, :n, x] = torch.mm(dy, k)
                dk[i, :m, x * g // h] += torch.mm(dy.t(), q)
                dv[i, :m, x * g // h] += torch.mm(w.t(), grad)
    return {"out": out, "lse": lse} if s["op"] == "cross" else {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_prefix(s):
    token = s["op"] == "prefix_token"
    q4 = s["q"][:, None] if token else s["q"]
    b, lq, h, d = q4.shape
    k4, v4 = ((s["k_cache"], s["v_cache"]) if token else (s["k"], s["v"]))
    k4, v4, g = k4.double(), v4.double(), k4.shape[2]
    out = _zeros(b, lq, h, d)
    for i, (n, m) in enumerate(zip(*_lengths(s))):
        if token:
            k4[i, m - 1], v4[i, m - 1] = s["k_new"][i].double(), s["v_new"][i].double()
        late = torch.arange(m, device="cuda")[None] > torch.arange(m - n, m, device="cuda")[:, None]
        hidden = torch.cat([torch.zeros(n, s["prefix"], dtype=torch.bool, device="cuda"), late], 1)
        for x in range(h):
            k = torch.cat([s["k_prefix"][:, x * g // h].double(), k4[i, :m, x * g // h]])
            v = torch.cat([s["v_prefix"][:, x * g // h].double(), v4[i, :m, x * g // h]])
            y = torch.mm(q4[i, :n, x].double(), k.t()) * s["scale"]
            out[i, :n, x] = torch.mm(torch.softmax(y.masked_fill_(hidden, -math.inf), 1), v)
    return {"out": out[:, 0], "k_cache": k4, "v_cache": v4} if token else out


def _exact_weights(s):
    b, lq, h, d = s["q"].shape
    lk, g = s["k"].shape[1:3]
    out = _zeros(b, g, lk)
    p, j = torch.arange(lk - lq, lk, device="cuda")[:, None], torch.arange(lk, device="cuda")[None]
    hidden = (j > p) | ((p - j >= (s["window"] or lk)) & (j >= s["sinks"]))
    for i in range(b):
        for x in range(h):
            y = torch.mm(s["q"][i, :, x].double(), s["k"][i, :, x * g // h].double().t()) * s["scale"]
            out[i, x * g // h] += torch.exp(y - s["lse"][i, x].double()[:, None]).masked_fill_(hidden, 0.0).sum(0)
    return out


def _exact_weights_token(s):
    b, h, d = s["q"].shape
    cap, g = s["k_cache"].shape[1:3]
    sinks, out = s["sinks"], _zeros(b, h, d)
    k, v, weights = s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()
    window = _window_of(s)
    for i, n in enumerate(_lengths(s)[1]):
        j = torch.cat([torch.arange(min(sinks, n)), torch.arange(max(min(sinks, n), n - window), n)])
        place = torch.where(j < cap, j, sinks + (j - sinks) % (cap - sinks)).cuda()
        k[i, place[-1]], v[i, place[-1]] = s["k_new"][i].double(), s["v_new"][i].double()
        weights[i, :, place[-1]] = 0
        keys, values = (x[i, place].repeat_interleave(h // g, 1) for x in (k, v))
        p = torch.softmax((s["q"][i].double() * keys).sum(2) * s["scale"], 0)
        out[i] = (p[..., None] * values).sum(0)
        weights[i, :, place] += p.view(-1, g, h // g).sum(2).t()
    return {"out": out, "weights": weights, "k_cache": k, "v_cache": v}


def _exact_evict(s):
    b, cap, g, d = s["k_cache"].shape
    keep, recent, sinks = s["keep"], s["recent"], s["sinks"]
    k, v, weights = _zeros(b, keep, g, d), _zeros(b, keep, g, d), _zeros(b, g, keep)
    rows = torch.full((b, g, keep), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")
    for i, n in enumerate(_lengths(s)[1]):
        kept = min(n, keep)
        lengths[i] = kept
        for x in range(g):
            at = torch.arange(n)
            if n > keep:
                w = s["weights"][i, x, sinks:n - recent].cpu().numpy()
                best = np.lexsort((np.arange(len(w)), -w))[:keep - sinks - recent]  # heaviest first, then lowest
                at = torch.cat([at[:sinks], torch.from_numpy(np.sort(best)) + sinks, at[n - recent:]])
            at = at.cuda()
            k[i, :kept, x], v[i, :kept, x] = s["k_cache"][i, at, x].double(), s["v_cache"][i, at, x].double()
            weights[i, x, :kept], rows[i, x, :kept] = s["weights"][i, x, at].double(), at.int()
    return {"k": k, "v": v, "weights": weights, "rows": rows, "lengths": lengths}


def exact(case, seed):
    s = prepare(case, seed)
    whole = {"cross": _exact_cross, "cross_train": _exact_cross, "prefix": _exact_prefix,
             "prefix_token": _exact_prefix, "weights": _exact_weights, "weights_token": _exact_weights_token,
             "evict": _exact_evict}
    return whole[case["op"]](s)
