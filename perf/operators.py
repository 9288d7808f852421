"""The operators around the fused chain that a transformer layer needs, as
cases to time and to compare: matrix products with bias, activation and
residual in their epilogue (``matmul_epilogue`` and its gradients), and
attention with a sliding window whose first tokens stay visible
(``window_attention`` for prompts and for training, ``window_attention_decode``
for single tokens against a cache).

    own                 False: run() computes the plain form; True: it calls the library
    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, made from the seed alone
    run(state)          one pass, and its outputs
    exact(case, seed)   the same outputs in 64 bits
    work(case)          bytes and floating-point operations a pass cannot do without

Kinds of case, by "op":

    "matmul"        out = round(act(a . b + bias) + residual)
    "matmul_train"  the same with the pre-activation kept, then da, db, dbias
    "attn"          out and the rows' log-sum-exp
    "attn_train"    out, then dq, dk, dv
    "decode"        one token a sequence against a cache that keeps the first
                    `sinks` tokens and the last capacity - sinks ones

A query at position p sees the keys j <= p with p - j < window or j < sinks.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]

# No drawn case does more than the largest listed product, and the plain form
# of attention holds scores of at most so many (query, key) pairs over heads.
_MOST_FLOPS = 2 * 8192 * 8192 * 4096
_MOST_SCORES = 1 << 30


def _matmul(name, op, m, n, k, dtype, out_dtype, activation, bias, residual, b_t):
    return {"name": name, "op": op, "m": m, "n": n, "k": k, "dtype": dtype, "out_dtype": out_dtype,
            "activation": activation, "bias": bias, "residual": residual, "b_t": b_t}


def _attn(name, op, batch, heads, kv_heads, lq, lk, dim, window, sinks, dtype, ragged):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "lq": lq,
            "lk": lk, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "ragged": ragged}


def _decode(name, batch, heads, kv_heads, capacity, longest, dim, window, sinks, dtype):
    return {"name": name, "op": "decode", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "capacity": capacity, "longest": longest, "dim": dim, "window": window, "sinks": sinks,
            "dtype": dtype}


def listed():
    return [
        # the output projection of one decode step of eight sequences, weights as [n, k]
        _matmul("proj_decode_bf16", "matmul", 8, 4096, 4096, "bf16", "bf16", "none", True, True, True),
        # an ordinary product of no particular size
        _matmul("ragged_f16", "matmul", 1500, 3000, 1000, "f16", "f16", "silu", True, True, False),
        # the largest product: a prompt's wide layer
        _matmul("up_prompt_bf16", "matmul", 8192, 8192, 4096, "bf16", "bf16", "gelu", True, False, False),
        # one training step of a layer of ordinary size, and one of odd size with weights as [n, k]
        _matmul("layer_train_bf16", "matmul_train", 4096, 4096, 2048, "bf16", "bf16", "gelu_tanh", True, True,
                False),
        _matmul("ragged_train_f16", "matmul_train", 777, 1304, 2064, "f16", "f16", "silu", True, False, True),
        # attention over prompts: four query heads a key head
        _attn("prompt_bf16", "attn", 2, 32, 8, 4096, 4096, 128, 1024, 4, "bf16", False),
        # a batch of padded prompts of odd lengths, head dim 64, a short window
        _attn("prompt_ragged_f16", "attn", 6, 8, 8, 777, 777, 64, 200, 8, "f16", True),
        # the next 128 tokens of one prompt against a long cache
        _attn("chunk_bf16", "attn", 1, 32, 8, 128, 8192, 128, 4096, 16, "bf16", False),
        # training: sequences of ordinary length; a padded batch with full causal rows and head dim 80
        _attn("train_bf16", "attn_train", 1, 32, 8, 4096, 4096, 128, 1024, 4, "bf16", False),
        _attn("train_ragged_f16", "attn_train", 3, 6, 3, 1000, 1000, 80, 0, 0, "f16", True),
        # one token of one sequence, where the launches count
        _decode("decode_one_f16", 1, 8, 8, 512, 300, 64, 256, 4, "f16"),
        # one token of 64 sequences, caches that have wrapped
        _decode("decode_batch_bf16", 64, 32, 8, 4100, 16384, 128, 4096, 4, "bf16"),
    ]


def _log_size(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(x / step)) * step))


def _drawn(rng):
    op = rng.choice(["matmul", "matmul", "matmul_train", "attn", "attn", "attn_train", "decode", "decode"])
    dtype = rng.choice(["bf16", "f16"])
    if op in ("matmul", "matmul_train"):
        few = op == "matmul" and rng.random() < 0.4
        m = _log_size(rng, 1, 64) if few else _log_size(rng, 65, 8192)
        return _matmul("", op, m, _log_size(rng, 64, 8192, 8), _log_size(rng, 64, 8192, 8), dtype,
                       dtype if op == "matmul_train" else rng.choice([dtype, dtype, "f32"]),
                       rng.choice(_ACTIVATIONS), rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 80, 96, 128, 128])
    sinks = rng.choice([0, 1, 4, 16, 100])
    if op == "decode":
        batch = _log_size(rng, 1, 128)
        capacity = _log_size(rng, 128, 8192)
        window = rng.choice([0, capacity - sinks, _log_size(rng, 16, 4096)])
        return _decode("", batch, heads, kv_heads, capacity, _log_size(rng, 16, 65536), dim,
                       max(0, window), sinks, dtype)
    batch = rng.choice([1, 1, 2, 3, 6])
    lk = _log_size(rng, 16, 8192)
    chunk = op == "attn" and rng.random() < 0.3
    lq = min(lk, _log_size(rng, 1, 512)) if chunk else lk
    window = rng.choice([0, _log_size(rng, 16, 4096), _log_size(rng, 16, 4096)])
    return _attn("", op, batch, heads, kv_heads, lq, lk, dim, window, sinks, dtype,
                 not chunk and rng.random() < 0.5)


def draw(rng):
    while True:
        case = _drawn(rng)
        del case["name"]
        if "lq" in case and case["batch"] * case["heads"] * case["lq"] * case["lk"] > _MOST_SCORES:
            continue
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= 1_300_000_000:
            return case


# ---------------------------------------------------------------------------
# lengths of a case's sequences
# ---------------------------------------------------------------------------
def _lengths(case):
    """Tokens of each sequence: of a padded batch all different, down to half
    of the longest; of a decode step from one token to the longest."""
    b = case["batch"]
    if case["op"] == "decode":
        return [1 + (case["longest"] - 1) * (i + 1) // b for i in range(b)]
    return [case["lk"] - (i * case["lk"]) // (2 * b) if case["ragged"] else case["lk"] for i in range(b)]


def _pairs(case):
    """(query, key) pairs that see each other, over the batch, for one head."""
    window, sinks, total = case["window"] or 1 << 40, case["sinks"], 0
    for n in _lengths(case):
        if case["op"] == "decode":
            window = min(window, case["capacity"] - sinks)
            p = np.array([n - 1], dtype=np.int64)
        else:
            p = np.arange(max(0, n - case["lq"]), n, dtype=np.int64)
        near = np.minimum(p + 1, window)
        total += int((near + np.minimum(sinks, p + 1 - near)).sum())
    return total


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] in ("matmul", "matmul_train"):
        m, n, k = case["m"], case["n"], case["k"]
        osize = _BYTES[case["out_dtype"]]
        small = n * size * case["bias"]
        forward = (m * k + k * n) * size + small + m * n * osize * (1 + case["residual"])
        if case["op"] == "matmul":
            return {"bytes": forward, "flops": 2 * m * n * k}
        return {"bytes": forward + m * n * size + (m * k + k * n) * size + n * 4, "flops": 6 * m * n * k}
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    pairs = _pairs(case)
    if case["op"] == "decode":
        new = 2 * b * g * d * size
        return {"bytes": 2 * pairs * g * d * size + 2 * new + 2 * b * h * d * size, "flops": 4 * pairs * h * d}
    rows = sum(min(n, case["lq"]) for n in _lengths(case))
    keys = sum(_lengths(case))
    q, kv = rows * h * d * size, keys * g * d * size
    if case["op"] == "attn":
        reach = min(keys, b * ((case["window"] or case["lk"]) + case["lq"] + case["sinks"]))
        return {"bytes": 2 * q + 2 * reach * g * d * size + rows * h * 4, "flops": 4 * pairs * h * d}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * h * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = _TORCH[case["dtype"]]

    def normal(*shape, by=1.0, to=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * by).to(to)

    state = dict(case)
    if case["op"] in ("matmul", "matmul_train"):
        m, n, k = case["m"], case["n"], case["k"]
        # activations of deviation 1, weights that keep it, a residual stream of its own size
        state["a"] = normal(m, k)
        weights = normal(n, k, by=1 / math.sqrt(k)) if case["b_t"] else normal(k, n, by=1 / math.sqrt(k))
        state["b"] = weights.t() if case["b_t"] else weights
        state["bias_v"] = normal(n, by=0.5) if case["bias"] else None
        state["residual_v"] = normal(m, n, to=_TORCH[case["out_dtype"]]) if case["residual"] else None
        if case["op"] == "matmul_train":
            state["dout"] = normal(m, n)
        return state
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    state["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["scale"] = 1 / math.sqrt(d)
    if case["op"] == "decode":
        state["q"] = normal(b, h, d)
        state["k_new"], state["v_new"] = normal(b, kv, d), normal(b, kv, d)
        state["k_cache"], state["v_cache"] = (normal(b, case["capacity"], kv, d) for _ in range(2))
        return state
    state["q"] = normal(b, case["lq"], h, d)
    state["k"], state["v"] = normal(b, case["lk"], kv, d), normal(b, case["lk"], kv, d)
    if case["op"] == "attn_train":
        state["dout"] = normal(b, case["lq"], h, d)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if s["op"] in ("matmul", "matmul_train"):
        from welder_typical_chain_amd import matmul_epilogue, matmul_epilogue_backward
        train = s["op"] == "matmul_train"
        got = matmul_epilogue(s["a"], s["b"], bias=s["bias_v"], residual=s["residual_v"],
                              activation=s["activation"], out_dtype=_TORCH[s["out_dtype"]],
                              return_pre=train and s["activation"] != "none")
        if not train:
            return got
        out, pre = got if s["activation"] != "none" else (got, None)
        da, db, dbias = matmul_epilogue_backward(s["dout"], s["a"], s["b"], pre=pre,
                                                 activation=s["activation"], need_bias=s["bias"])
        return {"out": out, "da": da, "db": db, "dbias": dbias}
    from welder_typical_chain_amd import window_attention, window_attention_backward, window_attention_decode
    mask = {"window": s["window"] or None, "sinks": s["sinks"], "scale": s["scale"]}
    if s["op"] == "decode":
        out = window_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["lens"], k_new=s["k_new"],
                                      v_new=s["v_new"], **mask)
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["ragged"]:
        mask.update(q_lens=s["lens"], k_lens=s["lens"])
    out, lse = window_attention(s["q"], s["k"], s["v"], return_lse=True, **mask)
    if s["op"] == "attn":
        return {"out": out, "lse": lse}
    dq, dk, dv = window_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **mask)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _act(z, kind):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z * torch.sigmoid(z) if kind == "silu" else z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        y = torch.sigmoid(z)
        return y * (1 + z * (1 - y))
    return torch.ones_like(z)


def _plain_matmul(s):
    a, b = s["a"].float(), s["b"].float()
    z = a @ b
    if s["bias_v"] is not None:
        z = z + s["bias_v"].float()
    out = _act(z, s["activation"])
    if s["residual_v"] is not None:
        out = out + s["residual_v"].float()
    out = out.to(_TORCH[s["out_dtype"]])
    if s["op"] == "matmul":
        return out
    dz = s["dout"].float() * _act_slope(z, s["activation"])
    dtype = s["a"].dtype
    return {"out": out, "da": (dz @ b.t()).to(dtype), "db": (a.t() @ dz).to(dtype),
            "dbias": dz.sum(0) if s["bias"] else None}


def _seen(q_pos, k_pos, window, sinks):
    """[.., queries, keys]: whether the query at position q_pos sees the key at k_pos."""
    back = q_pos[..., :, None] - k_pos[..., None, :]
    near = back < window if window else torch.ones_like(back, dtype=torch.bool)
    return (back >= 0) & (near | (k_pos[..., None, :] < sinks))


def _plain_attn(s):
    dtype = s["q"].dtype
    b, lq, h, d = s["q"].shape
    lk, kv = s["k"].shape[1:3]
    r = h // kv
    q = s["q"].float().transpose(1, 2).reshape(b, kv, r * lq, d)  # a key head's query heads, one after another
    k, v = (s[x].float().transpose(1, 2) for x in ("k", "v"))
    at = torch.arange(lq, device="cuda")
    n = s["lens"][:, None].long()
    first = 0 if s["ragged"] else lk - lq
    seen = _seen((at + first).expand(b, lq), torch.arange(lk, device="cuda").expand(b, lk), s["window"], s["sinks"])
    seen = seen & (at[None, :, None] + first < n[..., None])  # rows behind a sequence's end see nothing
    seen = seen[:, None, None]
    y = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, kv, r, lq, lk)
    y = torch.where(seen, y, -math.inf)
    top = y.amax(-1, keepdim=True)
    e = torch.exp(y - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(b, kv, r * lq, lk), v)

    def rows(x):  # [b, lq, h, d] of a key head's rows
        return x.reshape(b, h, lq, d).transpose(1, 2)

    if s["op"] == "attn":
        return {"out": rows(out).to(dtype), "lse": (top + torch.log(total)).view(b, h, lq)}
    dout = s["dout"].float().transpose(1, 2).reshape(b, kv, r * lq, d)
    p = p.view(b, kv, r * lq, lk)
    dp = torch.matmul(dout, v.transpose(2, 3))
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * s["scale"]
    return {"out": rows(out).to(dtype), "dq": rows(torch.matmul(ds, k)).to(dtype),
            "dk": torch.matmul(ds.transpose(2, 3), q).transpose(1, 2).to(dtype),
            "dv": torch.matmul(p.transpose(2, 3), dout).transpose(1, 2).to(dtype)}


def _plain_decode(s):
    b, h, d = s["q"].shape
    cap, kv = s["k_cache"].shape[1:3]
    sinks, rest = s["sinks"], s["k_cache"].shape[1] - s["sinks"]
    last = s["lens"].long()[:, None] - 1
    # a token's place: the first `sinks` stay, the others take turns in what is left
    new = torch.where(last < sinks, last, sinks + torch.remainder(last - sinks, rest))[:, 0]
    each = torch.arange(b, device="cuda")
    s["k_cache"][each, new] = s["k_new"]
    s["v_cache"][each, new] = s["v_new"]
    slot = torch.arange(cap, device="cuda")[None]
    at = torch.where(slot < sinks, slot, last - torch.remainder(last - slot, rest))
    seen = (at <= last) & ((slot < sinks) | (at >= sinks))
    if s["window"]:
        seen = seen & ((last - at < s["window"]) | (slot < sinks))
    q = s["q"].float().view(b, kv, h // kv, d)
    k, v = (s[x].float().transpose(1, 2) for x in ("k_cache", "v_cache"))
    y = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    y = torch.where(seen[:, None, None], y, -math.inf)
    e = torch.exp(y - y.amax(-1, keepdim=True))
    out = torch.matmul(e / e.sum(-1, keepdim=True), v).view(b, h, d).to(s["q"].dtype)
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_plain(s):
    if s["op"] in ("matmul", "matmul_train"):
        return _plain_matmul(s)
    return _plain_decode(s) if s["op"] == "decode" else _plain_attn(s)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_matmul(s):
    a, b = s["a"].double(), s["b"].double()
    z = torch.mm(a, b)
    if s["bias_v"] is not None:
        z += s["bias_v"].double()[None]
    x = z.clone().requires_grad_()
    kind = s["activation"]
    with torch.enable_grad():
        if kind == "gelu":
            y = x * 0.5 * torch.erfc(-x / math.sqrt(2.0))
        elif kind == "gelu_tanh":
            u = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
            y = x / (1 + torch.exp(-u))
        elif kind == "silu":
            y = x / (1 + torch.exp(-x))
        else:
            y = torch.relu(x) if kind == "relu" else x * 1
    out = y.detach() if s["residual_v"] is None else y.detach() + s["residual_v"].double()
    if s["op"] == "matmul":
        return out
    (dz,) = torch.autograd.grad(y, x, s["dout"].double())
    return {"out": out, "da": torch.mm(dz, b.t()), "db": torch.mm(a.t(), dz),
            "dbias": dz.sum(0) if s["bias"] else None}


def _exact_attn(s):
    """Row by row of the batch and head by head; the gradient by the chain rule
    of each row's softmax, rows of a sequence alone."""
    b, lq, h, d = s["q"].shape
    kv = s["k"].shape[2]
    out = torch.zeros(b, lq, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, lq), -math.inf, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, n in enumerate(_lengths(s)):
        rows = min(n, lq)
        j = torch.arange(n, device="cuda")
        p = j[n - rows:, None]
        hidden = j > p
        if s["window"]:
            hidden |= (p - j >= s["window"]) & (j >= s["sinks"])
        for x in range(h):
            q, k, v = s["q"][i, :rows, x].double(), s["k"][i, :n, x * kv // h].double(), s["v"][i, :n, x * kv // h].double()
            y = torch.mm(q, k.t()).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
            lse[i, x, :rows] = torch.logsumexp(y, 1)
            w = torch.exp(y - lse[i, x, :rows, None])
            out[i, :rows, x] = torch.mm(w, v)
            if s["op"] == "attn_train":
                g = s["dout"][i, :rows, x].double()
                dy = w * (torch.mm(g, v.t()) - (g * out[i, :rows, x]).sum(1, keepdim=True))
                dq[i, :rows, x] = torch.mm(dy, k) * s["scale"]
                dk[i, :n, x * kv // h] += torch.mm(dy.t(), q) * s["scale"]
                dv[i, :n, x * kv // h] += torch.mm(w.t(), g)
    return {"out": out, "lse": lse} if s["op"] == "attn" else {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_decode(s):
    b, h, d = s["q"].shape
    cap, kv = s["k_cache"].shape[1:3]
    sinks, out = s["sinks"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k, v = s["k_cache"].double(), s["v_cache"].double()
    window = min(s["window"] or cap, cap - sinks)
    for i, n in enumerate(_lengths(s)):
        j = torch.cat([torch.arange(min(sinks, n)), torch.arange(max(min(sinks, n), n - window), n)])
        place = torch.where(j < cap, j, sinks + (j - sinks) % (cap - sinks)).cuda()
        k[i, place[-1]], v[i, place[-1]] = s["k_new"][i].double(), s["v_new"][i].double()
        keys, values = (x[i, place].repeat_interleave(h // kv, 1) for x in (k, v))
        y = (s["q"][i].double() * keys).sum(2) * s["scale"]
        out[i] = (torch.softmax(y, 0)[..., None] * values).sum(0)
    return {"out": out, "k_cache": k, "v_cache": v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("matmul", "matmul_train"):
        return _exact_matmul(s)
    return _exact_decode(s) if case["op"] == "decode" else _exact_attn(s)
