"""Plain 64-bit forms of attention with any mask, of what its keys receive, and of a
cache's cut, with error bounds of the kernels from the roundings that the
documentation states (the symbols are those of tests/layer_util.py)."""
import math

import torch

from tests.layer_util import E32, ELEM, cache_row, half_step, least, rounded


def lengths_of(lens, b, most):
    return [most if lens is None else min(max(int(lens[i]), 0), most) for i in range(b)]


def cross_mask(b, lq, lk, q_lens, k_lens, device):
    nq, nk = lengths_of(q_lens, b, lq), lengths_of(k_lens, b, lk)
    i, j = torch.arange(lq, device=device)[:, None], torch.arange(lk, device=device)[None]
    return torch.stack([(i < nq[x]) & (j < nk[x]) for x in range(b)]) if b else torch.zeros(0, lq, lk, dtype=torch.bool, device=device)


def causal_mask(b, lq, lk, q_lens, k_lens, device, window=None, sinks=0):
    nq, nk = lengths_of(q_lens, b, lq), lengths_of(k_lens, b, lk)
    i, j = torch.arange(lq, device=device)[:, None], torch.arange(lk, device=device)[None]
    out = []
    for x in range(b):
        p = i + nk[x] - nq[x]
        m = (i < nq[x]) & (j < nk[x]) & (j <= p)
        if window:
            m = m & ((p - j < window) | (j < sinks))
        out.append(m)
    return torch.stack(out)


def prefix_inputs(kp, vp, k, v, mask):
    """Keys, values and mask of [prefix | own] for each sequence; a row that has no query sees nothing."""
    b = k.shape[0]
    return (torch.cat([kp[None].expand(b, *kp.shape), k], 1), torch.cat([vp[None].expand(b, *vp.shape), v], 1), mask)


def attention(q, k, v, mask, scale=None, dout=None):
    """{"out": (ref, bound), "lse", "weights" and with dout "dq", "dk", "dv"} under mask [b, lq, lk].

    What no mask lets through is taken out before any product, so that NaN there is not met."""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    dtype, u, dev = q.dtype, half_step(q.dtype), q.device
    scale = d ** -0.5 if scale is None else scale
    shape = {"out": q.shape, "lse": (b, h, lq), "weights": (b, kv, lk), "dq": q.shape, "dk": k.shape, "dv": k.shape}
    if dout is None:
        shape = {x: shape[x] for x in ("out", "lse", "weights")}
    res = {x: [torch.zeros(s, dtype=torch.float64, device=dev) for _ in range(2)] for x, s in shape.items()}
    for i in range(b):
        m = mask[i]
        rows, cols = m.any(1), m.any(0)
        for x in range(h):
            g = x * kv // h
            qq = torch.where(rows[:, None], q[i, :, x].double(), 0.0)
            kk = torch.where(cols[:, None], k[i, :, g].double(), 0.0)
            vv = torch.where(cols[:, None], v[i, :, g].double(), 0.0)
            s = torch.where(m, (qq @ kk.t()) * scale, -math.inf)
            lse = torch.logsumexp(s, 1) if lk else torch.full((lq,), -math.inf, dtype=torch.float64, device=dev)
            p = torch.where(m, torch.exp(s - torch.where(rows, lse, 0.0)[:, None]), 0.0)
            # error of a score, of a weight (relative), of the log-sum-exp; 16 E32: joins of waves and splits
            ds_ = abs(scale) * 2 * (d + 2) * E32 * (qq.abs() @ kk.abs().t()) + ELEM * torch.where(m, s.abs(), 0.0)
            score = torch.where(m, ds_, 0.0).amax(1, keepdim=True) if lk else torch.zeros(lq, 1, device=dev, dtype=torch.float64)
            n = m.sum(1, keepdim=True)
            rel = 2 * score + (2 * n + 64 + 16) * E32 + ELEM * 4
            out = p @ vv
            err = (u + rel) * (p @ vv.abs()) + least(dtype) * (m.double() @ vv.abs())
            size = torch.where(rows, lse.abs(), 0.0)
            res["out"][0][i, :, x], res["out"][1][i, :, x] = out, rounded(out, err, dtype)
            res["lse"][0][i, x], res["lse"][1][i, x] = lse, rel[:, 0] + 4 * E32 * size
            # what a key receives is summed in f32 from exp(score - lse), lse rounded to f32
            each = p * (rel + 8 * E32 * size[:, None])
            count = m.sum(0) * (h // kv)
            res["weights"][0][i, g] += p.sum(0)
            res["weights"][1][i, g] += each.sum(0) + 2 * (count + 2) * E32 * p.sum(0) + 2.0 ** -126 * (1 + count)
            if dout is None:
                continue
            gg = torch.where(rows[:, None], dout[i, :, x].double(), 0.0)
            dp = gg @ vv.t()
            delta = (gg * out).sum(1, keepdim=True)
            # delta is computed from the rounded out
            ddelta = (gg.abs() * rounded(out, err, dtype)).sum(1, keepdim=True) + 2 * (d + 2) * E32 * (gg.abs() * out.abs()).sum(1, keepdim=True)
            ds = p * (dp - delta)
            mass = p * (dp.abs() + delta.abs())
            dpe = 2 * (d + 2) * E32 * (gg.abs() @ vv.abs().t())
            dse = rel * mass + p * (ddelta + dpe) + u * ds.abs() + torch.where(m, least(dtype), 0.0)
            pe = (rel + u) * p + torch.where(m, least(dtype), 0.0)
            res["dq"][0][i, :, x] = scale * (ds @ kk)
            res["dq"][1][i, :, x] = abs(scale) * ((dse + 2 * n * E32 * mass) @ kk.abs())
            res["dk"][0][i, :, g] += scale * (ds.t() @ qq)
            res["dk"][1][i, :, g] += abs(scale) * ((dse + 2 * count * E32 * mass).t() @ qq.abs())
            res["dv"][0][i, :, g] += p.t() @ gg
            res["dv"][1][i, :, g] += (pe + 2 * count * E32 * p).t() @ gg.abs()
    for x in ("dq", "dk", "dv"):
        if x in res:
            res[x][1] = rounded(res[x][0], res[x][1], dtype)
    return {x: tuple(y) for x, y in res.items()}


def seen_tokens(n, cap, window, sinks):
    """Tokens that the newest of n sees in a cache of `cap` rows."""
    w = min(window or cap, cap - sinks)
    return list(range(min(sinks, n))) + list(range(max(min(sinks, n), n - w), n))


def decode(q, k_cache, v_cache, lengths, kp=None, vp=None, window=None, sinks=0, scale=None, k_new=None, v_new=None,
           weights=None):
    """{"out": (ref, bound), "k_cache", "v_cache", "weights": (ref, bound)} after one token."""
    b, h, d = q.shape
    cap, kv = k_cache.shape[1:3]
    kc, vc = k_cache.clone(), v_cache.clone()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    w = None if weights is None else weights.double()
    w_bound = None if weights is None else torch.zeros_like(w)
    for i in range(b):
        n = int(lengths[i])
        if n <= 0:
            continue
        if k_new is not None:
            kc[i, cache_row(n - 1, cap, sinks)] = k_new[i]
            vc[i, cache_row(n - 1, cap, sinks)] = v_new[i]
        at = torch.tensor([cache_row(j, cap, sinks) for j in seen_tokens(n, cap, window, sinks)], device=q.device)
        keys, values = kc[i:i + 1, at], vc[i:i + 1, at]
        if kp is not None:
            keys, values = torch.cat([kp[None], keys], 1), torch.cat([vp[None], values], 1)
        all_of = torch.ones(1, 1, keys.shape[1], dtype=torch.bool, device=q.device)
        got = attention(q[i:i + 1, None], keys, values, all_of, scale=scale)
        out[i], bound[i] = got["out"][0][0, 0], got["out"][1][0, 0]
        if w is not None:
            w[i, :, cache_row(n - 1, cap, sinks)] = 0
            w[i, :, at] += got["weights"][0][0]
            w_bound[i, :, at] = got["weights"][1][0] + 2 * E32 * w[i, :, at].abs()
    return {"out": (out, bound), "k_cache": kc, "v_cache": vc, "weights": (w, w_bound)}


def evict(k_cache, v_cache, weights, lengths, keep, recent=0, sinks=0):
    """(k, v, weights, rows, lengths) of cache_evict, row by row."""
    b, cap, kv, d = k_cache.shape
    k, v = (torch.zeros(b, keep, kv, d, dtype=k_cache.dtype) for _ in range(2))
    w, rows = torch.zeros(b, kv, keep), torch.full((b, kv, keep), -1, dtype=torch.int32)
    kept = torch.zeros(b, dtype=torch.int32)
    src_k, src_v, src_w = k_cache.cpu(), v_cache.cpu(), weights.cpu()
    for i in range(b):
        n = min(max(int(lengths[i]), 0), cap)
        kept[i] = min(n, keep)
        for g in range(kv):
            stay = list(range(n))
            if n > keep:
                x = src_w[i, g].tolist()
                between = sorted(range(sinks, n - recent), key=lambda r: (x[r] == x[r], -x[r] if x[r] == x[r] else 0, r))
                stay = sorted([*range(sinks), *between[:keep - sinks - recent], *range(n - recent, n)])
            at = torch.tensor(stay, dtype=torch.long)
            k[i, :len(stay), g], v[i, :len(stay), g] = src_k[i, at, g], src_v[i, at, g]
            w[i, g, :len(stay)], rows[i, g, :len(stay)] = src_w[i, g, at], at.int()
    return k, v, w, rows, kept
