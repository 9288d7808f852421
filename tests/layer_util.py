"""Plain 64-bit forms of the layer operators and error bounds of their kernels,
element by element, from the roundings that the documentation states.

u is half a step of the 16-bit type (bf16 2^-8, f16 2^-11) and e = 2^-24 that of
float32.  A float32 sum of n products in any order is off by at most
(n + 1) e sum|x||y| (to first order; the bounds take twice that).
"""
import math

import torch

E32 = 2.0 ** -24
#: exp2 and reciprocal instructions (1 step each) and the constants around them
ELEM = 16 * E32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the distance of the type's subnormals: what rounding adds near zero."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def act(z, kind):
    if kind == "relu":
        return torch.relu(z)
    if kind == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def act_slope(z, kind):
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        y = act(z, kind) if kind != "none" else z * 1
    return torch.autograd.grad(y.sum(), z)[0]


def matmul_reference(a, b, bias, residual, kind):
    """(out, z, bound of z, bound of act(z)) in 64 bits."""
    a, b = a.double(), b.double()
    z = a @ b
    size = a.abs() @ b.abs()
    if bias is not None:
        z = z + bias.double()
        size = size + bias.double().abs()
    dz = 2 * (a.shape[-1] + 2) * E32 * size
    y = act(z, kind)
    # slopes are at most 1.13; 1.5e-7 |z| is the error function's approximation
    dy = 1.13 * dz + (z.abs() * (2e-7 + 2 * ELEM) if kind not in ("none", "relu") else 0)
    if residual is not None:
        y = y + residual.double()
        dy = dy + E32 * y.abs()
    return y, z, dz, dy


def assert_within(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, what
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - ref).abs() - bound
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (f"{what}: element {worst} is {float(got.flatten()[worst])}, "
                                    f"should be {float(ref.flatten()[worst])} +- {float(bound.flatten()[worst]):.3g}")


def rounded(ref, err, dtype):
    """Bound of a value with error `err`, rounded once to `dtype`."""
    return err + half_step(dtype) * (ref.abs() + err) + least(dtype)


def seen_mask(lq, lk, nq, nk, window, sinks, device="cpu"):
    """[lq, lk]: does query i see key j, in a sequence of nq queries and nk keys."""
    p = torch.arange(lq, device=device)[:, None] + nk - nq
    j = torch.arange(lk, device=device)[None]
    m = (j <= p) & (j < nk) & (torch.arange(lq, device=device)[:, None] < nq)
    if window:
        m &= (p - j < window) | (j < sinks)
    return m


def attention_reference(q, k, v, window=None, sinks=0, scale=None, q_lens=None, k_lens=None, dout=None, kernel_out=None):
    """64-bit results and bounds: {"out": (ref, bound), "lse": ..., with dout also "dq", "dk", "dv"}.

    What no mask lets through is taken out before any product, so that NaN there is not met."""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    dtype, u, dev = q.dtype, half_step(q.dtype), q.device
    scale = d ** -0.5 if scale is None else scale
    names = ["out", "lse"] + (["dq", "dk", "dv"] if dout is not None else [])
    shape = {"out": q.shape, "lse": (b, h, lq), "dq": q.shape, "dk": k.shape, "dv": k.shape}
    res = {x: [torch.zeros(shape[x], dtype=torch.float64, device=dev) for _ in range(2)] for x in names}
    for i in range(b):
        nq = lq if q_lens is None else min(max(int(q_lens[i]), 0), lq)
        nk = lk if k_lens is None else min(max(int(k_lens[i]), 0), lk)
        m = seen_mask(lq, lk, nq, nk, window, sinks, dev)
        rows, cols = m.any(1), m.any(0)
        for x in range(h):
            g = x * kv // h
            qq = torch.where(rows[:, None], q[i, :, x].double(), 0.0)
            kk = torch.where(cols[:, None], k[i, :, g].double(), 0.0)
            vv = torch.where(cols[:, None], v[i, :, g].double(), 0.0)
            s = (qq @ kk.t()) * scale
            s = torch.where(m, s, -math.inf)
            lse = torch.logsumexp(s, 1) if lk else torch.full((lq,), -math.inf, dtype=torch.float64, device=dev)
            p = torch.where(m, torch.exp(s - torch.where(rows, lse, 0.0)[:, None]), 0.0)
            # error of a score, of a weight (relative), of the log-sum-exp
            ds_ = abs(scale) * 2 * (d + 2) * E32 * (qq.abs() @ kk.abs().t()) + ELEM * torch.where(m, s.abs(), 0.0)
            score = torch.where(m, ds_, 0.0).amax(1, keepdim=True) if lk else torch.zeros(lq, 1, device=dev, dtype=torch.float64)
            n = m.sum(1, keepdim=True)
            rel = 2 * score + (2 * n + 64) * E32 + ELEM * 4
            out = p @ vv
            # weights below the 16-bit type's normal range are rounded absolutely
            tiny = least(dtype) * (m.double() @ vv.abs())
            err = (u + rel) * (p @ vv.abs()) + tiny
            res["out"][0][i, :, x], res["out"][1][i, :, x] = out, rounded(out, err, dtype)
            res["lse"][0][i, x] = lse
            res["lse"][1][i, x] = rel[:, 0] + 4 * E32 * torch.where(rows, lse.abs(), 0.0)
            if dout is None:
                continue
            gg = torch.where(rows[:, None], dout[i, :, x].double(), 0.0)
            dp = gg @ vv.t()
            delta = (gg * out).sum(1, keepdim=True)
            # delta is computed from the rounded out
            ddelta = (gg.abs() * rounded(out, err, dtype)).sum(1, keepdim=True) + 2 * (d + 2) * E32 * (gg.abs() * out.abs()).sum(1, keepdim=True)
            ds = p * (dp - delta)
            size = p * (dp.abs() + delta.abs())
            dpe = 2 * (d + 2) * E32 * (gg.abs() @ vv.abs().t())
            dse = rel * size + p * (ddelta + dpe) + u * ds.abs() + torch.where(m, least(dtype), 0.0)
            pe = (rel + u) * p + torch.where(m, least(dtype), 0.0)
            res["dq"][0][i, :, x] = scale * (ds @ kk)
            res["dq"][1][i, :, x] = abs(scale) * ((dse + 2 * n * E32 * size) @ kk.abs())
            nr = m.sum(0) * (h // kv)
            res["dk"][0][i, :, g] += scale * (ds.t() @ qq)
            res["dk"][1][i, :, g] += abs(scale) * ((dse + 2 * nr * E32 * size).t() @ qq.abs())
            res["dv"][0][i, :, g] += p.t() @ gg
            res["dv"][1][i, :, g] += (pe + 2 * nr * E32 * p).t() @ gg.abs()
    for x in ("dq", "dk", "dv"):
        if x in res:
            res[x][1] = rounded(res[x][0], res[x][1], dtype)
    return {x: tuple(v) for x, v in res.items()}


def cache_row(j, capacity, sinks):
    return j if j < sinks else sinks + (j - sinks) % (capacity - sinks)


def decode_reference(q, k_cache, v_cache, lengths, window=None, sinks=0, scale=None, k_new=None, v_new=None):
    """(out, bound, k_cache, v_cache) after one token; the caches are copies."""
    b, h, d = q.shape
    cap, kv = k_cache.shape[1:3]
    kc, vc = k_cache.clone(), v_cache.clone()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    w = min(window or cap, cap - sinks)
    for i in range(b):
        n = int(lengths[i])
        if n <= 0:
            continue
        if k_new is not None:
            kc[i, cache_row(n - 1, cap, sinks)] = k_new[i]
            vc[i, cache_row(n - 1, cap, sinks)] = v_new[i]
        js = [j for j in range(min(sinks, n))] + [j for j in range(max(min(sinks, n), n - w), n)]
        at = torch.tensor([cache_row(j, cap, sinks) for j in js], device=q.device)
        # the tokens that are seen, as a sequence of their own
        got = attention_reference(q[i:i + 1, None], kc[i:i + 1, at], vc[i:i + 1, at], scale=scale)["out"]
        out[i], bound[i] = got[0][0, 0], got[1][0, 0]
    return out, bound, kc, vc
