"""PyTorch-facing entry points of the operators around the fused chain that a
transformer layer needs: matrix products with an epilogue, attention with a
sliding window whose first tokens stay visible, attention to another sequence
and behind a prefix that a batch shares, and a cache cut to the rows that
attention has weighed most.

As in ``chain.py``, PyTorch supplies device memory and the current HIP stream
and every byte is computed by the HIP kernels behind ``include/wtc/wtc_layer.h``.
Every call runs on the current stream of its tensors' device, may be captured
into a graph, and takes its scratch memory from PyTorch's allocator (so that
calls and graphs never share any).  The gradients are functions of their own:
a call on tensors that autograd would track, in reverse or in forward mode,
raises, instead of dropping the gradient in silence (``torch.no_grad()``, or
the ``forward`` of a ``torch.autograd.Function``, is where these are called; a
dual tensor's tangent needs the latter).
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_FLOATS = {**_DTYPES, torch.float32: _lib.DTYPE_F32}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}

# The C structs are eight-byte fields throughout, packed here into bytes.
_pack_matmul = struct.Struct("13q").pack
_pack_attention = struct.Struct("28q2qd").pack
_pack_prefix = struct.Struct("5q").pack
_pack_evict = struct.Struct("21q").pack
_SIZES_END = 28 * 8  # where sizes and strides end: addresses and the scale follow


# A decode step's kernels take 5 to 10 us, less than a careless host call, so
# the helpers read each property of a tensor once and build no intermediate
# objects: 16.8 -> 9.5 us on the host for a
# window_attention_decode with a new token.
def _check_inputs(dtype, *named):
    """Device index of the tensors (None among them are skipped), all of `dtype` if it is given."""
    grad = torch.is_grad_enabled()
    device = -2
    for name, t in named:
        if t is None:
            continue
        at = t.get_device()  # -1 on the CPU
        if at != device:
            if at < 0:
                raise ValueError(f"{name} must be on the GPU")
            if device >= 0:
                raise ValueError(f"{name} is on another device")
            device = at
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, is {t.dtype}")
        if grad and t.requires_grad:
            raise ValueError(f"{name} requires a gradient, which this call does not record: call it under "
                             "torch.no_grad() and use the backward function")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for name, t in named:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has a tangent (a forward-mode gradient), which this call does not carry on")
    return device


def _launch(device, fn, *args):
    """Calls a C entry point on `device` with its current stream as last argument."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:  # the library launches on the current device
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


_sizes: dict = {}  # (function, arguments without addresses) -> bytes


def _scratch(name, args, device, keyed=None, *more):
    """(tensor, pointer, bytes) of a call's workspace; none for size 0."""
    key = (name, device, args if keyed is None else args[:keyed], *more)
    size = _sizes.get(key)
    if size is None:
        with torch.cuda.device(device):  # the plan goes by its compute units
            size = getattr(_lib.lib(), name)(args, *more)
        if size < 0:
            _lib.check(_lib.WTC_ERR_ARG)
        if len(_sizes) >= 4096:
            _sizes.clear()
        _sizes[key] = size
    if size == 0:
        return None, None, 0
    t = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device))
    return t, t.data_ptr(), size


def _check_out(out, *named, what="out"):
    """Refuses an `out` (called `what`) that starts where an input does, or lies over one: of tensors
    without gaps that is known, of others only the start (columns side by side in one
    buffer share no element, but their ranges meet)."""
    size = out.numel() * out.element_size()
    if not size:
        return
    at = out.data_ptr()
    end = at + size if out.is_contiguous() else at
    for name, t in named:
        if t is None or not t.numel():
            continue
        first = t.data_ptr()
        if first == at or (end > at and t.is_contiguous() and first < end and
                           at < first + t.numel() * t.element_size()):
            raise ValueError(f"{what} may not be or lie over {name}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _row_stride(t, name):
    """The row stride of a 2-D tensor whose rows are contiguous."""
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    if rows <= 1 or cols == 0:
        return cols
    if t.stride(0) < cols:
        raise ValueError(f"{name}: rows overlap")
    return t.stride(0)


def _code_of(t, name):
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported {name} dtype {t.dtype}: float16 or bfloat16") from None


def _weights(b, k):
    """(n, ldb, b_trans) of a [K, N] matrix stored by rows, or of the transpose of one."""
    if b.dim() != 2 or b.shape[0] != k:
        raise ValueError(f"b must be [{k}, N], is {tuple(b.shape)}")
    n = b.shape[1]
    if n == 0 or k == 0:
        return n, n, 0
    if b.stride(1) == 1 and (b.stride(0) >= n or k <= 1):
        return n, max(b.stride(0) if k > 1 else n, n), 0
    if b.stride(0) == 1 and (b.stride(1) >= k or n <= 1):
        return n, max(b.stride(1) if n > 1 else k, k), 1
    raise ValueError("b must be stored by rows, or be the transpose of such a matrix")


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def matmul_epilogue(a: torch.Tensor, b: torch.Tensor, *, bias: torch.Tensor | None = None,
                    residual: torch.Tensor | None = None, activation: str = "none",
                    out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    return_pre: bool = False):
    """out = round(act(a @ b + bias) + residual), in one pass over a and b.

    a: [..., K] float16 or bfloat16 (2-D: rows may be strided); b: [K, N] of the
    same type, stored by rows or as the transpose of such a matrix (a
    ``weight.t()``); bias: [N] of that type or float32; residual: [..., N] of
    the output type.  K and N are multiples of 8.  activation: "none", "relu",
    "gelu" (z Phi(z)), "gelu_tanh" or "silu".  Products and epilogue are
    float32, rounded once to `out_dtype` (a's type, or float32).  `out` may be
    `residual` itself, and lie over no other input.  With return_pre=True the result is
    (out, pre), pre = a @ b + bias in float32, which matmul_epilogue_backward
    needs for an activation (rounded to 16 bits it would move dbias by 5e-4).
    """
    code = _code_of(a, "a")
    a_shape = a.shape
    if not a_shape:
        raise ValueError("a must have at least one dimension")
    k = a_shape[-1]
    flat = len(a_shape) == 2
    a2 = a if flat else a.reshape(-1, k) if a.numel() else a.new_empty((a_shape[:-1].numel(), k))
    m = a2.shape[0]
    n, ldb, trans = _weights(b, k)
    device = _check_inputs(None, ("a", a), ("b", b), ("bias", bias), ("residual", residual), ("out", out))
    dtype = a.dtype
    if b.dtype != dtype:
        raise TypeError("a and b must have the same element type")
    act = _activation(activation)
    if out_dtype is None:
        out_dtype = dtype if out is None else out.dtype
    if out_dtype != dtype and out_dtype != torch.float32:
        raise TypeError(f"out_dtype must be {dtype} or float32")
    shape = (m, n) if flat else (*a_shape[:-1], n)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=a.device)
    elif out.shape != shape or out.dtype != out_dtype:
        raise ValueError("out has the wrong shape or dtype")
    else:
        itself = residual is not None and residual.shape == shape and out.data_ptr() == residual.data_ptr() and \
            (out.stride() == residual.stride() or (out.is_contiguous() and residual.is_contiguous()))
        _check_out(out, ("a", a), ("b", b.t() if trans else b), ("bias", bias), ("residual", None if itself else residual))
    out2 = out if flat else out.view(-1, n) if out.numel() else out.new_empty((m, n))
    bias_code = code
    if bias is not None:
        if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            raise ValueError(f"bias must be a contiguous [{n}]")
        if bias.dtype != dtype and bias.dtype != torch.float32:
            raise TypeError(f"bias must be {dtype} or float32")
        bias_code = _FLOATS[bias.dtype]
    ldo = ldr = _row_stride(out2, "out")
    if residual is not None:
        if residual.shape != shape or residual.dtype != out_dtype:
            raise ValueError(f"residual must be {tuple(shape)} of {out_dtype}")
        r2 = residual if flat else residual.reshape(-1, n) if residual.numel() else out2
        ldr = _row_stride(r2, "residual")
        residual = r2
    pre = torch.empty(shape, dtype=torch.float32, device=a.device) if return_pre else None
    lib = _lib.lib()
    args = _pack_matmul(m, n, k, _row_stride(a2, "a"), ldb, ldr, ldo, trans, code, _FLOATS[out_dtype], bias_code,
                        act, n)
    ws, ws_ptr, ws_bytes = _scratch("wtc_matmul_epilogue_workspace_size", args, device)
    _launch(device, lib.wtc_matmul_epilogue, args, a2.data_ptr(), b.data_ptr(), _ptr(bias), _ptr(residual),
            out2.data_ptr(), _ptr(pre), ws_ptr, ws_bytes)
    return (out, pre) if return_pre else out


def matmul_epilogue_backward(dout: torch.Tensor, a: torch.Tensor, b: torch.Tensor, *,
                             pre: torch.Tensor | None = None, activation: str = "none", need_a: bool = True,
                             need_b: bool = True, need_bias: bool = True):
    """(da, db, dbias) of matmul_epilogue: with dz = dout * act'(pre),
    da = dz @ b.T, db = a.T @ dz (stored as b is) and dbias = the column sums of
    dz in float32; None for what is not needed.  dout: [..., N] of a's type; pre:
    what return_pre=True gave (not needed with activation "none").  The
    products take dz rounded to a's type and sum in float32: a float16 dz has
    float16's range, so dout is best scaled to well above 6e-5 and below 5e4.
    The residual's gradient is dout itself.
    """
    code = _code_of(a, "a")
    if a.dim() < 1:
        raise ValueError("a must have at least one dimension")
    k = a.shape[-1]
    lead = a.shape[:-1]
    a2 = a if a.dim() == 2 else a.reshape(-1, k) if a.numel() else a.new_empty((lead.numel(), k))
    m = a2.shape[0]
    n, ldb, trans = _weights(b, k)
    device = _check_inputs(a.dtype, ("dout", dout), ("a", a), ("b", b))
    _check_inputs(torch.float32, ("pre", pre))
    act = _activation(activation)
    if dout.shape != lead + (n,):
        raise ValueError(f"dout must be {tuple(lead + (n,))}")
    if act and pre is None:
        raise ValueError("the gradient of an activation needs pre")
    if pre is not None and (pre.shape != dout.shape or not pre.is_contiguous() or pre.get_device() != device):
        raise ValueError("pre must be contiguous, of dout's shape and on its device")
    if dout.dim() == 2:  # (a gradient that autograd broadcast is copied)
        d2 = dout if dout.stride(1) == 1 and dout.stride(0) >= n or not dout.numel() else dout.contiguous()
    else:
        d2 = dout.reshape(-1, n).contiguous() if dout.numel() else dout.new_empty((m, n))
    da = torch.empty(a.shape, dtype=a.dtype, device=a.device) if need_a else None
    db = None
    if need_b:
        db = torch.empty((n, k) if trans else (k, n), dtype=a.dtype, device=a.device)
    dbias = torch.empty(n, dtype=torch.float32, device=a.device) if need_bias else None
    lib = _lib.lib()
    args = _pack_matmul(m, n, k, _row_stride(a2, "a"), ldb, n, n, trans, code, code, code, act,
                        _row_stride(d2, "dout"))
    ws, ws_ptr, ws_bytes = _scratch("wtc_matmul_epilogue_backward_workspace_size", args, device)
    _launch(device, lib.wtc_matmul_epilogue_backward, args, d2.data_ptr(), a2.data_ptr(), b.data_ptr(),
            _ptr(pre) if act else None, _ptr(da), _ptr(db), _ptr(dbias), ws_ptr, ws_bytes)
    return da, db.t() if trans and db is not None else db, dbias


def matmul_epilogue_plan(m: int, n: int, k: int, *, b_trans: bool = False, part: str = "forward",
                         cu_count: int = 0) -> tuple:
    """(tile rows, tile columns, splits of k) of the kernel that matmul_epilogue runs for
    dense operands of these sizes on a device of `cu_count` compute units (0: the current
    one), or of part "da" or "db" of its gradients.  (16, 16, 1): few rows, no tiles."""
    args = _pack_matmul(m, n, k, k, k if b_trans else n, n, n, bool(b_trans), _lib.DTYPE_BF16, _lib.DTYPE_BF16,
                        _lib.DTYPE_BF16, 0, n)
    got = (ctypes.c_int64 * 3)()
    at = [ctypes.cast(ctypes.byref(got, 8 * i), ctypes.POINTER(ctypes.c_int64)) for i in range(3)]
    _lib.check(_lib.lib().wtc_matmul_epilogue_plan(args, ("forward", "da", "db").index(part), cu_count, *at))
    return tuple(got)


def window_attention_plan(batch: int, heads: int, kv_heads: int, lq: int, lk: int, dim: int, *,
                          window: int | None = None, sinks: int = 0, cu_count: int = 0) -> dict:
    """What window_attention and its gradients run for dense tensors of these sizes on a
    device of `cu_count` compute units (0: the current one): "row_waves" and "key_splits" of
    the forward pass, "dq_row_waves", "query_parts" and "far_parts" of the gradients."""
    got = (ctypes.c_int64 * 5)()
    _lib.check(_lib.lib().wtc_window_attention_plan(
        _dense_attention(batch, heads, kv_heads, lq, lk, dim, *_mask(window, sinks)), cu_count, got))
    return dict(zip(("row_waves", "key_splits", "dq_row_waves", "query_parts", "far_parts"), got))


def _dense_attention(batch, heads, kv_heads, lq, lk, dim, window=0, sinks=0):
    q, kv = (lq * heads * dim, heads * dim, dim), (lk * kv_heads * dim, kv_heads * dim, dim)
    return _pack_attention(batch, heads, kv_heads, lq, lk, dim, window, sinks, _lib.DTYPE_BF16, *q, *kv, *kv,
                           *q, *q, 0, 0, 0, 0, 0, 0, dim ** -0.5)


def cross_attention_plan(batch: int, heads: int, kv_heads: int, lq: int, lk: int, dim: int, *,
                         cu_count: int = 0) -> dict:
    """What cross_attention and its gradients run, as window_attention_plan: "few_rows"
    (the kernel for few rows takes the forward pass), "wave_blocks" (row blocks of 32 that a
    wave holds), "key_splits", "one_launch" (dq with dk and dv), "query_parts" of those."""
    got = (ctypes.c_int64 * 5)()
    _lib.check(_lib.lib().wtc_cross_attention_plan(_dense_attention(batch, heads, kv_heads, lq, lk, dim), cu_count, got))
    return dict(zip(("few_rows", "wave_blocks", "key_splits", "one_launch", "query_parts"), got))


def prefix_attention_plan(batch: int, heads: int, kv_heads: int, prefix: int, lq: int, lk: int, dim: int, *,
                          cu_count: int = 0) -> dict:
    """What prefix_attention runs, as window_attention_plan: "one_launch" (for prefix and own
    keys), "prefix_splits" (of the prefix's own launch), "key_splits" (of the other launch),
    "wave_blocks" (row blocks of 32 that a wave holds where the prefix is read)."""
    got = (ctypes.c_int64 * 4)()
    shared = _pack_prefix(prefix, kv_heads * dim, dim, kv_heads * dim, dim)
    _lib.check(_lib.lib().wtc_prefix_attention_plan(_dense_attention(batch, heads, kv_heads, lq, lk, dim), shared,
                                                    cu_count, got))
    return dict(zip(("one_launch", "prefix_splits", "key_splits", "wave_blocks"), got))


def _strides(t, name):
    """Strides of [batch, tokens, heads, dim], dim contiguous; dimensions of one element get a harmless one."""
    n0, n1, n2, n3 = t.shape
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 and n3 > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0


def _row_strides(t, name):
    """_strides of [batch, heads, dim]: sequence, token (one), head."""
    n0, n1, n2 = t.shape
    s0, s1, s2 = t.stride()
    if s2 != 1 and n2 > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return s0 if n0 > 1 else 0, 0, s1 if n1 > 1 else 0


def _lens(t, batch, name, device):
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.shape != (batch,) or t.get_device() != device or \
            (batch > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 [{batch}] on the tensors' device")
    return t.data_ptr()


def _mask(window, sinks):
    if window is not None and window < 1:
        raise ValueError("window must be at least 1 (None: no limit)")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    return min(int(window or 0), 1 << 40), min(int(sinks), 1 << 40)


def _attention_args(q, k, v, window, sinks, scale, q_lens, k_lens, device):
    k_shape = k.shape
    if q.dim() != 4 or len(k_shape) != 4 or v.shape != k_shape:
        raise ValueError("q must be [B, Lq, H, D], k and v [B, Lk, Hkv, D]")
    b, lq, h, d = q.shape
    bk, lk, kv, dk = k_shape
    if bk != b or dk != d or kv == 0 or h % kv:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k_shape)}")
    w, s = _mask(window, sinks)
    return (b, h, kv, lq, lk, d, w, s, _code_of(q, "q"), *_strides(q, "q"), *_strides(k, "k"),
            *_strides(v, "v")), (_lens(q_lens, b, "q_lens", device), _lens(k_lens, b, "k_lens", device),
                                 d ** -0.5 if scale is None else float(scale))


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None,
                     sinks: int = 0, scale: float | None = None, q_lens: torch.Tensor | None = None,
                     k_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     return_lse: bool = False):
    """Causal softmax attention, softmax_row(scale * q . k) . v, in which the query
    at position p sees the keys j <= p with p - j < window or j < sinks.

    q: [B, Lq, H, D]; k, v: [B, Lk, Hkv, D], float16 or bfloat16, any strides of
    16-byte multiples with D contiguous (so also transposed [B, H, L, D]
    tensors); H a multiple of Hkv (query head h reads key head
    h // (H / Hkv)); D a multiple of 8 up to 128.  window None: no limit.  scale
    None: D ** -0.5.  q_lens / k_lens: int32 [B] on the GPU, tokens of each
    sequence of a batch padded on the right.  The queries are the last tokens:
    query i stands at position i + k_len - q_len.  A query that sees no key,
    and one behind its sequence's end, gives zeros; keys behind the end are not
    read.  Statistics and sums are float32; the weights are rounded to q's
    type before the product with v.  With return_lse=True the result is
    (out, lse), lse the rows' log-sum-exp, float32 [B, H, Lq].
    """
    return _attention("wtc_window_attention", q, k, v, window, sinks, scale, q_lens, k_lens, out, return_lse)


def _attention(name, q, k, v, window, sinks, scale, q_lens, k_lens, out, return_lse):
    device = _check_inputs(q.dtype, ("q", q), ("k", k), ("v", v), ("out", out))
    head, tail = _attention_args(q, k, v, window, sinks, scale, q_lens, k_lens, device)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape")
    else:
        _check_out(out, ("q", q), ("k", k), ("v", v))
    b, lq, h, _ = q.shape
    lse = torch.empty((b, h, lq), dtype=torch.float32, device=q.device) if return_lse else None
    args = _pack_attention(*head, *_strides(out, "out"), 0, 0, 0, 0, 0, 0, 0, *tail)
    ws, ws_ptr, ws_bytes = _scratch(name + "_workspace_size", args, device, _SIZES_END)
    _launch(device, getattr(_lib.lib(), name), args, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            _ptr(lse), ws_ptr, ws_bytes)
    return (out, lse) if return_lse else out


def window_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                              out: torch.Tensor, lse: torch.Tensor, *, window: int | None = None,
                              sinks: int = 0, scale: float | None = None, q_lens: torch.Tensor | None = None,
                              k_lens: torch.Tensor | None = None):
    """(dq, dk, dv) of window_attention called with the same arguments, which gave
    `out` and `lse`.  Contiguous, in the shapes and type of q, k, v; a key
    head's gradient is the sum over the query heads that share it.  Sums are
    float32; the products take the weights and their gradients rounded to q's
    type (float16: times a power of two that keeps them in its range, so a
    gradient may have any size that its results have).  Two calls give the same
    bits.
    """
    return _attention_backward("wtc_window_attention_backward", dout, q, k, v, out, lse, window, sinks, scale,
                               q_lens, k_lens)


def _check_lse(lse, b, h, lq, device):
    if lse.shape != (b, h, lq) or lse.dtype != torch.float32 or not lse.is_contiguous() or \
            not lse.is_cuda or lse.get_device() != device:
        raise ValueError("lse must be the forward call's: float32, contiguous, [B, H, Lq]")
    _check_inputs(None, ("lse", lse))


def _attention_backward(name, dout, q, k, v, out, lse, window, sinks, scale, q_lens, k_lens):
    device = _check_inputs(q.dtype, ("dout", dout), ("q", q), ("k", k), ("v", v), ("out", out))
    head, tail = _attention_args(q, k, v, window, sinks, scale, q_lens, k_lens, device)
    b, lq, h, _ = q.shape
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError("dout and out must have q's shape")
    _check_lse(lse, b, h, lq, device)
    if dout.stride(3) != 1 or 0 in dout.stride():  # a gradient that autograd broadcast
        dout = dout.contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    args = _pack_attention(*head, *_strides(out, "out"), *_strides(dout, "dout"), 0, 0, 0, 0, *tail)
    ws, ws_ptr, ws_bytes = _scratch(name + "_workspace_size", args, device, _SIZES_END)
    _launch(device, getattr(_lib.lib(), name), args, dout.data_ptr(), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws_ptr,
            ws_bytes)
    return dq, dk, dv


def window_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            lengths: torch.Tensor, *, k_new: torch.Tensor | None = None,
                            v_new: torch.Tensor | None = None, window: int | None = None, sinks: int = 0,
                            scale: float | None = None, out: torch.Tensor | None = None,
                            weights: torch.Tensor | None = None) -> torch.Tensor:
    """window_attention for one token of each sequence, against a cache of fixed size.

    q: [B, H, D]; k_cache, v_cache: [B, C, Hkv, D], C > sinks.  Token j of a
    sequence stands in row j if j < sinks, else in row
    sinks + (j - sinks) % (C - sinks): a sequence longer than C keeps its first
    `sinks` and its newest C - sinks tokens, and the window is at most that.
    lengths: int32 [B] on the GPU, tokens of each sequence with the new one, any
    number; 0 is an idle sequence (its out is 0, its cache is left alone).
    k_new, v_new: [B, Hkv, D], the new token's key and value, written to the
    caches in the same pass; without them the caches hold it already.
    weights: float32 [B, Hkv, C], contiguous: every visible row's softmax weight,
    summed over the query heads of its key head, is added to it; the newest
    token's row is set to it (what that row held was another token's).
    """
    return _decode(q, k_cache, v_cache, lengths, k_new, v_new, window, sinks, scale, out, weights, None)


def _key_weights(weights, b, kv, n, device):
    if weights.shape != (b, kv, n) or weights.dtype != torch.float32 or not weights.is_contiguous() or \
            weights.get_device() != device:
        raise ValueError(f"weights must be float32, contiguous, {(b, kv, n)}, on the tensors' device")
    _check_inputs(None, ("weights", weights))


def _decode(q, k_cache, v_cache, lengths, k_new, v_new, window, sinks, scale, out, weights, prefix):
    shape, cache = q.shape, k_cache.shape
    if len(shape) != 3 or len(cache) != 4 or v_cache.shape != cache:
        raise ValueError("q must be [B, H, D], the caches [B, C, Hkv, D]")
    device = _check_inputs(q.dtype, ("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("k_new", k_new),
                           ("v_new", v_new), ("out", out), *(prefix or ()))
    if lengths is None:
        raise ValueError("lengths must be given")
    b, h, d = shape
    bk, cap, kv, dk = cache
    if bk != b or dk != d or kv == 0 or h % kv:
        raise ValueError(f"shape mismatch: q {tuple(shape)} caches {tuple(cache)}")
    w, s = _mask(window, sinks)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape:
        raise ValueError("out must have q's shape")
    else:
        _check_out(out, ("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("k_new", k_new), ("v_new", v_new),
                   ("weights", weights), *(prefix or ()))
    kn = vn = (0, 0, 0)
    if k_new is not None and v_new is not None:
        if k_new.shape != (b, kv, d) or v_new.shape != (b, kv, d):
            raise ValueError(f"k_new and v_new must be {(b, kv, d)}")
        kn, vn = _row_strides(k_new, "k_new"), _row_strides(v_new, "v_new")
    elif k_new is not v_new:
        raise ValueError("k_new and v_new go together")
    args = _pack_attention(b, h, kv, 1, cap, d, w, s, _code_of(q, "q"), *_row_strides(q, "q"),
                           *_strides(k_cache, "k_cache"), *_strides(v_cache, "v_cache"), *_row_strides(out, "out"),
                           0, 0, 0, kn[0], kn[2], vn[0], vn[2], 0, _lens(lengths, b, "lengths", device),
                           d ** -0.5 if scale is None else float(scale))
    tensors = k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_new), _ptr(v_new), out.data_ptr()
    if prefix is not None:
        (_, kp), (_, vp) = prefix
        common = _prefix_args(kp, vp, kv, d)
        if k_new is not None:
            _check_out(k_cache, *prefix, what="k_cache")
            _check_out(v_cache, *prefix, what="v_cache")
        ws, ws_ptr, ws_bytes = _scratch("wtc_prefix_attention_decode_workspace_size", args, device, _SIZES_END, common)
        _launch(device, _lib.lib().wtc_prefix_attention_decode, args, common, q.data_ptr(), kp.data_ptr(),
                vp.data_ptr(), *tensors, ws_ptr, ws_bytes)
    elif weights is not None:
        _key_weights(weights, b, kv, cap, device)
        _check_out(weights, ("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("k_new", k_new), ("v_new", v_new),
                   what="weights")
        ws, ws_ptr, ws_bytes = _scratch("wtc_window_attention_decode_weights_workspace_size", args, device, _SIZES_END)
        _launch(device, _lib.lib().wtc_window_attention_decode_weights, args, q.data_ptr(), *tensors,
                weights.data_ptr(), ws_ptr, ws_bytes)
    else:
        ws, ws_ptr, ws_bytes = _scratch("wtc_window_attention_decode_workspace_size", args, device, _SIZES_END)
        _launch(device, _lib.lib().wtc_window_attention_decode, args, q.data_ptr(), *tensors, ws_ptr, ws_bytes)
    return out


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None,
                    q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, return_lse: bool = False):
    """Softmax attention to another sequence, softmax_row(scale * q . k) . v: every query
    of a sequence sees every key of it.

    q: [B, Lq, H, D]; k, v: [B, Lk, Hkv, D]; types, strides, heads, dimensions,
    lengths, scale and results are window_attention's.  Lq and Lk have nothing
    to do with each other (Lq + Lk up to 2^30); one token a sequence is Lq = 1.
    The rows of a sequence of k, and of v, may not overlap.
    A query of a sequence without keys, and one behind its sequence's end, gives zeros.
    An infinite value of v makes what its sequence's queries get of it infinite or NaN
    (where its weight is rounded to 0).
    """
    return _attention("wtc_cross_attention", q, k, v, None, 0, scale, q_lens, k_lens, out, return_lse)


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             out: torch.Tensor, lse: torch.Tensor, *, scale: float | None = None,
                             q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None):
    """(dq, dk, dv) of cross_attention called with the same arguments, which gave `out`
    and `lse`; otherwise as window_attention_backward."""
    return _attention_backward("wtc_cross_attention_backward", dout, q, k, v, out, lse, None, 0, scale, q_lens, k_lens)


def _prefix_args(kp, vp, kv, d):
    if kp.dim() != 3 or kp.shape[1:] != (kv, d) or vp.shape != kp.shape:
        raise ValueError(f"k_prefix and v_prefix must be [P, {kv}, {d}]")
    (k0, _, k1), (v0, _, v1) = _row_strides(kp, "k_prefix"), _row_strides(vp, "v_prefix")
    return _pack_prefix(kp.shape[0], k0, k1, v0, v1)


def prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k: torch.Tensor,
                     v: torch.Tensor, *, scale: float | None = None, q_lens: torch.Tensor | None = None,
                     k_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     return_lse: bool = False):
    """Causal attention of a batch whose sequences go on from one prefix: each query sees
    the whole prefix and, as in window_attention, its own sequence up to itself.

    k_prefix, v_prefix: [P, Hkv, D], one for the batch; q: [B, Lq, H, D]; k, v:
    [B, Lk, Hkv, D], each sequence's own tokens, whose last ones the queries are.
    P and Lk may be 0; the prefix's rows may not overlap.  Everything else is window_attention's.  Where sequences
    have few query rows, the prefix is read once for all of them together.
    """
    common = ("k_prefix", k_prefix), ("v_prefix", v_prefix)
    device = _check_inputs(q.dtype, ("q", q), ("k", k), ("v", v), ("out", out), *common)
    head, tail = _attention_args(q, k, v, None, 0, scale, q_lens, k_lens, device)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape")
    else:
        _check_out(out, ("q", q), ("k", k), ("v", v), *common)
    b, lq, h, d = q.shape
    lse = torch.empty((b, h, lq), dtype=torch.float32, device=q.device) if return_lse else None
    args = _pack_attention(*head, *_strides(out, "out"), 0, 0, 0, 0, 0, 0, 0, *tail)
    shared = _prefix_args(k_prefix, v_prefix, k.shape[2], d)
    ws, ws_ptr, ws_bytes = _scratch("wtc_prefix_attention_workspace_size", args, device, _SIZES_END, shared)
    _launch(device, _lib.lib().wtc_prefix_attention, args, shared, q.data_ptr(), k_prefix.data_ptr(),
            v_prefix.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), ws_ptr, ws_bytes)
    return (out, lse) if return_lse else out


def prefix_attention_decode(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                            k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None,
                            scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """prefix_attention for one token of each sequence, against caches of the own tokens.

    q: [B, H, D]; k_prefix, v_prefix: [P, Hkv, D]; k_cache, v_cache: [B, C, Hkv, D],
    C at least 1; lengths: int32 [B] on the GPU, tokens of each sequence behind
    the prefix with the new one (0: an idle sequence, its out is 0).  Token j of
    them stands in row j % C.  k_new, v_new: as in window_attention_decode.
    """
    return _decode(q, k_cache, v_cache, lengths, k_new, v_new, None, 0, scale, out, None,
                   (("k_prefix", k_prefix), ("v_prefix", v_prefix)))


def window_attention_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, window: int | None = None,
                             sinks: int = 0, scale: float | None = None, q_lens: torch.Tensor | None = None,
                             k_lens: torch.Tensor | None = None, weights: torch.Tensor | None = None):
    """What each key has received in window_attention called with the same arguments, which
    gave `lse`: float32 [B, Hkv, Lk], the softmax weights of the queries that see it, summed
    over them and over the query heads of its key head (0 behind a sequence's end).

    weights: float32 [B, Hkv, Lk], contiguous: they are added to it, and it is the result.
    """
    device = _check_inputs(q.dtype, ("q", q), ("k", k))
    head, tail = _attention_args(q, k, k, window, sinks, scale, q_lens, k_lens, device)
    b, lq, h, d = q.shape
    _, lk, kv, _ = k.shape
    _check_lse(lse, b, h, lq, device)
    add = weights is not None
    if add:
        _key_weights(weights, b, kv, lk, device)
        _check_out(weights, ("q", q), ("k", k), ("lse", lse), what="weights")
    else:
        weights = torch.empty((b, kv, lk), dtype=torch.float32, device=q.device)
    args = _pack_attention(*head, lq * h * d, h * d, d, 0, 0, 0, 0, 0, 0, 0, *tail)
    ws, ws_ptr, ws_bytes = _scratch("wtc_window_attention_weights_workspace_size", args, device, _SIZES_END)
    _launch(device, _lib.lib().wtc_window_attention_weights, args, q.data_ptr(), k.data_ptr(), lse.data_ptr(),
            weights.data_ptr(), add, ws_ptr, ws_bytes)
    return weights


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, lengths: torch.Tensor,
                keep: int, *, recent: int = 0, sinks: int = 0, k_out: torch.Tensor | None = None,
                v_out: torch.Tensor | None = None, weights_out: torch.Tensor | None = None):
    """(k, v, weights, rows, lengths) of a smaller cache that holds the rows of most weight.

    k_cache, v_cache: [B, C, Hkv, D] (float16 or bfloat16, D contiguous), token j of a
    sequence in row j; weights: float32 [B, Hkv, C], contiguous, what each row has
    received (window_attention_weights, window_attention_decode); lengths: int32 [B]
    on the GPU.  A sequence of at most `keep` rows keeps them all.  Of a longer one
    each key head keeps its first `sinks` rows, its last `recent` ones and, of those
    between, the ones of greatest weight (of equal ones the lowest; a NaN is
    greater than any number), in their order.  recent + sinks <= keep.

    The results: k, v [B, keep, Hkv, D], zeros behind a sequence's end; weights
    [B, Hkv, keep], zeros there; rows, int32 [B, Hkv, keep]: which they were, -1
    behind the end; lengths, int32 [B], min(lengths, keep).  k_out, v_out
    [B, C', Hkv, D] and weights_out [B, Hkv, C'], C' >= keep, given together, take them
    instead, with room for new tokens: rows of k_out and v_out from `keep` on stay as
    they are, those of weights_out are 0.  They lie over no input.
    """
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("the caches must be [B, C, Hkv, D]")
    given = k_out is not None
    if given != (v_out is not None) or given != (weights_out is not None):
        raise ValueError("k_out, v_out and weights_out go together")
    device = _check_inputs(k_cache.dtype, ("k_cache", k_cache), ("v_cache", v_cache), ("k_out", k_out), ("v_out", v_out))
    b, cap, kv, d = shape
    code = _code_of(k_cache, "k_cache")
    _key_weights(weights, b, kv, cap, device)
    if lengths is None:
        raise ValueError("lengths must be given")
    lens = _lens(lengths, b, "lengths", device)
    if not 0 < keep or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError("keep must be at least 1, and hold recent + sinks rows")
    if given:
        if k_out.dim() != 4 or v_out.shape != k_out.shape or k_out.shape[0] != b or k_out.shape[2:] != shape[2:] or \
                k_out.shape[1] < keep:
            raise ValueError(f"k_out and v_out must be [{b}, C, {kv}, {d}], C at least {keep}")
        _key_weights(weights_out, b, kv, k_out.shape[1], device)
        inputs = ("k_cache", k_cache), ("v_cache", v_cache), ("weights", weights), ("lengths", lengths)
        _check_out(k_out, *inputs, what="k_out")
        _check_out(v_out, *inputs, ("k_out", k_out), what="v_out")
        _check_out(weights_out, *inputs, ("k_out", k_out), ("v_out", v_out), what="weights_out")
    else:
        k_out, v_out = (torch.empty((b, keep, kv, d), dtype=k_cache.dtype, device=k_cache.device) for _ in range(2))
        weights_out = torch.empty((b, kv, keep), dtype=torch.float32, device=k_cache.device)
    rows = torch.empty((b, kv, keep), dtype=torch.int32, device=k_cache.device)
    kept = torch.empty(b, dtype=torch.int32, device=k_cache.device)
    args = _pack_evict(b, kv, cap, k_out.shape[1], d, code, keep, recent, sinks, *_strides(k_cache, "k_cache"),
                       *_strides(v_cache, "v_cache"), *_strides(k_out, "k_out"), *_strides(v_out, "v_out"))
    _launch(device, _lib.lib().wtc_cache_evict, args, k_cache.data_ptr(), v_cache.data_ptr(), weights.data_ptr(), lens,
            k_out.data_ptr(), v_out.data_ptr(), weights_out.data_ptr(), rows.data_ptr(), kept.data_ptr())
    return k_out, v_out, weights_out, rows, kept
