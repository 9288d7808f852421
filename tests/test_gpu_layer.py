"""The layer operators on the GPU against plain 64-bit forms (tests/layer_util.py),
at the sizes, masks, strides and values where they can go wrong."""
import math

import pytest
import torch

from tests import layer_util as U

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


@pytest.fixture(scope="module")
def W(native_lib):
    import welder_typical_chain_amd as w
    return w


def rand(seed, *shape, dtype=F32, by=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * by).to(dtype)


# ---------------------------------------------------------------------------
# matmul_epilogue
# ---------------------------------------------------------------------------
def check_matmul(W, m, n, k, dtype, out_dtype, kind, bias, residual, trans, a=None, seed=1):
    a = rand(seed, m, k, dtype=dtype) if a is None else a
    b = rand(seed + 1, n, k, dtype=dtype, by=0.1).t() if trans else rand(seed + 1, k, n, dtype=dtype, by=0.1)
    bv = None if bias is None else rand(seed + 2, n, dtype=bias)
    r = rand(seed + 3, m, n, dtype=out_dtype) if residual else None
    out, pre = W.matmul_epilogue(a, b, bias=bv, residual=r, activation=kind, out_dtype=out_dtype, return_pre=True)
    y, z, dz, dy = U.matmul_reference(a, b, bv, r, kind)
    assert out.dtype == out_dtype and pre.dtype == F32
    U.assert_within(out, y, U.rounded(y, dy, out_dtype), "out")
    U.assert_within(pre, z, U.rounded(z, dz, F32), "pre")
    again = W.matmul_epilogue(a, b, bias=bv, residual=r, activation=kind, out_dtype=out_dtype)
    assert torch.equal(out, again), "two calls differ"


SIZES = [(1, 8, 8), (1, 64, 4096), (16, 24, 2056), (17, 40, 4160), (7, 4104, 1032), (3, 136, 72), (8, 1024, 512), (16, 4096, 256), (33, 264, 1000), (64, 128, 64),
         (65, 72, 40), (127, 520, 128), (128, 128, 128), (129, 136, 136), (256, 256, 32), (257, 264, 2056),
         (300, 1000, 96), (513, 776, 520), (1024, 2048, 256)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype,trans", [(BF16, False), (F16, True), (BF16, True), (F16, False)])
def test_matmul_sizes(W, m, n, k, dtype, trans):
    check_matmul(W, m, n, k, dtype, dtype, "none", dtype, True, trans)


@pytest.mark.parametrize("kind", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,out_dtype,bias,residual", [(5, F32, F32, True), (200, BF16, BF16, False), (200, F32, None, True),
                                                       (5, BF16, None, False)])
def test_matmul_epilogues(W, kind, m, out_dtype, bias, residual):
    check_matmul(W, m, 328, 256, BF16, out_dtype, kind, bias, residual, False)


def test_matmul_strided_rows_and_leading_dims(W):
    wide = rand(5, 70, 3 * 128, dtype=BF16)
    check_matmul(W, 70, 96, 128, BF16, BF16, "silu", BF16, True, True, a=wide[:, 128:256])
    a, b = rand(6, 2, 5, 64, dtype=F16), rand(7, 64, 40, dtype=F16)
    out = W.matmul_epilogue(a, b)
    assert out.shape == (2, 5, 40)
    assert torch.equal(out.view(10, 40), W.matmul_epilogue(a.view(10, 64), b))
    big = torch.full((70, 200), 7.0, dtype=F16, device="cuda")  # an out with strided rows: what is between them stays
    W.matmul_epilogue(rand(8, 70, 64, dtype=F16), rand(9, 64, 96, dtype=F16), out=big[:, 16:112])
    assert bool((big[:, :16] == 7).all()) and bool((big[:, 112:] == 7).all())


def test_matmul_in_place_residual_and_weights_stored_wide(W):
    a, wide = rand(1, 40, 64, dtype=BF16), rand(2, 64, 256, dtype=BF16)
    b, r = wide[:, 64:160], rand(3, 40, 96, dtype=BF16)
    want = W.matmul_epilogue(a, b.contiguous(), residual=r)
    got = W.matmul_epilogue(a, b, residual=r, out=r)
    assert got.data_ptr() == r.data_ptr() and torch.equal(got, want)


def test_matmul_empty(W):
    a, b = rand(1, 0, 64, dtype=F16), rand(2, 64, 32, dtype=F16)
    assert W.matmul_epilogue(a, b).shape == (0, 32)
    bias = rand(3, 32, dtype=F16)
    out = W.matmul_epilogue(rand(1, 5, 0, dtype=F16), rand(2, 0, 32, dtype=F16), bias=bias, activation="relu")
    assert torch.equal(out, torch.relu(bias).expand(5, 32))
    out = W.matmul_epilogue(rand(1, 5, 64, dtype=F16), rand(2, 64, 0, dtype=F16), activation="silu")
    assert out.shape == (5, 0)
    for m in (5, 40):
        x, w = rand(1, m, 64, dtype=F16), rand(2, 64, 0, dtype=F16)
        da, db, dbias = W.matmul_epilogue_backward(rand(1, m, 0, dtype=F16), x, w)
        assert bool((da == 0).all()) and db.shape == (64, 0) and dbias.shape == (0,)
    da, db, dbias = W.matmul_epilogue_backward(rand(1, 0, 32, dtype=F16), a, b)
    assert da.shape == (0, 64) and bool((db == 0).all()) and bool((dbias == 0).all())


def test_matmul_extreme_values(W):
    """An infinite pre-activation gives the activation's limit; NaN stays in its row."""
    z = torch.zeros(6, 8, device="cuda")
    z[:, 0] = torch.tensor([math.inf, -math.inf, NAN, 1e30, -1e30, 60.0])
    a = z.to(BF16)
    b = torch.eye(8, dtype=BF16, device="cuda")
    b[1:] = 0  # only column 0 of a counts
    b[0, 0] = 1
    for kind in ("relu", "gelu", "gelu_tanh", "silu"):
        x = a[:, :1].float().expand(6, 8).contiguous()
        # every entry of a row of `a` other than the first is 0, and 0 * b is 0
        out = W.matmul_epilogue(a, torch.cat([b[:1, :1].expand(1, 8), b[1:]]), activation=kind, out_dtype=F32)
        assert bool((out[0] == math.inf).all()) and bool((out[1] == 0).all()) and bool(out[2].isnan().all()), kind
        assert bool((out[3] == x[3]).all()) and bool((out[4] == 0).all()) and bool((out[5] == x[5]).all()), kind


@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (5, 136, 72), (64, 128, 256), (130, 264, 136), (257, 72, 520),
                                   (300, 512, 256), (1000, 264, 1032), (2048, 256, 256)])
@pytest.mark.parametrize("dtype,trans,kind", [(BF16, False, "gelu_tanh"), (F16, True, "silu"), (BF16, True, "none"),
                                              (F16, False, "gelu"), (BF16, False, "relu")])
def test_matmul_backward(W, m, n, k, dtype, trans, kind):
    a = rand(1, m, k, dtype=dtype)
    b = rand(2, n, k, dtype=dtype, by=0.1).t() if trans else rand(2, k, n, dtype=dtype, by=0.1)
    dout, pre = rand(3, m, n, dtype=dtype), rand(4, m, n)
    da, db, dbias = W.matmul_epilogue_backward(dout, a, b, pre=None if kind == "none" else pre, activation=kind)
    assert db.stride() == b.stride() or min(n, k) == 1
    dz = dout.double() * U.act_slope(pre.double(), kind)
    # slope: absolute error of the formulas in f32, then the rounding of dz
    ez = dout.double().abs() * (0 if kind in ("none", "relu") else 2e-7 + 4 * U.ELEM * (1 + pre.double().abs() ** 3))
    u = 0 if kind == "none" else U.half_step(dtype)
    err = ez + u * (dz.abs() + ez) + (0 if kind == "none" else U.least(dtype))
    size = dz.abs() + err
    bd, ad = b.double(), a.double()
    ref = dz @ bd.t()
    U.assert_within(da, ref, U.rounded(ref, (err + 2 * (n + 2) * U.E32 * size) @ bd.t().abs(), dtype), "da")
    ref = ad.t() @ dz
    U.assert_within(db, ref, U.rounded(ref, ad.t().abs() @ (err + 2 * (m + 2) * U.E32 * size), dtype), "db")
    assert dbias.dtype == F32
    U.assert_within(dbias, dz.sum(0), (ez + 2 * (m + 2) * U.E32 * size).sum(0), "dbias")
    again = W.matmul_epilogue_backward(dout, a, b, pre=None if kind == "none" else pre, activation=kind)
    assert all(torch.equal(x, y) for x, y in zip((da, db, dbias), again)), "two calls differ"
    one = W.matmul_epilogue_backward(dout, a, b, pre=pre, activation=kind, need_a=False, need_bias=False)
    assert one[0] is None and one[2] is None and torch.equal(one[1], db)
    one = W.matmul_epilogue_backward(dout, a, b, pre=pre, activation=kind, need_b=False, need_bias=False)
    assert one[1] is None and torch.equal(one[0], da)
    one = W.matmul_epilogue_backward(dout, a, b, pre=pre, activation=kind, need_a=False, need_b=False)
    assert torch.equal(one[2], dbias)


def test_matmul_backward_strided(W):
    wide_d, wide_a = rand(1, 90, 304, dtype=BF16), rand(2, 90, 200, dtype=BF16)
    dout, a = wide_d[:, 8:144], wide_a[:, 64:192]
    b = rand(3, 128, 136, dtype=BF16)
    got = W.matmul_epilogue_backward(dout, a, b)
    want = W.matmul_epilogue_backward(dout.contiguous(), a.contiguous(), b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # a gradient that autograd broadcast from one value
    got = W.matmul_epilogue_backward(torch.ones((), dtype=BF16, device="cuda").expand(90, 136), a, b)
    want = W.matmul_epilogue_backward(torch.ones(90, 136, dtype=BF16, device="cuda"), a, b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---------------------------------------------------------------------------
# window_attention
# ---------------------------------------------------------------------------
def check_attention(W, q, k, v, dout=None, **kw):
    ref = U.attention_reference(q, k, v, dout=dout, **kw)
    out, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    U.assert_within(out, *ref["out"], "out")
    empty = ref["lse"][0] == -math.inf
    assert torch.equal(lse == -math.inf, empty), "rows without keys"
    U.assert_within(torch.where(empty, 0.0, lse), torch.where(empty, 0.0, ref["lse"][0]), ref["lse"][1], "lse")
    assert torch.equal(out, W.window_attention(q, k, v, **kw)), "two calls differ"
    if dout is None:
        return out
    got = W.window_attention_backward(dout, q, k, v, out, lse, **kw)
    for name, x in zip(("dq", "dk", "dv"), got):
        U.assert_within(x, *ref[name], name)
    again = W.window_attention_backward(dout, q, k, v, out, lse, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, again)), "two calls differ"
    return (out, *got)


def qkv(seed, b, lq, lk, h, kv, d, dtype):
    return (rand(seed, b, lq, h, d, dtype=dtype), rand(seed + 1, b, lk, kv, d, dtype=dtype),
            rand(seed + 2, b, lk, kv, d, dtype=dtype), rand(seed + 3, b, lq, h, d, dtype=dtype))


@pytest.mark.parametrize("lq,lk,window,sinks", [
    (1, 1, None, 0), (1, 1, 1, 1), (2, 2, 1, 0), (7, 7, 3, 1), (31, 31, None, 0), (33, 33, 32, 4), (64, 64, 64, 0),
    (65, 65, 1, 0), (65, 65, 1, 65), (127, 127, 16, 3), (128, 128, 40, 100), (129, 129, None, 5), (200, 200, 64, 64),
    (257, 257, 65, 1), (300, 300, 100, 130), (300, 300, 1000, 4), (511, 511, 7, 70), (513, 513, 128, 16),
    (1, 300, 64, 4), (5, 300, None, 0), (17, 700, 130, 9), (100, 612, 65, 200), (40, 20, None, 0), (40, 20, 4, 2)])
@pytest.mark.parametrize("dtype,h,kv,d", [(BF16, 4, 2, 128), (F16, 3, 3, 64), (F16, 5, 1, 80)])
def test_attention_masks(W, lq, lk, window, sinks, dtype, h, kv, d):
    q, k, v, g = qkv(11, 2, lq, lk, h, kv, d, dtype)
    check_attention(W, q, k, v, g, window=window, sinks=sinks)


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 56, 72, 96, 104, 120, 128])
def test_attention_dims(W, d):
    q, k, v, g = qkv(21, 1, 150, 150, 4, 2, d, BF16)
    check_attention(W, q, k, v, g, window=40, sinks=2, scale=0.2)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attention_scales(W, scale):
    q, k, v, g = qkv(25, 1, 130, 130, 2, 2, 64, BF16)
    check_attention(W, q, k, v, g, window=50, sinks=2, scale=scale)
    check_decode(W, [3, 100, 300], 120, 2, 2, 64, BF16, window=50, sinks=2, scale=scale)


@pytest.mark.parametrize("h,kv", [(1, 1), (8, 1), (6, 2), (7, 7), (12, 4), (32, 2), (64, 1), (80, 1), (140, 1)])
def test_attention_heads(W, h, kv):
    q, k, v, g = qkv(31, 2, 90, 90, h, kv, 64, F16)
    check_attention(W, q, k, v, g, window=33, sinks=3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4), (20, 80)])
def test_attention_padded_batch_with_nan_behind_the_ends(W, dtype, window, sinks):
    q, k, v, g = qkv(41, 6, 190, 190, 4, 2, 64, dtype)
    lens = torch.tensor([190, 0, 1, 100, 64, 129], dtype=torch.int32, device="cuda")
    for i, n in enumerate(lens.tolist()):
        for t in (q, k, v, g):
            t[i, n:] = NAN
    out, dq, dk, dv = check_attention(W, q, k, v, g, window=window, sinks=sinks, q_lens=lens, k_lens=lens)
    for i, n in enumerate(lens.tolist()):
        assert all(bool((t[i, n:] == 0).all()) for t in (out, dq, dk, dv))


def test_attention_lens_apart(W):
    """Queries that are the last ones of longer sequences, and of shorter ones (the first see nothing)."""
    q, k, v, g = qkv(51, 5, 70, 260, 4, 4, 96, BF16)
    q_lens = torch.tensor([70, 3, 60, 70, 500], dtype=torch.int32, device="cuda")
    k_lens = torch.tensor([260, 200, 20, 0, 300], dtype=torch.int32, device="cuda")
    check_attention(W, q, k, v, g, window=90, sinks=6, q_lens=q_lens, k_lens=k_lens)
    check_attention(W, q, k, v, g, q_lens=q_lens, k_lens=k_lens)


def test_attention_strides(W):
    """[B, H, L, D] tensors, slices of a joint projection, broadcast keys."""
    b, n, h, kv, d = 2, 150, 4, 2, 64
    joint = rand(61, b, n, (h + 2 * kv) * d, dtype=BF16).view(b, n, h + 2 * kv, d)
    q, k, v = joint[:, :, :h], joint[:, :, h:h + kv], joint[:, :, h + kv:]
    g = rand(62, b, h, n, d, dtype=BF16).transpose(1, 2)
    got = check_attention(W, q, k, v, g, window=60, sinks=4)
    want = W.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=60, sinks=4)
    assert torch.equal(got[0], want)
    out = torch.empty(b, h, n, d, dtype=BF16, device="cuda").transpose(1, 2)
    assert torch.equal(W.window_attention(q, k, v, window=60, sinks=4, out=out), want)
    one_k, one_v = (x[:1].expand(b, n, kv, d) for x in (k, v))
    check_attention(W, q, one_k, one_v, g, window=60, sinks=4)


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("name", ["k", "v", "q", "g"])
@pytest.mark.parametrize("lq", [200, 20])
def test_attention_bad_values_stay_where_they_are_seen(W, bad, name, lq):
    """A NaN or an infinity in a key, a value, a query or a gradient reaches no row whose
    mask hides it: those rows stay within the bounds of the clean inputs (not bit for bit:
    rows next to a bad value may be computed again, in another order of the same sums)."""
    lk, at, window, sinks = 200, 190, 30, 2
    q, k, v, g = qkv(71, 1, lq, lk, 2, 1, 64, BF16)
    kw = dict(window=window, sinks=sinks)
    ref = U.attention_reference(q, k, v, dout=g, **kw)
    t = dict(q=q, k=k, v=v, g=g)
    row = at if name in ("k", "v") else at - (lk - lq)
    t[name][0, row, 0, 5] = bad
    out, lse = W.window_attention(t["q"], t["k"], t["v"], return_lse=True, **kw)
    got = (out, *W.window_attention_backward(t["g"], t["q"], t["k"], t["v"], out, lse, **kw))
    pos = torch.arange(lq, device="cuda") + lk - lq
    one_head = name in ("q", "g")
    touched_q = pos == at if one_head else (pos >= at) & (pos < at + window)
    # keys that some touched query sees
    touched_k = U.seen_mask(lq, lk, lq, lk, window, sinks, "cuda")[touched_q].any(0)
    nothing = torch.zeros_like(touched_q)
    for what, x, touched in (("out", got[0], nothing if name == "g" else touched_q), ("dq", got[1], touched_q),
                             ("dk", got[2], touched_k), ("dv", got[3], nothing[:0] if name == "v" else touched_k)):
        want, bound = ref[what]
        if touched.numel() == 0:  # a value's gradient does not depend on values
            touched = torch.zeros_like(touched_k)
        U.assert_within(x[:, ~touched], want[:, ~touched], bound[:, ~touched], (name, what))
        if one_head and x.shape[2] == 2:
            U.assert_within(x[:, :, 1], want[:, :, 1], bound[:, :, 1], (name, what, "other head"))


def test_attention_full_of_nan(W):
    """Everything NaN stays NaN (and ends soon)."""
    q, k, v, g = qkv(75, 1, 700, 700, 4, 2, 64, BF16)
    out, lse = W.window_attention(q, k, torch.full_like(v, NAN), return_lse=True)
    assert bool(out.isnan().all()) and bool(lse.isfinite().all())
    nan = torch.full_like(q, NAN)
    out, lse = W.window_attention(nan, k, v, return_lse=True)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    out, lse = W.window_attention(q, k, v, return_lse=True)
    dq, dk, dv = W.window_attention_backward(nan, q, k, v, out, lse)
    assert bool(dq.isnan().all()) and bool(dk.isnan().all()) and bool(dv.isnan().all())


def test_attention_bad_value_in_a_first_token(W):
    """A NaN in one column of a first token's value reaches that column of every row and no other."""
    q, k, v, g = qkv(76, 1, 600, 600, 2, 2, 64, F16)
    kw = dict(window=40, sinks=2)
    ref = U.attention_reference(q, k, v, **kw)["out"]
    v[0, 1, 0, 7] = NAN
    out = W.window_attention(q, k, v, **kw)
    assert bool(out[0, 1:, 0, 7].isnan().all())
    clean = out.clone()
    clean[0, 1:, 0, 7] = ref[0][0, 1:, 0, 7].to(F16)
    U.assert_within(clean, *ref, "out")


@pytest.mark.parametrize("b,lq,lk,window,sinks", [(1, 900, 900, 5, 850), (2, 40, 900, 17, 300), (1, 1500, 1500, 1, 1)])
def test_attention_many_or_far_first_tokens(W, b, lq, lk, window, sinks):
    q, k, v, g = qkv(77, b, lq, lk, 2, 1, 32, BF16)
    check_attention(W, q, k, v, g, window=window, sinks=sinks)


def test_attention_backward_of_a_broadcast_gradient(W):
    q, k, v, _ = qkv(78, 1, 70, 70, 2, 2, 64, BF16)
    out, lse = W.window_attention(q, k, v, return_lse=True)
    one = torch.ones((), dtype=BF16, device="cuda").expand(q.shape)
    got = W.window_attention_backward(one, q, k, v, out, lse)
    want = W.window_attention_backward(one.contiguous(), q, k, v, out, lse)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_past_32_bits(W):
    """A cache of over 4 GiB: its last rows, its wrapped rows and its first ones."""
    kv, d, cap, sinks = 32, 128, 600_000, 3
    cache = torch.zeros(1, cap, kv, d, dtype=BF16, device="cuda")  # 4.9 GB, keys and values alike
    assert cache.numel() * 2 > 1 << 32
    cache[:, :400] = rand(1, 1, 400, kv, d, dtype=BF16)
    cache[:, -400:] = rand(2, 1, 400, kv, d, dtype=BF16)
    q = rand(3, 1, 64, d, dtype=BF16)
    for n in (cap, cap + 150):  # the second wraps: 150 rows behind the first ones, the rest at the end
        n_t = torch.tensor([n], dtype=torch.int32, device="cuda")
        ref, bound, _, _ = U.decode_reference(q, cache, cache, [n], window=300, sinks=sinks)
        U.assert_within(W.window_attention_decode(q, cache, cache, n_t, window=300, sinks=sinks), ref, bound, f"n {n}")
    # the last tokens of a prompt of that length, and the same with heads before tokens
    q = rand(4, 1, 5, 32, d, dtype=BF16)
    rows = torch.cat([torch.arange(sinks), torch.arange(cap - 104, cap)]).cuda()
    ref = U.attention_reference(q, cache[:, rows], cache[:, rows], window=100, sinks=sinks)["out"]
    U.assert_within(W.window_attention(q, cache, cache, window=100, sinks=sinks), *ref, "prompt")
    turned = cache.view(1, kv, cap, d)  # another tensor of the same values: [B, H, L, D]
    turned = turned.transpose(1, 2)
    ref = U.attention_reference(q, turned[:, rows], turned[:, rows], window=100, sinks=sinks)["out"]
    U.assert_within(W.window_attention(q, turned, turned, window=100, sinks=sinks), *ref, "turned")


def test_attention_all_scores_minus_infinity(W):
    """A row whose visible scores are all -inf is a row without keys."""
    q = torch.ones(1, 40, 1, 64, dtype=F16, device="cuda")
    k, v = torch.ones_like(q), torch.ones_like(q)
    k[0, :10, 0, 0] = -math.inf
    out, lse = W.window_attention(q, k, v, return_lse=True)
    assert bool((out[0, :10] == 0).all()) and bool((lse[0, 0, :10] == -math.inf).all())
    assert bool((out[0, 10:] == 1).all())


def test_attention_large_scores(W):
    """Scores of several hundred: the running maximum moves from tile to tile."""
    q, k, v, g = qkv(81, 1, 300, 300, 2, 2, 64, BF16)
    ramp = torch.linspace(0, 40, 300, device="cuda")
    k = (k.float() + ramp[None, :, None, None] * q.float().mean(1, keepdim=True)).to(BF16)
    check_attention(W, q * 4, k, v, window=200, sinks=3)
    check_attention(W, q * 4, k.flip(1).contiguous(), v, window=200, sinks=3)


def test_attention_empty(W):
    q, k, v, _ = qkv(1, 2, 5, 0, 2, 2, 64, F16)
    out, lse = W.window_attention(q, k, v, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = W.window_attention_backward(q, q, k, v, out, lse)
    assert bool((dq == 0).all()) and dk.shape == k.shape
    q, k, v, _ = qkv(1, 2, 0, 5, 2, 2, 64, F16)
    out, lse = W.window_attention(q, k, v, return_lse=True)
    dq, dk, dv = W.window_attention_backward(q, q, k, v, out, lse)
    assert out.numel() == 0 and bool((dk == 0).all()) and bool((dv == 0).all())
    q, k, v, _ = qkv(1, 0, 5, 5, 2, 2, 64, F16)
    assert W.window_attention(q, k, v).numel() == 0


# ---------------------------------------------------------------------------
# window_attention_decode
# ---------------------------------------------------------------------------
def check_decode(W, lengths, cap, h, kv, d, dtype, new=True, seed=1, q=None, kc=None, vc=None, **kw):
    b = len(lengths)
    q = rand(seed, b, h, d, dtype=dtype) if q is None else q
    kc = rand(seed + 1, b, cap, kv, d, dtype=dtype) if kc is None else kc
    vc = rand(seed + 2, b, cap, kv, d, dtype=dtype) if vc is None else vc
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    extra = {}
    if new:
        extra = dict(k_new=rand(seed + 3, b, kv, d, dtype=dtype), v_new=rand(seed + 4, b, kv, d, dtype=dtype))
    ref, bound, rk, rv = U.decode_reference(q, kc, vc, lengths, **kw, **extra)
    for _ in range(2):  # a second call finds the token already there and gives the same
        out = W.window_attention_decode(q, kc, vc, n, **kw, **extra)
        U.assert_within(out, ref, bound, "out")
        assert torch.equal(kc, rk) and torch.equal(vc, rv), "caches"
    return out


@pytest.mark.parametrize("cap,window,sinks", [(1, None, 0), (2, 1, 1), (40, None, 0), (64, 16, 4), (100, 100, 0),
                                              (300, 296, 4), (300, 50, 70), (1000, None, 1), (1000, 3, 990)])
@pytest.mark.parametrize("dtype,h,kv,d", [(BF16, 8, 2, 128), (F16, 3, 3, 64), (F16, 5, 1, 80)])
def test_decode(W, cap, window, sinks, dtype, h, kv, d):
    lengths = [1, 2, 0, max(1, cap // 2), cap, cap + 1, 3 * cap + 5, 100000]
    check_decode(W, lengths, cap, h, kv, d, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("b,h,kv,cap", [(1, 8, 8, 5000), (1, 64, 1, 3000), (2, 40, 8, 2500), (130, 8, 2, 200), (3, 17, 1, 700)])
def test_decode_batches(W, b, h, kv, cap):
    check_decode(W, [(i * 977 + cap) % (2 * cap) for i in range(b)], cap, h, kv, 128, BF16, sinks=4)


@pytest.mark.parametrize("d", [8, 16, 40, 96, 104, 120])
def test_decode_dims(W, d):
    check_decode(W, [90, 33, 200], 120, 4, 2, d, F16, window=70, sinks=2, scale=0.3)


def test_decode_reads_only_what_is_seen(W):
    """NaN in rows that hold nothing yet, and in rows of tokens outside the window."""
    cap, sinks, window = 200, 3, 40
    kc, vc = rand(1, 2, cap, 2, 64, dtype=BF16), rand(2, 2, cap, 2, 64, dtype=BF16)
    lengths = [90, 1000]
    for i, n in enumerate(lengths):
        seen = {U.cache_row(j, cap, sinks) for j in list(range(sinks)) + list(range(n - window, n))}
        hidden = [r for r in range(cap) if r not in seen]
        kc[i, hidden] = NAN
        vc[i, hidden] = NAN
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = rand(3, 2, 4, 64, dtype=BF16)
    ref, bound, _, _ = U.decode_reference(q, kc, vc, lengths, window=window, sinks=sinks)
    U.assert_within(W.window_attention_decode(q, kc, vc, n, window=window, sinks=sinks), ref, bound, "out")


def test_decode_strides_and_shared_q(W):
    """Caches as [B, Hkv, C, D], new rows as slices of a joint projection."""
    b, cap, h, kv, d = 3, 150, 4, 2, 64
    kc = rand(1, b, kv, cap, d, dtype=F16).transpose(1, 2)
    vc = rand(2, b, kv, cap, d, dtype=F16).transpose(1, 2)
    joint = rand(3, b, (h + 2 * kv) * d, dtype=F16).view(b, h + 2 * kv, d)
    q, kn, vn = joint[:, :h], joint[:, h:h + kv], joint[:, h + kv:]
    lengths = [5, 150, 777]
    ref, bound, rk, rv = U.decode_reference(q, kc, vc, lengths, sinks=2, k_new=kn, v_new=vn)
    out = W.window_attention_decode(q, kc, vc, torch.tensor(lengths, dtype=torch.int32, device="cuda"), k_new=kn,
                                    v_new=vn, sinks=2)
    U.assert_within(out, ref, bound, "out")
    assert torch.equal(kc, rk) and torch.equal(vc, rv)


def test_decode_follows_the_prompt(W):
    """Token by token, decode gives what window_attention gives for the whole prompt."""
    n, h, kv, d, window, sinks, cap = 90, 4, 2, 64, 24, 3, 30
    q, k, v, _ = qkv(91, 1, n, n, h, kv, d, BF16)
    ref = U.attention_reference(q, k, v, window=window, sinks=sinks)["out"]
    kc, vc = (torch.full((1, cap, kv, d), NAN, dtype=BF16, device="cuda") for _ in range(2))
    for t in range(n):
        out = W.window_attention_decode(q[:, t], kc, vc, torch.tensor([t + 1], dtype=torch.int32, device="cuda"),
                                        k_new=k[:, t], v_new=v[:, t], window=window, sinks=sinks)
        U.assert_within(out, ref[0][:, t], ref[1][:, t], f"token {t}")


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------
def layer_weights(dim, h, kv, d, hidden, dtype):
    return dict(qkv=rand(1, dim, (h + 2 * kv) * d, dtype=dtype, by=dim ** -0.5),
                qkv_bias=rand(2, (h + 2 * kv) * d, dtype=dtype, by=0.1),
                proj=rand(3, h * d, dim, dtype=dtype, by=(h * d) ** -0.5),
                up=rand(4, hidden, dim, dtype=dtype, by=dim ** -0.5), up_bias=rand(5, hidden, dtype=dtype, by=0.1),
                down=rand(6, dim, hidden, dtype=dtype, by=hidden ** -0.5))


def layer_forward(W, x, w, h, kv, d, **kw):
    """A transformer layer (without norms): project, attend, project, two wide products."""
    b, n, _ = x.shape
    y = W.matmul_epilogue(x, w["qkv"], bias=w["qkv_bias"]).view(b, n, h + 2 * kv, d)
    q, k, v = y[:, :, :h], y[:, :, h:h + kv], y[:, :, h + kv:]
    o, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    x1 = W.matmul_epilogue(o.view(b, n, h * d), w["proj"], residual=x)
    u, pre = W.matmul_epilogue(x1, w["up"].t(), bias=w["up_bias"], activation="gelu_tanh", return_pre=True)
    x2 = W.matmul_epilogue(u, w["down"].t(), residual=x1)
    return x2, (q, k, v, o, lse, x1, u, pre)


def layer_backward(W, g, x, w, kept, h, kv, d, **kw):
    b, n, _ = x.shape
    q, k, v, o, lse, x1, u, pre = kept
    du, ddown, _ = W.matmul_epilogue_backward(g, u, w["down"].t(), need_bias=False)
    dx1, dup, dup_bias = W.matmul_epilogue_backward(du, x1, w["up"].t(), pre=pre, activation="gelu_tanh")
    dx1 = dx1 + g
    do, dproj, _ = W.matmul_epilogue_backward(dx1, o.view(b, n, h * d), w["proj"], need_bias=False)
    dq, dk, dv = W.window_attention_backward(do.view(b, n, h, d), q, k, v, o, lse, **kw)
    dy = torch.cat([dq, dk, dv], 2).view(b, n, -1)
    dx, dqkv, dqkv_bias = W.matmul_epilogue_backward(dy, x, w["qkv"])
    return dict(x=dx + dx1, qkv=dqkv, qkv_bias=dqkv_bias, proj=dproj, up=dup.t(), up_bias=dup_bias, down=ddown.t())


def plain_layer(x, w, h, kv, d, window, sinks):
    b, n, _ = x.shape
    y = (x @ w["qkv"] + w["qkv_bias"]).view(b, n, h + 2 * kv, d).transpose(1, 2)
    q, k, v = y[:, :h], y[:, h:h + kv].repeat_interleave(h // kv, 1), y[:, h + kv:].repeat_interleave(h // kv, 1)
    s = (q @ k.transpose(2, 3)) * d ** -0.5
    s = s.masked_fill(~U.seen_mask(n, n, n, n, window, sinks, x.device), -math.inf)
    o = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(b, n, h * d)
    x1 = x + o @ w["proj"]
    u = U.act(x1 @ w["up"].t() + w["up_bias"], "gelu_tanh")
    return x1 + u @ w["down"].t()


def test_a_layer_forward_and_backward(W):
    """The operators together against autograd in 64 bits; between them values are
    rounded to bf16 about ten times a path, each off by at most 2^-8: 5 % in norm is
    ten such roundings and more than their random sum."""
    h, kv, d, kw = 4, 2, 64, dict(window=50, sinks=4)
    x, w = rand(9, 2, 140, 256, dtype=BF16), layer_weights(256, h, kv, d, 512, BF16)
    y, kept = layer_forward(W, x, w, h, kv, d, **kw)
    g = rand(10, *y.shape, dtype=BF16)
    got = layer_backward(W, g, x, w, kept, h, kv, d, **kw)
    leaves = {"x": x.double().requires_grad_(), **{n: t.double().requires_grad_() for n, t in w.items()}}
    ref = plain_layer(leaves["x"], leaves, h, kv, d, 50, 4)
    ref.backward(g.double())
    for name, a, b in [("y", y, ref)] + [(n, got[n], leaves[n].grad) for n in got]:
        rel = float(((a.double() - b).norm() / b.norm()).detach())
        assert a.shape == b.shape and rel < 10 * 2.0 ** -8, (name, rel)


def test_a_layer_captured_and_replayed(W):
    """Prefill, training step and decode in one graph, replayed with new inputs among eager work."""
    h, kv, d, kw = 4, 2, 64, dict(window=50, sinks=4)
    x, w = rand(9, 1, 140, 256, dtype=BF16), layer_weights(256, h, kv, d, 512, BF16)
    g = rand(10, 1, 140, 256, dtype=BF16)
    kc, vc = rand(11, 3, 60, kv, d, dtype=BF16), rand(12, 3, 60, kv, d, dtype=BF16)
    n = torch.tensor([5, 60, 200], dtype=torch.int32, device="cuda")
    row = rand(13, 3, (h + 2 * kv), d, dtype=BF16)
    small = rand(14, 3, 256, dtype=BF16)

    def step():
        y, kept = layer_forward(W, x, w, h, kv, d, **kw)
        grads = layer_backward(W, g, x, w, kept, h, kv, d, **kw)
        o = W.window_attention_decode(row[:, :h], kc, vc, n, k_new=row[:, h:h + kv], v_new=row[:, h + kv:], **kw)
        z = W.matmul_epilogue(o.view(3, h * d), w["proj"], residual=small)
        return [y, *grads.values(), o, z]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        x.copy_(rand(100 + seed, *x.shape, dtype=BF16))
        row.copy_(rand(200 + seed, *row.shape, dtype=BF16))
        n += 1
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {seed}"


def test_two_graphs_and_streams_at_once(W):
    """Calls on two streams and two graphs replayed together do not share scratch memory."""
    q, k, v, g = qkv(1, 1, 700, 700, 4, 1, 64, BF16)
    q2, k2, v2, g2 = qkv(5, 1, 700, 700, 4, 1, 64, BF16)
    kc, vc = rand(3, 1, 4000, 1, 64, dtype=BF16), rand(4, 1, 4000, 1, 64, dtype=BF16)
    n = torch.tensor([4000], dtype=torch.int32, device="cuda")
    a, b = rand(7, 8, 2048, dtype=BF16), rand(8, 2048, 512, dtype=BF16)

    def work(q, k, v, g):
        out, lse = W.window_attention(q, k, v, window=64, sinks=4, return_lse=True)
        return [out, *W.window_attention_backward(g, q, k, v, out, lse, window=64, sinks=4),
                W.window_attention_decode(q[0, :1], kc, vc, n), W.matmul_epilogue(a, b)]

    want1, want2 = work(q, k, v, g), work(q2, k2, v2, g2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, got = [], []
    for s, args in zip(streams, ((q, k, v, g), (q2, k2, v2, g2))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got.append(work(*args))
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got[0], want1))
        assert all(torch.equal(x, y) for x, y in zip(got[1], want2))
    eager = []
    for s, args in zip(streams, ((q, k, v, g), (q2, k2, v2, g2))):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager.append([work(*args) for _ in range(3)])
    torch.cuda.synchronize()
    for rounds, want in zip(eager, (want1, want2)):
        for r in rounds:
            assert all(torch.equal(x, y) for x, y in zip(r, want))


def test_calls_from_several_host_threads(W):
    import threading
    args = []
    for i in range(4):
        q, k, v, g = qkv(20 + 10 * i, 1, 300 + 50 * i, 300 + 50 * i, 4, 2, 64, BF16)
        args.append((q, k, v, g, rand(5 + i, 8 + 30 * i, 512, dtype=BF16), rand(50 + i, 256, 512, dtype=BF16).t()))

    def work(q, k, v, g, a, b):
        out, lse = W.window_attention(q, k, v, window=70, sinks=4, return_lse=True)
        n = torch.full((1,), k.shape[1], dtype=torch.int32, device="cuda")
        return [out, *W.window_attention_backward(g, q, k, v, out, lse, window=70, sinks=4),
                W.window_attention_decode(q[:, 0], k, v, n), W.matmul_epilogue(a, b, activation="gelu")]

    want = [work(*x) for x in args]
    torch.cuda.synchronize()
    got, streams = [[] for _ in args], [torch.cuda.Stream() for _ in args]

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i].append(work(*args[i]))
        streams[i].synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for rounds, ref in zip(got, want):
        assert len(rounds) == 10
        for r in rounds:
            assert all(torch.equal(x, y) for x, y in zip(r, ref))


def test_refusals_on_the_gpu(W):
    a, b = rand(1, 16, 64, dtype=F16), rand(2, 64, 32, dtype=F16)
    for kw, err in [(dict(activation="tanh"), ValueError), (dict(out_dtype=BF16), TypeError),
                    (dict(bias=rand(1, 31, dtype=F16)), ValueError), (dict(bias=rand(1, 32, dtype=BF16)), TypeError),
                    (dict(residual=rand(1, 16, 32)), ValueError), (dict(out=rand(1, 16, 40, dtype=F16)), ValueError)]:
        with pytest.raises(err):
            W.matmul_epilogue(a, b, **kw)
    with pytest.raises(TypeError):
        W.matmul_epilogue(a.float(), b.float())
    with pytest.raises(TypeError):
        W.matmul_epilogue(a, b.to(BF16))
    with pytest.raises(ValueError):
        W.matmul_epilogue(a, b.cpu())
    with pytest.raises(W._lib.WtcError):
        W.matmul_epilogue(rand(1, 4, 60, dtype=F16), rand(1, 60, 32, dtype=F16))
    with pytest.raises(W._lib.WtcError):
        W.matmul_epilogue(rand(1, 4, 65, dtype=F16)[:, 1:], b)  # rows not 16-byte aligned
    square = rand(2, 64, 64, dtype=F16)
    with pytest.raises(ValueError):
        W.matmul_epilogue(a, square, out=a)
    with pytest.raises(ValueError):
        W.matmul_epilogue(a.requires_grad_(), b)
    a = a.detach()
    with pytest.raises(ValueError):
        W.matmul_epilogue_backward(rand(1, 16, 32, dtype=F16), a, b, activation="silu")
    q, k, v, _ = qkv(1, 1, 8, 8, 2, 2, 64, F16)
    with pytest.raises(ValueError):
        W.window_attention(q, k[:, :, :, :32], v)
    with pytest.raises(ValueError):
        W.window_attention(q, k, v, out=q)
    with pytest.raises(ValueError):
        W.window_attention(q, k, v, window=0)
    with pytest.raises(ValueError):
        W.window_attention(q, k, v, k_lens=torch.tensor([8], device="cuda"))
    with pytest.raises(TypeError):
        W.window_attention(q, k, v.to(BF16))
    with pytest.raises(W._lib.WtcError):
        W.window_attention(*qkv(1, 1, 8, 8, 2, 2, 136, F16)[:3])
    with pytest.raises(W._lib.WtcError):
        W.window_attention(q, k, v, out=q[:, :1].expand(1, 8, 2, 64).clone()[:, :1].expand(1, 8, 2, 64))
    with pytest.raises(W._lib.WtcError):
        W.window_attention_decode(q[:, 0], k, v, torch.tensor([8], dtype=torch.int32, device="cuda"), sinks=8)
