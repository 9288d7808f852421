"""The layer operators on the GPU at values, sizes and calls at the edges of what
their documentation allows, against plain 64-bit forms (tests/layer_util.py)."""
import math
from unittest import mock

import pytest
import torch

from tests import layer_util as U
from tests.layer_sizes import FULL_CHIP, LARGE_GRADIENTS, LARGE_PRODUCTS
from welder_typical_chain_amd.layer import matmul_epilogue_plan, window_attention_plan

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


def qkv(seed, b, lq, lk, h, kv, d, dtype):
    return (rand(seed, b, lq, h, d, dtype=dtype), rand(seed + 1, b, lk, kv, d, dtype=dtype),
            rand(seed + 2, b, lk, kv, d, dtype=dtype), rand(seed + 3, b, lq, h, d, dtype=dtype))


# ---------------------------------------------------------------------------
# a NaN that a token sees is in its result, whichever wave or split meets it
# ---------------------------------------------------------------------------
def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cap,n", [(40, 1), (40, 33), (200, 150), (3000, 2900), (3000, 7000)])
def test_decode_nan_query(W, dtype, cap, n):
    """One workgroup and several splits: the NaN head is NaN, the others are not touched."""
    q, kc, vc = rand(1, 1, 4, 64, dtype=dtype), rand(2, 1, cap, 2, 64, dtype=dtype), rand(3, 1, cap, 2, 64, dtype=dtype)
    clean = W.window_attention_decode(q, kc, vc, lens(n), sinks=3)
    q[0, 2, 11] = NAN
    out = W.window_attention_decode(q, kc, vc, lens(n), sinks=3)
    assert bool(out[0, 2].isnan().all())
    others = [0, 1, 3]
    assert torch.equal(out[0, others], clean[0, others])


@pytest.mark.parametrize("n,new", [(1, True), (1, False), (33, True), (33, False), (65, True), (129, False), (2900, False)])
def test_decode_nan_key_alone(W, n, new):
    """The newest key is alone in its tile (and wave): its NaN reaches the heads that read it."""
    cap = 3000
    q, kc, vc = rand(1, 1, 4, 64, dtype=BF16), rand(2, 1, cap, 2, 64, dtype=BF16), rand(3, 1, cap, 2, 64, dtype=BF16)
    kn, vn = rand(4, 1, 2, 64, dtype=BF16), rand(5, 1, 2, 64, dtype=BF16)
    if new:
        kn[0, 1, 3] = NAN
        out = W.window_attention_decode(q, kc, vc, lens(n), k_new=kn, v_new=vn)
    else:
        kc[0, n - 1, 1, 3] = NAN
        out = W.window_attention_decode(q, kc, vc, lens(n))
    assert bool(out[0, 2:].isnan().all()) and bool(out[0, :2].isfinite().all())


def test_decode_nan_first_token_alone(W):
    """A first token in a tile of its own."""
    q, kc, vc = rand(1, 1, 2, 64, dtype=F16), rand(2, 1, 500, 2, 64, dtype=F16), rand(3, 1, 500, 2, 64, dtype=F16)
    kc[0, 0, 0, 0] = NAN
    out = W.window_attention_decode(q, kc, vc, lens(400), window=90, sinks=1)
    assert bool(out[0, 0].isnan().all()) and bool(out[0, 1].isfinite().all())


@pytest.mark.parametrize("cap,n", [(300, 256), (4000, 4000)])
@pytest.mark.parametrize("where", ["key", "value"])
def test_decode_nan_beside_far_larger_scores(W, cap, n, where):
    """A NaN at a key whose wave (or split) has far smaller scores than another: 0 * NaN and
    a sum of NaN stay NaN although that wave's weight in the row is 0."""
    q = torch.full((1, 1, 64), 8.0, dtype=BF16, device="cuda")
    kc, vc = rand(2, 1, cap, 1, 64, dtype=BF16, by=0.1), rand(3, 1, cap, 1, 64, dtype=BF16)
    kc[0, :32] += 40  # the first tile's scores: 8 * 40 * 64 / 8
    if where == "key":
        kc[0, n - 1, 0, 5] = NAN
    else:
        vc[0, n - 1, 0] = NAN
    out = W.window_attention_decode(q, kc, vc, lens(n))
    assert bool(out.isnan().all())
    if where == "value":  # the prompt form says the same
        out = W.window_attention(q[:, None], kc[:, :n], vc[:, :n])
        assert bool(out.isnan().all())


@pytest.mark.parametrize("dtype,h,kv,d", [(BF16, 2, 2, 64), (F16, 40, 1, 80), (BF16, 4, 2, 128)])
@pytest.mark.parametrize("cap,n", [(1, 1), (1, 7), (2, 2), (33, 33), (33, 70)])
def test_decode_over_stale_nan(W, dtype, h, kv, d, cap, n):
    """What the new token's row held before does not matter, in a cache of one row either."""
    q, kn, vn = rand(1, 2, h, d, dtype=dtype), rand(2, 2, kv, d, dtype=dtype), rand(3, 2, kv, d, dtype=dtype)
    kc, vc = rand(4, 2, cap, kv, d, dtype=dtype), rand(5, 2, cap, kv, d, dtype=dtype)
    want, bound, rk, rv = U.decode_reference(q, kc, vc, [n, n], k_new=kn, v_new=vn)
    kc[:, U.cache_row(n - 1, cap, 0)] = NAN
    vc[:, U.cache_row(n - 1, cap, 0)] = NAN
    out = W.window_attention_decode(q, kc, vc, lens(n, n), k_new=kn, v_new=vn)
    U.assert_within(out, want, bound, "out")
    assert torch.equal(kc, rk) and torch.equal(vc, rv)


@pytest.mark.parametrize("cap,window,sinks", [(300, None, 3), (64, 16, 0), (5000, 4000, 100)])
def test_decode_of_the_longest_sequences(W, cap, window, sinks):
    """Lengths up to what int32 holds, and negative ones (idle)."""
    n = [2 ** 31 - 1, 2 ** 31 - 17, 2 ** 30, -5]
    q, kn, vn = rand(1, 4, 4, 64, dtype=BF16), rand(2, 4, 2, 64, dtype=BF16), rand(3, 4, 2, 64, dtype=BF16)
    kc, vc = rand(4, 4, cap, 2, 64, dtype=BF16), rand(5, 4, cap, 2, 64, dtype=BF16)
    want, bound, rk, rv = U.decode_reference(q, kc, vc, n, window=window, sinks=sinks, k_new=kn, v_new=vn)
    out = W.window_attention_decode(q, kc, vc, lens(*n), window=window, sinks=sinks, k_new=kn, v_new=vn)
    U.assert_within(out, want, bound, "out")
    assert torch.equal(kc, rk) and torch.equal(vc, rv)


def test_decode_all_scores_minus_infinity(W):
    """Keys of -inf alone: a row without keys, as in the prompt form; beside others they count nothing."""
    q = torch.ones(1, 1, 64, dtype=F16, device="cuda")
    kc, vc = torch.ones(1, 100, 1, 64, dtype=F16, device="cuda"), torch.ones(1, 100, 1, 64, dtype=F16, device="cuda")
    kc[0, :40, 0, 0] = -math.inf
    assert bool((W.window_attention_decode(q, kc, vc, lens(40)) == 0).all())
    assert bool((W.window_attention_decode(q, kc, vc, lens(100)) == 1).all())
    assert bool((W.window_attention_decode(q, kc, vc, lens(0)) == 0).all())


# ---------------------------------------------------------------------------
# activations: relative to their own size, also in the tails
# ---------------------------------------------------------------------------
E = U.E32
#: error of an activation relative to |act(z)| besides the argument's own, in half
#: steps of float32.  gelu: the tail's variable t = 1 / (1 + p u) is off by 3 (an fma, a
#: reciprocal of one step), which the tail takes 3.4 times at most (near u = 0); its ten
#: Horner steps 6; exp 2 and two roundings of its correction; three products.
#: sigmoid: exp 4, sum 1, reciprocal 2, products 3.
ACT_STEPS = {"gelu": 28, "silu": 14, "gelu_tanh": 14}


#: exponentials and sigmoids below float32's normal numbers may become 0
FLUSH = 2.0 ** -126


def tanh_argument(z):
    return 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)


def act64(z, kind):
    if kind == "gelu_tanh":  # (1 + tanh loses the negative tail even in 64 bits)
        return z * torch.sigmoid(tanh_argument(z))
    return U.act(z, kind)


def slope64(z, kind):
    if kind == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    x = tanh_argument(z) if kind == "gelu_tanh" else z
    dx = c * (1 + 3 * 0.044715 * z * z) if kind == "gelu_tanh" else 1.0
    return torch.sigmoid(x) * (1 + z * dx * torch.sigmoid(-x))


def argument_error(z, kind):
    """Relative change of the tail by what the argument of the exponential is off: gelu_tanh
    takes a polynomial that five roundings touch; the others keep theirs whole."""
    if kind != "gelu_tanh":
        return 0.0
    return 5 * E * tanh_argument(z).abs()


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [16, 4096])
def test_activation_values_relative(W, kind, out_dtype, rows):
    """z over [-12, 12], exact in 16 bits: what a (one column) times ones gives."""
    dtype = BF16 if out_dtype == BF16 else F16
    a = torch.zeros(rows, 8, dtype=dtype, device="cuda")
    a[:, 0] = torch.linspace(-12, 12, rows, device="cuda").to(dtype)
    trans = rows <= 16  # (few rows against [n, k] weights: the kernel without tiles)
    b = torch.zeros(264, 8, dtype=dtype, device="cuda") if trans else torch.zeros(8, 264, dtype=dtype, device="cuda")
    if trans:
        b[:, 0] = 1
        b = b.t()
    else:
        b[0] = 1
    out = W.matmul_epilogue(a, b, activation=kind, out_dtype=out_dtype)
    z = a[:, :1].double()
    y = act64(z, kind)
    err = (ACT_STEPS[kind] * E + argument_error(z, kind)) * y.abs() + FLUSH * z.abs()
    if out_dtype != F32:
        # for a 16-bit result the exponential's argument has three roundings more, and
        # gelu's polynomial is off by 1.1e-6
        size = {"gelu": z * z / 2, "silu": z.abs(), "gelu_tanh": tanh_argument(z).abs()}[kind]
        err = err + (1.2e-6 + 3 * E * size) * y.abs()
    bound = U.rounded(y, err, out_dtype)
    U.assert_within(out, y.expand(out.shape), bound.expand(out.shape), kind)


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation_slopes_relative(W, kind):
    """dbias of one row with dout 1 is the slope, in float32.  Each of its two terms is off by
    its own share, so near its zero the bound is that of the terms."""
    n = 8192
    pre = torch.linspace(-12, 12, n, device="cuda")[None].contiguous()
    dout = torch.ones(1, n, dtype=F16, device="cuda")
    a, b = torch.zeros(1, 8, dtype=F16, device="cuda"), torch.zeros(8, n, dtype=F16, device="cuda")
    _, _, slope = W.matmul_epilogue_backward(dout, a, b, pre=pre, activation=kind, need_a=False, need_b=False)
    z = pre[0].double()
    want = slope64(z, kind)
    first = act64(z, kind) / z  # Phi or the sigmoid
    steps = ACT_STEPS[kind] + 6
    # (what is flushed goes into the result times 1 + z times the argument's slope: 400 at most)
    U.assert_within(slope, want, (steps * E + argument_error(z, kind)) * (first.abs() + (want - first).abs()) + 400 * FLUSH, kind)


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("z,value,slope", [(math.inf, math.inf, 1.0), (-math.inf, 0.0, 0.0), (3e38, 3e38, 1.0), (-3e38, 0.0, 0.0),
                                           (1e19, 1e19, 1.0), (-1e19, 0.0, 0.0), (-200.0, 0.0, 0.0), (200.0, 200.0, 1.0), (0.0, 0.0, 0.5),
                                           (NAN, NAN, NAN)])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_activation_limits(W, kind, z, value, slope, out_dtype):
    a, b = torch.zeros(5, 0, dtype=BF16, device="cuda"), torch.zeros(0, 8, dtype=BF16, device="cuda")
    bias = torch.full((8,), z, device="cuda")
    out = W.matmul_epilogue(a, b, bias=bias, activation=kind, out_dtype=out_dtype)
    want = torch.full_like(out, value)
    assert bool(out.isnan().all()) if z != z else torch.equal(out, want), out[0, 0]
    pre = bias[None].contiguous()
    got = W.matmul_epilogue_backward(torch.ones(1, 8, dtype=BF16, device="cuda"), torch.zeros(1, 8, dtype=BF16, device="cuda"),
                                     torch.zeros(8, 8, dtype=BF16, device="cuda"), pre=pre, activation=kind)[2]
    assert bool(got.isnan().all()) if z != z else bool((got == slope).all()), got[0]


# ---------------------------------------------------------------------------
# float16 gradients of any size that their results have
# ---------------------------------------------------------------------------
def check_gradients(W, q, k, v, g, **kw):
    """Bounds without the absolute error that weights and their gradients would have as plain
    float16 numbers (2^-25): only the results' own rounding has one."""
    with mock.patch.object(U, "least", lambda dtype: 0.0):
        ref = U.attention_reference(q, k, v, dout=g, **kw)
    out, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    for name, x in zip(("dq", "dk", "dv"), W.window_attention_backward(g, q, k, v, out, lse, **kw)):
        want, bound = ref[name]
        # a packed gradient below 2^-37 of its row's largest, a weight below 2^-28, keeps 2^-39 at least
        bound = bound + U.least(q.dtype) + 2.0 ** -37 * want.abs().max()
        assert float(want.abs().max()) < 6e4, "the test's own results leave float16's range"
        U.assert_within(x, want, bound, name)


SHAPES = [(1, 40, 40, 2, 1, 64, dict()), (1, 300, 300, 4, 2, 80, dict(window=100, sinks=4)),
          (1, 1000, 1000, 2, 1, 128, dict(window=90, sinks=140)), (1, 20, 700, 6, 2, 32, dict())]


@pytest.mark.parametrize("b,lq,lk,h,kv,d,kw", SHAPES)
def test_large_gradients(W, b, lq, lk, h, kv, d, kw):
    """Loss-scaled: dP - D of 10^5 and more, whose product with the weights passes 65504, while
    dq, dk and dv fit float16."""
    q, k, v, g = qkv(5, b, lq, lk, h, kv, d, F16)
    q, k = q * 0.02, k * 0.02
    v, g = v * 30, g * (4000 if lq < lk else 1500)
    check_gradients(W, q, k, v, g, **kw)


@pytest.mark.parametrize("b,lq,lk,h,kv,d,kw", SHAPES)
@pytest.mark.parametrize("big", ["q", "k"])
def test_small_gradients(W, b, lq, lk, h, kv, d, kw, big):
    """dS of 10^-8 and below, whose sums with large keys or queries are ordinary numbers."""
    q, k, v, g = qkv(6, b, lq, lk, h, kv, d, F16)
    q, k = (q * 60, k * 0.01) if big == "q" else (q * 0.01, k * 60)
    check_gradients(W, q, k, v * 0.02, g * 2e-4, **kw)


def test_gradients_of_rows_of_very_different_size(W):
    """Rows of 10^4 and rows of 10^-5 in one call: where only the small ones meet, they keep
    their size; a key that both see has the large ones' error."""
    q, k, v, g = qkv(7, 1, 600, 600, 2, 2, 64, F16)
    g = g * torch.logspace(-5, 3, 600, device="cuda")[None, :, None, None].to(F16)
    check_gradients(W, q * 0.3, k * 0.3, v, g, window=30)
    check_gradients(W, q * 0.3, k * 0.3, v, g.flip(1).contiguous(), window=30)


def test_gradients_of_small_weights(W):
    """Beside a key of weight 1 all others have about e^-14 = 8e-7, less than float16's normal
    numbers: the values' gradient adds them as they are."""
    q, k, v, g = qkv(8, 1, 700, 700, 1, 1, 64, F16)
    q, k = q * 0.1 + 1, k * 0.1
    k[0, 0] = 1.75
    check_gradients(W, q, k, v, g * 200)


# ---------------------------------------------------------------------------
# calls that autograd would track
# ---------------------------------------------------------------------------
def test_tangents_are_refused(W):
    """A dual tensor does not require a gradient, and its tangent would be lost."""
    import torch.autograd.forward_ad as fwad
    a, b = rand(1, 16, 64, dtype=F16), rand(2, 64, 32, dtype=F16)
    q, k, v, g = qkv(1, 1, 8, 8, 2, 2, 64, F16)
    out, lse = W.window_attention(q, k, v, return_lse=True)
    n = torch.tensor([8], dtype=torch.int32, device="cuda")
    want = W.matmul_epilogue(a, b)

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return W.matmul_epilogue(x, b)

        @staticmethod
        def jvp(ctx, dx):
            return W.matmul_epilogue(dx.contiguous(), b)

    with fwad.dual_level():
        def dual(t):
            return fwad.make_dual(t, torch.ones_like(t))
        for call in (lambda: W.matmul_epilogue(dual(a), b), lambda: W.matmul_epilogue(a, dual(b)),
                     lambda: W.matmul_epilogue(a, b, bias=dual(rand(3, 32, dtype=F16))),
                     lambda: W.matmul_epilogue_backward(want, dual(a), b),
                     lambda: W.window_attention(dual(q), k, v), lambda: W.window_attention(q, k, dual(v)),
                     lambda: W.window_attention_backward(dual(g), q, k, v, out, lse),
                     lambda: W.window_attention_backward(g, q, k, v, out, dual(lse)),
                     lambda: W.window_attention_decode(dual(q)[:, 0], k, v, n)):
            with pytest.raises(ValueError, match="gradient"):
                call()
            with pytest.raises(ValueError, match="gradient"), torch.no_grad():  # (which keeps tangents)
                call()
        assert torch.equal(W.matmul_epilogue(a, b), want)  # others are not held up
        y, dy = fwad.unpack_dual(Product.apply(dual(a)))  # inside a Function's forward they are its own affair
        assert torch.equal(y, want) and torch.equal(dy, W.matmul_epilogue(torch.ones_like(a), b))
    assert torch.equal(W.matmul_epilogue(a, b), want)


def test_lse_that_requires_a_gradient_is_refused(W):
    q, k, v, g = qkv(1, 1, 8, 8, 2, 2, 64, F16)
    out, lse = W.window_attention(q, k, v, return_lse=True)
    want = W.window_attention_backward(g, q, k, v, out, lse)
    lse.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        W.window_attention_backward(g, q, k, v, out, lse)
    with torch.no_grad():
        got = W.window_attention_backward(g, q, k, v, out, lse)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---------------------------------------------------------------------------
# outputs that lie over inputs
# ---------------------------------------------------------------------------
def test_outputs_over_inputs_are_refused(W):
    flat = rand(1, 4096 + 64, dtype=F16)
    a, b = flat[:4096].view(64, 64), rand(2, 64, 64, dtype=F16)
    over = flat[64:].view(64, 64)  # one row further on
    bias = over[3]
    with pytest.raises(ValueError, match="out may not"):
        W.matmul_epilogue(a, b, out=over)
    with pytest.raises(ValueError, match="out may not"):
        W.matmul_epilogue(b, a, out=over)
    with pytest.raises(ValueError, match="out may not"):
        W.matmul_epilogue(b, a.t(), out=over)
    with pytest.raises(ValueError, match="out may not"):
        W.matmul_epilogue(b, b, bias=bias, out=over)
    with pytest.raises(ValueError, match="out may not"):
        W.matmul_epilogue(b, b, residual=a, out=over)
    wide = rand(3, 64, 128, dtype=F16)
    with pytest.raises(ValueError, match="out may not"):  # the same start, other rows
        W.matmul_epilogue(b, b, residual=wide.view(128, 64)[:64], out=wide[:, :64])
    want = W.matmul_epilogue(b, b, residual=wide[:, :64].contiguous())
    assert torch.equal(W.matmul_epilogue(b, b, residual=wide[:, :64], out=wide[:, :64]), want)
    # columns side by side of one buffer do not overlap
    joint = rand(4, 64, 192, dtype=F16)
    want = W.matmul_epilogue(joint[:, :64], b)
    assert torch.equal(W.matmul_epilogue(joint[:, :64], b, out=joint[:, 64:128]), want)

    buf = rand(5, 2 * 8 * 2 * 64 + 128, dtype=F16)
    q, o = buf[:2048].view(2, 8, 2, 64), buf[128:].view(2, 8, 2, 64)
    k, v = rand(6, 2, 8, 2, 64, dtype=F16), rand(7, 2, 8, 2, 64, dtype=F16)
    for x in ((q, k, v), (k, q, v), (k, v, q)):
        with pytest.raises(ValueError, match="out may not"):
            W.window_attention(*x, out=o)
    n = torch.tensor([8, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="out may not"):
        W.window_attention_decode(k[:, 0], q, v, n, out=buf[128:384].view(2, 2, 64))
    with pytest.raises(ValueError, match="out may not"):
        W.window_attention_decode(k[:, 0], k, v, n, k_new=buf[:256].view(2, 2, 64), v_new=v[:, 1], out=buf[128:384].view(2, 2, 64))


def test_one_cache_for_keys_and_values_cannot_take_a_token(W):
    q, kc, kn = rand(1, 1, 2, 64, dtype=F16), rand(2, 1, 8, 2, 64, dtype=F16), rand(3, 1, 2, 64, dtype=F16)
    n = torch.tensor([5], dtype=torch.int32, device="cuda")
    with pytest.raises(W._lib.WtcError, match="same"):
        W.window_attention_decode(q, kc, kc, n, k_new=kn, v_new=kn + 1)
    want = W.window_attention_decode(q, kc, kc.clone(), n)
    assert torch.equal(W.window_attention_decode(q, kc, kc, n), want)


@pytest.mark.parametrize("n", [40, 400])
def test_a_nan_value_of_weight_0_in_the_gradients(W, n):
    """0 * NaN in a row's result makes its D NaN, and with it the gradient of every key that the
    row sees: also in rows of few keys, which sum D themselves."""
    q, k = torch.ones(1, n, 1, 64, dtype=BF16, device="cuda"), rand(1, 1, n, 1, 64, dtype=BF16, by=0.1)
    v, g = rand(2, 1, n, 1, 64, dtype=BF16), rand(3, 1, n, 1, 64, dtype=BF16)
    k[0, 3] = -40  # its scores are 320 below the others'
    v[0, 3, 0] = NAN
    out, lse = W.window_attention(q, k, v, return_lse=True)
    dq, dk, dv = W.window_attention_backward(g, q, k, v, out, lse)
    assert bool(out[0, 3:].isnan().all()) and bool(out[0, :3].isfinite().all())
    assert bool(dq[0, 3:].isnan().all()) and bool(dk.isnan().all())
    assert bool(dq[0, :3].isfinite().all()) and bool(dv.isfinite().all())


# ---------------------------------------------------------------------------
# the kernels that large calls run
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("size,tile", LARGE_PRODUCTS)
@pytest.mark.parametrize("dtype,out_dtype,kind,bias,residual,trans", [
    (BF16, BF16, "gelu", BF16, True, False), (F16, F32, "silu", F32, True, True), (BF16, F32, "none", None, False, False),
    (F16, F16, "gelu_tanh", F16, True, True), (BF16, BF16, "relu", None, False, True), (F16, F32, "gelu", F16, True, False)])
def test_large_products(W, size, tile, dtype, out_dtype, kind, bias, residual, trans):
    m, n, k = size
    assert matmul_epilogue_plan(m, n, k, b_trans=trans)[:2] == tile
    a = rand(1, m, k, dtype=dtype)
    b = rand(2, n, k, dtype=dtype, by=0.1).t() if trans else rand(2, k, n, dtype=dtype, by=0.1)
    bv = None if bias is None else rand(3, n, dtype=bias)
    r = rand(4, m, n, dtype=out_dtype) if residual else None
    out, pre = W.matmul_epilogue(a, b, bias=bv, residual=r, activation=kind, out_dtype=out_dtype, return_pre=True)
    y, z, dz, dy = U.matmul_reference(a, b, bv, r, kind)
    U.assert_within(out, y, U.rounded(y, dy, out_dtype), "out")
    U.assert_within(pre, z, U.rounded(z, dz, F32), "pre")
    wide = torch.full((m, n + 16), 7.0, dtype=out_dtype, device="cuda")  # what is between an out's rows stays
    again = W.matmul_epilogue(a, b, bias=bv, residual=r, activation=kind, out=wide[:, 8:n + 8])
    assert torch.equal(out, again) and bool((wide[:, :8] == 7).all()) and bool((wide[:, n + 8:] == 7).all())


@pytest.mark.parametrize("size,part,tile,split", LARGE_GRADIENTS)
@pytest.mark.parametrize("dtype,trans,kind", [(BF16, False, "none"), (F16, True, "silu"), (BF16, True, "relu"), (F16, False, "gelu")])
def test_large_gradients_of_products(W, size, part, tile, split, dtype, trans, kind):
    m, n, k = size
    *got, splits = matmul_epilogue_plan(m, n, k, b_trans=trans, part=part)
    assert tuple(got) == tile and (splits > 1) == split
    a, dout, pre = rand(1, m, k, dtype=dtype), rand(3, m, n, dtype=dtype), rand(4, m, n)
    b = rand(2, n, k, dtype=dtype, by=0.1).t() if trans else rand(2, k, n, dtype=dtype, by=0.1)
    da, db, dbias = W.matmul_epilogue_backward(dout, a, b, pre=None if kind == "none" else pre, activation=kind)
    dz = dout.double() * U.act_slope(pre.double(), kind)
    # the slope's own error (64 half steps of its terms, which are at most 1 and |z| in size), then dz's rounding
    ez = dout.double().abs() * (0 if kind in ("none", "relu") else 64 * U.E32 * (1 + pre.double().abs()))
    err = 0 * dz if kind == "none" else ez + U.half_step(dtype) * (dz.abs() + ez) + U.least(dtype)
    size_of = dz.abs() + err
    bd, ad = b.double(), a.double()
    ref = dz @ bd.t()
    U.assert_within(da, ref, U.rounded(ref, (err + 2 * (n + 2) * U.E32 * size_of) @ bd.t().abs(), dtype), "da")
    ref = ad.t() @ dz
    U.assert_within(db, ref, U.rounded(ref, ad.t().abs() @ (err + 2 * (m + 2) * U.E32 * size_of), dtype), "db")
    U.assert_within(dbias, dz.sum(0), (ez + 2 * (m + 2) * U.E32 * size_of).sum(0), "dbias")
    again = W.matmul_epilogue_backward(dout, a, b, pre=None if kind == "none" else pre, activation=kind)
    assert all(torch.equal(x, y) for x, y in zip((da, db, dbias), again))


@pytest.mark.parametrize("b,h,kv,lq,lk,d,kw", FULL_CHIP)
@pytest.mark.parametrize("dtype,ragged", [(BF16, False), (F16, True)])
def test_attention_on_a_full_chip(W, b, h, kv, lq, lk, d, kw, dtype, ragged):
    """A wave to each row: rings of three stages forward, four waves a block in dq."""
    plan = window_attention_plan(b, h, kv, lq, lk, d, **kw)
    assert plan["row_waves"] == 1 and plan["dq_row_waves"] == 1
    q, k, v, g = qkv(91, b, lq, lk, h, kv, d, dtype)
    if ragged:
        q_lens = torch.tensor([(lq + 1) * i // b for i in range(b)], dtype=torch.int32, device="cuda")
        k_lens = torch.tensor([(lk + 1) * ((7 * i + 3) % b + 1) // b for i in range(b)], dtype=torch.int32, device="cuda")
        for i in range(b):  # nothing behind the ends is read
            for t, n in ((q, q_lens), (g, q_lens), (k, k_lens), (v, k_lens)):
                t[i, int(n[i]):] = NAN
        kw = dict(kw, q_lens=q_lens, k_lens=k_lens)
    ref = U.attention_reference(q, k, v, dout=g, **kw)
    out, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    U.assert_within(out, *ref["out"], "out")
    empty = ref["lse"][0] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    U.assert_within(torch.where(empty, 0.0, lse), torch.where(empty, 0.0, ref["lse"][0]), ref["lse"][1], "lse")
    got = W.window_attention_backward(g, q, k, v, out, lse, **kw)
    for name, x in zip(("dq", "dk", "dv"), got):
        U.assert_within(x, *ref[name], name)
    assert torch.equal(out, W.window_attention(q, k, v, **kw))
    again = W.window_attention_backward(g, q, k, v, out, lse, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("bad", [NAN, -math.inf])
@pytest.mark.parametrize("name", ["k", "v", "q", "g"])
def test_bad_values_on_a_full_chip(W, bad, name):
    """As with two waves a row: a bad value in one sequence reaches the rows of that sequence
    that see it and no other."""
    b, n, window, sinks, at = 280, 200, 30, 2, 150
    kw = dict(window=window, sinks=sinks)
    plan = window_attention_plan(b, 2, 1, n, n, 64, **kw)
    assert plan["row_waves"] == 1 and plan["dq_row_waves"] == 1
    q, k, v, g = qkv(95, b, n, n, 2, 1, 64, F16)
    clean, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    want = (clean, *W.window_attention_backward(g, q, k, v, clean, lse, **kw))
    dict(q=q, k=k, v=v, g=g)[name][5, at, 0, 9] = bad
    out, lse = W.window_attention(q, k, v, return_lse=True, **kw)
    got = (out, *W.window_attention_backward(g, q, k, v, out, lse, **kw))
    pos = torch.arange(n, device="cuda")
    one_head = name in ("q", "g")
    rows = pos == at if one_head else (pos >= at) & (pos < at + window)
    keys = U.seen_mask(n, n, n, n, window, sinks, "cuda")[rows].any(0)
    none = torch.zeros_like(rows)
    touched = (none if name == "g" else rows, rows, keys, none if name == "v" else keys)
    others = [i for i in range(b) if i != 5]
    clean5 = [t[5:6].clone() for t in qkv(95, b, n, n, 2, 1, 64, F16)]
    ref = U.attention_reference(*clean5[:3], dout=clean5[3], **kw)
    for what, x, y, t in zip(("out", "dq", "dk", "dv"), got, want, touched):
        assert torch.equal(x[others], y[others]), (name, what)
        r, bound = ref[what]
        U.assert_within(x[5:6, ~t], r[:, ~t], bound[:, ~t], (name, what))
