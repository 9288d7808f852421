"""Cross attention, attention behind a shared prefix and their gradients where kernels change
hands, on the GPU against plain 64-bit forms (tests/masked_util.py)."""
import pytest
import torch

from tests import layer_util as U
from tests.layer_util import E32, ELEM, half_step, least
from tests.test_gpu_masked import BF16, F16, W, check_prefix, cross_inputs, lens, prefix_inputs, rand  # noqa: F401

pytestmark = pytest.mark.gpu


# one launch, at most as many workgroups as CUs: one row block a wave, whose loop is shortest
# (two k-steps) up to dim 32
@pytest.mark.parametrize("b,n,lq,lk,h,kv,d", [(16, 500, 200, 200, 16, 2, 32), (2, 8000, 70, 70, 4, 2, 32), (1, 16000, 130, 135, 2, 1, 16),
                                              (8, 2100, 100, 160, 8, 4, 8)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefix_small_dims(W, b, n, lq, lk, h, kv, d, dtype):  # noqa: F811
    args = prefix_inputs(301, b, n, lq, lk, h, kv, d, dtype)
    out = check_prefix(W, *args)
    cold = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for _ in range(3):  # keys and values from memory, later than the loop would like
        cold.zero_()
        assert torch.equal(out, W.prefix_attention(*args))


def gradients_of_few_keys(q, k, v, g, scale):
    """(dq, dk) of one sequence and their bounds where D = sum_j P dP is summed in float32, not
    taken from the rounded `out`: dS keeps float32's error of P, dP and D and the one rounding
    before its products.  q, g [lq, h, d]; k, v [lk, kv, d]."""
    (lq, h, d), (lk, kv, _) = q.shape, k.shape
    u = half_step(q.dtype)
    dq, dk = torch.zeros(2, lq, h, d, dtype=torch.float64, device="cuda"), torch.zeros(2, lk, kv, d, dtype=torch.float64, device="cuda")
    for x in range(h):
        y = x * kv // h
        qq, kk, vv, gg = q[:, x].double(), k[:, y].double(), v[:, y].double(), g[:, x].double()
        s = qq @ kk.t() * scale
        lse = torch.logsumexp(s, 1, keepdim=True)
        p, dp = torch.exp(s - lse), gg @ vv.t()
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        # relative error of a weight: its score's, the log-sum-exp's with its own rounding, the exponential
        dot = 2 * (d + 2) * E32
        score = scale * dot * (qq.abs() @ kk.abs().t()) + ELEM * s.abs()
        rel = 2 * score.amax(1, keepdim=True) + (2 * lk + 80) * E32 + 4 * ELEM + 12 * E32 * lse.abs()
        dpe = dot * (gg.abs() @ vv.abs().t())
        # of D: that of each P dP, and of their sum
        de = (p * (rel * dp.abs() + dpe)).sum(1, keepdim=True) + 2 * (lk + 2) * E32 * (p * dp.abs()).sum(1, keepdim=True)
        # the products start from -D: two more roundings at its size
        size = dp.abs() + (p * dp).sum(1, keepdim=True).abs()
        dse = rel * ds.abs() + p * (dpe + de + 4 * E32 * size)
        err = dse + u * (ds.abs() + dse) + least(q.dtype)
        mass = p * size
        dq[0, :, x] = scale * (ds @ kk)
        dq[1, :, x] = scale * ((err + 2 * lk * E32 * mass) @ kk.abs())
        dk[0, :, y] += scale * (ds.t() @ qq)
        dk[1, :, y] += scale * ((err + 2 * (lq * h // kv + 2) * E32 * mass).t() @ qq.abs())
    return [(r, U.rounded(r, e, q.dtype)) for r, e in (dq, dk)]


# Sequences of few keys beside longer ones.  The values differ by one step of their type, so
# that `out` is off by up to half of what they differ by: a D from it is far outside the bound.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lk,n", [(300, (1, 5, 300)), (300, (40, 128, 129)), (140, (2, 64, 65)), (128, (1, 40, 128))])
@pytest.mark.parametrize("lq,h,kv,d", [(100, 4, 2, 64), (7, 3, 1, 128), (333, 1, 1, 24)])
def test_cross_gradients_of_few_keys_in_a_padded_batch(W, lq, h, kv, d, lk, n, dtype):  # noqa: F811
    q, k, _, g = cross_inputs(311, 3, lq, lk, h, kv, d, dtype)
    step = 2 * torch.finfo(dtype).eps  # of numbers from 2 to 4
    v = (2 + rand(315, 1, 1, kv, d).abs().clamp(max=1.5) + step * (rand(316, 3, lk, kv, d) > 0)).to(dtype)
    queries = (lq, lq, lq - lq // 2)
    nq, nk = lens(*queries), lens(*n)
    out, lse = W.cross_attention(q, k, v, q_lens=nq, k_lens=nk, return_lse=True)
    dq, dk, dv = W.cross_attention_backward(g, q, k, v, out, lse, q_lens=nq, k_lens=nk)
    for i, (x, y) in enumerate(zip(queries, n)):
        if y <= 128:
            refs = gradients_of_few_keys(q[i, :x], k[i, :y], v[i, :y], g[i, :x], d ** -0.5)
            U.assert_within(dq[i, :x], *refs[0], f"dq of {y} keys")
            U.assert_within(dk[i, :y], *refs[1], f"dk of {y} keys")
        assert not dq[i, x:].any() and not dk[i, y:].any() and not dv[i, y:].any() and not out[i, x:].any()
        assert bool(torch.isneginf(lse[i, :, x:]).all()) and bool(torch.isfinite(lse[i, :, :x]).all())


def test_heads_over_2_gib_apart(W):  # noqa: F811
    """Each key head has one query head, and the heads of q and dout are further apart than 32-bit offsets reach."""
    b, lq, lk, h, d = 2, 70, 150, 2, 64
    q, k, v, g = cross_inputs(321, b, lq, lk, h, h, d, BF16)
    strides = (lq * d, d, (1 << 30) + 64, 1)
    far = []
    for x in (q, g):
        buffer = torch.empty(strides[2] + b * lq * d, dtype=BF16, device="cuda")
        far.append(buffer.as_strided(x.shape, strides).copy_(x))
    nk = lens(150, 90)
    out, lse = W.cross_attention(q, k, v, k_lens=nk, return_lse=True)
    assert torch.equal(out, W.cross_attention(far[0], k, v, k_lens=nk))
    for x, y in zip(W.cross_attention_backward(g, q, k, v, out, lse, k_lens=nk),
                    W.cross_attention_backward(far[1], far[0], k, v, out, lse, k_lens=nk)):
        assert torch.equal(x, y)
    out, lse = W.window_attention(q, k, v, window=40, k_lens=nk, return_lse=True)
    for x, y in zip(W.window_attention_backward(g, q, k, v, out, lse, window=40, k_lens=nk),
                    W.window_attention_backward(far[1], far[0], k, v, out, lse, window=40, k_lens=nk)):
        assert torch.equal(x, y)
    assert torch.equal(W.window_attention_weights(q, k, lse, window=40, k_lens=nk),
                       W.window_attention_weights(far[0], k, lse, window=40, k_lens=nk))
