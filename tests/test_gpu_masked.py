"""Cross attention, attention behind a shared prefix, what keys receive and a cache cut
by it, on the GPU against plain 64-bit forms (tests/masked_util.py)."""
import math

import pytest
import torch

from tests import layer_util as U
from tests import masked_util as M
from welder_typical_chain_amd import _lib

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")
KINDS = [(BF16, 4, 2, 128), (F16, 3, 3, 64), (F16, 5, 1, 80)]


@pytest.fixture(scope="module")
def W(native_lib):
    import welder_typical_chain_amd as w
    return w


def rand(seed, *shape, dtype=F32, by=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * by).to(dtype)


def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def within(got, ref, what):
    """As U.assert_within, where the reference may be -inf (a row that sees nothing)."""
    value, bound = ref
    empty = torch.isneginf(value)
    assert torch.equal(torch.isneginf(got), empty), what
    U.assert_within(torch.where(empty, 0.0, got.double()), torch.where(empty, 0.0, value), torch.where(empty, 0.0, bound), what)


# ---------------------------------------------------------------------------
# cross attention
# ---------------------------------------------------------------------------
def check_cross(W, q, k, v, g=None, **kw):
    at = {x: kw[x] for x in ("q_lens", "k_lens") if x in kw}
    mask = M.cross_mask(q.shape[0], q.shape[1], k.shape[1], kw.get("q_lens"), kw.get("k_lens"), q.device)
    ref = M.attention(q, k, v, mask, scale=kw.get("scale"), dout=g)
    out, lse = W.cross_attention(q, k, v, return_lse=True, **kw)
    within(out, ref["out"], "out")
    within(lse, ref["lse"], "lse")
    assert torch.equal(out, W.cross_attention(q, k, v, **kw)), "two calls differ"
    if g is not None:
        got = W.cross_attention_backward(g, q, k, v, out, lse, **kw)
        for x, y in zip(("dq", "dk", "dv"), got):
            within(y, ref[x], x)
        for y, z in zip(got, W.cross_attention_backward(g, q, k, v, out, lse, **kw)):
            assert torch.equal(y, z), "two calls differ"
    assert set(at) <= {"q_lens", "k_lens"}
    return out


def cross_inputs(seed, b, lq, lk, h, kv, d, dtype):
    return (rand(seed, b, lq, h, d, dtype=dtype), rand(seed + 1, b, lk, kv, d, dtype=dtype),
            rand(seed + 2, b, lk, kv, d, dtype=dtype), rand(seed + 3, b, lq, h, d, dtype=dtype))


@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 65), (1, 1030), (2, 33), (7, 700), (64, 64), (65, 1), (130, 70), (257, 63),
                                   (300, 513)])
@pytest.mark.parametrize("dtype,h,kv,d", KINDS)
def test_cross_sizes(W, lq, lk, dtype, h, kv, d):
    check_cross(W, *cross_inputs(1, 2, lq, lk, h, kv, d, dtype))


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 72, 96, 120, 128])
@pytest.mark.parametrize("lq", [1, 70])
def test_cross_dims(W, d, lq):
    check_cross(W, *cross_inputs(5, 2, lq, 150, 4, 2, d, BF16))


@pytest.mark.parametrize("h,kv", [(1, 1), (8, 1), (6, 2), (7, 7), (33, 1), (64, 1), (70, 1), (140, 2)])
@pytest.mark.parametrize("lq", [1, 3, 40])
def test_cross_heads(W, h, kv, lq):
    check_cross(W, *cross_inputs(9, 1, lq, 200, h, kv, 32, F16))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("lq", [1, 50])
def test_cross_scales(W, scale, lq):
    check_cross(W, *cross_inputs(13, 1, lq, 90, 2, 2, 64, F16), scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,lk", [(90, 200), (1, 200), (4, 1000)])
def test_cross_padded_batch_with_nan_behind_the_ends(W, dtype, lq, lk):
    q, k, v, g = cross_inputs(17, 6, lq, lk, 4, 2, 64, dtype)
    nq, nk = lens(lq, max(1, lq // 2), 0, lq, lq + 9, -3), lens(lk, 0, lk // 3, 1, lk + 5, 17)
    for i in range(6):
        q[i, max(0, int(nq[i])):] = NAN
        g[i, max(0, int(nq[i])):] = NAN
        k[i, max(0, int(nk[i])):] = NAN
        v[i, max(0, int(nk[i])):] = math.inf
    out = check_cross(W, q, k, v, g, q_lens=nq, k_lens=nk)
    assert not out[1].any() and not out[2].any()
    check_cross(W, q[:1], k[:1], v[:1], g[:1], q_lens=nq[:1])
    check_cross(W, q[3:4], k[3:4], v[3:4], g[3:4], k_lens=nk[3:4])


def test_cross_strides(W):
    wide = rand(21, 2, 4, 150, 3 * 64, dtype=BF16)  # [B, H, L, D] inside wider rows
    k, v = (wide[:, :2, :, x:x + 64].transpose(1, 2) for x in (0, 64))
    q = wide[:, :, 20:60, 128:].transpose(1, 2)
    g = rand(22, 2, 40, 4, 64, dtype=BF16)
    check_cross(W, q, k, v, g)
    into = torch.full((2, 4, 40, 64), 7.0, dtype=BF16, device="cuda").transpose(1, 2)
    assert torch.equal(W.cross_attention(q, k, v, out=into), W.cross_attention(q.contiguous(), k.contiguous(), v.contiguous()))
    one = rand(23, 1, 40, 4, 64, dtype=BF16)
    out, lse = W.cross_attention(one, k[:1], v[:1], return_lse=True)
    same = W.cross_attention_backward(rand(24, 1, 1, 4, 64, dtype=BF16).expand(1, 40, 4, 64), one, k[:1], v[:1], out, lse)
    again = W.cross_attention_backward(rand(24, 1, 1, 4, 64, dtype=BF16).expand(1, 40, 4, 64).contiguous(), one, k[:1], v[:1], out, lse)
    assert all(torch.equal(x, y) for x, y in zip(same, again))
    states = rand(25, 1, 300, 2, 64, dtype=BF16).expand(3, 300, 2, 64)  # one sequence of states for a batch
    check_cross(W, rand(26, 3, 2, 4, 64, dtype=BF16), states, states)


@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("lq", [1, 90])
def test_cross_bad_values_stay_in_their_sequence(W, bad, lq):
    q, k, v, g = cross_inputs(31, 3, lq, 140, 4, 2, 64, F16)
    clean = W.cross_attention(q, k, v)
    v[1, 77, 1, 5] = bad
    out, lse = W.cross_attention(q, k, v, return_lse=True)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert torch.equal(out[1, :, :2], clean[1, :, :2])  # the query heads of the other key head
    hit = out[1, :, 2:, 5]
    assert bool((torch.isnan(hit) if bad != bad else hit == bad).all())
    assert bool(torch.isfinite(out[1, :, 2:, :5]).all())
    q[0, 0, 0, 3] = bad
    out, lse = W.cross_attention(q, k, v, return_lse=True)
    assert bool(torch.isnan(out[0, 0, 0]).all()) and torch.equal(out[2], clean[2])
    assert torch.equal(out[0, 1:], clean[0, 1:]) and torch.equal(out[0, 0, 1:], clean[0, 0, 1:])
    dq, dk, dv = W.cross_attention_backward(g, q, k, v, out, lse)
    assert bool(torch.isfinite(dq[2]).all()) and bool(torch.isfinite(dk[2]).all()) and bool(torch.isfinite(dv[2]).all())


def test_cross_all_scores_minus_infinity_and_large_ones(W):
    q, k, v, _ = cross_inputs(35, 1, 40, 100, 2, 2, 64, BF16)
    q[0, :, :, 0], k[0, :, :, 0] = -1e30, 3e38
    q[0, :, :, 1:] = 0
    out, lse = W.cross_attention(q, k, v, return_lse=True)
    assert bool(torch.isneginf(lse).all()) and not out.any()
    q, k, v, g = cross_inputs(36, 1, 40, 300, 2, 2, 64, F16)
    check_cross(W, 30 * q, k, v)


def test_cross_empty(W):
    for b, lq, lk in [(0, 4, 4), (2, 0, 5), (2, 5, 0)]:
        q, k, v, g = cross_inputs(39, b, lq, lk, 4, 2, 32, F16)
        out, lse = W.cross_attention(q, k, v, return_lse=True)
        assert not out.any() and bool(torch.isneginf(lse).all())
        dq, dk, dv = W.cross_attention_backward(g, q, k, v, out, lse)
        assert not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("b,lq,lk,h,kv,d", [(40, 130, 150, 8, 8, 64), (30, 1, 300, 32, 8, 128), (3, 1000, 700, 6, 3, 80),
                                            (1, 2100, 90, 8, 2, 128), (1, 64, 5000, 4, 4, 64), (200, 2, 65, 4, 2, 96),
                                            # more workgroups than CUs: two row blocks a wave, at every width
                                            (70, 150, 200, 8, 4, 128), (90, 100, 130, 6, 3, 96), (130, 140, 100, 4, 4, 40),
                                            (300, 70, 33, 1, 1, 16),
                                            # few workgroups: keys split, gradients in one launch or in two
                                            (1, 300, 3000, 2, 2, 128), (1, 90, 2500, 5, 5, 24), (2, 400, 129, 4, 4, 96), (2, 600, 900, 12, 4, 64),
                                            # a group of over 64 heads in tiles of 128 rows
                                            (1, 30, 300, 100, 1, 64), (1, 9, 200, 260, 2, 32)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cross_large(W, b, lq, lk, h, kv, d, dtype):
    check_cross(W, *cross_inputs(43, b, lq, lk, h, kv, d, dtype))


# ---------------------------------------------------------------------------
# a shared prefix
# ---------------------------------------------------------------------------
def prefix_inputs(seed, b, n, lq, lk, h, kv, d, dtype):
    return (rand(seed, b, lq, h, d, dtype=dtype), rand(seed + 1, n, kv, d, dtype=dtype), rand(seed + 2, n, kv, d, dtype=dtype),
            rand(seed + 3, b, lk, kv, d, dtype=dtype), rand(seed + 4, b, lk, kv, d, dtype=dtype))


def check_prefix(W, q, kp, vp, k, v, **kw):
    b, lq = q.shape[:2]
    own = M.causal_mask(b, lq, k.shape[1], kw.get("q_lens"), kw.get("k_lens"), q.device)
    query = M.cross_mask(b, lq, kp.shape[0], kw.get("q_lens"), None, q.device)
    ref = M.attention(q, *M.prefix_inputs(kp, vp, k, v, torch.cat([query, own], 2)), scale=kw.get("scale"))
    out, lse = W.prefix_attention(q, kp, vp, k, v, return_lse=True, **kw)
    within(out, ref["out"], "out")
    within(lse, ref["lse"], "lse")
    assert torch.equal(out, W.prefix_attention(q, kp, vp, k, v, **kw)), "two calls differ"
    return out


@pytest.mark.parametrize("n", [0, 1, 63, 65, 700, 2100])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 40), (5, 5), (33, 130), (200, 200), (3, 2), (4, 0)])
@pytest.mark.parametrize("dtype,h,kv,d", KINDS)
def test_prefix_sizes(W, n, lq, lk, dtype, h, kv, d):
    check_prefix(W, *prefix_inputs(51, 3, n, lq, lk, h, kv, d, dtype))


@pytest.mark.parametrize("b", [1, 2, 17, 130])
@pytest.mark.parametrize("lq", [1, 6])
def test_prefix_batches(W, b, lq):
    check_prefix(W, *prefix_inputs(55, b, 1000, lq, 20, 8, 2, 64, BF16))


@pytest.mark.parametrize("b,n,lq,lk,h,kv,d", [
    (70, 90, 100, 100, 4, 4, 128), (90, 65, 90, 130, 6, 3, 96), (300, 40, 130, 130, 2, 2, 64), (300, 33, 140, 140, 1, 1, 24),  # full chips
    (1, 5000, 150, 300, 2, 2, 128), (2, 3000, 64, 64, 8, 2, 80), (1, 4001, 500, 500, 1, 1, 64),  # keys split
    (2, 31, 200, 200, 2, 1, 128), (2, 32, 200, 231, 2, 1, 96), (2, 95, 130, 130, 1, 1, 64), (2, 96, 257, 300, 1, 1, 32),  # units' ends
    (130, 5000, 32, 40, 8, 2, 128), (70, 4000, 20, 20, 16, 4, 96)])  # over 64 rows a sequence, in two launches
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefix_large(W, b, n, lq, lk, h, kv, d, dtype):
    check_prefix(W, *prefix_inputs(57, b, n, lq, lk, h, kv, d, dtype))


@pytest.mark.parametrize("d", [8, 24, 40, 96, 120])
@pytest.mark.parametrize("h,kv", [(3, 1), (70, 1)])
def test_prefix_dims_and_heads(W, d, h, kv):
    check_prefix(W, *prefix_inputs(59, 2, 300, 9, 20, h, kv, d, F16), scale=-0.2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,n", [(50, 300), (2, 1500), (150, 64)])
def test_prefix_padded_batch_with_nan_behind_the_ends(W, dtype, lq, n):
    q, kp, vp, k, v = prefix_inputs(63, 5, n, lq, lq + 30, 4, 2, 64, dtype)
    nq, nk = lens(lq, lq // 2, 0, 1, lq), lens(lq + 30, lq // 2, 5, 20, 0)
    for i in range(5):
        q[i, int(nq[i]):] = NAN
        k[i, int(nk[i]):] = NAN
        v[i, int(nk[i]):] = math.inf
    out = check_prefix(W, q, kp, vp, k, v, q_lens=nq, k_lens=nk)
    assert not out[2].any() and not out[3, 1:].any()


def test_prefix_hides_later_tokens(W):
    q, kp, vp, k, v = prefix_inputs(67, 2, 500, 100, 100, 4, 2, 64, F16)
    own = M.causal_mask(2, 100, 100, None, None, "cuda")
    keys, values, mask = M.prefix_inputs(kp, vp, k, v, torch.cat([torch.ones(2, 100, 500, dtype=torch.bool, device="cuda"), own], 2))
    clean = M.attention(q, keys, values, mask)["out"]
    v[0, 60, 0, 3], k[1, 70, 1] = NAN, math.inf
    out = W.prefix_attention(q, kp, vp, k, v)

    def unchanged(*at):
        within(out[at], (clean[0][at], clean[1][at]), f"rows {at}")

    every = slice(None)
    unchanged(0, slice(0, 60))
    unchanged(1, slice(0, 70))
    assert bool(torch.isnan(out[0, 60:, :2, 3]).all()) and bool(torch.isnan(out[1, 70:, 2:]).all())
    unchanged(0, every, slice(2, 4))
    unchanged(1, every, slice(0, 2))
    vp[499, 1, 0] = NAN
    out = W.prefix_attention(q, kp, vp, k, v)
    assert bool(torch.isnan(out[:, :, 2:, 0]).all())
    unchanged(0, slice(0, 60), slice(0, 2))


def test_prefix_strides(W):
    store = rand(71, 2, 600, 2, 3, 64, dtype=BF16)  # keys and values beside each other in one buffer
    kp, vp = store[0, :500, :, 0], store[0, :500, :, 2]
    k, v = store[:, 500:540, :, 1], store[:, 520:560, :, 0]
    q = rand(72, 2, 4, 40, 64, dtype=BF16).transpose(1, 2)
    check_prefix(W, q, kp, vp, k, v)
    check_prefix(W, q[:, 39:], kp, vp, k, v)
    heads_first = rand(73, 2, 500, 64, dtype=BF16).transpose(0, 1)
    check_prefix(W, q, heads_first, heads_first, k, v)


def check_prefix_decode(W, b, n, cap, lengths, h, kv, d, dtype, new, seed=81):
    q, kp, vp = rand(seed, b, h, d, dtype=dtype), rand(seed + 1, n, kv, d, dtype=dtype), rand(seed + 2, n, kv, d, dtype=dtype)
    kc, vc = rand(seed + 3, b, cap, kv, d, dtype=dtype), rand(seed + 4, b, cap, kv, d, dtype=dtype)
    kn, vn = (rand(seed + 5 + x, b, kv, d, dtype=dtype) if new else None for x in range(2))
    ref = M.decode(q, kc, vc, lengths, kp, vp, k_new=kn, v_new=vn)
    out = W.prefix_attention_decode(q, kp, vp, kc, vc, lengths, k_new=kn, v_new=vn)
    within(out, ref["out"], "out")
    assert torch.equal(kc, ref["k_cache"]) and torch.equal(vc, ref["v_cache"])
    assert torch.equal(out, W.prefix_attention_decode(q, kp, vp, kc, vc, lengths)), "two calls differ"


@pytest.mark.parametrize("n", [0, 1, 64, 333, 3000])
@pytest.mark.parametrize("cap,lengths", [(1, (1, 0, 3)), (40, (1, 40, 0)), (64, (100, 64, 33)), (700, (650, 1, 90))])
@pytest.mark.parametrize("dtype,h,kv,d", KINDS)
def test_prefix_decode(W, n, cap, lengths, dtype, h, kv, d):
    for new in (True, False):
        check_prefix_decode(W, 3, n, cap, lens(*lengths), h, kv, d, dtype, new)


@pytest.mark.parametrize("b,n,h,kv,d", [(1, 5000, 8, 8, 128), (130, 200, 8, 2, 64), (64, 2000, 32, 8, 128), (5, 900, 40, 1, 80),
                                        (2, 700, 70, 1, 24)])
def test_prefix_decode_batches(W, b, n, h, kv, d):
    check_prefix_decode(W, b, n, 90, torch.arange(b, dtype=torch.int32, device="cuda") % 91, h, kv, d, BF16, True)


def test_prefix_decode_reads_only_what_is_seen(W):
    b, n, cap = 3, 200, 80
    q, kp, vp = rand(85, b, 4, 64, dtype=F16), rand(86, n, 2, 64, dtype=F16), rand(87, n, 2, 64, dtype=F16)
    kc, vc = rand(88, b, cap, 2, 64, dtype=F16), rand(89, b, cap, 2, 64, dtype=F16)
    at = lens(10, 0, 77)
    want = W.prefix_attention_decode(q, kp, vp, kc, vc, at)
    for i, m in enumerate((10, 0, 77)):
        kc[i, m:], vc[i, m:] = NAN, NAN
    q[1] = NAN
    got = W.prefix_attention_decode(q, kp, vp, kc, vc, at)
    assert torch.equal(got, want) and not got[1].any()
    kp[5, 1] = NAN
    got = W.prefix_attention_decode(q, kp, vp, kc, vc, at)
    assert torch.equal(got[:, :2], want[:, :2]) and not got[1].any() and bool(torch.isnan(got[0, 2:]).all())


# ---------------------------------------------------------------------------
# what the keys receive
# ---------------------------------------------------------------------------
def check_weights(W, q, k, window=None, sinks=0, scale=None, q_lens=None, k_lens=None):
    b, lq = q.shape[:2]
    kw = dict(window=window, sinks=sinks, scale=scale, q_lens=q_lens, k_lens=k_lens)
    mask = M.causal_mask(b, lq, k.shape[1], q_lens, k_lens, q.device, window, sinks)
    ref = M.attention(q, k, k, mask, scale=scale)["weights"]
    _, lse = W.window_attention(q, k, k, return_lse=True, **kw)
    got = W.window_attention_weights(q, k, lse, **kw)
    within(got, ref, "weights")
    before = rand(7, *got.shape).abs()
    into = before.clone()
    assert W.window_attention_weights(q, k, lse, weights=into, **kw) is into
    assert torch.equal(into, before + got)
    return got, lse


@pytest.mark.parametrize("lq,lk,window,sinks", [
    (1, 1, None, 0), (1, 300, None, 0), (1, 700, 100, 4), (5, 64, None, 0), (64, 65, 3, 0), (130, 130, None, 0),
    (257, 257, 60, 5), (300, 1000, 200, 300), (600, 600, 1, 0), (40, 20, None, 0), (700, 700, None, 0)])
@pytest.mark.parametrize("dtype,h,kv,d", KINDS)
def test_weights_masks(W, lq, lk, window, sinks, dtype, h, kv, d):
    got, _ = check_weights(W, rand(91, 2, lq, h, d, dtype=dtype), rand(92, 2, lk, kv, d, dtype=dtype), window, sinks)
    rows = min(lq, lk)  # (further queries stand before the first key)
    # a row's weights sum to 1: lq h / kv roundings of up to lk terms
    assert bool(((got.double().sum(2) - rows * h // kv).abs() < 1e-4 * rows * h).all())


@pytest.mark.parametrize("d", [8, 24, 32, 96, 104])
@pytest.mark.parametrize("h,kv", [(6, 2), (33, 1), (64, 1), (140, 1)])
def test_weights_dims_and_heads(W, d, h, kv):
    check_weights(W, rand(95, 1, 45, h, d, dtype=F16), rand(96, 1, 310, kv, d, dtype=F16), scale=0.3)


@pytest.mark.parametrize("scale", [0.0, -0.4, 3.0])
def test_weights_scales(W, scale):
    check_weights(W, rand(97, 2, 100, 4, 64, dtype=BF16), rand(98, 2, 140, 2, 64, dtype=BF16), 50, 2, scale)


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_weights_padded_batch_with_nan_behind_the_ends(W, window, sinks):
    q, k = rand(99, 5, 120, 4, 64, dtype=BF16), rand(100, 5, 300, 2, 64, dtype=BF16)
    nq, nk = lens(120, 50, 0, 120, 3), lens(300, 200, 100, 20, 0)
    for i in range(5):
        q[i, int(nq[i]):], k[i, int(nk[i]):] = NAN, NAN
    got, lse = check_weights(W, q, k, window, sinks, q_lens=nq, k_lens=nk)
    assert not got[2].any() and not got[4].any() and not got[1, :, 200:].any()


def test_weights_bad_values_stay_where_they_are_seen(W):
    q, k = rand(101, 1, 300, 2, 64, dtype=F16), rand(102, 1, 300, 1, 64, dtype=F16)
    _, lse = W.window_attention(q, k, k, window=50, return_lse=True)
    clean = W.window_attention_weights(q, k, lse, window=50)
    q[0, 200, 1, 3] = NAN  # a query: the keys that it sees
    _, lse = W.window_attention(q, k, k, window=50, return_lse=True)
    got = W.window_attention_weights(q, k, lse, window=50)
    assert bool(torch.isnan(got[0, 0, 151:201]).all())
    assert torch.equal(got[0, 0, :151], clean[0, 0, :151]) and torch.equal(got[0, 0, 201:], clean[0, 0, 201:])


def test_weights_of_rows_without_any(W):
    q, k = rand(103, 1, 70, 2, 64, dtype=BF16), rand(104, 1, 70, 2, 64, dtype=BF16)
    q[..., 0], k[..., 0] = -1e30, 3e38  # every score -inf
    q[..., 1:] = 0
    _, lse = W.window_attention(q, k, k, return_lse=True)
    assert bool(torch.isneginf(lse).all()) and not W.window_attention_weights(q, k, lse).any()
    none = W.window_attention_weights(q[:, :0], k, lse[:, :, :0].contiguous())
    assert none.shape == (1, 2, 70) and not none.any()
    assert W.window_attention_weights(q[:0], k[:0], lse[:0]).shape == (0, 2, 70)
    keep = torch.ones(1, 2, 70, device="cuda")
    W.window_attention_weights(q[:, :0], k, lse[:, :, :0].contiguous(), weights=keep)
    assert bool((keep == 1).all())


def test_weights_large(W):
    check_weights(W, rand(105, 1, 2000, 8, 128, dtype=BF16), rand(106, 1, 2000, 2, 128, dtype=BF16))
    check_weights(W, rand(107, 3, 1500, 4, 64, dtype=F16), rand(108, 3, 1500, 4, 64, dtype=F16), 300, 600)


def check_decode_weights(W, b, cap, lengths, h, kv, d, dtype, window=None, sinks=0, new=True, seed=111):
    q = rand(seed, b, h, d, dtype=dtype)
    kc, vc = rand(seed + 1, b, cap, kv, d, dtype=dtype), rand(seed + 2, b, cap, kv, d, dtype=dtype)
    kn, vn = (rand(seed + 3 + x, b, kv, d, dtype=dtype) if new else None for x in range(2))
    w = rand(seed + 5, b, kv, cap).abs()
    ref = M.decode(q, kc, vc, lengths, window=window, sinks=sinks, k_new=kn, v_new=vn, weights=w)
    kw = dict(k_new=kn, v_new=vn, window=window, sinks=sinks)
    out = W.window_attention_decode(q, kc, vc, lengths, weights=w, **kw)
    within(out, ref["out"], "out")
    within(w, ref["weights"], "weights")
    assert torch.equal(kc, ref["k_cache"]) and torch.equal(vc, ref["v_cache"])


@pytest.mark.parametrize("cap,window,sinks,lengths", [
    (1, None, 0, (1, 0, 9)), (2, 1, 1, (1, 2, 7)), (40, None, 0, (40, 1, 33)), (64, 16, 4, (3, 64, 500)),
    (100, None, 60, (61, 150, 99)), (300, 256, 5, (290, 299, 1000)), (2000, None, 0, (2000, 1900, 5)),
    (1500, 1000, 100, (1400, 9000, 40))])
@pytest.mark.parametrize("dtype,h,kv,d", KINDS)
def test_decode_weights(W, cap, window, sinks, lengths, dtype, h, kv, d):
    for new in (True, False):
        check_decode_weights(W, 3, cap, lens(*lengths), h, kv, d, dtype, window, sinks, new)


@pytest.mark.parametrize("b,cap,h,kv,d", [(1, 4000, 8, 8, 64), (130, 100, 8, 2, 64), (2, 700, 40, 1, 80), (2, 300, 140, 2, 24)])
def test_decode_weights_batches(W, b, cap, h, kv, d):
    check_decode_weights(W, b, cap, torch.arange(b, dtype=torch.int32, device="cuda") * 7 % cap + 1, h, kv, d, BF16)


def test_decode_weights_of_nan_and_of_no_weight(W):
    q, kc = rand(121, 3, 4, 64, dtype=F16), rand(122, 3, 90, 2, 64, dtype=F16)
    q[1] = NAN
    w = torch.ones(3, 2, 90, device="cuda")
    W.window_attention_decode(q, kc, kc.clone(), lens(90, 50, 30), weights=w)
    assert bool(torch.isnan(w[1, :, :50]).all()) and bool((w[1, :, 50:] == 1).all())
    assert bool(torch.isfinite(w[0]).all()) and bool(torch.isfinite(w[2]).all())
    q, kc = torch.zeros(1, 2, 64, dtype=BF16, device="cuda"), torch.zeros(1, 50, 2, 64, dtype=BF16, device="cuda")
    q[..., 0], kc[..., 0] = -1e30, 3e38
    w = torch.ones(1, 2, 50, device="cuda")
    out = W.window_attention_decode(q, kc, kc.clone(), lens(50), weights=w)
    assert not out.any() and bool((w[..., :49] == 1).all()) and not w[..., 49].any()


# ---------------------------------------------------------------------------
# the smaller cache
# ---------------------------------------------------------------------------
def check_evict(W, k, v, w, lengths, keep, **kw):
    want = M.evict(k, v, w, lengths, keep, **kw)
    got = W.cache_evict(k, v, w, lengths, keep, **kw)
    for x, y, z in zip(("k", "v", "weights", "rows", "lengths"), got, want):
        y = y.cpu()
        same = (y == z) | ((y != y) & (z != z)) if y.is_floating_point() else y == z
        assert y.shape == z.shape and y.dtype == z.dtype and bool(same.all()), x
    return got


def cache(seed, b, cap, kv, d, dtype=BF16):
    return rand(seed, b, cap, kv, d, dtype=dtype), rand(seed + 1, b, cap, kv, d, dtype=dtype), rand(seed + 2, b, kv, cap).exp()


@pytest.mark.parametrize("cap,keep,recent,sinks", [(1, 1, 0, 0), (10, 4, 1, 1), (64, 64, 10, 4), (100, 1, 0, 0), (300, 50, 50, 0),
                                                   (300, 50, 0, 50), (300, 50, 30, 20), (1025, 1024, 5, 0), (1500, 700, 100, 4),
                                                   (5000, 2500, 32, 4), (2100, 30, 7, 2), (40, 60, 5, 3)])
@pytest.mark.parametrize("dtype,kv,d", [(BF16, 2, 128), (F16, 3, 24)])
def test_evict_sizes(W, cap, keep, recent, sinks, dtype, kv, d):
    check_evict(W, *cache(131, 3, cap, kv, d, dtype), lens(cap, max(1, cap // 2), cap + 7), keep, recent=recent, sinks=sinks)


@pytest.mark.parametrize("levels", [1, 2, 5])
@pytest.mark.parametrize("cap", [700, 3001])
def test_evict_ties(W, levels, cap):
    k, v, _ = cache(135, 2, cap, 2, 32)
    w = torch.randint(0, levels, (2, 2, cap), device="cuda").float()
    check_evict(W, k, v, w, lens(cap, cap - 13), cap // 3, recent=20, sinks=3)


def test_evict_special_weights(W):
    k, v, w = cache(139, 2, 400, 2, 32)
    w[0, 0, ::7], w[0, 0, 1::9], w[0, 1, ::3], w[0, 1, 1::3] = NAN, math.inf, 0.0, -0.0
    w[1, 0] = NAN
    w[1, 1] = torch.linspace(-3, 3, 400, device="cuda")
    w[0, 1, 3:30] = 1e-41  # subnormal
    check_evict(W, k, v, w, lens(400, 390), 100, recent=10, sinks=2)
    check_evict(W, k, v, w, lens(400, 390), 300, recent=0, sinks=0)


def test_evict_short_and_empty_sequences(W):
    k, v, w = cache(143, 5, 200, 2, 64)
    for i, n in enumerate((0, -4, 30, 50, 51)):  # rows behind the end are not read
        k[i, max(n, 0):], v[i, max(n, 0):], w[i, :, max(n, 0):] = NAN, NAN, NAN
    got = check_evict(W, k, v, w, lens(0, -4, 30, 50, 51), 50, recent=8, sinks=1)
    assert got[4].tolist() == [0, 0, 30, 50, 50]
    empty = W.cache_evict(k[:0], v[:0], w[:0], lens(), 50)
    assert empty[0].shape == (0, 50, 2, 64) and empty[3].shape == (0, 2, 50)
    none = W.cache_evict(k[:, :0], v[:, :0], w[:, :, :0].contiguous(), lens(0, 0, 0, 0, 0), 4)
    assert not none[0].any() and bool((none[3] == -1).all())


def test_evict_into_a_cache_with_room_and_strides(W):
    store = rand(147, 3, 2, 500, 2, 80, dtype=F16)  # [B, Hkv, C, k or v, D]
    k, v = store[:, :, :, 0].transpose(1, 2), store[:, :, :, 1].transpose(1, 2)
    w = rand(148, 3, 2, 500).exp()
    at = lens(500, 20, 333)
    want = M.evict(k, v, w, at, 100, recent=9, sinks=2)
    ko, vo = (torch.full((3, 2, 130, 80), 7.0, dtype=F16, device="cuda").transpose(1, 2) for _ in range(2))
    wo = torch.full((3, 2, 130), 7.0, device="cuda")
    got = W.cache_evict(k, v, w, at, 100, recent=9, sinks=2, k_out=ko, v_out=vo, weights_out=wo)
    assert got[0] is ko and got[1] is vo and got[2] is wo
    assert torch.equal(ko[:, :100].cpu(), want[0]) and torch.equal(vo[:, :100].cpu(), want[1])
    assert torch.equal(wo[:, :, :100].cpu(), want[2]) and not wo[:, :, 100:].any()
    assert bool((ko[:, 100:] == 7).all()) and bool((vo[:, 100:] == 7).all())
    assert torch.equal(got[3].cpu(), want[3]) and got[4].tolist() == [100, 20, 100]


def test_evict_past_32_bits(W):
    rows, d = (1 << 24) + 100, 128  # 4.3 GB a cache: the last rows lie past 2^32 bytes
    k = torch.zeros(1, rows, 1, d, dtype=BF16, device="cuda")
    k[0, -50:] = rand(151, 50, 1, d, dtype=BF16)
    w = torch.zeros(1, 1, rows, device="cuda")
    w[0, 0, -40:-30] = 5
    got = W.cache_evict(k, k.clone(), w, lens(rows), 30, recent=4)
    at = [*range(16), *range(rows - 40, rows - 30), *range(rows - 4, rows)]
    assert got[3].flatten().tolist() == at
    assert torch.equal(got[0][0], k[0, torch.tensor(at, device="cuda")]) and torch.equal(got[0], got[1])


def test_offsets_past_32_bits(W):
    """Sequences, and tokens of one sequence, more than 2^32 bytes apart."""
    far = torch.zeros(5 << 29, dtype=F16, device="cuda")  # 5.4 GB
    apart = far.as_strided((2, 200, 1, 64), ((1 << 31) + 4096, 64, 64, 1))
    strided = far.as_strided((1, 300, 1, 64), (0, 1 << 23, 64, 1))  # 300 tokens over 5 GB
    for k, lq in ((apart, 1), (apart, 90), (strided, 1), (strided, 300)):
        b, n = k.shape[:2]
        k.copy_(rand(153, *k.shape, dtype=F16))
        q, g = rand(154, b, lq, 1, 64, dtype=F16), rand(155, b, lq, 1, 64, dtype=F16)
        check_cross(W, q, k, k, g)
        check_prefix(W, q, k[0], k[0], k, k)
        check_weights(W, q, k)
        w = torch.ones(b, 1, n, device="cuda")
        ref = M.decode(q[:, 0], k.contiguous(), k.contiguous(), lens(*[n] * b), kp=k[0].contiguous(), vp=k[0].contiguous())
        within(W.prefix_attention_decode(q[:, 0], k[0], k[0], k, k, lens(*[n] * b)), ref["out"], "decode")
        ref = M.decode(q[:, 0], k.contiguous(), k.contiguous(), lens(*[n] * b), weights=w.clone())
        W.window_attention_decode(q[:, 0], k, k, lens(*[n] * b), weights=w)
        within(w, ref["weights"], "weights")
        check_evict(W, k.contiguous(), k.contiguous(), w, lens(*[n] * b), 50)
        got = W.cache_evict(k, k, w, lens(*[n] * b), 50, recent=3)
        assert all(torch.equal(x, y) for x, y in zip(got, W.cache_evict(k.contiguous(), k.contiguous(), w, lens(*[n] * b), 50, recent=3)))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def serve(W, s, steps):
    """A prompt, its keys' weights, the cache cut, then tokens that attend to encoder states,
    to a shared text and to the cut cache, which goes on counting."""
    _, lse = W.window_attention(s["q"], s["k"], s["v"], return_lse=True, k_lens=s["n"], q_lens=s["n"])
    w = W.window_attention_weights(s["q"], s["k"], lse, k_lens=s["n"], q_lens=s["n"])
    s["w"].zero_()
    _, _, _, rows, n = W.cache_evict(s["k"], s["v"], w, s["n"], 60, recent=10, sinks=2, k_out=s["kc"], v_out=s["vc"],
                                     weights_out=s["w"])
    outs = [rows]
    for i in range(steps):
        n = n + 1
        x = s["tokens"][i]
        a = W.window_attention_decode(x, s["kc"], s["vc"], n, k_new=s["kn"][i], v_new=s["vn"][i], weights=s["w"])
        c = W.cross_attention(a[:, None], s["states"], s["states"], k_lens=s["n"])[:, 0]
        outs.append(W.prefix_attention_decode(c, s["text"], s["text"], s["k2"], s["v2"], n, k_new=s["kn"][i], v_new=s["vn"][i]))
    cut = W.cache_evict(s["kc"], s["vc"], s["w"], n, 40, recent=5)
    return [*outs, s["w"].clone(), *cut]


def serving(seed):
    b, h, kv, d = 3, 8, 2, 64
    s = {"q": rand(seed, b, 200, h, d, dtype=BF16), "n": lens(200, 150, 40)}
    for i, x in enumerate(("k", "v", "states")):
        s[x] = rand(seed + 1 + i, b, 200, kv, d, dtype=BF16)
    s["kc"], s["vc"], s["k2"], s["v2"] = (torch.zeros(b, 80, kv, d, dtype=BF16, device="cuda") for _ in range(4))
    s["w"] = torch.zeros(b, kv, 80, device="cuda")
    s["text"] = rand(seed + 4, 300, kv, d, dtype=BF16)
    s["tokens"] = rand(seed + 5, 4, b, h, d, dtype=BF16)
    s["kn"], s["vn"] = rand(seed + 6, 4, b, kv, d, dtype=BF16), rand(seed + 7, 4, b, kv, d, dtype=BF16)
    return s


def test_serving_follows_the_plain_forms(W):
    s = serving(161)
    got = serve(W, s, 4)
    ref = serving(161)
    mask = M.causal_mask(3, 200, 200, ref["n"], ref["n"], "cuda")
    weights = M.attention(ref["q"], ref["k"], ref["v"], mask)["weights"]
    want = M.evict(ref["k"], ref["v"], weights[0].float(), ref["n"], 60, recent=10, sinks=2)
    # the same rows, but where the weight of the last one that stays is within the bound of the next one's
    for b in range(3):
        for g in range(2):
            mine, theirs = set(got[0][b, g].tolist()), set(want[3][b, g].tolist())
            x, e = weights[0][b, g], weights[1][b, g]
            for r in mine - theirs:
                t = min(theirs - mine, key=lambda t: float(x[t]))
                assert float(x[t] - x[r]) <= float(e[t] + e[r])
    # the steps from the library's own cut, which the rows name
    kc, vc, w = (torch.zeros_like(ref[x]) for x in ("kc", "vc", "w"))
    for b in range(3):
        for g in range(2):
            at = got[0][b, g][got[0][b, g] >= 0].long()
            kc[b, :len(at), g], vc[b, :len(at), g], w[b, g, :len(at)] = ref["k"][b, at, g], ref["v"][b, at, g], weights[0][b, g, at].float()
    n = ref["n"].clamp(max=60)
    k2, v2 = ref["k2"], ref["v2"]
    for i in range(4):
        n = n + 1
        step = M.decode(ref["tokens"][i], kc, vc, n, k_new=ref["kn"][i], v_new=ref["vn"][i], weights=w)
        kc, vc, w = step["k_cache"], step["v_cache"], step["weights"][0].float()
        a = step["out"][0]
        c = M.attention(a.to(BF16)[:, None], ref["states"], ref["states"], M.cross_mask(3, 1, 200, None, ref["n"], "cuda"))["out"][0][:, 0]
        last = M.decode(c.to(BF16), k2, v2, n, ref["text"], ref["text"], k_new=ref["kn"][i], v_new=ref["vn"][i])
        k2, v2 = last["k_cache"], last["v_cache"]
        # an input that is a rounding (2^-8) away moves a result of softmax by about its size: all of them are
        # averages of values of deviation 1 by nearly even weights
        assert float((got[1 + i].double() - last["out"][0]).abs().max()) < 0.03
    assert float((got[5].double() - w.double()).abs().max()) < 0.05 * float(w.max())
    assert torch.equal(s["kc"], kc) and torch.equal(s["vc"], vc) and torch.equal(s["k2"], k2)


def test_serving_captured_and_replayed(W):
    s = serving(171)
    want = [x.clone() for x in serve(W, s, 4)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        serve(W, s, 4)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serve(W, s, 4)
    other = serving(172)
    for _ in range(4):
        for x in got:
            x.fill_(3)
        graph.replay()
        eager = serve(W, other, 4)  # between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert not torch.equal(eager[1], want[1])
    for x in ("tokens", "states", "k"):  # the graph reads what stands there then
        s[x].copy_(other[x])
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, serve(W, s, 4)))


def test_training_captured_and_replayed(W):
    q, k, v, g = cross_inputs(181, 2, 150, 333, 4, 2, 64, F16)

    def step():
        out, lse = W.cross_attention(q, k, v, return_lse=True)
        return [out, *W.cross_attention_backward(g, q, k, v, out, lse)]

    want = [x.clone() for x in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_streams_at_once(W):
    a, b = serving(191), serving(192)
    want = [[x.clone() for x in serve(W, s, 4)] for s in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = serve(W, s, 4)
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(x, y) for x, y in zip(got[i], want[i]))


def test_gradients_against_differences(W):
    """Central differences of the 64-bit form along a direction: off by h^2 and 2^-53 / h, about 1e-10; the kernel's
    gradients by 2^-11 of the sum of the terms' sizes for each of the three roundings that it makes."""
    q, k, v, g = cross_inputs(195, 1, 9, 14, 2, 1, 16, F16)
    out, lse = W.cross_attention(q, k, v, return_lse=True)
    grads = W.cross_attention_backward(g, q, k, v, out, lse)
    mask = M.cross_mask(1, 9, 14, None, None, "cuda")
    for name, grad, at in zip("qkv", grads, ("dq", "dk", "dv")):
        x = dict(q=q.double(), k=k.double(), v=v.double())
        step, ends = rand(196, *x[name].shape).double(), []
        for sign in (1, -1):
            y = dict(x)
            y[name] = x[name] + sign * 1e-5 * step
            s = torch.matmul(y["q"].transpose(1, 2), y["k"].transpose(1, 2).transpose(2, 3)) * 16 ** -0.5
            o = torch.matmul(torch.softmax(s, -1), y["v"].transpose(1, 2)).transpose(1, 2)
            ends.append(float((o * g.double()).sum()))
        bound = M.attention(q, k, v, mask, dout=g)[at][1]
        assert abs((ends[0] - ends[1]) / 2e-5 - float((grad.double() * step).sum())) < float((bound * step.abs()).sum()) + 1e-7


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals_on_the_gpu(W):
    q, k, v, g = cross_inputs(201, 2, 8, 16, 4, 2, 64, F16)
    out, lse = W.cross_attention(q, k, v, return_lse=True)
    kp = rand(205, 10, 2, 64, dtype=F16)
    kc, n = k.clone(), lens(3, 3)
    w = torch.ones(2, 2, 16, device="cuda")

    def refused(error, f, *args, **kw):
        with pytest.raises(error):
            f(*args, **kw)

    refused(TypeError, W.cross_attention, q, k.bfloat16(), v)
    refused(TypeError, W.cross_attention, q.float(), k.float(), v.float())
    refused(ValueError, W.cross_attention, q, k[:1], v[:1])
    refused(ValueError, W.cross_attention, q, k, v[:, :8])
    refused(ValueError, W.cross_attention, q, k, v, out=q)
    refused(ValueError, W.cross_attention, q, k, v, k_lens=lens(1))
    refused(ValueError, W.cross_attention, q, k, v, k_lens=n.long())
    refused(ValueError, W.cross_attention, q.requires_grad_(), k, v)
    q.requires_grad_(False)
    refused(ValueError, W.cross_attention, q[..., ::2], k[..., ::2], v[..., ::2])
    refused(ValueError, W.cross_attention_backward, g[:, :4], q, k, v, out, lse)
    refused(ValueError, W.cross_attention_backward, g, q, k, v, out, lse.double())
    refused(ValueError, W.prefix_attention, q, kp[:, :1], kp[:, :1], k, v)
    refused(ValueError, W.prefix_attention, q, kp, kp[:5], k, v)
    refused(TypeError, W.prefix_attention, q, kp.bfloat16(), kp, k, v)
    refused(ValueError, W.prefix_attention, q, kp[None], kp[None], k, v)
    refused(ValueError, W.prefix_attention, q, kp.cpu(), kp, k, v)
    refused(ValueError, W.prefix_attention, q, kp.clone().requires_grad_(), kp, k, v)
    refused(ValueError, W.prefix_attention_decode, q[:, 0], kp, kp, k, v, None)
    refused(ValueError, W.prefix_attention_decode, q[:, 0], kp, kp, k, v, n, k_new=k[:, 0])
    refused(_lib.WtcError, W.prefix_attention_decode, q[:, 0], kp, kp, kc, kc, n, k_new=v[:, 0], v_new=v[:, 0])
    refused(_lib.WtcError, W.prefix_attention_decode, q[:, 0], kp, kp, k[:, :0], v[:, :0], n)
    refused(ValueError, W.prefix_attention_decode, q[:, 0], kp, kp, k, v, n, out=kp[:2].expand(2, 2, 64).repeat(1, 2, 1)[:1])
    refused(ValueError, W.window_attention_weights, q, k, lse[:1])
    refused(ValueError, W.window_attention_weights, q, k, lse, weights=w[:, :, :8])
    refused(ValueError, W.window_attention_weights, q, k, lse, weights=w.double())
    refused(ValueError, W.window_attention_weights, q, k, lse, weights=w.transpose(0, 1))
    refused(ValueError, W.window_attention_weights, q, k, lse, window=0)
    refused(ValueError, W.window_attention_weights, q, k, lse, weights=w.clone().requires_grad_())
    refused(ValueError, W.window_attention_decode, q[:, 0], k, v, n, weights=w[..., :9])
    refused(ValueError, W.window_attention_decode, q[:, 0], k, v, n, weights=w.half())
    refused(ValueError, W.cache_evict, k, v, w, n, 0)
    refused(ValueError, W.cache_evict, k, v, w, n, 4, recent=3, sinks=2)
    refused(ValueError, W.cache_evict, k, v, w, n, 4, recent=-1)
    refused(ValueError, W.cache_evict, k, v, w, None, 4)
    refused(ValueError, W.cache_evict, k, v, w, n.long(), 4)
    refused(ValueError, W.cache_evict, k, v, w[:, :1], n, 4)
    refused(ValueError, W.cache_evict, k, v[:1], w, n, 4)
    refused(TypeError, W.cache_evict, k, v.bfloat16(), w, n, 4)
    refused(TypeError, W.cache_evict, k.float(), v.float(), w, n, 4)
    refused(ValueError, W.cache_evict, k, v, w, n, 4, k_out=k[:, :4].clone())
    refused(ValueError, W.cache_evict, k, v, w, n, 4, k_out=k[:, :4], v_out=v[:, :4].clone(), weights_out=w[..., :4].clone())
    refused(ValueError, W.cache_evict, k, v, w, n, 16, k_out=kc, v_out=kc, weights_out=w.clone())
    refused(ValueError, W.cache_evict, k, v, w, n, 16, k_out=kc, v_out=kc.clone(), weights_out=w)
    refused(ValueError, W.cache_evict, k, v, w, n, 17, k_out=kc, v_out=kc.clone(), weights_out=w.clone())
