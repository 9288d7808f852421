"""The layer operators on the GPU at values, sizes and calls at the edges of what
their documentation allows, against plain 64-bit forms (tests/layer_util.py)."""
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


def test_decode_all_scores_minus_infinity(W):
    """Keys of -inf alone: a row without keys, as in the prompt form; beside others they count nothing."""
    q = torch.ones(1, 1, 64, dtype=F16, device="cuda")
    kc, vc = torch.ones(1, 100, 1, 64, dtype=F16, device="cuda"), torch.ones(1, 100, 1, 64, dtype=F16, device="cuda")
    kc[0, :40, 0, 0] = -math.inf
    assert bool((W.window_attention_decode(q, kc, vc, lens(40)) == 0).all())
    assert bool((W.window_attention_decode(q, kc, vc, lens(100)) == 1).all())
    assert bool((W.window_attention_decode(q, kc, vc, lens(0)) == 0).all())
