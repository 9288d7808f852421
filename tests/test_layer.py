"""The layer operators without a GPU: what the C entry points and the Python
functions refuse, workspace sizes, and the plain forms that the GPU tests
compare with (their gradients against differences)."""
import math

import pytest
import torch

from tests import layer_util as U
from welder_typical_chain_amd import _lib, layer

ERR_ARG, ERR_WS, ERR_UNSUPPORTED = _lib.WTC_ERR_ARG, _lib.WTC_ERR_WORKSPACE, _lib.WTC_ERR_UNSUPPORTED
A = 1 << 20  # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def L(native_lib):
    return _lib.lib()


def matmul_args(**kw):
    x = dict(m=16, n=32, k=64, lda=64, ldb=32, ldr=32, ldo=32, b_trans=0, dtype=1, out_dtype=1, bias_dtype=1,
             activation=0, ldd=32)
    assert set(kw) <= set(x)
    x.update(kw)
    return layer._pack_matmul(*x.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), ERR_ARG), (dict(dtype=3), ERR_ARG), (dict(out_dtype=2), ERR_ARG), (dict(bias_dtype=2), ERR_ARG),
    (dict(activation=5), ERR_ARG), (dict(activation=-1), ERR_ARG), (dict(m=-1), ERR_ARG), (dict(n=-8), ERR_ARG),
    (dict(n=28, ldb=32), ERR_ARG), (dict(k=60), ERR_ARG), (dict(lda=56), ERR_ARG), (dict(lda=68), ERR_ARG),
    (dict(ldb=24), ERR_ARG), (dict(ldo=24), ERR_ARG), (dict(ldr=24), ERR_ARG), (dict(b_trans=1), ERR_ARG),
    (dict(m=1 << 31), ERR_UNSUPPORTED), (dict(m=1 << 25), ERR_UNSUPPORTED), (dict(lda=1 << 27), ERR_UNSUPPORTED),
    (dict(ldb=1 << 26), ERR_UNSUPPORTED), (dict(lda=1 << 62), ERR_UNSUPPORTED)])
def test_matmul_refusals(L, kw, code):
    args = matmul_args(**kw)
    assert L.wtc_matmul_epilogue(args, A, A, None, None, A, None, A, 1 << 40, None) == code
    assert L.wtc_last_error()
    assert L.wtc_matmul_epilogue_workspace_size(args) == -1


def test_matmul_pointer_refusals(L):
    ok = matmul_args()
    assert L.wtc_matmul_epilogue_workspace_size(ok) >= 0
    for k in range(5):
        ptrs = [A, A, A, A, A]
        ptrs[k] += 8
        assert L.wtc_matmul_epilogue(ok, *ptrs, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_matmul_epilogue(ok, None, A, None, None, A, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_matmul_epilogue(ok, A, A, None, None, None, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_matmul_epilogue(None, A, A, None, None, A, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_matmul_epilogue(matmul_args(m=0), None, None, None, None, None, None, None, 0, None) == 0


def test_matmul_backward_refusals(L):
    f = L.wtc_matmul_epilogue_backward
    assert f(matmul_args(ldd=24), A, A, A, None, A, A, A, A, 1 << 40, None) == ERR_ARG
    assert f(matmul_args(ldd=36), A, A, A, None, A, A, A, A, 1 << 40, None) == ERR_ARG
    assert f(matmul_args(), None, A, A, None, A, A, A, A, 1 << 40, None) == ERR_ARG
    assert f(matmul_args(activation=2), A, A, A, None, A, A, A, A, 1 << 40, None) == ERR_ARG  # no pre
    need = L.wtc_matmul_epilogue_backward_workspace_size(matmul_args(activation=2))
    assert need >= 16 * 32 * 2
    assert f(matmul_args(activation=2), A, A, A, A, A, A, A, A, need - 1, None) == ERR_WS
    assert f(matmul_args(activation=2), A, A, A, A, A, A, A, None, need, None) == ERR_WS
    assert f(matmul_args(activation=2), A, A, A, A, A, A, A, A + 16, need, None) == ERR_ARG
    assert L.wtc_matmul_epilogue_backward_workspace_size(matmul_args(activation=9)) == -1


def attention_args(**kw):
    x = dict(batch=2, heads=4, kv_heads=2, lq=8, lk=16, dim=64, window=0, sinks=0, dtype=2,
             q=(2048, 256, 64), k=(2048, 128, 64), v=(2048, 128, 64), o=(2048, 256, 64), do=(2048, 256, 64),
             kn=(128, 64), vn=(128, 64), q_lens=0, k_lens=0, scale=0.125)
    assert set(kw) <= set(x)
    x.update(kw)
    flat = []
    for t in x.values():
        flat += list(t) if isinstance(t, tuple) else [t]
    return layer._pack_attention(*flat)


BAD_ATTENTION = [
    (dict(dtype=0), ERR_ARG), (dict(dtype=3), ERR_ARG), (dict(batch=-1), ERR_ARG), (dict(lk=-1), ERR_ARG),
    (dict(window=-1), ERR_ARG), (dict(sinks=-1), ERR_ARG), (dict(heads=5), ERR_ARG), (dict(kv_heads=0), ERR_ARG),
    (dict(heads=0), ERR_ARG), (dict(dim=4), ERR_ARG), (dict(dim=136), ERR_ARG), (dict(dim=60), ERR_ARG),
    (dict(scale=math.inf), ERR_ARG), (dict(scale=math.nan), ERR_ARG), (dict(q=(2048, 252, 64)), ERR_ARG),
    (dict(k=(2048, -128, 64)), ERR_ARG), (dict(v=(2048, 128, 60)), ERR_ARG),
    (dict(k=(2048, 1 << 24, 64)), ERR_UNSUPPORTED), (dict(batch=1 << 31), ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + [
    (dict(o=(2048, 0, 64)), ERR_ARG), (dict(o=(2048, 256, 32)), ERR_ARG), (dict(o=(0, 256, 64)), ERR_ARG),
    (dict(lq=1 << 31), ERR_UNSUPPORTED)])
def test_attention_refusals(L, kw, code):
    assert L.wtc_window_attention(attention_args(**kw), A, A, A, A, None, A, 1 << 40, None) == code
    assert L.wtc_last_error()


def test_attention_pointer_refusals(L):
    ok = attention_args()
    for k in range(4):
        ptrs = [A, A, A, A]
        ptrs[k] += 2
        assert L.wtc_window_attention(ok, *ptrs, None, A, 1 << 40, None) == ERR_ARG
        ptrs[k] = None
        assert L.wtc_window_attention(ok, *ptrs, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_window_attention(attention_args(batch=0), None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + [(dict(do=(2048, 250, 64)), ERR_ARG)])
def test_attention_backward_refusals(L, kw, code):
    assert L.wtc_window_attention_backward(attention_args(**kw), *[A] * 9, A, 1 << 40, None) == code


def test_attention_backward_workspace(L):
    ok = attention_args()
    need = L.wtc_window_attention_backward_workspace_size(ok)
    assert need >= 2 * 4 * 8 * 4
    assert L.wtc_window_attention_backward(ok, *[A] * 9, A, need - 1, None) == ERR_WS
    assert L.wtc_window_attention_backward(ok, *[A] * 9, None, need, None) == ERR_WS
    assert L.wtc_window_attention_backward(ok, *[A] * 9, A + 8, need, None) == ERR_ARG
    assert L.wtc_window_attention_backward_workspace_size(attention_args(dim=4)) == -1


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + [
    (dict(lq=2), ERR_ARG), (dict(sinks=16), ERR_ARG), (dict(k_lens=0), ERR_ARG), (dict(kn=(100, 64)), ERR_ARG),
    (dict(k=(0, 128, 64)), ERR_ARG), (dict(v=(2048, 64, 64)), ERR_ARG)])
def test_decode_refusals(L, kw, code):
    args = attention_args(**{**dict(lq=1, k_lens=A), **kw})
    assert L.wtc_window_attention_decode(args, A, A, A, A, A, A, A, 1 << 40, None) == code


def test_decode_pointer_refusals(L):
    ok = attention_args(lq=1, k_lens=A)
    for k in range(6):
        ptrs = [A] * 6
        ptrs[k] = None
        assert L.wtc_window_attention_decode(ok, *ptrs, A, 1 << 40, None) == ERR_ARG
        ptrs[k] = A + 8
        assert L.wtc_window_attention_decode(ok, *ptrs, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_window_attention_decode_workspace_size(attention_args(lq=2)) == -1


def test_python_functions_refuse_cpu_tensors():
    a, b = torch.zeros(16, 64, dtype=torch.float16), torch.zeros(64, 32, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        layer.matmul_epilogue(a, b)
    with pytest.raises(ValueError, match="GPU"):
        layer.matmul_epilogue_backward(a[:, :32], a, b)
    q = torch.zeros(1, 8, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        layer.window_attention(q, q, q)
    with pytest.raises(ValueError, match="GPU"):
        layer.window_attention_decode(q[:, 0], q, q, torch.tensor([1], dtype=torch.int32))
    with pytest.raises(TypeError):
        layer.matmul_epilogue(a.float(), b.float())


def test_the_package_offers_them():
    import welder_typical_chain_amd as w
    for name in ("matmul_epilogue", "matmul_epilogue_backward", "window_attention", "window_attention_backward",
                 "window_attention_decode"):
        assert getattr(w, name) is getattr(layer, name) and name in w.__all__


# ---- the plain forms themselves ------------------------------------------------
def test_reference_gradients_against_differences():
    """Central differences of the 64-bit form, h = 1e-5: off by h^2 and 2^-53 / h, about 1e-10."""
    torch.manual_seed(3)
    q, k, v, g = (torch.randn(1, 9, n, 8).half() for n in (4, 2, 2, 4))
    kw = dict(window=4, sinks=2)
    ref = U.attention_reference(q, k, v, dout=g, **kw)
    h = 1e-5
    for name, at in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        x = dict(q=q.double(), k=k.double(), v=v.double())
        step = torch.randn_like(x[name])
        ends = []
        for sign in (1, -1):
            y = dict(x)
            y[name] = x[name] + sign * h * step
            # the 64-bit form itself, on values that float16 does not hold
            s = torch.einsum("bihd,bjhd->bhij", y["q"], y["k"].repeat_interleave(2, 2)) * 8 ** -0.5
            s = s.masked_fill(~U.seen_mask(9, 9, 9, 9, 4, 2), -math.inf)
            o = torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), y["v"].repeat_interleave(2, 2))
            ends.append(float((o * g.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * h)
        assert abs(slope - float((ref[at][0] * step).sum())) < 1e-7, name
    for kind in ("relu", "gelu", "gelu_tanh", "silu"):
        z = torch.linspace(-4, 4, 64, dtype=torch.float64) + 1e-3
        slope = (U.act(z + h, kind) - U.act(z - h, kind)) / (2 * h)
        assert float((slope - U.act_slope(z, kind)).abs().max()) < 1e-8


def test_reference_mask():
    m = U.seen_mask(3, 6, 3, 5, 2, 1)
    assert m.tolist() == [[True, True, True, False, False, False], [True, False, True, True, False, False],
                          [True, False, False, True, True, False]]
    assert [U.cache_row(j, 5, 2) for j in range(9)] == [0, 1, 2, 3, 4, 2, 3, 4, 2]
