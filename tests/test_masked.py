"""Cross attention, the shared prefix, what keys receive and cache_evict without a GPU:
refusals of the C entry points and the Python functions, workspace sizes, and the plain
forms that the GPU tests compare with."""
import math

import pytest
import torch

from tests import layer_util as U
from tests import masked_util as M
from tests.test_layer import BAD_ATTENTION, A, attention_args
from welder_typical_chain_amd import _lib, layer

ERR_ARG, ERR_WS, ERR_UNSUPPORTED = _lib.WTC_ERR_ARG, _lib.WTC_ERR_WORKSPACE, _lib.WTC_ERR_UNSUPPORTED
NONE = (dict(window=3), ERR_ARG), (dict(sinks=1), ERR_ARG)  # what attention without a window refuses
BIG = 1 << 40


@pytest.fixture(scope="module")
def L(native_lib):
    return _lib.lib()


def prefix_args(**kw):
    x = dict(prefix=100, kp=(128, 64), vp=(128, 64))
    assert set(kw) <= set(x)
    x.update(kw)
    return layer._pack_prefix(x["prefix"], *x["kp"], *x["vp"])


def evict_args(**kw):
    x = dict(batch=2, kv_heads=2, rows=100, out_rows=20, dim=64, dtype=2, keep=20, recent=5, sinks=2,
             k=(12800, 128, 64), v=(12800, 128, 64), ko=(2560, 128, 64), vo=(2560, 128, 64))
    assert set(kw) <= set(x)
    x.update(kw)
    flat = []
    for t in x.values():
        flat += list(t) if isinstance(t, tuple) else [t]
    return layer._pack_evict(*flat)


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + [
    *NONE, (dict(o=(2048, 0, 64)), ERR_ARG), (dict(o=(0, 256, 64)), ERR_ARG), (dict(batch=1, kv_heads=1, heads=1, lq=1 << 29, lk=(1 << 29) + 1), ERR_UNSUPPORTED),
    (dict(k=(2048, 56, 64)), ERR_ARG), (dict(v=(2048, 0, 64)), ERR_ARG)])
def test_cross_refusals(L, kw, code):
    assert L.wtc_cross_attention(attention_args(**kw), A, A, A, A, None, A, BIG, None) == code
    assert L.wtc_last_error()


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + [*NONE, (dict(do=(2048, 250, 64)), ERR_ARG), (dict(k=(2048, 0, 64)), ERR_ARG)])
def test_cross_backward_refusals(L, kw, code):
    args = attention_args(**kw)
    assert L.wtc_cross_attention_backward(args, A, A, A, A, A, A, A, A, A, A, BIG, None) == code
    assert L.wtc_cross_attention_backward_workspace_size(args) == -1


def test_cross_pointer_and_workspace_refusals(L):
    ok = attention_args()
    assert L.wtc_cross_attention_workspace_size(ok) >= 0
    assert L.wtc_cross_attention_workspace_size(None) == -1
    for k in range(4):
        for bad in (A + 8, None):
            ptrs = [A] * 4
            ptrs[k] = bad
            assert L.wtc_cross_attention(ok, *ptrs, None, A, BIG, None) == ERR_ARG
    assert L.wtc_cross_attention(None, A, A, A, A, None, A, BIG, None) == ERR_ARG
    assert L.wtc_cross_attention(attention_args(lq=0), None, None, None, None, None, None, 0, None) == 0
    need = L.wtc_cross_attention_backward_workspace_size(ok)
    assert need >= 2 * 4 * 8 * 8  # two numbers a row
    f = L.wtc_cross_attention_backward
    assert f(ok, *[A] * 9, A, need - 1, None) == ERR_WS and f(ok, *[A] * 9, None, need, None) == ERR_WS
    assert f(ok, *[A] * 9, A + 16, need, None) == ERR_ARG
    many = attention_args(batch=1, lq=1, lk=8192)  # few rows against many keys: splits
    need = L.wtc_cross_attention_workspace_size(many)
    assert need > 0 and L.wtc_cross_attention(many, A, A, A, A, None, A, need - 1, None) == ERR_WS


BAD_PREFIX = [(dict(prefix=-1), ERR_ARG), (dict(kp=(120, 60)), ERR_ARG), (dict(vp=(-128, 64)), ERR_ARG), (dict(vp=(0, 64)), ERR_ARG), (dict(kp=(56, 64)), ERR_ARG),
              (dict(kp=(1 << 24, 64)), ERR_UNSUPPORTED), (dict(prefix=1 << 30), ERR_UNSUPPORTED), (dict(prefix=1 << 40), ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + list(NONE) + [(dict(o=(2048, 0, 64)), ERR_ARG)])
def test_prefix_refusals(L, kw, code):
    assert L.wtc_prefix_attention(attention_args(**kw), prefix_args(), A, A, A, A, A, A, None, A, BIG, None) == code


@pytest.mark.parametrize("kw,code", BAD_ATTENTION + list(NONE) + [(dict(lq=2), ERR_ARG), (dict(lk=0), ERR_ARG), (dict(k_lens=0), ERR_ARG)])
def test_prefix_decode_refusals(L, kw, code):
    args = attention_args(**{"lq": 1, "k_lens": A, **kw})
    assert L.wtc_prefix_attention_decode(args, prefix_args(), *[A] * 8, A, BIG, None) == code


@pytest.mark.parametrize("kw,code", BAD_PREFIX)
def test_prefix_extent_refusals(L, kw, code):
    x = prefix_args(**kw)
    assert L.wtc_prefix_attention(attention_args(), x, A, A, A, A, A, A, None, A, BIG, None) == code
    assert L.wtc_prefix_attention_workspace_size(attention_args(), x) == -1
    token = attention_args(lq=1, k_lens=A)
    assert L.wtc_prefix_attention_decode(token, x, *[A] * 8, A, BIG, None) == code
    assert L.wtc_prefix_attention_decode_workspace_size(token, x) == -1


def test_prefix_pointer_and_workspace_refusals(L):
    ok, x = attention_args(), prefix_args()
    for k in range(6):
        for bad in (A + 8, None):
            ptrs = [A] * 6
            ptrs[k] = bad
            assert L.wtc_prefix_attention(ok, x, *ptrs, None, A, BIG, None) == ERR_ARG
    assert L.wtc_prefix_attention(ok, None, *[A] * 6, None, A, BIG, None) == ERR_ARG
    need = L.wtc_prefix_attention_workspace_size(ok, x)
    assert need > 0 and L.wtc_prefix_attention(ok, x, *[A] * 6, None, A, need - 1, None) == ERR_WS
    token = attention_args(lq=1, k_lens=A)
    for k in range(8):
        ptrs = [A, A, A, A, 2 * A, A, A, A]
        ptrs[k] += 8
        assert L.wtc_prefix_attention_decode(token, x, *ptrs, A, BIG, None) == ERR_ARG
    f = L.wtc_prefix_attention_decode
    assert f(token, x, A, A, A, A, 2 * A, None, A, A, A, BIG, None) == ERR_ARG  # k_new alone
    assert f(token, x, A, A, A, A, A, A, A, A, A, BIG, None) == ERR_ARG         # one cache takes k_new and v_new
    need = L.wtc_prefix_attention_decode_workspace_size(token, x)
    assert need > 0 and f(token, x, A, A, A, A, 2 * A, A, A, A, A, need - 1, None) == ERR_WS


@pytest.mark.parametrize("kw,code", BAD_ATTENTION)
def test_weights_refusals(L, kw, code):
    args = attention_args(**kw)
    assert L.wtc_window_attention_weights(args, A, A, A, A, 0, A, BIG, None) == code
    assert L.wtc_window_attention_weights_workspace_size(args) == -1


def test_weights_pointer_and_workspace_refusals(L):
    ok = attention_args()
    for k in range(4):
        ptrs = [A] * 4
        ptrs[k] = None
        assert L.wtc_window_attention_weights(ok, *ptrs, 0, A, BIG, None) == ERR_ARG
    assert L.wtc_window_attention_weights(ok, A + 8, A, A, A, 0, A, BIG, None) == ERR_ARG
    many = attention_args(batch=1, lq=8192, lk=8192, q=(0, 256, 64))
    need = L.wtc_window_attention_weights_workspace_size(many)
    assert need > 0 and L.wtc_window_attention_weights(many, A, A, A, A, 0, A, need - 1, None) == ERR_WS
    token = attention_args(lq=1, k_lens=A)
    need = L.wtc_window_attention_decode_weights_workspace_size(token)
    f = L.wtc_window_attention_decode_weights
    assert need > 0 and f(token, A, A, 2 * A, A, A, A, A, A, need - 1, None) == ERR_WS
    assert f(token, A, A, 2 * A, A, A, A, None, A, need, None) == ERR_ARG
    assert f(token, A, A, A, A, A, A, A, A, need, None) == ERR_ARG
    assert f(attention_args(lq=2, k_lens=A), A, A, 2 * A, A, A, A, A, A, BIG, None) == ERR_ARG


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), ERR_ARG), (dict(batch=-1), ERR_ARG), (dict(rows=-1), ERR_ARG), (dict(kv_heads=0), ERR_ARG), (dict(dim=60), ERR_ARG),
    (dict(dim=136), ERR_ARG), (dict(keep=0), ERR_ARG), (dict(recent=-1), ERR_ARG), (dict(sinks=-1), ERR_ARG), (dict(recent=19), ERR_ARG),
    (dict(recent=1 << 62, sinks=1 << 62), ERR_ARG), (dict(out_rows=19), ERR_ARG), (dict(k=(12800, 130, 64)), ERR_ARG),
    (dict(v=(-12800, 128, 64)), ERR_ARG), (dict(ko=(2560, 120, 64)), ERR_ARG), (dict(vo=(2560, 64, 64)), ERR_ARG),
    (dict(ko=(0, 128, 64)), ERR_ARG), (dict(rows=1 << 31), ERR_UNSUPPORTED), (dict(out_rows=1 << 31), ERR_UNSUPPORTED),
    (dict(batch=1 << 30), ERR_UNSUPPORTED),
    (dict(batch=1 << 20, kv_heads=8, rows=1, keep=1, recent=0, sinks=0, out_rows=1, ko=(512, 512, 64), vo=(512, 512, 64)), ERR_UNSUPPORTED)])
def test_evict_refusals(L, kw, code):
    assert L.wtc_cache_evict(evict_args(**kw), *[A] * 9, None) == code
    assert L.wtc_last_error()


def test_evict_pointer_refusals(L):
    for k in range(9):
        ptrs = [A] * 9
        ptrs[k] = None
        assert L.wtc_cache_evict(evict_args(), *ptrs, None) == ERR_ARG
    for k in (0, 1, 4, 5):
        ptrs = [A] * 9
        ptrs[k] += 8
        assert L.wtc_cache_evict(evict_args(), *ptrs, None) == ERR_ARG
    assert L.wtc_cache_evict(None, *[A] * 9, None) == ERR_ARG
    assert L.wtc_cache_evict(evict_args(batch=0), *[None] * 9, None) == 0


def test_python_functions_refuse_cpu_tensors():
    q, n = torch.zeros(1, 8, 2, 64, dtype=torch.float16), torch.tensor([1], dtype=torch.int32)
    lse, w = torch.zeros(1, 2, 8), torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="GPU"):
        layer.cross_attention(q, q, q)
    with pytest.raises(ValueError, match="GPU"):
        layer.cross_attention_backward(q, q, q, q, q, lse)
    with pytest.raises(ValueError, match="GPU"):
        layer.prefix_attention(q, q[0], q[0], q, q)
    with pytest.raises(ValueError, match="GPU"):
        layer.prefix_attention_decode(q[:, 0], q[0], q[0], q, q, n)
    with pytest.raises(ValueError, match="GPU"):
        layer.window_attention_weights(q, q, lse)
    with pytest.raises(ValueError, match="GPU"):
        layer.cache_evict(q, q, w, n, 4)


def test_the_package_offers_them():
    import welder_typical_chain_amd as w
    for name in ("cross_attention", "cross_attention_backward", "prefix_attention", "prefix_attention_decode",
                 "window_attention_weights", "cache_evict"):
        assert getattr(w, name) is getattr(layer, name) and name in w.__all__


# ---- the plain forms themselves ------------------------------------------------
def test_plain_forms_agree_with_the_causal_one():
    torch.manual_seed(5)
    q, k, v, g = (torch.randn(2, n, h, 8).half() for n, h in ((7, 4), (9, 2), (9, 2), (7, 4)))
    nq, nk = torch.tensor([7, 3]), torch.tensor([9, 5])
    kw = dict(window=4, sinks=2, q_lens=nq, k_lens=nk)
    want = U.attention_reference(q, k, v, dout=g, **kw)
    mask = M.causal_mask(2, 7, 9, nq, nk, "cpu", 4, 2)
    got = M.attention(q, k, v, mask, dout=g)
    for x in want:
        assert torch.equal(want[x][0], got[x][0]), x
    # each row's weights sum to 1
    assert torch.allclose(got["weights"][0].sum(2), torch.tensor([[14.0, 14.0], [6.0, 6.0]]).double())
    # a prefix is a part of the keys that every query sees
    own = M.causal_mask(2, 7, 9, None, None, "cpu")
    keys, values, _ = M.prefix_inputs(k[0, :3], v[0, :3], k, v, None)
    both = torch.cat([torch.ones(2, 7, 3, dtype=torch.bool), own], 2)
    assert torch.equal(M.attention(q, keys, values, both)["out"][0], U.attention_reference(q, keys, values)["out"][0])
    assert M.cross_mask(1, 2, 3, torch.tensor([1]), torch.tensor([2]), "cpu").tolist() == [[[True, True, False], [False] * 3]]


def test_plain_decode_and_evict():
    torch.manual_seed(7)
    q, kc, vc = torch.randn(2, 2, 8).half(), torch.randn(2, 5, 1, 8).half(), torch.randn(2, 5, 1, 8).half()
    n = torch.tensor([4, 9])
    want = U.decode_reference(q, kc, vc, n, window=3, sinks=1)
    got = M.decode(q, kc, vc, n, window=3, sinks=1, weights=torch.ones(2, 1, 5))
    assert torch.equal(want[0], got["out"][0])
    w = got["weights"][0]
    # three of the rows below the newest token's take their share; its own is set
    assert math.isclose(float(w[0].sum()), 4 + 2, rel_tol=1e-12) and math.isclose(float(w[1].sum()), 4 + 2, rel_tol=1e-12)
    x = torch.tensor([[[1.0, 5.0, 2.0, 5.0, float("nan"), 0.0]]])
    k = torch.arange(6.0).view(1, 6, 1, 1).expand(1, 6, 1, 8).half()
    rows = lambda *a, **kw: M.evict(k, k, x, *a, **kw)[3].flatten().tolist()  # noqa: E731
    assert rows([6], 2) == [1, 4] and rows([6], 3) == [1, 3, 4] and rows([4], 2) == [1, 3] and rows([3], 4) == [0, 1, 2, -1]
    assert rows([6], 3, recent=1, sinks=1) == [0, 4, 5] and rows([6], 2, recent=1, sinks=1) == [0, 5] and rows([99], 1) == [4]
