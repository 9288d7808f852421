"""Refusals and plans of the layer operators at the edges of what their C entry
points take (no GPU)."""
import pytest

from tests.layer_sizes import FULL_CHIP, LARGE_GRADIENTS, LARGE_PRODUCTS
from tests.test_layer import A, ERR_ARG, ERR_UNSUPPORTED, attention_args
from welder_typical_chain_amd import _lib, layer


@pytest.fixture(scope="module")
def L(native_lib):
    return _lib.lib()


def test_one_cache_cannot_take_a_key_and_a_value(L):
    args = attention_args(lq=1, k_lens=A)
    assert L.wtc_window_attention_decode(args, A, A, A, A, A, A, None, 0, None) == ERR_ARG
    assert b"same cache" in L.wtc_last_error()


@pytest.mark.parametrize("kw", [dict(k=(2048, 8, 64)), dict(v=(2048, 56, 64))])
def test_decode_refuses_caches_of_overlapping_rows(L, kw):
    args = attention_args(**{**dict(lq=1, k_lens=A), **kw})
    assert L.wtc_window_attention_decode_workspace_size(args) == -1
    assert L.wtc_window_attention_decode(args, A, A, 2 * A, None, None, A, A, 1 << 40, None) == ERR_ARG
    same = attention_args(lq=1, k_lens=A, k=(2048, 0, 64), v=(2048, 0, 64))  # one row for all tokens
    assert L.wtc_window_attention_decode_workspace_size(same) >= 0


# A launch takes fewer than 2^32 threads: 2^23 workgroups of 512, 2^24 of 256.
ONE = dict(heads=1, kv_heads=1, dim=8, q=(8, 8, 8), k=(8, 8, 8), v=(8, 8, 8), o=(8, 8, 8), do=(8, 8, 8), kn=(8, 8), vn=(8, 8))


@pytest.mark.parametrize("kw", [dict(batch=1 << 23, lq=1, lk=1), dict(batch=1 << 13, lq=1 << 17, lk=1),
                                dict(batch=1 << 23, lq=1, lk=64)])
def test_attention_of_too_many_workgroups(L, kw):
    wide = {**ONE, "q": (1 << 21, 8, 8), "o": (1 << 21, 8, 8), "do": (1 << 21, 8, 8)} if kw["lq"] > 1 else ONE
    args = attention_args(**{**wide, **kw})
    assert L.wtc_window_attention_workspace_size(args) == -1
    assert L.wtc_window_attention(args, A, A, A, A, None, A, 1 << 50, None) == ERR_UNSUPPORTED
    assert L.wtc_window_attention_backward_workspace_size(args) == -1
    assert L.wtc_window_attention_backward(args, *[A] * 9, A, 1 << 50, None) == ERR_UNSUPPORTED
    less = attention_args(**{**wide, **kw, "batch": kw["batch"] - 1})
    assert L.wtc_window_attention_workspace_size(less) >= 0


@pytest.mark.parametrize("kw", [dict(batch=1 << 17, lq=1, lk=1 << 13, window=0), dict(batch=1 << 19, lq=1, lk=256, window=1, sinks=128)])
def test_attention_gradient_of_too_many_keys(L, kw):
    """Key blocks of all sequences (2^23), sums of first tokens in parts (64 threads a key)."""
    args = attention_args(**{**ONE, **kw})
    assert L.wtc_window_attention_workspace_size(args) >= 0
    assert L.wtc_window_attention_backward_workspace_size(args) == -1
    assert L.wtc_window_attention_backward(args, *[A] * 9, A, 1 << 50, None) == ERR_UNSUPPORTED


def test_decode_of_too_many_workgroups(L):
    args = attention_args(**{**ONE, "batch": 1 << 24, "lq": 1, "lk": 1, "k_lens": A})
    assert L.wtc_window_attention_decode_workspace_size(args) == -1
    assert L.wtc_window_attention_decode(args, A, A, 2 * A, A, A, A, A, 1 << 50, None) == ERR_UNSUPPORTED
    assert L.wtc_window_attention_decode_workspace_size(attention_args(**{**ONE, "batch": (1 << 24) - 1, "lq": 1, "lk": 1, "k_lens": A})) >= 0


@pytest.mark.parametrize("scale", [1e39, -1e300, 3.5e38])
def test_scale_beyond_float32(L, scale):
    assert L.wtc_window_attention(attention_args(scale=scale), A, A, A, A, None, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_window_attention_backward(attention_args(scale=scale), *[A] * 9, A, 1 << 40, None) == ERR_ARG
    assert L.wtc_window_attention_decode(attention_args(lq=1, k_lens=A, scale=scale), A, A, 2 * A, A, A, A, A, 1 << 40, None) == ERR_ARG


@pytest.mark.parametrize("size,tile", LARGE_PRODUCTS)
@pytest.mark.parametrize("b_trans", [False, True])
def test_plan_of_large_products(L, size, tile, b_trans):
    assert layer.matmul_epilogue_plan(*size, b_trans=b_trans, cu_count=256) == (*tile, 1)


@pytest.mark.parametrize("size,part,tile,split", LARGE_GRADIENTS)
@pytest.mark.parametrize("b_trans", [False, True])
def test_plan_of_large_gradients(L, size, part, tile, split, b_trans):
    *got, splits = layer.matmul_epilogue_plan(*size, b_trans=b_trans, part=part, cu_count=256)
    assert tuple(got) == tile and (splits > 1) == split


def test_plan_of_few_rows(L):
    assert layer.matmul_epilogue_plan(8, 4096, 4096, b_trans=True, cu_count=256) == (16, 16, 1)
    assert layer.matmul_epilogue_plan(8, 4096, 4096, cu_count=256)[0] == 64


@pytest.mark.parametrize("b,h,kv,lq,lk,d,kw", FULL_CHIP)
def test_plan_of_a_full_chip(L, b, h, kv, lq, lk, d, kw):
    plan = layer.window_attention_plan(b, h, kv, lq, lk, d, cu_count=256, **kw)
    assert plan["row_waves"] == 1 and plan["dq_row_waves"] == 1 and plan["key_splits"] == 1
    few = layer.window_attention_plan(1, h, kv, 90, 90, d, cu_count=256, **kw)
    assert few["row_waves"] == 2 and few["dq_row_waves"] == 2


def test_plan_refusals(L):
    with pytest.raises(_lib.WtcError):
        layer.matmul_epilogue_plan(8, 12, 8)
    with pytest.raises(ValueError):
        layer.matmul_epilogue_plan(8, 16, 8, part="dc")
    with pytest.raises(_lib.WtcError):
        layer.window_attention_plan(1, 3, 2, 8, 8, 64)
    args = attention_args()
    assert L.wtc_window_attention_plan(None, 0, None) == ERR_ARG and L.wtc_window_attention_plan(args, 0, None) == ERR_ARG
    assert L.wtc_matmul_epilogue_plan(None, 0, 0, None, None, None) == ERR_ARG
