"""Refusals and plans of the layer operators at the edges of what their C entry
points take (no GPU)."""
import pytest

from tests.test_layer import A, ERR_ARG, ERR_UNSUPPORTED, attention_args
from welder_typical_chain_amd import _lib


@pytest.fixture(scope="module")
def L(native_lib):
    return _lib.lib()


def test_one_cache_cannot_take_a_key_and_a_value(L):
    args = attention_args(lq=1, k_lens=A)
    assert L.wtc_window_attention_decode(args, A, A, A, A, A, A, None, 0, None) == ERR_ARG
    assert b"same cache" in L.wtc_last_error()


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
