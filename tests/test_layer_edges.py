"""Refusals and plans of the layer operators at the edges of what their C entry
points take (no GPU)."""
import pytest

from tests.test_layer import A, ERR_ARG, attention_args
from welder_typical_chain_amd import _lib


@pytest.fixture(scope="module")
def L(native_lib):
    return _lib.lib()


def test_one_cache_cannot_take_a_key_and_a_value(L):
    args = attention_args(lq=1, k_lens=A)
    assert L.wtc_window_attention_decode(args, A, A, A, A, A, A, None, 0, None) == ERR_ARG
    assert b"same cache" in L.wtc_last_error()
