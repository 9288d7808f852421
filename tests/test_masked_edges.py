"""Limits of the attention calls without a GPU."""
import pytest

from tests.test_layer import attention_args
from tests.test_masked import L  # noqa: F401

TILES = ("wtc_cross_attention_backward", "wtc_window_attention_backward", "wtc_window_attention_weights")


# A tile of query rows holds the query heads of one key head: the distance between other heads
# is no limit.
@pytest.mark.parametrize("name", TILES)
@pytest.mark.parametrize("tensor", ["q", "do"])
def test_heads_far_apart(L, name, tensor):  # noqa: F811
    far = (64, 64, (1 << 30) + 64)
    size = getattr(L, name + "_workspace_size")
    assert size(attention_args(heads=2, kv_heads=2, **{tensor: far})) >= 0, L.wtc_last_error()
    if tensor == "q" or name != TILES[2]:  # (weights has no dout)
        assert size(attention_args(heads=4, kv_heads=2, **{tensor: far})) == -1
        assert b"query heads span" in L.wtc_last_error()
