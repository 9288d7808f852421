"""Limits and plans of the attention calls without a GPU."""
import ctypes

import pytest

from tests.test_layer import attention_args
from tests.test_masked import ERR_ARG, L, prefix_args  # noqa: F401
from welder_typical_chain_amd import _lib, layer

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


# What the GPU tests' sizes run on 256 CUs (test_gpu_masked.py's and test_gpu_masked_edges.py's):
# each form of prefix_attention, of cross_attention and of its gradients is among them.
@pytest.mark.parametrize("size,want", [
    ((300, 2, 2, 40, 130, 130, 64), (1, 0, 1, 2)), ((300, 1, 1, 33, 140, 140, 24), (1, 0, 1, 2)), ((70, 4, 4, 90, 100, 100, 128), (1, 0, 1, 2)),
    ((2, 2, 1, 31, 200, 200, 128), (1, 0, 1, 1)), ((16, 16, 2, 500, 200, 200, 32), (1, 0, 1, 1)), ((8, 8, 4, 2100, 100, 160, 8), (1, 0, 15, 2)),
    ((1, 2, 2, 5000, 150, 300, 128), (1, 0, 28, 1)), ((2, 4, 2, 8000, 70, 70, 32), (1, 0, 32, 1)), ((1, 2, 1, 16000, 130, 135, 16), (1, 0, 32, 1)),
    ((130, 8, 2, 5000, 32, 40, 128), (0, 1, 1, 1)), ((70, 16, 4, 4000, 20, 20, 96), (0, 2, 1, 1)), ((3, 5, 1, 700, 5, 5, 80), (0, 5, 1, 1)),
    ((3, 3, 3, 0, 200, 200, 64), (0, 0, 1, 1)), ((3, 3, 3, 700, 4, 0, 64), (0, 2, 0, 1))])
def test_prefix_plan(L, size, want):  # noqa: F811
    assert tuple(layer.prefix_attention_plan(*size, cu_count=256).values()) == want


@pytest.mark.parametrize("size,want", [
    ((40, 8, 8, 130, 150, 64), (0, 2, 1, 0, 1)), ((30, 32, 8, 1, 300, 128), (1, 1, 1, 0, 1)), ((1, 4, 4, 64, 5000, 64), (1, 1, 16, 1, 1)),
    ((1, 2, 2, 300, 3000, 128), (0, 1, 19, 1, 1)), ((2, 12, 4, 600, 900, 64), (0, 1, 3, 0, 4)), ((1, 8, 2, 2100, 90, 128), (0, 1, 1, 0, 16)),
    # the gradients of test_cross_gradients_of_few_keys_in_a_padded_batch
    ((3, 4, 2, 100, 300, 64), (0, 1, 1, 1, 1)), ((3, 3, 1, 7, 140, 128), (1, 1, 1, 1, 1)), ((3, 1, 1, 333, 128, 24), (0, 1, 1, 0, 1))])
def test_cross_plan(L, size, want):  # noqa: F811
    assert tuple(layer.cross_attention_plan(*size, cu_count=256).values()) == want


def test_plan_refusals(L):  # noqa: F811
    got = (ctypes.c_int64 * 5)()
    ok, shared = attention_args(), prefix_args()
    assert L.wtc_cross_attention_plan(ok, 256, got) == 0 and L.wtc_prefix_attention_plan(ok, shared, 256, got) == 0
    for bad in (None, attention_args(window=3), attention_args(dim=60)):
        assert L.wtc_cross_attention_plan(bad, 256, got) == ERR_ARG and L.wtc_prefix_attention_plan(bad, shared, 256, got) == ERR_ARG
    assert L.wtc_cross_attention_plan(ok, 256, None) == ERR_ARG and L.wtc_prefix_attention_plan(ok, shared, 256, None) == ERR_ARG
    assert L.wtc_prefix_attention_plan(ok, None, 256, got) == ERR_ARG and L.wtc_prefix_attention_plan(ok, prefix_args(prefix=-1), 256, got) == ERR_ARG
    with pytest.raises(_lib.WtcError):
        layer.cross_attention_plan(1, 3, 2, 4, 4, 64)
