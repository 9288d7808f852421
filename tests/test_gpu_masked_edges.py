"""Cross attention, attention behind a shared prefix and their gradients where kernels change
hands, on the GPU against plain 64-bit forms (tests/masked_util.py)."""
import pytest
import torch

from tests.test_gpu_masked import BF16, F16, W, check_prefix, prefix_inputs  # noqa: F401

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
