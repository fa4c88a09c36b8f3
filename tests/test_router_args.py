"""Arguments of router_losses at the ends of their ranges, without a GPU."""
import pytest
import torch

from oxidizr_amd import _lib, ops
from oxidizr_amd.moe import ModelError

P = 1 << 20  # an aligned address that a refused call never touches


@pytest.mark.parametrize("tau", [1e-60, 1e-45, 1e-39, 2.0 ** -128, 2.0 ** -127, 1.1e-38, 2.0 ** 128, 1e39])
def test_a_temperature_beyond_fp32_or_whose_inverse_is(tau):
    # the scores were NaN: the kernels multiply by log2(e) / tau, and 0 times infinity is none
    with pytest.raises(ModelError, match="temperature must be"):
        ops.router_losses(torch.zeros(4, 6), torch.zeros(4, 2, dtype=torch.int32), temperature=tau)
    L = _lib.load()
    args = (0, None, _lib.MOE_DTYPE_F32, 4, 6, 2, 4, P, P, 0, tau)
    assert L.moe_router_losses(*args, 1.0, 1.0, None, 1, P, P, P, None, None, P) == 1
    assert b"temperature" in L.moe_last_error()
    assert L.moe_router_losses_backward(*args, None, 1, P, P, P, P, P) == 1
    assert b"temperature" in L.moe_last_error()


@pytest.mark.parametrize("tau", [2.0 ** -126, 1e-37, 3e38])
def test_the_ends_are_accepted(tau):
    with pytest.raises(ModelError, match="CUDA"):  # the next check
        ops.router_losses(torch.zeros(4, 6), torch.zeros(4, 2, dtype=torch.int32), temperature=tau)
