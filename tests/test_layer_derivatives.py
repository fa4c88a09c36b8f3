"""MoeLayer and MoeBlock under forward-mode differentiation and traces, which they do not have: a
derivative or a result may not get lost without an error."""
import pytest
import torch
from torch.autograd import forward_ad

from oxidizr_amd import moe
from oxidizr_amd.moe import ModelError, MoeBlock, MoeConfig, MoeLayer

CFG = dict(hidden_size=64, num_experts=4, experts_per_tok=2, intermediate_size=32)


def modules(device):
    """Frozen modules: nothing in them requires a gradient."""
    return [m.requires_grad_(False) for m in (
        MoeLayer(MoeConfig(**CFG), torch.float32, device), MoeBlock(MoeConfig(**CFG), torch.float32, device),
        MoeBlock(MoeConfig(**CFG, residual_scale=0.5), torch.float32, device))]


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("which", range(3))
def test_traces_are_refused(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    m, x = modules("cpu")[which], torch.ones(1, 3, 64)
    with pytest.raises(ModelError, match="traced"):
        torch.jit.trace(lambda t: m(t)[0], x, check_trace=False)
    with pytest.raises(ModelError, match="traced"):
        make_fx(lambda t: m(t)[0])(x)


@pytest.mark.parametrize("which,function", [(0, "_MoeFunction"), (1, "_MoeBlockFunction")])
def test_forward_mode_goes_through_the_autograd_function(which, function, monkeypatch):
    class Reached(Exception):
        pass

    class Function:
        @staticmethod
        def apply(*args):
            raise Reached
    monkeypatch.setattr(moe, function, Function)
    m = modules("cpu")[which]
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(1, 3, 64), torch.ones(1, 3, 64))
        with pytest.raises(Reached):
            m(x)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused_on_the_device(which):
    m = modules("cuda")[which]
    x = torch.randn(2, 9, 64, device="cuda")
    want = m(x)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            m(forward_ad.make_dual(x, x))
        for a, b in zip(m(x), want):  # without a derivative there is nothing to lose
            assert torch.equal(a, b)
