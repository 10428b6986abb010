"""What the leaf decoder's operators refuse rather than get wrong: ways of torch to take a function apart (up to the device check)."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import svox_amd as svox


@pytest.mark.parametrize("gradients", [False, True])
def test_tracing_is_refused(gradients):
    x, w = torch.ones(3, 8), torch.ones(8, 8)
    with torch.set_grad_enabled(gradients):
        for call in (lambda x: svox.layer_norm(x) * 2, lambda x: svox.gated_ffn(x, w, w, w) * 2, svox.LeafDecoder(8, 4)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(call, (x.requires_grad_(gradients),), check_trace=False)
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call)(x)
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            svox.layer_norm(x)


@pytest.mark.gpu
def test_tangents_are_refused(gpu):
    x, w = torch.randn(3, 8, device=gpu), torch.randn(8, 8, device=gpu)
    for call in (lambda x: svox.layer_norm(x), lambda x: svox.gated_ffn(x, w, w, w)):
        for leaf in (x, x.clone().requires_grad_()):
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
                call(forward_ad.make_dual(leaf, torch.ones_like(x)))
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(x), x))
        torch.autograd.grad(call(leaf), leaf, torch.ones_like(x))
