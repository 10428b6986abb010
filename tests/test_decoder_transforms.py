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


@pytest.mark.gpu
def test_tensors_that_are_turned_around_where_they_are_read(gpu):
    """Views whose numbers are the negatives of what lies in memory (the imaginary part of a conjugate), as every argument and as a gradient."""
    g = torch.Generator().manual_seed(0)
    t = [torch.randn(*shape, generator=g).to(gpu) for shape in ((5, 8), (12, 8), (12, 8), (8, 12), (12,), (12,), (8,), (5, 8))]
    grad = torch.randn(5, 8, generator=g).to(gpu)

    def step(call, tensors, grad):
        leaves = [v.detach().requires_grad_() for v in tensors]
        y = call(*leaves)
        return [y, *torch.autograd.grad(y, leaves, grad)]

    turned = lambda v: torch._neg_view(-v)  # noqa: E731
    for call, tensors in ((svox.gated_ffn, t), (svox.layer_norm, (t[0], t[6], t[1][0]))):
        want = step(call, tensors, grad)
        for i in range(len(tensors) + 1):
            some = [turned(v) if j == i else v for j, v in enumerate(tensors)]
            got = step(call, some, turned(grad) if i == len(tensors) else grad)
            assert all(torch.equal(a, b) for a, b in zip(want, got)), i
            assert torch.equal(call(*some), want[0])
    assert torch.complex(t[0], -t[0]).conj().imag.is_neg()
    assert torch.equal(svox.layer_norm(torch.complex(t[0], -t[0]).conj().imag), svox.layer_norm(t[0]))
