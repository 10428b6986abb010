"""What the operators of networks over cells refuse rather than get wrong: derivatives in forward mode, and transforms of functions."""
import pytest
import torch
from torch.autograd import forward_ad

import svox_amd as svox

pytestmark = pytest.mark.gpu


def calls(gpu):
    p, f = torch.rand(3, device=gpu), torch.rand(4, device=gpu)
    w = torch.ones(8, device=gpu)
    return {
        "attention q": lambda x: svox.attention(x, x.detach(), x.detach()),
        "attention k": lambda x: svox.attention(torch.ones_like(x).detach(), x, torch.ones(3, 2, 8, device=gpu)),
        "attention v": lambda x: svox.attention(torch.ones(3, 2, 8, device=gpu), torch.ones(3, 2, 8, device=gpu), x),
        "rotate_heads": lambda x: svox.rotate_heads(x, torch.ones(3, 1, 8, device=gpu), p, f)[0],
        "rotate_heads k": lambda x: svox.rotate_heads(torch.ones(3, 1, 8, device=gpu), x, p, f, w, w)[1],
    }


NAMES = ["attention q", "attention k", "attention v", "rotate_heads", "rotate_heads k"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(gpu, name):
    call, x = calls(gpu)[name], torch.randn(3, 2, 8, device=gpu)
    for leaf in (x, x.clone().requires_grad_()):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            call(forward_ad.make_dual(leaf, torch.ones_like(x)))
    leaf = x.clone().requires_grad_()
    y = call(leaf)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    torch.autograd.grad(call(leaf), leaf, torch.ones_like(y))


def test_tangents_of_weights_positions_and_clipped_tensors_are_refused(gpu):
    x, p, f, w = torch.randn(3, 2, 8, device=gpu), torch.rand(3, device=gpu), torch.rand(4, device=gpu), torch.ones(8, device=gpu)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    with forward_ad.dual_level():
        for call in (lambda: svox.rotate_heads(x, x, dual(p), f), lambda: svox.rotate_heads(x, x, p, dual(f)), lambda: svox.rotate_heads(x, x, p, f, dual(w)),
                     lambda: svox.rotate_heads(x, x, p, f, w, dual(w)), lambda: svox.clip_norm([x, dual(w)], 1.0)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()


def test_transforms_of_functions_are_refused(gpu):
    x = torch.randn(5, 3, 2, 8, device=gpu)
    for name, call in calls(gpu).items():
        with pytest.raises(RuntimeError, match="transforms of functions"):
            torch.vmap(call)(x) if name != "attention q" else torch.vmap(lambda t: svox.attention(t, t, t))(x)
        with pytest.raises(RuntimeError, match="transforms of functions"):
            torch.func.grad(lambda t: call(t).sum())(x[0])
    for call in (lambda t: svox.clip_norm([t], 1.0)[0], svox.layer_norm, lambda t: svox.gated_ffn(t, torch.ones(8, 8, device=gpu), torch.ones(8, 8, device=gpu), torch.ones(8, 8, device=gpu))):
        with pytest.raises(RuntimeError, match="transforms of functions"):
            torch.vmap(call)(x)
        with pytest.raises(RuntimeError, match="transforms of functions"):
            torch.func.grad(lambda t: call(t).sum())(x[0])
    with pytest.raises(RuntimeError, match="transforms of functions|Batching rule|vmap"):
        torch.autograd.functional.jacobian(lambda t: svox.attention(t, t, t), x[0], vectorize=True)


def test_second_derivatives_are_refused(gpu):
    for name, call in calls(gpu).items():
        leaf = torch.randn(3, 2, 8, device=gpu, requires_grad=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(call(leaf).sum(), leaf, create_graph=True)


def test_tensors_that_are_not_dense_are_named_so(gpu):
    x = torch.randn(3, 2, 8, device=gpu)
    for call in (lambda: svox.attention(x, x.to_sparse(), x), lambda: svox.rotate_heads(x.to_sparse(), x, torch.zeros(3, device=gpu), torch.zeros(4, device=gpu)),
                 lambda: svox.layer_norm(x.to_sparse()), lambda: svox.clip_norm([x.to_sparse()], 1.0)):
        with pytest.raises(RuntimeError, match="dense"):
            call()
