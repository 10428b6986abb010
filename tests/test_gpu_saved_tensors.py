"""Tensors that the operators keep for their backward passes, and hooks that give back others: what has the same numbers gives the same gradients,
however it lies; what is of another device, type or shape is refused before a kernel sees it."""
import pytest
import torch

import svox_amd as svox

pytestmark = pytest.mark.gpu


def operators(dtype):
    g = torch.Generator().manual_seed(0)
    some = lambda *shape: torch.randn(*shape, generator=g).to(dtype).to("cuda:0")  # noqa: E731
    positions, frequencies = torch.rand(40, 3, generator=g).to("cuda:0"), torch.rand(3, 12, generator=g).to("cuda:0")
    offsets = torch.tensor([0, 7, 7, 40], device="cuda:0")
    heads = [some(40, 4, 24), some(40, 2, 24)]
    return {
        "attention": (lambda q, k, v: svox.attention(q, k, v, offsets, causal=True), [*heads, some(40, 2, 24)]),
        "key_offsets": (lambda q, k, v: svox.attention(q, k, v, offsets, offsets.clone()), [*heads, some(40, 2, 24)]),
        "rotate_heads": (lambda *x: torch.cat(svox.rotate_heads(x[0], x[1], positions, frequencies, *x[2:]), 1), [*heads, some(24), some(24)]),
        "layer_norm": (svox.layer_norm, [some(40, 24), some(24), some(24)]),
        "gated_ffn": (svox.gated_ffn, [some(40, 24), some(30, 24), some(30, 24), some(16, 30), some(30), some(30), some(16)]),
    }


NAMES = ["attention", "key_offsets", "rotate_heads", "layer_norm", "gated_ffn"]


def gradients(call, inputs, pack, unpack):
    """Of inputs that are given as tensors of their own, so that hooks see those the operator keeps."""
    leaves = [x.detach().requires_grad_() for x in inputs]
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = call(*leaves)
    grad = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(y.dtype).to(y.device)
    return torch.autograd.grad(y, leaves, grad)


def turned(x):
    """The same numbers, the last dimension's farthest apart in memory."""
    return x if x.dim() < 2 else x.movedim(-1, 0).contiguous().movedim(0, -1)


def apart(x):
    """The same numbers, each a few places from the next."""
    wide = x.new_zeros(*x.shape, 3)
    wide[..., 1] = x
    return wide[..., 1]


same = lambda x: x  # noqa: E731


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("name", NAMES)
def test_the_same_numbers_in_other_places(gpu, name, dtype):
    call, inputs = operators(dtype)[name]
    want = gradients(call, inputs, same, same)
    for pack, unpack in ((turned, same), (same, apart), (lambda x: x.cpu(), lambda x: x.cuda()), (lambda x: torch._neg_view(-x) if x.is_floating_point() else x, same)):
        assert all(torch.equal(a, b) for a, b in zip(want, gradients(call, inputs, pack, unpack)))
    with torch.autograd.graph.save_on_cpu():
        leaves = [x.detach().requires_grad_() for x in inputs]
        y = call(*leaves)
    grad = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(y.dtype).to(y.device)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, leaves, grad)))


@pytest.mark.parametrize("name", NAMES)
def test_other_tensors_are_refused(gpu, name):
    call, inputs = operators(torch.float32)[name]
    kept = []
    gradients(call, inputs, lambda x: kept.append(x) or x, same)
    count = len(kept)
    assert count >= 3
    for change in (lambda x: x.cpu(), lambda x: x.double() if x.is_floating_point() else x.int(), lambda x: x[:-1], lambda x: x.unsqueeze(0), lambda x: x.to_sparse()):
        for i in range(count):
            seen = []
            pack = lambda x: (seen.append(0), (len(seen) - 1, x))[1]  # noqa: E731
            unpack = lambda p: change(p[1]) if p[0] == i else p[1]  # noqa: E731
            with pytest.raises(RuntimeError, match="hook on saved tensors"):
                gradients(call, inputs, pack, unpack)


@pytest.mark.parametrize("name", NAMES)
def test_checkpoints_compute_the_same_again(gpu, name):
    """Nothing is kept but the inputs; the operator runs again for its backward pass."""
    from torch.utils.checkpoint import checkpoint

    call, inputs = operators(torch.bfloat16)[name]
    want = gradients(call, inputs, same, same)
    leaves = [x.detach().requires_grad_() for x in inputs]
    y = checkpoint(call, *leaves, use_reentrant=False)
    grad = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(y.dtype).to(y.device)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, leaves, grad)))
