"""A leaf decoder trained through the renderer: the operators together as a program uses them."""
import copy

import pytest
import torch

import svox_amd as svox
from decoder_reference import gated_ffn, layer_norm

pytestmark = pytest.mark.gpu


def scene(gpu, dtype=torch.float32, depth=1):
    torch.manual_seed(0)
    features = svox.N3Tree(data_format=None, data_dim=12, init_refine=2, device=gpu)
    features.data.data.normal_()
    tree = svox.N3Tree(data_format="SH1", init_refine=2, device=gpu)
    decoder = svox.LeafDecoder(12, tree.data_dim, hidden=40, depth=depth, device=gpu, dtype=dtype)
    return features, tree, decoder


def some_rays(gpu, n, seed):
    g = torch.Generator().manual_seed(seed)
    origins = torch.nn.functional.normalize(torch.randn(n, 3, generator=g), dim=1) * 2 + 0.5
    dirs = torch.nn.functional.normalize(torch.rand(n, 3, generator=g) - origins, dim=1)
    return svox.Rays(origins.to(gpu), dirs.to(gpu), dirs.to(gpu))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_records_are_those_of_the_definitions(gpu, dtype):
    """With the operators' own numbers in between, every step lies within the bounds of its definition in 64 bits."""
    features, tree, decoder = scene(gpu, dtype)
    with torch.no_grad():
        records = decoder.decode_tree(features, tree)
        x = features.data.reshape(-1, 12).to(dtype)
        for norm, ffn, last in zip(decoder.norms, decoder.ffns, (False, True)):
            n = norm(x)
            layer_norm(x, norm.weight, norm.bias)[0].holds(n)
            t = {"x": n, "residual": None if last else x, **dict(ffn.named_parameters())}
            y = ffn(n, residual=t["residual"])
            gated_ffn(t, "silu")[0].holds(y)
            x = y
    assert torch.equal(records, x) and torch.equal(tree.data.reshape(-1, tree.data_dim), records.float())


def test_gradients_of_a_rendering_reach_weights_and_features(gpu):
    """The gradients backward_through leaves are those of torch's own float32 network with the renderer's gradient of the records."""
    features, tree, decoder = scene(gpu)
    renderer, rays = svox.VolumeRenderer(tree, step_size=1e-2), some_rays(gpu, 500, 1)
    target = torch.rand(500, 3, generator=torch.Generator().manual_seed(2)).to(gpu)
    loss = decoder.backward_through(features, tree, lambda: ((renderer(rays) - target) ** 2).mean())
    # the renderer's gradient of the records, on the records as they are
    value = ((renderer(rays) - target) ** 2).mean()
    assert abs(float(value) - float(loss)) <= 1e-6 * float(loss)
    value.backward()
    grad = tree.data.grad.reshape(-1, tree.data_dim)
    f = copy.deepcopy(decoder).double()
    data = features.data.detach().double().requires_grad_()
    x = data.reshape(-1, 12)
    for i, (norm, ffn) in enumerate(zip(f.norms, f.ffns)):
        n = torch.nn.functional.layer_norm(x, (12,), norm.weight, norm.bias)
        h = torch.nn.functional.silu(n @ ffn.w_gate.t() + ffn.b_gate) * (n @ ffn.w_up.t() + ffn.b_up)
        x = h @ ffn.w_down.t() + ffn.b_down + (x if i == 0 else 0)
    f.zero_grad()
    x.backward(grad.double())
    pairs = [(features.data.grad, data.grad)] + [(a.grad, b.grad) for a, b in zip(decoder.parameters(), f.parameters())]
    for got, want in pairs:
        # the renderer's atomic sums differ by some 2^-20 from call to call, the chain of six float32 products by as much again
        assert float((got.double() - want).norm()) <= 1e-4 * float(want.norm()) + 1e-12


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_through_the_renderer_brings_the_loss_down(gpu, dtype):
    features, tree, decoder = scene(gpu, dtype)
    truth = svox.N3Tree(data_format="SH1", init_refine=2, device=gpu)
    g = torch.Generator().manual_seed(3)
    truth.data.data.copy_(torch.randn(truth.data.shape, generator=g) * 2)
    renderer, model = svox.VolumeRenderer(truth, step_size=1e-2), svox.VolumeRenderer(tree, step_size=1e-2)
    optimizer = torch.optim.Adam([features.data, *decoder.parameters()], lr=1e-2)
    losses = []
    for step in range(60):
        rays = some_rays(gpu, 400, 10 + step)
        with torch.no_grad():
            target = renderer(rays)
        optimizer.zero_grad(set_to_none=True)
        losses.append(float(decoder.backward_through(features, tree, lambda: ((model(rays) - target) ** 2).mean())))
        optimizer.step()
    assert all(v == v for v in losses) and sum(losses[-10:]) < 0.5 * sum(losses[:10]), losses


def test_decode_tree_refuses_other_structures(gpu):
    features, tree, decoder = scene(gpu)
    with pytest.raises(ValueError, match="same structure"):
        decoder.decode_tree(features, svox.N3Tree(data_format="SH1", init_refine=1, device=gpu))
    with pytest.raises(ValueError, match="records of 4 numbers"):
        decoder.decode_tree(features, svox.N3Tree(data_format="SH4", init_refine=2, device=gpu))
