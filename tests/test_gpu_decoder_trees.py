"""A leaf decoder between trees of different spare capacity."""
import pytest
import torch

import svox_amd as svox
from test_gpu_leaf_decoder import scene, some_rays

pytestmark = pytest.mark.gpu


def test_spare_capacity_is_left_as_it_is(gpu):
    features, tree, decoder = scene(gpu)
    records = decoder.decode_tree(features, tree)
    roomy = svox.N3Tree(data_format="SH1", init_refine=2, init_reserve=9, device=gpu)
    wide = svox.N3Tree(data_format=None, data_dim=12, init_refine=2, init_reserve=5, device=gpu)
    nodes = tree.n_internal
    assert tree.capacity == nodes and roomy.capacity == nodes + 8 and wide.capacity == nodes + 4
    roomy.data.data[nodes:] = 7.0
    wide.data.data[:nodes] = features.data.data
    wide.data.data[nodes:] = float("nan")
    assert torch.equal(decoder.decode_tree(wide, roomy), records)
    assert torch.equal(roomy.data[:nodes], tree.data) and bool((roomy.data[nodes:] == 7).all())
    target = torch.rand(300, 3, generator=torch.Generator().manual_seed(2)).to(gpu)
    rays, grads = some_rays(gpu, 300, 1), []
    for f, t in ((features, tree), (wide, roomy)):
        renderer = svox.VolumeRenderer(t, step_size=1e-2)
        decoder.zero_grad()
        decoder.backward_through(f, t, lambda: ((renderer(rays) - target) ** 2).mean())
        grads.append([f.data.grad[:nodes].clone()] + [p.grad.clone() for p in decoder.parameters()])
    assert bool((wide.data.grad[nodes:] == 0).all())
    for a, b in zip(*grads):    # (the renderer's atomic sums differ by some 2^-20 from call to call)
        assert float((a - b).norm()) <= 1e-4 * float(a.norm()) + 1e-12
