"""What a leaf decoder with heads refuses when it is made or called, before anything runs on a GPU."""
import pytest
import torch

import svox_amd as svox


def test_heads_that_attention_cannot_take():
    for features, heads in ((256, 1), (129, 1), (390, 3), (1024, 4)):
        with pytest.raises(ValueError, match="128"):
            svox.LeafDecoder(features, 28, heads=heads)
    for features, heads in ((128, 1), (256, 2), (1024, 8)):
        assert svox.LeafDecoder(features, 28, heads=heads).attends[0].dim == 128
    assert not hasattr(svox.LeafDecoder(256, 28), "attends")


def test_a_step_whose_norm_cannot_be_bounded_is_refused_before_it_begins():
    """(Trees without a GPU: what comes after the checks would fail.)"""
    decoder = svox.LeafDecoder(8, 28, hidden=8)
    for kw in ({"with_norm": True}, {"max_norm": -1.0}, {"max_norm": float("nan")}, {"max_norm": -1.0, "with_norm": True}):
        with pytest.raises(ValueError, match="norm"):
            decoder.backward_through(None, None, None, **kw)


def test_features_whose_gradients_cannot_be_clipped_are_refused_before_the_step_begins():
    features, tree = svox.N3Tree(data_format=None, data_dim=8, dtype=torch.float64), svox.N3Tree(data_format="SH1")
    called = []
    with pytest.raises(ValueError, match="float64"):
        svox.LeafDecoder(8, tree.data_dim, hidden=8).backward_through(features, tree, lambda: called.append(1), max_norm=1.0)
    assert not called and features.data.grad is None


@pytest.mark.gpu
def test_a_step_tells_its_norm(gpu):
    """The norm of the gradients before they are clipped; where a batch has none that is finite, the step says so and leaves them as they are."""
    torch.manual_seed(0)
    features, tree = svox.N3Tree(data_format=None, data_dim=24, init_refine=1, device=gpu), svox.N3Tree(data_format="SH1", init_refine=1, device=gpu)
    features.data.data.normal_()
    decoder = svox.LeafDecoder(24, tree.data_dim, hidden=40, device=gpu, heads=4, window=16)
    weight = torch.randn(tree.data.shape, generator=torch.Generator().manual_seed(1)).to(gpu)
    nodes = tree._structure().nodes
    everything = [features.data, *decoder.parameters()]
    loss = lambda: (tree.data[:nodes] * weight[:nodes]).sum()  # noqa: E731
    alone = decoder.backward_through(features, tree, loss)
    whole = [p.grad.clone() for p in everything]
    want = float(torch.stack([g.double().square().sum() for g in whole]).sum().sqrt())
    for most, with_norm in ((0.5 * want, True), (2 * want, True), (0.5 * want, False)):
        for p in everything:
            p.grad = None
        out = decoder.backward_through(features, tree, loss, max_norm=most, with_norm=with_norm)
        value, norm = out if with_norm else (out, None)
        assert torch.equal(value, alone) and value.shape == ()
        if with_norm:
            assert norm.shape == () and norm.device == features.data.device and float(norm) == pytest.approx(want, rel=1e-5)
        factor = min(1.0, most / want)
        assert all(float((p.grad - factor * g).norm()) <= 1e-5 * float(g.norm()) for p, g in zip(everything, whole))
    for p in everything:
        p.grad = None
    weight[0, 0, 0, 0, 1] = float("inf")
    _, norm = decoder.backward_through(features, tree, loss, max_norm=1.0, with_norm=True)
    assert not torch.isfinite(norm) and not all(torch.isfinite(p.grad).all() for p in everything)


@pytest.mark.gpu
def test_the_widest_heads_run(gpu):
    decoder = svox.LeafDecoder(256, 28, hidden=64, device=gpu, heads=2, window=10)
    y = decoder(torch.randn(35, 256, device=gpu), torch.rand(35, 3, device=gpu))
    y.sum().backward()
    assert y.shape == (35, 28) and all(torch.isfinite(p.grad).all() for p in decoder.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [0, 2])
def test_a_decoder_is_of_its_weights_type_under_autocast(gpu, heads):
    decoder = svox.LeafDecoder(32, 28, hidden=64, device=gpu, heads=heads, window=10)
    x, positions = torch.randn(35, 32, device=gpu), torch.rand(35, 3, device=gpu)
    want = decoder(x, positions)
    wanted = torch.autograd.grad(want.sum(), list(decoder.parameters()))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = decoder(x, positions)
    assert got.dtype == torch.float32 and torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got.sum(), list(decoder.parameters())), wanted))
