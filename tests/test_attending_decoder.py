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


@pytest.mark.gpu
def test_the_widest_heads_run(gpu):
    decoder = svox.LeafDecoder(256, 28, hidden=64, device=gpu, heads=2, window=10)
    y = decoder(torch.randn(35, 256, device=gpu), torch.rand(35, 3, device=gpu))
    y.sum().backward()
    assert y.shape == (35, 28) and all(torch.isfinite(p.grad).all() for p in decoder.parameters())
