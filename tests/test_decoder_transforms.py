"""What the leaf decoder's operators refuse rather than get wrong: ways of torch to take a function apart (up to the device check)."""
import pytest
import torch
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
