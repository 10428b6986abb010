"""svox_amd -- N^3-tree queries and differentiable volume rendering on AMD MI355X (gfx950).

Use it where `import svox` was used:  `import svox_amd as svox`.
"""
from .decoder import LeafDecoder, gated_ffn, layer_norm
from .formats import DataFormat, LocalIndex, NDCConfig, Rays
from .network import attention, clip_grad_norm, clip_norm, rotate_heads
from .renderer import VolumeRenderer
from .tree import N3Tree
from .view import N3TreeView

__version__ = "0.1.0"
__all__ = ["N3Tree", "N3TreeView", "VolumeRenderer", "NDCConfig", "Rays", "LocalIndex", "DataFormat",
           "LeafDecoder", "layer_norm", "gated_ffn", "attention", "rotate_heads", "clip_norm", "clip_grad_norm"]
