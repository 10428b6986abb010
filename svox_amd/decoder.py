"""A leaf decoder: a small network that turns the features kept in the leaves of a tree into records a renderer reads.

A tree may hold any numbers (`N3Tree(data_format=None, data_dim=D)`); what the renderer reads are records of basis
coefficients and density.  `LeafDecoder` makes the one from the other with two operators, `layer_norm` and `gated_ffn`, each a
few HIP kernels with its gradient, and, where cells are to see their neighbours, with those of `svox_amd.network`; the gradient of the records that a rendering leaves goes back through it to the network's
weights and to the features.  The reference has no such operators.
"""
import math

import torch
from torch import nn

from .csrc import decoder as _D
from .network import attention, clip_grad_norm, rotate_heads

__all__ = ["layer_norm", "gated_ffn", "LeafDecoder"]

_native = None


def _calls():
    global _native
    if _native is None:
        _native = _D.native()
    return _native


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x.

    :param x: (..., D) float32, float16 or bfloat16, on a GPU; rows may lie any distance apart
    :param weight: (D,) or None (1), of x's type
    :param bias: (D,) or None (0), of x's type
    :return: (..., D), differentiable once with respect to x, weight and bias

    Mean, variance and the sums of the gradients are held in 32 bits and do not depend on the order in which the GPU works.
    """
    return (_native or _calls()).layer_norm(x, weight, bias, eps)


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, residual=None, activation="silu"):
    """(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down + residual.

    :param x: (..., D) float32, float16 or bfloat16, on a GPU; rows may lie any distance apart
    :param w_gate, w_up: (H, D); :param w_down: (K, H)
    :param b_gate, b_up: (H,) or None; :param b_down: (K,) or None
    :param residual: (..., K) or None; added to the result before it is rounded
    :param activation: "silu", "gelu" (with the error function), "relu" or "sigmoid"
    :return: (..., K), differentiable once with respect to every tensor

    All tensors have x's type.  Products are summed in 32 bits; float16 and bfloat16 round the hidden numbers (and, in the
    backward pass, their gradients) to that type between the two products, as the matrix cores take them: the result is off by 1.4
    times what one rounding of it is, and in float16 a hidden number or a gradient beyond 65504 becomes infinite and one below 2^-25
    zero (scale the loss).  float32 keeps 24 bits throughout; there numbers from 3.396e38 on make NaN, as infinite ones do.
    Training keeps x alone: the backward pass computes the hidden numbers again.
    """
    code = _D.ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(_D.ACTIVATIONS)}")
    return (_native or _calls()).gated_ffn(x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, code)


class _Norm(nn.Module):
    def __init__(self, dim, eps, **kw):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, **kw))
        self.bias = nn.Parameter(torch.zeros(dim, **kw))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class _Ffn(nn.Module):
    def __init__(self, dim, hidden, out, activation, **kw):
        super().__init__()
        self.activation = activation
        self.w_gate = nn.Parameter(torch.randn(hidden, dim, **kw) * dim ** -0.5)
        self.w_up = nn.Parameter(torch.randn(hidden, dim, **kw) * dim ** -0.5)
        self.w_down = nn.Parameter(torch.randn(out, hidden, **kw) * hidden ** -0.5)
        self.b_gate = nn.Parameter(torch.zeros(hidden, **kw))
        self.b_up = nn.Parameter(torch.zeros(hidden, **kw))
        self.b_down = nn.Parameter(torch.zeros(out, **kw))

    def forward(self, x, residual=None):
        return gated_ffn(x, self.w_gate, self.w_up, self.w_down, self.b_gate, self.b_up, self.b_down, residual=residual,
                         activation=self.activation)


class _Attend(nn.Module):
    def __init__(self, features, heads, kv_heads, eps, **kw):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, features // heads
        self.norm = _Norm(features, eps, **kw)
        self.w_qkv = nn.Parameter(torch.randn((heads + 2 * kv_heads) * self.dim, features, **kw) * features ** -0.5)
        self.w_out = nn.Parameter(torch.randn(features, features, **kw) * features ** -0.5)
        self.q_weight = nn.Parameter(torch.ones(self.dim, **kw))
        self.k_weight = nn.Parameter(torch.ones(self.dim, **kw))

    def forward(self, x, positions, frequencies, offsets):
        wide, narrow = self.heads * self.dim, self.kv_heads * self.dim
        heads = lambda t: t.unflatten(1, (-1, self.dim))  # noqa: E731
        with torch.autocast(x.device.type, enabled=False):      # (a decoder is of its weights' type, whatever a caller has torch's products in)
            q, k, v = nn.functional.linear(self.norm(x), self.w_qkv).split([wide, narrow, narrow], dim=1)
            q, k = rotate_heads(heads(q), heads(k), positions, frequencies, self.q_weight, self.k_weight)
            return torch.addmm(x, attention(q, k, heads(v), offsets).flatten(1), self.w_out.t())


def _cell_centres(tree):
    """(cells, 3) float32, the centres of all cells of the tree's nodes in tree coordinates."""
    at = tree._unpack_index(torch.arange(tree._structure().nodes * tree.N ** 3, device=tree.data.device))
    depth = tree.parent_depth[:, 1].to(at.device)[at[:, 0]]
    return tree._calc_corners(at).float() + 0.5 * float(tree.N) ** -(depth + 1.0)[:, None]


def _cells(data, tree):
    """The cells of the tree's nodes in `data`, without its spare capacity."""
    nodes = tree._structure().nodes
    return data if nodes == data.shape[0] else data[:nodes]


class LeafDecoder(nn.Module):
    """Features of a leaf to its record: `depth` blocks x + ffn(norm(x)) over the features, then ffn(norm(x)) to the record.  With `heads`, each
    block begins with x + attention among the cells of a window, of queries and keys that are rotated by the cells' centres.

    A decoder that is trained through a renderer, with the features of every leaf:

        features = svox.N3Tree(data_format=None, data_dim=16, init_refine=4, device="cuda:0")
        tree = svox.N3Tree(data_format="SH4", init_refine=4, device="cuda:0")
        decoder = svox.LeafDecoder(16, tree.data_dim, hidden=64).cuda()
        renderer = svox.VolumeRenderer(tree)
        optimizer = torch.optim.Adam([features.data, *decoder.parameters()], lr=1e-2)
        for rays, target in batches:
            optimizer.zero_grad()
            loss = decoder.backward_through(features, tree, lambda: ((renderer(rays) - target) ** 2).mean())
            optimizer.step()

    :param features: numbers of a leaf's features
    :param record: numbers of a record (`tree.data_dim`)
    :param hidden: hidden units of every block (default: four for each feature)
    :param heads: heads of the attention in every block, of up to 128 features each; 0: cells are decoded by themselves
    :param kv_heads: heads of its keys and values (default: as many)
    :param window: cells of a window: consecutive ones, which lie near one another in space, as a node's children follow one another.  Cells that
        are divided are among them: their records nobody reads, but the leaves of their window see their features
    """

    def __init__(self, features, record, hidden=None, depth=1, activation="silu", eps=1e-5, device=None, dtype=torch.float32, heads=0, kv_heads=None,
                 window=512):
        super().__init__()
        if activation not in _D.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(_D.ACTIVATIONS)}")
        kw = dict(device=device, dtype=dtype)
        hidden = 4 * features if hidden is None else hidden
        self.norms = nn.ModuleList(_Norm(features, eps, **kw) for _ in range(depth + 1))
        self.ffns = nn.ModuleList([_Ffn(features, hidden, features, activation, **kw) for _ in range(depth)]
                                  + [_Ffn(features, hidden, record, activation, **kw)])
        self.window = window
        if heads:
            kv_heads = heads if kv_heads is None else kv_heads
            if heads < 0 or kv_heads < 1 or features % heads or heads % kv_heads or window < 1:
                raise ValueError(f"{features} features do not make {heads} heads for {kv_heads} heads of keys, or a window of {window} cells is none")
            if features // heads > 128:
                raise ValueError(f"{features} features make heads of {features // heads} numbers of {heads} heads, more than the 128 that attention takes")
            self.attends = nn.ModuleList(_Attend(features, heads, kv_heads, eps, **kw) for _ in range(depth))
            # pairs of a head take turns among the three axes, from one turn over the tree to 2^8 (kept as whole numbers, whose type stays
            # where a module's is changed)
            pairs = torch.arange(features // heads // 2)
            waves = 2 * math.pi * 2.0 ** (8.0 * (pairs // 3) / max(1, (len(pairs) + 2) // 3 - 1))
            frequencies = torch.where(pairs % 3 == torch.arange(3)[:, None], waves, torch.zeros(())).float()
            self.register_buffer("frequencies", frequencies.to(device).view(torch.int32), persistent=False)

    def forward(self, x, positions=None, offsets=None):
        """(..., features) to (..., record), in the type of the weights.

        :param positions: (rows, 3), of a decoder with heads: where the cells are, in tree coordinates
        :param offsets: where the windows of a decoder with heads begin and end, as of `attention` (default: every `window` rows)
        """
        x = x.to(self.norms[0].weight.dtype)
        shape = x.shape
        if self._attends():
            if positions is None:
                raise ValueError("a decoder with heads needs the positions of the cells")
            x = x.reshape(-1, shape[-1])
            if offsets is None:
                rows = x.shape[0]
                offsets = torch.arange(0, rows + self.window, self.window, device=x.device).clamp_(max=rows) if rows else None
        for i, (norm, ffn) in enumerate(zip(self.norms[:-1], self.ffns[:-1])):
            if self._attends():
                x = self.attends[i](x, positions, self.frequencies.view(torch.float32), offsets)
            x = ffn(norm(x), residual=x)
        y = self.ffns[-1](self.norms[-1](x))
        return y.reshape(*shape[:-1], y.shape[-1]) if self._attends() else y

    def _attends(self):
        return hasattr(self, "attends")

    def decode_tree(self, features, tree):
        """Writes the records of the features in the tree `features` into `tree`, a tree of the same structure (the same nodes, the
        same cells divided; their spare capacity may differ), and returns them, (cells, record), for a backward pass.  Every cell of
        a node is decoded, also those that have children and are not read."""
        if not features._divided_like(tree):
            raise ValueError("features and tree must have the same structure")
        source = _cells(features.data, features)
        rows = source.reshape(-1, features.data_dim)
        records = self(rows, _cell_centres(features)) if self._attends() else self(rows)
        if records.shape[1] != tree.data_dim:
            raise ValueError(f"the decoder makes records of {records.shape[1]} numbers, the tree's have {tree.data_dim}")
        with torch.no_grad():
            _cells(tree.data, tree).copy_(records.view(*source.shape[:-1], -1))
        return records

    def backward_through(self, features, tree, loss, max_norm=None, with_norm=False):
        """One pass of training: decodes `features` into `tree`, calls `loss` (a function of no arguments that renders `tree`) and
        adds the gradients of what it returns to those of the decoder's weights and of `features.data`, and to those of whatever else
        it was made of.  Returns the loss.  The records' gradient takes the decoder's type: in float16 what is below 2^-25 becomes zero,
        so scale the loss there.  With `max_norm` the gradients of the weights and of `features.data`, as they then stand, are clipped together
        (`clip_grad_norm`); where their norm is not finite they stay as they are.  `with_norm` returns (loss, norm before), by which the caller
        tells a batch whose step it had better leave out.  (`tree.data` has to require its gradient, which is that of the records; what
        `tree.data.grad` holds stays as it is.)"""
        if with_norm and max_norm is None:
            raise ValueError("with_norm is the norm that max_norm bounds: give both")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"max_norm must be >= 0, got {max_norm}")
        if max_norm is not None and features.data.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise ValueError(f"gradients of {features.data.dtype} cannot be clipped: features need float32, float16 or bfloat16 for max_norm")
        if not (tree.data.requires_grad and tree.data.is_leaf):
            raise ValueError("tree.data does not require a gradient, or is computed from something else: that of the records has to come through it")
        records = self.decode_tree(features, tree)
        kept, tree.data.grad = tree.data.grad, None
        try:
            value = loss()
            value.backward()
            grad = tree.data.grad
        finally:
            tree.data.grad = kept
        if grad is not None and records.requires_grad:    # (None: the loss does not depend on the records)
            records.backward(_cells(grad, tree).reshape(records.shape).to(records.dtype))
        if max_norm is None:
            return value.detach()
        norm = clip_grad_norm([features.data, *self.parameters()], max_norm)
        return (value.detach(), norm) if with_norm else value.detach()
