"""A leaf decoder: a small network that turns the features kept in the leaves of a tree into records a renderer reads.

A tree may hold any numbers (`N3Tree(data_format=None, data_dim=D)`); what the renderer reads are records of basis
coefficients and density.  `LeafDecoder` makes the one from the other with two operators, `layer_norm` and `gated_ffn`, each a
few HIP kernels with its gradient; the gradient of the records that a rendering leaves goes back through it to the network's
weights and to the features.  The reference has no such operators.
"""
import torch
from torch import nn

from .csrc import decoder as _D

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


def _cells(data, tree):
    """The cells of the tree's nodes in `data`, without its spare capacity."""
    nodes = tree._structure().nodes
    return data if nodes == data.shape[0] else data[:nodes]


class LeafDecoder(nn.Module):
    """Features of a leaf to its record: `depth` blocks x + ffn(norm(x)) over the features, then ffn(norm(x)) to the record.

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
    """

    def __init__(self, features, record, hidden=None, depth=1, activation="silu", eps=1e-5, device=None, dtype=torch.float32):
        super().__init__()
        if activation not in _D.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(_D.ACTIVATIONS)}")
        kw = dict(device=device, dtype=dtype)
        hidden = 4 * features if hidden is None else hidden
        self.norms = nn.ModuleList(_Norm(features, eps, **kw) for _ in range(depth + 1))
        self.ffns = nn.ModuleList([_Ffn(features, hidden, features, activation, **kw) for _ in range(depth)]
                                  + [_Ffn(features, hidden, record, activation, **kw)])

    def forward(self, x):
        """(..., features) to (..., record), in the type of the weights."""
        x = x.to(self.norms[0].weight.dtype)
        for norm, ffn in zip(self.norms[:-1], self.ffns[:-1]):
            x = ffn(norm(x), residual=x)
        return self.ffns[-1](self.norms[-1](x))

    def decode_tree(self, features, tree):
        """Writes the records of the features in the tree `features` into `tree`, a tree of the same structure (the same nodes, the
        same cells divided; their spare capacity may differ), and returns them, (cells, record), for a backward pass.  Every cell of
        a node is decoded, also those that have children and are not read."""
        if not features._divided_like(tree):
            raise ValueError("features and tree must have the same structure")
        source = _cells(features.data, features)
        records = self(source.reshape(-1, features.data_dim))
        if records.shape[1] != tree.data_dim:
            raise ValueError(f"the decoder makes records of {records.shape[1]} numbers, the tree's have {tree.data_dim}")
        with torch.no_grad():
            _cells(tree.data, tree).copy_(records.view(*source.shape[:-1], -1))
        return records

    def backward_through(self, features, tree, loss):
        """One pass of training: decodes `features` into `tree`, calls `loss` (a function of no arguments that renders `tree`) and
        adds the gradients of what it returns to those of the decoder's weights and of `features.data`, and to those of whatever else
        it was made of.  Returns the loss.  The records' gradient takes the decoder's type: in float16 what is below 2^-25 becomes zero,
        so scale the loss there.  (`tree.data` has to require its gradient, which is that of the records; what `tree.data.grad`
        holds stays as it is.)"""
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
        return value.detach()
