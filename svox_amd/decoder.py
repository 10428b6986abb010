"""The operators of a leaf decoder, a small network that turns the features kept in the leaves of a tree into records a
renderer reads: layer norm and the gated feed-forward block, each a few HIP kernels with its gradient.  The reference has no
such operators.
"""
from .csrc import decoder as _D

__all__ = ["layer_norm", "gated_ffn"]

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
    backward pass, their gradients) to that type between the two products, float32 keeps 24 bits throughout.  Training keeps x
    alone: the backward pass computes the hidden numbers again.
    """
    code = _D.ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(_D.ACTIVATIONS)}")
    return (_native or _calls()).gated_ffn(x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, code)
