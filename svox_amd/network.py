"""Operators of networks over the cells of a tree, beside those of the leaf decoder: attention within packed sequences of cells, heads of
queries and keys rotated by their cells' positions, and the norm of many gradients together with its clipping.  Each is a few HIP kernels.  The reference has no such operators.
"""
import torch

from .csrc import network as _N

__all__ = ["attention", "rotate_heads", "clip_norm", "clip_grad_norm"]

_native = None


def _calls():
    global _native
    if _native is None:
        _native = _N.native()
    return _native


def attention(q, k, v, offsets=None, key_offsets=None, causal=False, scale=None):
    """softmax(scale q . k) v for every query, over the keys of its own sequence.

    :param q: (T, H, D) float32, float16 or bfloat16, on a GPU, D up to 128; rows and heads may lie any distance apart
    :param k, v: (S, G, D) of q's type; H a multiple of G, heads h of q go with head h // (H / G) of k and v
    :param offsets: (sequences + 1,) int32 or int64 on the GPU: sequence s holds rows offsets[s] to offsets[s + 1] - 1 of q; None: one of all
    :param key_offsets: the same of k and v; None: they are packed as q is
    :param causal: a query sees the keys up to its own place, counted from the ends of its sequence's queries and keys
    :param scale: > 0; None: 1 / sqrt(D)
    :return: (T, H, D), differentiable once with respect to q, k and v; 0 for rows that see no key or belong to no sequence

    Scores, their exponentials and all sums are held in 32 bits; 16-bit types round exponentials and the gradients of scores once, as operands of
    the next product, float16 times powers of two that keep them among its normal numbers: result and gradients are off by 1 to 1.7 times what
    one rounding to the type is, in the mean.  The same call gives the same bits.  Rows that a query does not see have no influence on it, whatever they hold.  The
    offsets are read on the GPU: nothing waits for it.
    """
    return (_native or _calls()).attention(q, k, v, offsets, key_offsets, causal, scale)


def rotate_heads(q, k, positions, frequencies, q_weight=None, k_weight=None, interleaved=False, eps=1e-6):
    """Every head of q and k divided by the root of the mean of its squares, times a weight, and rotated by its row's positions.

        n = x / sqrt(mean(x^2) + eps) * weight
        angle_i = sum over axes of positions[row, axis] * frequencies[axis, i]
        (y_a, y_b) = (n_a cos(angle_i) - n_b sin(angle_i), n_b cos(angle_i) + n_a sin(angle_i))

    :param q: (T, H, D) float32, float16 or bfloat16, on a GPU, D up to 256; rows and heads may lie any distance apart
    :param k: (T, G, D), of q's type
    :param positions: (T, axes), up to four axes, or (T,): float32, float64, int32 or int64
    :param frequencies: (axes, R / 2) or (R / 2,) float32, R up to D; numbers of a head from R on are not rotated
    :param q_weight, k_weight: (D,) or None (1), of q's type
    :param interleaved: pairs (a, b) are (2 i, 2 i + 1); else (i, i + R / 2)
    :return: (T, H, D) and (T, G, D), differentiable once with respect to q, k and the weights

    Angles are computed in 64 bits, sums are held in 32 bits and do not depend on the order in which the GPU works.
    """
    return (_native or _calls()).rotate_heads(q, k, positions, frequencies, q_weight, k_weight, interleaved, eps)


def clip_norm(tensors, max_norm):
    """The norm of all numbers of many tensors together, and the tensors scaled to `max_norm` where it is larger.

    :param tensors: float32, float16 or bfloat16 tensors of one GPU, of any shapes and also of different types, or one of them
    :param max_norm: >= 0
    :return: the norm, a float32 tensor without dimensions, and a list of new tensors: x * (max_norm / norm) where the norm exceeds max_norm
        and is finite, else copies of x

    The squares are summed in 64 bits and in an order of their own; a norm beyond float32's largest number scales x and is returned as infinite.  Nothing waits for the GPU.  Not differentiable.
    """
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.zeros(()), []
    return (_native or _calls()).clip_norm(tensors, max_norm)


def clip_grad_norm(parameters, max_norm):
    """`clip_norm` of the gradients of `parameters` (tensors, or one), in place; those without a gradient are left out.

    :return: the norm before, a float32 tensor without dimensions on the gradients' device

    Where the norm is not finite the gradients stay as they are: the caller sees it by the norm.  A gradient that several parameters
    hold counts once.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return (_native or _calls()).clip_in_place(grads, max_norm)
