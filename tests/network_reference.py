"""The operators of svox_amd.network in 64 bits, each number with a bound of how far a computation may be from it that rounds where the
operators say they do (`Near` of decoder_reference.py).  Nothing in the bounds is measured: a sum of n numbers in 32 bits is off by at most
(n + 16) 2^-24 of the sum of their magnitudes, whatever its order, a rounding to p bits by 2^-p of the value, a division, a root or an
exponential of float32 by 2^-20 (2^-18 where results have 16 bits)."""
import math

import numpy as np

from decoder_reference import EVAL, U32, Near


def array(x):
    return x.detach().double().cpu().numpy()


# ---- clipping
def clip_norm(tensors, max_norm):
    """(norm, tensors): the norm is rounded once to 32 bits; a scaled number is off by the factor's rounding, the product's and that of its type."""
    total = math.sqrt(math.fsum(float((array(x) ** 2).sum()) for x in tensors))
    factor = max_norm / total if math.isfinite(total) and total > max_norm else 1.0
    near = [Near(array(x) * factor, np.zeros(x.shape) if factor == 1.0 else np.abs(array(x)) * factor * 2 * U32) for x in tensors]
    return Near(total, 2 * U32 * total), [n if factor == 1.0 else n.rounded(x.dtype) for n, x in zip(near, tensors)]


# ---- rotation of heads
def _pairs(rotated, interleaved):
    i = np.arange(rotated // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotated // 2)


def rotate_heads(x, positions, frequencies, weight=None, interleaved=False, eps=1e-6, grad=None, dtype=None):
    """(y, {"x": , "weight": }) of the heads x (T, H, D); positions (T, axes), frequencies (axes, pairs)."""
    dtype, (rows, heads, d) = dtype or x.dtype, x.shape
    v, w = array(x), np.ones(d) if weight is None else array(weight)
    # the mean of squares is off by (d + 16) 2^-24 of itself, its root by half that; the root and the division add theirs
    rel = (d + 16) * U32 / 2 + 2 * EVAL[dtype]
    r = 1 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    n = v * r
    angle = (array(positions)[:, :, None] * array(frequencies)[None]).sum(1)[:, None]
    c, s = np.cos(angle), np.sin(angle)
    size = (np.abs(array(positions))[:, :, None] * np.abs(array(frequencies))[None]).sum(1)[:, None]
    off = 2 * EVAL[dtype] + size * 2.0 ** -50          # of a sine or cosine
    a, b = _pairs(2 * frequencies.shape[1], interleaved)

    def turned(t, err, s):
        y, e = t.copy(), err.copy()
        y[..., a], y[..., b] = t[..., a] * c - t[..., b] * s, t[..., b] * c + t[..., a] * s
        spread = (off + 2 * U32) * (np.abs(t[..., a]) + np.abs(t[..., b])) + err[..., a] + err[..., b]
        e[..., a], e[..., b] = spread, spread
        return y, e

    y, y_off = turned(n * w, np.abs(n * w) * (rel + 2 * U32), s)
    if grad is None:
        return Near(y, y_off).rounded(dtype), {}
    dn, dn_off = turned(array(grad), np.zeros(x.shape), -s)
    g, g_off = dn * w, dn_off * np.abs(w) + U32 * np.abs(dn * w)
    m = (g * n).mean(-1, keepdims=True)
    m_off = (g_off * np.abs(n) + np.abs(g * n) * (rel + 2 * U32)).mean(-1, keepdims=True) + (d + 16) * U32 * np.abs(g * n).mean(-1, keepdims=True)
    dx = r * (g - n * m)
    dx_off = r * (g_off + np.abs(n) * m_off + (np.abs(g) + np.abs(n * m)) * (2 * rel + 4 * U32))
    grads = {"x": Near(dx, dx_off)}
    if weight is not None:
        terms = np.abs(dn * n)
        grads["weight"] = Near((dn * n).sum((0, 1)), (dn_off * np.abs(n) + terms * (rel + 2 * U32)).sum((0, 1)) + (rows * heads + 16) * U32 * terms.sum((0, 1)))
    return Near(y, y_off).rounded(dtype), {name: near.rounded(dtype) for name, near in grads.items()}
