"""The operators of svox_amd.network in 64 bits, each number with a bound of how far a computation may be from it that rounds where the
operators say they do (`Near` of decoder_reference.py).  Nothing in the bounds is measured: a sum of n numbers in 32 bits is off by at most
(n + 16) 2^-24 of the sum of their magnitudes, whatever its order, a rounding to p bits by 2^-p of the value, a division, a root or an
exponential of float32 by 2^-20 (2^-18 where results have 16 bits)."""
import math

import numpy as np

from decoder_reference import EVAL, ROUND, SMALL, U32, Near


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


# ---- attention
def seen_by(a, b, causal):
    """(a, b): which of b keys each of a queries sees."""
    i, j = np.arange(a)[:, None], np.arange(b)[None]
    return (j - i <= b - a) if causal else np.ones((a, b), dtype=bool)


def _attend(q, k, v, seen, scale, dtype, grad):
    """One head of one sequence: ((o, off), [(dq, off), (dk, off), (dv, off)])."""
    (a, d), b = q.shape, k.shape[0]
    # (an exponential, relative to the largest, that is below the type's smallest normal number, or half its smallest, may be 0: exp(-88) is
    # 2^-126, and the hardware's exponential returns no number below that)
    round_, small = ROUND[dtype] if dtype.itemsize == 2 else 0.0, SMALL[dtype]
    if a == 0 or b == 0:
        zero = [(np.zeros(x.shape), np.zeros(x.shape)) for x in (q, q, k, v)]
        return zero[0], zero[1:]
    s = scale * (q @ k.T)
    some = seen.any(1, keepdims=True)
    top = np.where(some, np.where(seen, s, -np.inf).max(1, keepdims=True), 0.0)
    p = np.where(seen, np.exp(np.where(seen, s, 0.0) - top), 0.0)
    total = p.sum(1, keepdims=True)
    p = p / np.where(some, total, 1.0)
    # a score's error is that of its exponential in parts; the scores' maximum cancels, what it is rounded to does not
    size = np.where(seen, np.abs(s), 0.0).max(1, keepdims=True)
    off = ((d + 16) * U32 * scale * np.where(seen, np.abs(q) @ np.abs(k).T, 0.0)).max(1, keepdims=True) + 8 * U32 * size
    rel = 2 * off + 2 * EVAL[dtype] + (b + 16) * U32
    av = np.abs(v)
    o = p @ v
    o_off = (rel + round_ + (b + 16) * U32) * (p @ av) + small * (seen @ av)
    if grad is None:
        return (o, o_off), None
    o_all = o_off + (ROUND[dtype] * (np.abs(o) + o_off) + SMALL[dtype])     # as the backward pass has it
    delta, dp = (grad * o).sum(1, keepdims=True), grad @ v.T
    ag = np.abs(grad)
    lse = np.abs(top + np.log(np.where(some, total, 1.0)))
    rel_b = 2 * rel + 8 * U32 * (size + lse + 1)
    ds = p * (dp - delta)
    ds_off = p * (rel_b * np.abs(dp - delta) + (d + 16) * U32 * (ag @ av.T + (ag * np.abs(o)).sum(1, keepdims=True)) + (ag * o_all).sum(1, keepdims=True))
    ds_off = np.where(seen, ds_off + (round_ + 4 * U32) * (np.abs(ds) + ds_off) + small * (1 + np.abs(dp - delta)), 0.0)
    p_off = np.where(seen, p * (rel_b + round_ + 4 * U32) + small, 0.0)
    dq, dk, dv = scale * (ds @ k), scale * (ds.T @ q), p.T @ grad
    dq_off = scale * (ds_off @ np.abs(k) + (b + 16) * U32 * (np.abs(ds) @ np.abs(k)))
    dk_off = scale * (ds_off.T @ np.abs(q) + (a + 16) * U32 * (np.abs(ds).T @ np.abs(q)))
    dv_off = p_off.T @ ag + (a + 16) * U32 * (p.T @ ag)
    return (o, o_off), [(dq, dq_off), (dk, dk_off), (dv, dv_off)]


def attention(q, k, v, offsets=None, key_offsets=None, causal=False, scale=None, grad=None):
    """(y, {"q": , "k": , "v": }); offsets are lists.  Gradients of keys add up over the heads that share them, one sum of all."""
    dtype, (t, h, d), (n, g, _) = q.dtype, q.shape, k.shape
    scale = d ** -0.5 if scale is None else scale
    offsets = [0, t] if offsets is None else list(offsets)
    key_offsets = ([0, n] if len(offsets) == 2 and t != n else offsets) if key_offsets is None else list(key_offsets)
    qq, kk, vv = array(q), array(k), array(v)
    dy = None if grad is None else array(grad)
    y = [np.zeros((t, h, d)) for _ in range(2)]
    grads = {"q": [np.zeros((t, h, d)) for _ in range(2)], "k": [np.zeros((n, g, d)) for _ in range(2)], "v": [np.zeros((n, g, d)) for _ in range(2)]}
    for q0, q1, k0, k1 in zip(offsets, offsets[1:], key_offsets, key_offsets[1:]):
        seen = seen_by(q1 - q0, k1 - k0, causal)
        for one in range(h):
            kv = one // (h // g)
            rows, keys = (slice(q0, q1), one), (slice(k0, k1), kv)
            o, parts = _attend(qq[rows], kk[keys], vv[keys], seen, scale, dtype, None if dy is None else dy[rows])
            for to, x in zip(y, o):
                to[rows] = x
            for name, at, part in zip("qkv", (rows, keys, keys), parts or ()):
                for to, x in zip(grads[name], part):
                    to[at] += x
    if grad is None:
        return Near(*y).rounded(dtype), {}
    for name in "kv":    # (the group's rows are one sum)
        grads[name][1] *= 1 + 2 * (h // g) * U32
        grads[name][1] += (h // g) * 16 * U32 * np.abs(grads[name][0])
    return Near(*y).rounded(dtype), {name: Near(*both).rounded(dtype) for name, both in grads.items()}
