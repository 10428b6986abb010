"""Layer norm, the gated feed-forward block and their gradients in 64 bits, each number with a bound of how far a computation
may be from it that rounds where the operators say they do.

A `Near` is a value and such a bound.  The rules are those of rounding analysis: a sum of n products in 32 bits is off by at most
(n + 16) 2^-24 of the sum of their magnitudes, whatever its order (16: what the float32 products of three bfloat16 planes leave
out, and the additions of parts); a rounding to p significant bits by 2^-p of the value; errors of factors multiply up as the
product rule has it.  Nothing in the bounds is measured.
"""
import math

import numpy as np
import torch

U32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALL = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}   # where a type's numbers run out
EVAL = {torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -18, torch.bfloat16: 2.0 ** -18}      # exp, erf and division in 32 bits


class Near:
    def __init__(self, v, e=None, most=math.inf):
        self.v = np.asarray(v, dtype=np.float64)
        self.e = np.zeros_like(self.v) if e is None else np.asarray(e, dtype=np.float64)
        self.most = most    # the type's largest number: what may lie beyond it may be infinite

    @property
    def T(self):
        return Near(self.v.T, self.e.T)

    @property
    def size(self):
        return np.abs(self.v) + self.e

    def __matmul__(self, o):
        n = self.v.shape[1]
        spread = np.abs(self.v) @ o.e + self.e @ np.abs(o.v) + self.e @ o.e
        return Near(self.v @ o.v, spread + (n + 16) * U32 * (self.size @ o.size))

    def __add__(self, o):
        v = self.v + o.v
        return Near(v, self.e + o.e + U32 * np.abs(v))

    def __mul__(self, o):
        v = self.v * o.v
        return Near(v, np.abs(self.v) * o.e + self.e * np.abs(o.v) + self.e * o.e + U32 * np.abs(v))

    def column_sums(self):
        n = self.v.shape[0]
        return Near(self.v.sum(0), self.e.sum(0) + (n + 16) * U32 * self.size.sum(0))

    def rounded(self, dtype):
        return Near(self.v, self.e + ROUND[dtype] * self.size + SMALL[dtype], torch.finfo(dtype).max)

    def holds(self, got, what=""):
        """Asserts that `got` (a tensor) lies within the bound everywhere."""
        got = got.detach().double().cpu().numpy()
        assert got.shape == self.v.shape, f"{what}: shape {got.shape}, expected {self.v.shape}"
        beyond = (self.size >= self.most) & np.isinf(got) & (np.sign(got) == np.sign(self.v))
        off = np.where(beyond, 0.0, np.abs(got - self.v))
        bad = ~(off <= self.e)
        if bad.any():
            at = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(self.e, 1e-300), 0)), off.shape)
            raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} numbers outside their bound, the worst at {at}: "
                                 f"{got[at]!r}, expected {self.v[at]!r} within {self.e[at]:.3e}")


def _erf(x):
    return np.vectorize(math.erf, otypes=[np.float64])(x) if x.size else x


def activation(name, g, dtype):
    """act(g) and act'(g)"""
    x, e = g.v, g.e
    with np.errstate(over="ignore"):
        s = 1.0 / (1.0 + np.exp(-x))
    if name == "relu":
        unsure = (np.abs(x) <= e) & (e > 0)
        return Near(np.maximum(x, 0), e), Near((x > 0).astype(float), unsure.astype(float))
    if name == "sigmoid":      # |act'| <= 1/4, |act''| < 0.1
        a, slope, first, second = s, s * (1 - s), 0.25, 0.1
    elif name == "silu":       # |act'| < 1.1, |act''| <= 1/2
        a, slope, first, second = x * s, s * (1 + x * (1 - s)), 1.1, 0.5
    else:                      # gelu: |act'| < 1.13, |act''| < 0.8
        below, density = 0.5 * (1 + _erf(x / math.sqrt(2))), np.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
        a, slope, first, second = x * below, below + x * density, 1.13, 0.8
    eps = EVAL[dtype]
    # (of factors that cancel, as 1 + erf and 1 - s do, the error is one of a number near 1)
    return Near(a, first * e + eps * np.maximum(1.0, np.abs(x))), Near(slope, second * e + eps * np.maximum(1.0, np.abs(x)))


def slope_by_differences(loss, tensors, name, direction, step=2.0 ** -13):
    """The derivative of `loss`, a function of a dict of float64 arrays, by array `name` along `direction`: from differences of the
    fourth order, in 64 bits (off by some step^4 of the fifth derivative and 2^-52 / step of the loss)."""
    at = lambda s: loss({**tensors, name: tensors[name] + s * step * direction})  # noqa: E731
    return (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * step)


def _near(t):
    return Near(t.detach().double().cpu().numpy())


def gated_ffn(t, act, grad=None, dtype=None):
    """(y, gradients by name) of the tensors in `t`, of any floating type; rows flattened."""
    dtype = dtype or t["x"].dtype
    hold = (lambda n: n) if dtype == torch.float32 else (lambda n: n.rounded(dtype))
    flat = lambda n: _near(t[n].reshape(-1, t[n].shape[-1]))  # noqa: E731
    x, wg, wu, wd = flat("x"), _near(t["w_gate"]), _near(t["w_up"]), _near(t["w_down"])
    none = Near(np.zeros(1))
    bias = lambda n: _near(t[n]) if t.get(n) is not None else none  # noqa: E731
    g, u = x @ wg.T + bias("b_gate"), x @ wu.T + bias("b_up")
    a, slope = activation(act, g, dtype)
    h = hold(a * u)
    y = h @ wd.T + bias("b_down")
    if t.get("residual") is not None:
        y = y + flat("residual")
    y = y.rounded(dtype)
    if grad is None:
        return y, {}
    dy = _near(grad.reshape(-1, grad.shape[-1]))
    dh = dy @ wd
    dg, du = hold(dh * u * slope), hold(dh * a)
    grads = {"x": dg @ wg + du @ wu, "w_gate": dg.T @ x, "w_up": du.T @ x, "w_down": dy.T @ h,
             "b_gate": dg.column_sums(), "b_up": du.column_sums(), "b_down": dy.column_sums(), "residual": dy}
    return y, {n: v.rounded(dtype) for n, v in grads.items() if n in ("x", "w_gate", "w_up", "w_down") or t.get(n) is not None}


def layer_norm(x, weight=None, bias=None, eps=1e-5, grad=None):
    """(y, gradients by name); rows flattened.  A row's sums are of depth 64 at most for each 256 numbers."""
    dtype, d = x.dtype, x.shape[-1]
    depth = (64 + d / 256) * U32
    v = x.detach().double().cpu().numpy().reshape(-1, d)
    w = np.ones(d) if weight is None else weight.detach().double().cpu().numpy()
    b = np.zeros(d) if bias is None else bias.detach().double().cpu().numpy()
    mean = v.mean(1, keepdims=True)
    c = v - mean
    rstd = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    n = c * rstd
    mean_off = depth * np.abs(v).mean(1, keepdims=True)
    # a wrong mean moves the differences by as much and the variance by its square; the variance itself is off by depth
    n_off = mean_off * rstd + np.abs(n) * (4 * depth + mean_off * rstd * mean_off * rstd) + 4 * U32 * (np.abs(v) * rstd + np.abs(n))
    y = Near(n, n_off) * Near(w) + Near(b)
    if grad is None:
        return y.rounded(dtype), {}
    dy = grad.detach().double().cpu().numpy().reshape(-1, d)
    rows = v.shape[0]
    dn = dy * w
    m1, m2 = dn.mean(1, keepdims=True), (dn * n).mean(1, keepdims=True)
    dx = rstd * (dn - m1 - n * m2)
    m1_off = depth * np.abs(dn).mean(1, keepdims=True)
    m2_off = (np.abs(dn) * n_off).mean(1, keepdims=True) + depth * np.abs(dn * n).mean(1, keepdims=True)
    dx_off = rstd * (m1_off + np.abs(n) * m2_off + n_off * (np.abs(m2) + m2_off) + 4 * U32 * (np.abs(dn) + np.abs(m1) + np.abs(n * m2)))
    dx_off = dx_off + np.abs(dx) * (4 * depth + mean_off * rstd * mean_off * rstd)
    terms = (rows + 16) * U32
    dw = Near((dy * n).sum(0), (np.abs(dy) * n_off).sum(0) + terms * np.abs(dy * n).sum(0))
    db = Near(dy.sum(0), terms * np.abs(dy).sum(0))
    grads = {"x": Near(dx, dx_off)}
    if weight is not None:
        grads["weight"] = dw
    if bias is not None:
        grads["bias"] = db
    return y.rounded(dtype), {k: g.rounded(dtype) for k, g in grads.items()}
