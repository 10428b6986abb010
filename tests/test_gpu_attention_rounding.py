"""How far attention and its gradients are from the definition in 64 bits in the mean, against one rounding of it to the type: the bounds of
network_reference.py are for the worst case, in which a number below the smallest of its type counts as often as there are keys."""
import math

import pytest
import torch

import svox_amd as svox

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]
name_of = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def exact(q, k, v, grad, causal=False):
    """(y, dq, dk, dv) in float64: every head by itself, its rows a few at a time."""
    (t, h, d), (n, kv_heads, _) = q.shape, k.shape
    group, scale, some = h // kv_heads, d ** -0.5, max(1, (1 << 25) // n)
    y, dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in (q, q, k, v))
    for i in range(h):
        kk, vv = k[:, i // group].double().contiguous(), v[:, i // group].double().contiguous()
        kt, vt = kk.t().contiguous(), vv.t().contiguous()
        for a in range(0, t, some):
            qq, gg = q[a:a + some, i].double().contiguous(), grad[a:a + some, i].double().contiguous()
            s = qq @ kt * scale
            if causal:
                s.masked_fill_(torch.arange(n, device=q.device)[None] > torch.arange(a, a + len(qq), device=q.device)[:, None] + n - t, -math.inf)
            p = torch.softmax(s, 1)
            y[a:a + some, i] = p @ vv
            ds = p * (gg @ vt - (gg * y[a:a + some, i]).sum(1, keepdim=True))
            dq[a:a + some, i] = ds @ kk * scale
            dk[:, i // group] += ds.t().contiguous() @ qq * scale
            dv[:, i // group] += p.t().contiguous() @ gg
    return y, dq, dk, dv


def roundings(got, want):
    """The root of the mean square of the error, in those of one rounding of `want`."""
    one = (want.to(got.dtype).double() - want).square().mean().sqrt()
    return float((got.double() - want).square().mean().sqrt() / one)


def inputs(t, n, h, kv_heads, d, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*shape, generator=g).to("cuda:0").to(dtype) for shape in ((t, h, d), (n, kv_heads, d), (n, kv_heads, d))], \
        (torch.randn(t, h, d, generator=g) * size).to("cuda:0").to(dtype)


def step(x, grad, **kw):
    leaves = [v.detach().requires_grad_() for v in x]
    y = svox.attention(*leaves, **kw)
    return [y.detach(), *torch.autograd.grad(y, leaves, grad)]


# A sum of many products of which one factor is rounded to the type is off by what one rounding of it is, in the mean, and the result is rounded once
# more: 1.42 times one rounding.  dq and dk have a part of the result's own error besides.  Twice one rounding is more than all of it.
TWO = 2.0

LONG = [(20, 262144, 8, 1, 32), (20, 32768, 8, 1, 64), (3, 100003, 4, 2, 128), (50, 70001, 2, 1, 33), (2100, 30011, 2, 2, 64)]


@pytest.mark.parametrize("dtype", HALVES, ids=name_of)
@pytest.mark.parametrize("t,n,h,kv_heads,d", LONG)
def test_values_gradients_over_long_rows(gpu, t, n, h, kv_heads, d, dtype):
    """Each p is some 1 / keys: below float16's normal numbers from 16 384 keys on."""
    x, grad = inputs(t, n, h, kv_heads, d, dtype, seed=n)
    want = exact(*x, grad)
    got = step(x, grad)
    assert roundings(got[0], want[0]) <= TWO
    assert roundings(got[3], want[3]) <= TWO
