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


SHAPES = [(200, 4096, 2, 1, 64), (200, 32768, 2, 1, 128), (70, 20011, 4, 2, 33), (300, 9000, 2, 2, 32), (40, 33000, 3, 1, 100)]


@pytest.mark.parametrize("dtype", HALVES, ids=name_of)
@pytest.mark.parametrize("size", [1e-3, 1.0, 300.0])
@pytest.mark.parametrize("t,n,h,kv_heads,d", SHAPES)
def test_gradients_of_every_size_over_long_rows(gpu, t, n, h, kv_heads, d, size, dtype):
    """Influences of single scores, some 1 / keys of the gradient's, below what float16 holds, or beyond it."""
    x, grad = inputs(t, n, h, kv_heads, d, dtype, seed=n, size=size)
    for got, want in zip(step(x, grad), exact(*x, grad)):
        assert roundings(got, want) <= TWO


@pytest.mark.parametrize("dtype", HALVES, ids=name_of)
@pytest.mark.parametrize("size", [1e-4, 1.0, 4000.0])
@pytest.mark.parametrize("d,kv_heads", [(16, 2), (32, 1), (64, 1), (128, 2), (100, 1)])
def test_gradients_of_every_size_of_causal_rows(gpu, d, kv_heads, size, dtype):
    """Few keys to a row and many."""
    x, grad = inputs(1500, 1500, 2, kv_heads, d, dtype, seed=d, size=size)
    want = exact(*x, grad, causal=True)
    assert all(float(w.abs().max()) < torch.finfo(torch.float16).max for w in want)
    for got, w in zip(step(x, grad, causal=True), want):
        assert roundings(got, w) <= TWO


@pytest.mark.parametrize("d", [32, 64, 128, 33])
@pytest.mark.parametrize("falling", [False, True])
def test_sizes_that_differ_from_row_to_row_and_along_a_row(gpu, d, falling):
    """Rows' gradients of all sizes from 2^-9 to 2^9, in either order, so that sums over rows grow by 2^18 on their way, and so do values along the keys:
    each row is as exact as if it were alone, and so is each key whose values are small."""
    t, n = 600, 5000
    x, grad = inputs(t, n, 2, 1, d, torch.float16, seed=d)
    along = 2.0 ** torch.linspace(9, -9, t, device="cuda:0") if falling else 2.0 ** torch.linspace(-9, 9, t, device="cuda:0")
    grad = (grad * along[:, None, None]).half()
    got, want = step(x, grad), exact(*x, grad)
    for a, b in zip(got, want):
        assert roundings(a, b) <= TWO
    for a in range(0, t, 50):
        assert roundings(got[1][a:a + 50], want[1][a:a + 50]) <= TWO
    x[2] = (x[2] * (2.0 ** torch.linspace(5 if falling else -5, -5 if falling else 5, n, device="cuda:0"))[:, None, None]).half()
    grad = (grad / along[:, None, None]).half()
    got, want = step(x, grad), exact(*x, grad)
    for a, b in zip(got, want):
        assert roundings(a, b) <= TWO


def test_rows_do_not_depend_on_what_their_neighbours_are(gpu):
    """Bit for bit, where the other sequences' gradients and values are 2^12 times as large or as small."""
    lengths = [30, 50, 7, 90, 41]
    offsets = torch.tensor([0, 30, 80, 87, 177, 218], device="cuda:0")
    for d in (32, 64, 128, 33):
        x, grad = inputs(218, 218, 4, 2, d, torch.float16, seed=d, size=1e-2)
        mine = slice(80, 87)
        clean = step(x, grad, offsets=offsets, causal=True)
        for factor in (2.0 ** 12, 2.0 ** -12):
            other, dy = [v.clone() for v in x], grad * factor
            other[2] = other[2] * factor
            for v, w in ((other[2], x[2]), (dy, grad)):
                v[mine] = w[mine]
            for a, b in zip(clean, step(other, dy, offsets=offsets, causal=True)):
                assert torch.equal(a[mine], b[mine])
    assert sum(lengths) == 218


@pytest.mark.parametrize("d", [32, 64, 128, 33])
def test_influences_beyond_float16(gpu, d):
    """do . v beyond 65 504 for keys so small that no gradient is."""
    x, grad = inputs(700, 700, 2, 1, d, torch.float16, seed=d, size=4000.0)
    x[0], x[1], x[2] = x[0] / 16, x[1] / 64, x[2] * 8
    want = exact(*x, grad, causal=True)
    assert all(float(w.abs().max()) < torch.finfo(torch.float16).max for w in want[1:])
    assert float((grad[:, 0].double() @ x[2][:, 0].double().t().contiguous()).abs().max()) > 2 * torch.finfo(torch.float16).max
    for got, w in zip(step(x, grad, causal=True), want):
        assert roundings(got, w) <= TWO


@pytest.mark.parametrize("dtype", HALVES, ids=name_of)
@pytest.mark.parametrize("d", [32, 64, 128, 33])
def test_a_row_of_small_exponentials(gpu, d, dtype):
    """Each e^-8 to e^-15 of the first, times values 100 times as large, in rows that no blocks share.  They are alike and rounded alike, by half a step,
    which is 2^-p of them at most (p bits); the root of the mean square of one rounding of the result is 2^-p-1 / sqrt(3) of it at least, and the
    result is rounded itself: at most sqrt(1 + 12) roundings, if they are all of the row.  A sum of 4096 numbers one after another, a lane's, is off by
    4096 2^-24 of itself at most, two roundings of float16.  Together less than 6."""
    g = torch.Generator().manual_seed(d)
    t, n = 16384, 8192
    q, k = torch.ones(t, 8, d, device="cuda:0", dtype=dtype), torch.zeros(n, 1, d, device="cuda:0", dtype=dtype)
    v = (100 * torch.linspace(0.7, 1.3, d) + torch.randn(n, 1, d, generator=g)).to("cuda:0").to(dtype)     # (so that results lie anywhere between steps)
    v[0] = 1
    for below in (8.0, 9.5, 10.4, 11.0, 12.0, 13.0, 14.2, 15.0):
        k.fill_(-below * d ** -0.5)
        k[0] = 0
        want = exact(q[:1, :1], k, v, torch.zeros_like(q[:1, :1]))[0]
        assert roundings(svox.attention(q, k, v), want.expand(t, 8, d)) <= 6.0, below


@pytest.mark.parametrize("d", [32, 64, 128, 30, 50, 99])
def test_long_sums_in_32_bits(gpu, d):
    """float32: a row's sums go over 65 536 keys in tiles of 32 or more, a key's over 16 384 rows.  An addition is a rounding of what the sum is by then: of
    n / 32 one after another each of two sums (a row's exponentials and their products with values) has the root of n / 64 roundings' error, those within
    a tile, a score's and an exponential's are some 200 more, a logarithm of a sum of some 2^14 as many again.  Twice the root of all of them, as they
    are not all by themselves; of n / 4 or n / 2 additions one after another it would be more than that."""
    t, n, h = 16384, 65536, 8
    x, grad = inputs(t, n, h, h, d, torch.float32, seed=d)
    got, want = step(x, grad), exact(*(v[:, :1] for v in (*x, grad)))
    for name, a, b, along in zip(("y", "q", "k", "v"), got, want, (n, n, t, t)):
        assert roundings(a[:, :1], b) <= 2 * math.sqrt(400 + along / 32), name


@pytest.mark.parametrize("dtype", HALVES, ids=name_of)
@pytest.mark.parametrize("n,d", [(300, 64), (4000, 32), (4000, 128), (2000, 33)])
@pytest.mark.parametrize("values", [1e-2, 1e-4, 1e-5])
def test_small_values_and_large_gradients(gpu, n, d, values, dtype):
    """A loss that is scaled, as float16 asks for, over values whose mean float16 holds a few bits of: the influences of scores are of both's product."""
    x, grad = inputs(300, n, 2, 1, d, dtype, seed=d, size=2000.0)
    x[2] = (x[2].float() * values).to(dtype)
    for got, want in zip(step(x, grad), exact(*x, grad)):
        assert roundings(got, want) <= TWO
