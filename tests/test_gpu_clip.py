"""The norm of many tensors and its clipping against their definition in 64 bits."""
import math

import pytest
import torch

import svox_amd as svox
from network_reference import clip_norm

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
name_of = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def some(sizes, dtypes, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtypes[i % len(dtypes)]).to("cuda:0") for i, n in enumerate(sizes)]


def check(tensors, max_norm):
    near, wanted = clip_norm(tensors, max_norm)
    before = [x.clone() for x in tensors]
    norm, out = svox.clip_norm(tensors, max_norm)
    assert norm.dtype == torch.float32 and norm.shape == ()
    near.holds(norm, "norm")
    assert len(out) == len(tensors)
    for i, (x, y, want) in enumerate(zip(tensors, out, wanted)):
        assert y.dtype == x.dtype and y.shape == x.shape and y.data_ptr() != x.data_ptr() or x.numel() == 0
        want.holds(y, f"tensor {i}")
    assert all(torch.equal(x, b) for x, b in zip(tensors, before))
    leaves = []
    for x in tensors:
        leaves.append(torch.zeros_like(x).requires_grad_())
        leaves[-1].grad = x.clone()
    at = [p.grad.data_ptr() for p in leaves]
    norm2 = svox.clip_grad_norm(leaves, max_norm)
    assert torch.equal(norm2, norm) and at == [p.grad.data_ptr() for p in leaves]
    assert all(torch.equal(p.grad, y) for p, y in zip(leaves, out))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("sizes", [[1], [0, 3, 0], [7, 1, 4095, 4096, 4097], [8191, 16384, 8193, 5], [300007]], ids=str)
@pytest.mark.parametrize("share", [0.25, 0.9999, 4.0])
def test_sizes(gpu, sizes, share, dtype):
    tensors = some(sizes, [dtype])
    check(tensors, share * math.sqrt(sum(float((x.double() ** 2).sum()) for x in tensors)))


@pytest.mark.parametrize("n", [2, 95, 96, 97, 193, 500])
def test_many_tensors_of_several_types(gpu, n):
    check(some([1 + 37 * i % 1000 for i in range(n)], DTYPES, seed=n), 3.0)


def test_more_chunks_than_blocks(gpu):
    check(some([9_000_003, 2, 10_000_000], [torch.float32], seed=1), 100.0)
    check(some([30_000_007], [torch.bfloat16], seed=2), 100.0)


def test_numbers_whose_squares_leave_float32(gpu):
    for scale in (1e30, 1e-30):
        tensors = some([100, 5000], [torch.float32], scale=scale)
        check(tensors, scale)
    huge = torch.full((10,), 3e38, device="cuda:0")
    norm, (y,) = svox.clip_norm([huge], 1.0)         # (the norm is beyond float32, the factor is not)
    assert torch.isinf(norm) and torch.allclose(y, torch.full_like(y, 10 ** -0.5), rtol=2.0 ** -21, atol=0)


def test_bounds_at_the_ends(gpu):
    x, = some([1000], [torch.float32])
    norm, (y,) = svox.clip_norm([x], 0.0)
    assert torch.equal(y, torch.zeros_like(y)) and norm > 0
    for most in (float(norm) * 1.001, math.inf):
        assert torch.equal(svox.clip_norm([x], most)[1][0], x)
    zero = torch.zeros(5, device="cuda:0")
    norm, (y,) = svox.clip_norm([zero], 0.0)
    assert norm == 0 and torch.equal(y, zero)
    assert svox.clip_norm([], 1.0)[1] == [] and svox.clip_grad_norm([], 1.0) == 0
    assert svox.clip_norm([zero[:0]], 1.0)[0] == 0
    norm, out = svox.clip_norm(x, 1.0)
    assert len(out) == 1 and torch.equal(out[0], svox.clip_norm([x], 1.0)[1][0])
    norm, (a, b) = svox.clip_norm([x, x], 1.0)     # (twice is twice)
    assert torch.equal(a, b) and a.data_ptr() != b.data_ptr() and abs(float(norm) - float(x.norm()) * 2 ** 0.5) <= 1e-4


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_what_is_not_finite_stays(gpu, bad, dtype):
    tensors = some([10, 20000], [dtype])
    tensors[1][777] = bad
    norm, out = svox.clip_norm(tensors, 0.1)
    assert not torch.isfinite(norm) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(tensors, out))
    leaf = torch.zeros_like(tensors[1]).requires_grad_()
    leaf.grad = tensors[1].clone()
    assert not torch.isfinite(svox.clip_grad_norm(leaf, 0.1))
    assert torch.equal(leaf.grad.view(torch.uint8), tensors[1].view(torch.uint8))


def test_layouts(gpu):
    """Turned, sliced, broadcast and negated tensors, one that does not begin at 16 bytes."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(61, 48, generator=g).to("cuda:0")
    odd = torch.randn(1001, generator=g).to(torch.float16).to("cuda:0")[1:]
    tensors = [x.t(), x[:, 3:20], x[::2], x[:1].expand(5, 48), odd, torch._neg_view(x), x[:0], x[0, 0]]
    near, wanted = clip_norm(tensors, 1.0)
    norm, out = svox.clip_norm(tensors, 1.0)
    near.holds(norm)
    for x_, y, want in zip(tensors, out, wanted):
        assert y.shape == x_.shape
        want.holds(y)


def test_gradients_where_they_lie(gpu):
    """A gradient in a slice, one that two parameters hold, one in turned order; what lies between stays, versions move on."""
    def leaf(grad):
        p = torch.zeros(grad.shape, device="cuda:0", dtype=grad.dtype).requires_grad_()
        p.grad = grad
        return p

    g = torch.Generator().manual_seed(4)
    wide = torch.randn(50, 20, generator=g).to("cuda:0")
    turned = torch.randn(7, 9, generator=g).to("cuda:0").t()
    shared = torch.randn(33, generator=g).to("cuda:0")
    kept = wide.clone()
    near, (a, b, c) = clip_norm([wide[:, 2:9].clone(), turned.clone(), shared.clone()], 0.5)
    without = torch.zeros(3, device="cuda:0", requires_grad=True)
    versions = [t._version for t in (wide, turned, shared)]
    norm = svox.clip_grad_norm((p for p in [leaf(wide[:, 2:9]), without, leaf(turned), leaf(shared), leaf(shared)]), 0.5)
    near.holds(norm)
    a.holds(wide[:, 2:9]), b.holds(turned), c.holds(shared)
    assert torch.equal(wide[:, :2], kept[:, :2]) and torch.equal(wide[:, 9:], kept[:, 9:]) and without.grad is None
    assert all(t._version > v for t, v in zip((wide, turned, shared), versions))
    for pair in ([shared, shared[1:]], [wide[:, 0], wide[:, 1]], [shared[:20], shared[:10]]):
        with pytest.raises(RuntimeError, match="share memory"):
            svox.clip_grad_norm([leaf(x) for x in pair], 0.5)
    with pytest.raises(RuntimeError, match="expand"):
        svox.clip_grad_norm(leaf(shared[:1].expand(9)), 0.5)


def test_refusals(gpu):
    x = torch.zeros(4, device="cuda:0")
    for tensors, most, error, text in [([x, x.cpu()], 1.0, RuntimeError, "CUDA tensor"), ([x.double()], 1.0, RuntimeError, "float32, float16 or bfloat16"),
                                       ([x], -1.0, RuntimeError, "max_norm"), ([x], math.nan, RuntimeError, "max_norm"), ([x, None], 1.0, TypeError, "tensor"),
                                       ([x.clone().requires_grad_()], 1.0, RuntimeError, "no gradient"), ([x.to_sparse()], 1.0, RuntimeError, "dense"),
                                       ([x], "1", TypeError, "real number")]:
        with pytest.raises(error, match=text):
            svox.clip_norm(tensors, most)
    with torch.no_grad():
        svox.clip_norm([x.clone().requires_grad_()], 1.0)


def test_a_captured_call_follows_its_inputs(gpu):
    tensors = some([5000, 3, 70001], DTYPES, seed=5)
    clipped = lambda: svox.clip_norm(tensors, 1.0)  # noqa: E731
    clipped()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, out = clipped()
    for i in range(3):
        for x in tensors:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to("cuda:0") * 10.0 ** i)
        graph.replay()
        torch.cuda.synchronize()
        want, wanted = clipped()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, wanted))


def test_two_streams_at_once(gpu):
    sets = [some([200000 + i, 31], DTYPES, seed=i) for i in range(2)]
    want = [svox.clip_norm(s, 2.0) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            got.append([svox.clip_norm(s, 2.0) for _ in range(5)])
    torch.cuda.synchronize()
    for (norm, out), several in zip(want, got):
        for n, o in several:
            assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(o, out))
