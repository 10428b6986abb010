"""Operators of networks over cells where numbers lie beyond what 32 bits count, and where tiles are put in order by what they have to do."""
import math

import pytest
import torch

import svox_amd as svox
from test_gpu_attention import check, inputs, normal, packed, step

pytestmark = pytest.mark.gpu


def far_apart(rows, heads, d, stride, dtype, seed):
    """Heads whose rows lie `stride` numbers apart, and the same side by side."""
    room = torch.empty(rows, stride, dtype=dtype, device="cuda:0")
    x = room[:, :heads * d].unflatten(1, (heads, d))
    x.copy_(normal(torch.Generator().manual_seed(seed), rows, heads, d, dtype=dtype))
    return x, x.contiguous()


@pytest.mark.parametrize("d", [64, 40])
def test_rows_beyond_32_bits(gpu, d):
    """Keys and queries of more than 2^32 numbers from first to last, with and without direct loads: bit for bit what dense ones give."""
    rows, stride = 70000, 65536 + 8
    k, kd = far_apart(rows, 1, d, stride, torch.bfloat16, 1)
    q, qd = far_apart(rows, 2, d, stride, torch.bfloat16, 2)
    assert k.stride(0) * rows > 1 << 32
    few, fewd = q[-3:], qd[-3:]
    assert torch.equal(svox.attention(few, k, k), svox.attention(fewd, kd, kd))
    offsets = torch.tensor([0, 1000, 69000, 69600, 70000], device=gpu)
    grad = normal(torch.Generator().manual_seed(3), rows, 2, d, dtype=torch.bfloat16)
    lengths = packed([500] * 140)
    for o in (lengths, offsets):
        y, grads = step({"q": q, "k": k, "v": k}, grad, o, causal=True)
        yd, gradsd = step({"q": qd, "k": kd, "v": kd}, grad, o, causal=True)
        assert torch.equal(y, yd) and all(torch.equal(grads[n], gradsd[n]) for n in grads)
    positions, frequencies = torch.arange(rows, device=gpu), torch.rand(d // 2, device=gpu)
    a, b = svox.rotate_heads(q, k, positions, frequencies)
    ad, bd = svox.rotate_heads(qd, kd, positions, frequencies)
    assert torch.equal(a, ad) and torch.equal(b, bd)


def test_rows_beyond_32_bits_are_right_at_their_end(gpu):
    rows, stride = 70000, 65536 + 8
    k, kd = far_apart(rows, 1, 64, stride, torch.float16, 4)
    x, grad = inputs(5, 40, 2, 1, 64, torch.float16, seed=5)
    x["k"], x["v"] = k[-40:], k[-80:-40]
    check(x, grad)
    q = {"q": normal(torch.Generator().manual_seed(6), 5, 2, 64, dtype=torch.float16), "k": k, "v": k}
    want, _ = step({**q, "k": kd, "v": kd}, grad)
    got, _ = step(q, grad)
    assert torch.equal(want, got)


def test_clip_norm_of_more_than_2_to_32_numbers(gpu):
    n = (1 << 32) + 12345
    x = torch.empty(n, dtype=torch.float16, device=gpu)
    part = normal(torch.Generator().manual_seed(7), 1 << 20, dtype=torch.float16)
    for at in range(0, n, 1 << 28):
        x[at:at + (1 << 28)] = part.repeat(256)[:n - at]
    whole, left = divmod(n, 1 << 20)
    squares = float((part.double() ** 2).sum()) * whole + float((part[:left].double() ** 2).sum())
    norm, (y,) = svox.clip_norm([x], 0.25 * math.sqrt(squares))
    assert abs(float(norm) - math.sqrt(squares)) <= 2.0 ** -22 * math.sqrt(squares)
    assert torch.equal(y[:1 << 20], (part.float() * 0.25).half()) and torch.equal(y[-left:], (part[:left].float() * 0.25).half())
    middle = n // 2 // (1 << 20) * (1 << 20)
    assert torch.equal(y[middle:middle + (1 << 20)], y[:1 << 20])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_tiles_in_order(gpu, causal, dtype):
    """Sequences of different lengths, one of them empty, on as many blocks as make the operator put tiles in order: forward and both gradients."""
    lengths = [900, 3, 0, 1500, 64, 500, 1, 1200]
    x, grad = inputs(sum(lengths), sum(lengths), 32, 16, 16, dtype, seed=8)
    check(x, grad, packed(lengths), causal=causal)
    # orders differ from call to call where tiles have as much to do; results do not
    first = step(x, grad, packed(lengths), causal=causal)
    for _ in range(3):
        again = step(x, grad, packed(lengths), causal=causal)
        assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][n], again[1][n]) for n in first[1])


def test_tiles_in_order_within_a_graph(gpu):
    lengths = [[900, 3, 0, 1500, 64, 500, 1, 1200], [0, 0, 0, 0, 0, 0, 0, 4168], [521] * 8, [4160, 1, 1, 1, 1, 1, 1, 2]]
    x, grad = inputs(4168, 4168, 32, 16, 16, torch.bfloat16, seed=9)
    offsets = packed(lengths[0])
    leaves = {n: v.detach().requires_grad_() for n, v in x.items()}

    def run():
        y = svox.attention(leaves["q"], leaves["k"], leaves["v"], offsets, causal=True)
        return [y, *torch.autograd.grad(y, list(leaves.values()), grad)]

    with torch.cuda.stream(torch.cuda.Stream()):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for n in lengths:
        offsets.copy_(packed(n))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_a_result_that_was_changed_has_no_gradient(gpu):
    x, grad = inputs(20, 20, 2, 2, 32, torch.float32)
    leaf = x["q"].requires_grad_()
    y = svox.attention(leaf, x["k"], x["v"])
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(grad)


def test_offsets_of_any_kind_with_tiles_in_order(gpu):
    """Places outside of the arrays and out of order, on many blocks: other memory is not touched."""
    q, k = torch.randn(4100, 32, 16, device=gpu), torch.randn(4100, 16, 16, device=gpu)
    for offsets in ([4000, 0, 2000, -7, 1 << 40, 3], [5, 5, 5], [1 << 50, -(1 << 50), 100, 50]):
        t = {"q": q[2:4098].detach().requires_grad_(), "k": k[2:4098].detach().requires_grad_(), "v": k[2:4098].detach().clone().requires_grad_()}
        y = svox.attention(t["q"], t["k"], t["v"], torch.tensor(offsets, device=gpu), causal=True)
        grads = torch.autograd.grad(y, list(t.values()), torch.ones_like(y))
        assert all(torch.isfinite(v).all() for v in (y, *grads))


def test_a_graph_that_is_kept_gives_the_same_gradients_again(gpu):
    x, grad = inputs(300, 300, 4, 2, 64, torch.bfloat16, seed=10)
    leaves = [v.requires_grad_() for v in x.values()]
    y = svox.attention(*leaves, packed([200, 0, 100]))
    first = torch.autograd.grad(y, leaves, grad, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, grad)))
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        torch.autograd.grad(y, leaves, grad)


def test_sequences_without_any_key(gpu):
    x, grad = inputs(50, 0, 4, 2, 32, torch.float16)
    y, grads = step(x, grad, packed([20, 30]), packed([0, 0]), causal=True)
    assert not y.any() and not grads["q"].any() and grads["k"].shape == (0, 2, 32)
    x, grad = inputs(0, 50, 4, 2, 32, torch.float16)
    y, grads = step(x, grad, packed([0, 0]), packed([20, 30]))
    assert y.shape == (0, 4, 32) and not grads["k"].any() and not grads["v"].any()


def test_calls_from_two_threads(gpu):
    """Each with a stream of its own; errors of one thread are not the other's."""
    import threading

    sets = [inputs(500 + i, 2000, 4, 2, 64, torch.bfloat16, seed=i) for i in range(2)]
    want = [step(x, grad) for x, grad in sets]
    torch.cuda.synchronize()
    got, errors = [[], []], [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i].append(step(*sets[i]))
                try:
                    svox.attention(sets[i][0]["q"], sets[i][0]["k"], sets[i][0]["v"], scale=-1.0 - i)
                except RuntimeError as e:
                    errors[i].append(str(e))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(errors[i]) == 5 and all(f"{-1.0 - i:.6f}" in e for e in errors[i])
        for y, grads in got[i]:
            assert torch.equal(y, want[i][0]) and all(torch.equal(grads[n], want[i][1][n]) for n in grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_rows_between_that_see_nothing(gpu, d, bad, dtype):
    """Whatever the queries of a sequence without keys hold, and the keys of one without queries, between others of the same tiles."""
    for queries, keys, names in (([40, 5, 40], [40, 0, 40], ("q", "grad")), ([40, 0, 40], [40, 5, 40], ("k", "v"))):
        x, grad = inputs(sum(queries), sum(keys), 4, 2, d, dtype, seed=11)
        clean_y, clean = step(x, grad, packed(queries), packed(keys))
        for name in names:
            broken, dy = {n: v.clone() for n, v in x.items()}, grad.clone()
            (dy if name == "grad" else broken[name])[40:45, :, 1:4] = bad
            y, grads = step(broken, dy, packed(queries), packed(keys))
            assert torch.equal(y, clean_y), name
            assert torch.equal(grads["q"], clean["q"]), name
            assert torch.equal(grads["k"], clean["k"]) and torch.equal(grads["v"], clean["v"]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 33, 64, 128])
def test_what_other_sequences_hold_in_larger_launches(gpu, d, causal, dtype):
    """Tiles of 128 rows that hold several sequences, of which one is not finite."""
    lengths = [1 + 37 * i % 170 for i in range(103)]
    rows, first = sum(lengths), sum(lengths[:50])
    x, grad = inputs(rows, rows, 8, 8, d, dtype, seed=12)
    offsets, mine = packed(lengths), slice(first, first + lengths[50])
    others = torch.ones(rows, dtype=torch.bool)
    others[mine] = False
    clean_y, clean = step(x, grad, offsets, causal=causal)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for name in ("q", "k", "v", "grad"):
            broken, dy = {n: v.clone() for n, v in x.items()}, grad.clone()
            (dy if name == "grad" else broken[name])[mine, :, d // 2] = bad
            y, grads = step(broken, dy, offsets, causal=causal)
            assert torch.equal(y[others], clean_y[others]), name
            assert all(torch.equal(grads[n][others], clean[n][others]) for n in grads), name
            assert not torch.isfinite(grads[{"grad": "v", "v": "q"}.get(name, name)][mine]).all(), name
