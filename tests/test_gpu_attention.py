"""Attention within packed sequences, and its gradients, against the definition in 64 bits (network_reference.py, whose bounds are derived from
where the operator rounds), at the sizes, layouts, masks and numbers where kernels like these go wrong."""
import numpy as np
import pytest
import torch

import svox_amd as svox
from decoder_reference import slope_by_differences
from network_reference import _attend, attention, seen_by

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
name_of = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to("cuda:0")


def inputs(t, n, h, g, d, dtype, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    return {"q": normal(gen, t, h, d, scale=spread, dtype=dtype), "k": normal(gen, n, g, d, dtype=dtype), "v": normal(gen, n, g, d, dtype=dtype)}, \
        normal(gen, t, h, d, dtype=dtype)


def packed(lengths, kind=torch.int32):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(kind).to("cuda:0")


def step(t, grad, *args, **kw):
    t = {n: v.detach().requires_grad_() for n, v in t.items()}
    y = svox.attention(t["q"], t["k"], t["v"], *args, **kw)
    return y, dict(zip(t, torch.autograd.grad(y, list(t.values()), grad)))


def check(t, grad, offsets=None, key_offsets=None, **kw):
    listed = lambda x: None if x is None else x.tolist()  # noqa: E731
    want, wanted = attention(t["q"], t["k"], t["v"], listed(offsets), listed(key_offsets), grad=grad, **kw)
    with torch.no_grad():
        without = svox.attention(t["q"], t["k"], t["v"], offsets, key_offsets, **kw)
    y, grads = step(t, grad, offsets, key_offsets, **kw)
    assert torch.equal(without, y)
    want.holds(y, "y")
    for name, got in grads.items():
        assert got.shape == t[name].shape and got.dtype == t[name].dtype
        wanted[name].holds(got, f"gradient of {name}")


# one sequence: lengths on both sides of 32, 64 and 128, heads of every width, groups of every kind
SIZES = [(1, 1, 1, 1, 1), (1, 1, 1, 1, 64), (2, 3, 2, 1, 8), (31, 33, 3, 3, 16), (32, 32, 4, 2, 32), (64, 64, 2, 2, 33), (65, 63, 6, 2, 64), (128, 128, 1, 1, 128),
         (129, 127, 5, 1, 100), (1, 300, 8, 2, 64), (1, 5000, 4, 1, 128), (7, 1000, 2, 1, 20), (300, 1, 3, 1, 48), (257, 260, 7, 7, 7), (200, 20, 8, 1, 96),
         (1000, 150, 2, 2, 65), (40, 700, 16, 4, 24), (3, 3, 21, 3, 127), (600, 600, 1, 1, 32)]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t,n,h,g,d", SIZES)
def test_one_sequence(gpu, t, n, h, g, d, causal, dtype):
    x, grad = inputs(t, n, h, g, d, dtype, seed=t + n + d, spread=2.0)
    check(x, grad, causal=causal)


LENGTHS = [[1], [1, 1, 1, 1, 1], [0, 5, 0, 0, 70, 0], [64, 64, 64], [128, 128], [33, 1, 200, 64, 2, 9], [8] * 40, [3, 130, 0, 257, 31, 32, 33], [1] * 150, [500, 12]]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: f"{len(x)}of{sum(x)}")
def test_packed_sequences(gpu, lengths, causal, dtype):
    h, g, d = [(2, 1, 32), (4, 4, 16), (3, 1, 64), (4, 2, 80)][len(lengths) % 4]
    x, grad = inputs(sum(lengths), sum(lengths), h, g, d, dtype, seed=sum(lengths))
    check(x, grad, packed(lengths, torch.int64 if len(lengths) % 2 else torch.int32), causal=causal)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("causal", [False, True])
def test_queries_and_keys_of_different_lengths(gpu, causal, dtype):
    """Sequences without queries, without keys, with more of the one or the other: rows that see nothing are zeros."""
    for of_q, of_k, d in [([1] * 9, [300, 0, 1, 64, 65, 2, 1000, 31, 5], 64), ([4, 0, 40, 7, 0], [9, 30, 0, 3, 0], 32), ([100, 3, 60], [10, 200, 59], 128)]:
        x, grad = inputs(sum(of_q), sum(of_k), 4, 2, d, dtype, seed=sum(of_k))
        check(x, grad, packed(of_q), packed(of_k), causal=causal)
        empty = [i for i, (a, b) in enumerate(zip(of_q, of_k)) if a and not b]
        y = svox.attention(x["q"], x["k"], x["v"], packed(of_q), packed(of_k), causal=causal)
        for i in empty:
            assert not y[sum(of_q[:i]):sum(of_q[:i + 1])].any()


def test_many_sequences_and_blocks(gpu):
    """More tiles than the GPU has places for, sequences found among thousands."""
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 20, (3000,), generator=g).tolist()
    x, grad = inputs(sum(lengths), sum(lengths), 2, 1, 16, torch.bfloat16, seed=2)
    check(x, grad, packed(lengths))
    check(x, grad, packed(lengths), causal=True)
    lengths = [700, 1, 900, 40, 3, 1100]
    x, grad = inputs(sum(lengths), sum(lengths), 16, 8, 32, torch.float16, seed=3)
    check(x, grad, packed(lengths), causal=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_rows_of_no_sequence(gpu, dtype):
    """Rows before the first and behind the last sequence are zeros, have no gradient and no influence."""
    x, grad = inputs(150, 150, 2, 1, 40, dtype, seed=4)
    for offsets in ([10, 30, 100], [0, 64, 64, 70], [149, 150], [70, 70]):
        check(x, grad, torch.tensor(offsets, device="cuda:0"), causal=True)
        bad = {n: v.clone() for n, v in x.items()}
        for v in bad.values():
            v[:offsets[0]] = float("nan")
            v[offsets[-1]:] = float("nan")
        bad_grad = grad.clone()
        bad_grad[:offsets[0]] = float("nan")
        bad_grad[offsets[-1]:] = float("inf")
        y, grads = step(x, grad, torch.tensor(offsets, device="cuda:0"))
        y2, grads2 = step(bad, bad_grad, torch.tensor(offsets, device="cuda:0"))
        assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_what_masked_rows_hold_has_no_influence(gpu, bad, d, dtype):
    lengths = [20, 7, 90, 1, 60]
    x, grad = inputs(178, 178, 2, 1, d, dtype, seed=5)
    offsets, at = packed(lengths), 20 + 7 + 40       # a row of the third sequence
    for causal in (False, True):
        clean_y, clean = step(x, grad, offsets, causal=causal)
        others = torch.ones(178, dtype=torch.bool)
        others[27:117] = False
        before = torch.arange(178) < at
        for name in ("q", "k", "v", "grad"):
            broken, dy = {n: v.clone() for n, v in x.items()}, grad.clone()
            (dy if name == "grad" else broken[name])[at, :, 3] = bad
            y, grads = step(broken, dy, offsets, causal=causal)
            keep = others | before if causal and name in ("k", "v") else others
            if name in ("q", "grad"):
                keep = torch.arange(178) != at
            assert torch.equal(y[keep], clean_y[keep]), name
            assert torch.equal(grads["q"][keep], clean["q"][keep]), name
            seen = others | (torch.arange(178) > at) if causal and name in ("q", "grad") else others
            if name in ("q", "grad"):
                assert torch.equal(grads["k"][seen], clean["k"][seen]) and torch.equal(grads["v"][seen], clean["v"][seen]), name
                assert not torch.isfinite(grads["v" if name == "grad" else "k"][27:at + 1]).all()
            else:
                assert torch.equal(grads["k"][others], clean["k"][others]) and torch.equal(grads["v"][others], clean["v"][others]), name
            if name == "v":                          # what does see it gets it
                want = torch.full_like(y[at:117, :, 3] if causal else y[27:117, :, 3], bad)
                assert torch.equal(y[at:117, :, 3] if causal else y[27:117, :, 3], want) or bad != bad and y[at:117, :, 3].isnan().all()
                assert torch.equal(y[27:117, :, :3], clean_y[27:117, :, :3])


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_large_scores(gpu, dtype):
    """Scores of hundreds, where exp overflows, and rows that see one key alone."""
    x, grad = inputs(100, 100, 2, 2, 32, dtype, seed=6)
    x["q"] = x["q"] * 16
    x["k"] = x["k"] * 4
    check(x, grad, causal=True)
    check(x, grad, packed([1] * 100))
    check({**x, "q": torch.zeros_like(x["q"])}, grad, causal=True, scale=3.0)


def test_layouts(gpu):
    """Heads as slices of one product, an odd beginning, turned, broadcast and negated ones, a gradient of one number."""
    for dtype in DTYPES:
        g = torch.Generator().manual_seed(7)
        x, grad = inputs(70, 70, 4, 2, 24, dtype, seed=8)
        wide = normal(g, 70, 8 * 24 + 5, dtype=dtype)
        for at in (0, 1, 5):
            q, k, v = wide[:, at:at + 192].split([96, 48, 48], dim=1)
            check({"q": q.unflatten(1, (4, 24)), "k": k.unflatten(1, (2, 24)), "v": v.unflatten(1, (2, 24))}, grad, causal=True)
        check({**x, "q": normal(g, 4, 70, 24, dtype=dtype).transpose(0, 1), "k": normal(g, 70, 24, 2, dtype=dtype).transpose(1, 2)}, grad)
        check({**x, "k": x["k"][:, :1].expand(70, 2, 24), "v": x["v"][:1].expand(70, 2, 24)}, grad)
        check(x, grad.new_ones(1, 1, 1).expand(70, 4, 24))
        check(x, normal(g, 70, 4, 31, dtype=dtype)[..., 3:27])
        check({**x, "v": torch._neg_view(x["v"])}, grad)
        check(x, grad, torch.tensor([0, 9, 30, 9, 70, 9], device="cuda:0")[::2], causal=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(gpu, causal, dtype):
    lengths, d = [9, 30, 1], 20
    x, grad = inputs(40, 40, 2, 1, d, dtype, seed=9)
    offsets = packed(lengths)
    _, grads = step(x, grad, offsets, causal=causal)
    _, wanted = attention(x["q"], x["k"], x["v"], offsets.tolist(), grad=grad, causal=causal)
    f64 = {n: v.double().cpu() for n, v in x.items()}
    c = grad.double().cpu().numpy()

    def loss(t):
        total, at = 0.0, 0
        for n in lengths:
            for h in range(2):
                q, k, v = t["q"][at:at + n, h].numpy(), t["k"][at:at + n, 0].numpy(), t["v"][at:at + n, 0].numpy()
                total += float((_attend(q, k, v, seen_by(n, n, causal), d ** -0.5, torch.float32, None)[0][0] * c[at:at + n, h]).sum())
            at += n
        return total

    g = torch.Generator().manual_seed(10)
    for n in f64:
        v = torch.randn(f64[n].shape, generator=g).sign().double()
        slope = slope_by_differences(loss, f64, n, v)
        along = float((grads[n].double().cpu() * v).sum())
        assert abs(slope - along) <= float(wanted[n].e.sum()) + 2.0 ** -20 * float(np.abs(wanted[n].v).sum()), n


def test_only_what_is_asked_for(gpu):
    x, grad = inputs(130, 130, 4, 2, 64, torch.bfloat16, seed=11)
    _, all_grads = step(x, grad, causal=True)
    for names in (["q"], ["k"], ["v"], ["k", "v"], ["v", "q"]):
        leaves = {n: v.detach().requires_grad_(n in names) for n, v in x.items()}
        got = torch.autograd.grad(svox.attention(leaves["q"], leaves["k"], leaves["v"], causal=True), [leaves[n] for n in names], grad)
        assert all(torch.equal(a, all_grads[n]) for n, a in zip(names, got)), names


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_no_queries_and_no_keys(gpu, dtype):
    x, grad = inputs(0, 50, 4, 2, 32, dtype)
    y, grads = step(x, grad)
    assert y.shape == (0, 4, 32) and not grads["k"].any() and not grads["v"].any() and grads["q"].shape == (0, 4, 32)
    x, grad = inputs(50, 0, 4, 2, 32, dtype)
    y, grads = step(x, grad)
    assert not y.any() and not grads["q"].any() and grads["k"].shape == (0, 2, 32)


def test_offsets_that_make_no_sense_stay_within_the_arrays(gpu):
    """Places outside of the arrays and out of order: results are unspecified, other memory is not touched."""
    for offsets, of_k in [([-5, 1000000, 3], None), ([0, 50, 20, 70, 10, 90], None), ([90, 0], None), ([0, 40, 90], [80, -1, 200])]:
        q = torch.randn(92, 2, 32, device=gpu)
        k = torch.randn(94, 2, 32, device=gpu)
        t = {"q": q[1:91].detach().requires_grad_(), "k": k[2:92].detach().requires_grad_(), "v": k[2:92].detach().clone().requires_grad_()}
        of = lambda x: None if x is None else torch.tensor(x, device=gpu)  # noqa: E731
        y = svox.attention(t["q"], t["k"], t["v"], of(offsets), of(of_k), causal=True)
        grads = torch.autograd.grad(y, list(t.values()), torch.ones_like(y))
        assert all(torch.isfinite(x).all() for x in (y, *grads))


def test_refusals(gpu):
    x, grad = inputs(6, 6, 4, 2, 32, torch.float32)
    q, k, v = x["q"], x["k"], x["v"]
    o = packed([2, 4])
    for args, text in [((q[0], k, v), "3-D"), ((q, k[:5], v), "shape"), ((q, k[..., :31], v[..., :31]), "same numbers of a head"), ((q, k.half(), v), "scalar type"),
                       ((q, k.cpu(), v), "CUDA tensor"), ((q.double(), k, v), "float32, float16"), ((q[:, :3], k, v), "multiple"), ((q, k, v, o.float()), "int32 or int64"),
                       ((q, k, v, o[:1]), "sequences"), ((q, k, v, o[None]), "sequences"), ((q, k, v, o.cpu()), "device of q"), ((q, k, v, None, o), "need offsets"),
                       ((q, k[:5], v[:5], o), "as many keys"), ((q, k, v, o, o.long()), "same shape and type"), ((q, k, v, o, packed([6])), "same shape and type"),
                       ((q, k, v, None, None, False, 0.0), "scale"), ((q, k, v, None, None, False, -1.0), "scale"), ((q, k, v, None, None, False, float("nan")), "scale")]:
        with pytest.raises(RuntimeError, match=text):
            svox.attention(*args)
    wide = torch.zeros(3, 1, 129, device=gpu)
    with pytest.raises(RuntimeError, match="dim must be <= 128"):
        svox.attention(wide, wide, wide)
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(svox.attention(leaf, k, v).sum(), leaf, create_graph=True)
    y = svox.attention(leaf, k, v, o)
    o.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), leaf)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_a_captured_step_follows_its_inputs(gpu, dtype):
    lengths = [100, 3, 200, 17]
    x, grad = inputs(320, 320, 4, 2, 64, dtype, seed=12)
    offsets = packed(lengths)
    leaves = {n: v.detach().requires_grad_() for n, v in x.items()}
    few, many = normal(torch.Generator().manual_seed(1), 1, 4, 64, dtype=dtype), normal(torch.Generator().manual_seed(2), 4000, 2, 64, dtype=dtype)

    def run():
        y = svox.attention(leaves["q"], leaves["k"], leaves["v"], offsets, causal=True)
        with torch.no_grad():
            split = svox.attention(few, many, many)
        return [y, split, *torch.autograd.grad(y, list(leaves.values()), grad)]

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            for v in (*leaves.values(), many):
                v.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(i)))
            offsets.copy_(packed([[100, 3, 200, 17], [1, 318, 0, 1], [320, 0, 0, 0]][i]))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_two_streams_at_once(gpu):
    sets = [inputs(400 + i, 3000, 4, 2, 64, torch.bfloat16, seed=i) for i in range(2)]
    want = [step(x, grad) for x, grad in sets]
    torch.cuda.synchronize()
    got = []
    for x, grad in sets:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append([step(x, grad) for _ in range(4)])
    torch.cuda.synchronize()
    for (y, grads), several in zip(want, got):
        for y2, grads2 in several:
            assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("d", [32, 64, 128, 24])
def test_heads_that_begin_anywhere(gpu, d, dtype):
    """Whole and partial widths whose numbers do not lie at whole numbers of 16 bytes, or rows of which do not."""
    g = torch.Generator().manual_seed(13)
    for shift, more in ((1, 0), (0, 1), (8, 8), (2, 6)):
        wide = normal(g, 140, 6 * d + shift + more, dtype=dtype)
        q, k, v = wide[:, shift:shift + 6 * d].split([2 * d, 2 * d, 2 * d], dim=1)
        grads = normal(g, 140, 2 * d + shift + more, dtype=dtype)[:, shift:shift + 2 * d].unflatten(1, (2, d))
        check({"q": q.unflatten(1, (2, d)), "k": k.unflatten(1, (2, d)), "v": v.unflatten(1, (2, d))}, grads, packed([100, 3, 37]), causal=True)
        grads = normal(g, 140, 2, d, dtype=dtype)
        check({"q": q.unflatten(1, (2, d)), "k": k.unflatten(1, (2, d)), "v": v.unflatten(1, (2, d))}, grads)


def test_tiles_that_are_shared_out_and_tiles_that_are_not(gpu):
    """Sequences of very different lengths: long ones' tiles are split and joined, short ones' are not, forward and backward."""
    for lengths, h, g, d in [([2000, 3, 0, 10, 1500, 1], 2, 1, 64), ([1, 3000], 3, 1, 16), ([5] * 30 + [2500], 1, 1, 128)]:
        x, grad = inputs(sum(lengths), sum(lengths), h, g, d, torch.float16, seed=sum(lengths))
        check(x, grad, packed(lengths), causal=True)
        check(x, grad, packed(lengths))
    of_q, of_k = [1, 3, 0, 2], [4000, 5, 60, 900]
    x, grad = inputs(sum(of_q), sum(of_k), 8, 2, 64, torch.bfloat16, seed=1)
    check(x, grad, packed(of_q), packed(of_k), causal=True)
    of_q, of_k = [4000, 5, 60, 900], [1, 3, 0, 2]
    x, grad = inputs(sum(of_q), sum(of_k), 2, 2, 64, torch.bfloat16, seed=1)
    check(x, grad, packed(of_q), packed(of_k))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,t,n", [(128, 1100, 1200), (113, 1100, 1200), (60, 2900, 2910), (128, 400, 400)])
def test_rows_between_few_and_many(gpu, d, t, n, causal, dtype):
    """Too few tiles for the GPU, but keys enough for tiles of 128 rows, or not."""
    x, grad = inputs(t, n, 8, 1 if d > 64 else 2, d, dtype, seed=13)
    check(x, grad, packed([t - 300, 0, 300]), packed([n - 350, 50, 300]), causal=causal)
