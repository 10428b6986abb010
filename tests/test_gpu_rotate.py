"""Norms of queries' and keys' heads with their rotation, and the gradients, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import svox_amd as svox
from decoder_reference import slope_by_differences
from network_reference import rotate_heads

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
name_of = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def normal(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to("cuda:0")


def inputs(rows, h, hk, d, rotated, axes, dtype, seed=0, weights=True):
    g = torch.Generator().manual_seed(seed)
    t = {"q": normal(g, rows, h, d, scale=1.5, dtype=dtype), "k": normal(g, rows, hk, d, scale=0.7, dtype=dtype)}
    if weights:
        t.update(q_weight=normal(g, d, scale=0.2, shift=1.0, dtype=dtype), k_weight=normal(g, d, scale=0.2, shift=1.0, dtype=dtype))
    positions = torch.rand(rows, axes, generator=g).to("cuda:0") * 50 - 10
    frequencies = (torch.rand(axes, rotated // 2, generator=g) * 6).to("cuda:0")
    grads = [normal(g, rows, h, d, dtype=dtype), normal(g, rows, hk, d, dtype=dtype)]
    return t, positions, frequencies, grads


def call(t, positions, frequencies, **kw):
    return svox.rotate_heads(t["q"], t["k"], positions, frequencies, t.get("q_weight"), t.get("k_weight"), **kw)


def step(t, positions, frequencies, grads, **kw):
    t = {n: v.detach().requires_grad_() for n, v in t.items()}
    y = call(t, positions, frequencies, **kw)
    return y, dict(zip(t, torch.autograd.grad(y, list(t.values()), grads)))


def check(t, positions, frequencies, grads, **kw):
    y, got = step(t, positions, frequencies, grads, **kw)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(call(t, positions, frequencies, **kw), y))
    p = positions[:, None] if positions.dim() == 1 else positions
    f = frequencies[None] if frequencies.dim() == 1 else frequencies
    for name, out, grad in zip("qk", y, grads):
        want, wanted = rotate_heads(t[name], p, f, t.get(name + "_weight"), grad=grad, **kw)
        want.holds(out, name)
        wanted["x"].holds(got[name], f"gradient of {name}")
        if name + "_weight" in t:
            wanted["weight"].holds(got[name + "_weight"], f"gradient of {name}_weight")


SIZES = [(1, 1, 1, 1, 0), (1, 1, 1, 2, 2), (3, 2, 1, 7, 4), (5, 4, 4, 8, 8), (17, 8, 2, 16, 16), (65, 3, 3, 31, 30), (33, 6, 3, 44, 30), (70, 4, 1, 32, 32),
         (50, 8, 2, 64, 64), (9, 5, 1, 96, 48), (21, 2, 2, 127, 126), (130, 4, 2, 128, 128), (13, 3, 1, 200, 66), (40, 2, 1, 256, 256), (11, 1, 3, 255, 2),
         (6, 1, 1, 256, 0), (2, 40, 7, 20, 12), (300, 1, 1, 64, 34)]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,h,hk,d,rotated", SIZES)
def test_sizes(gpu, rows, h, hk, d, rotated, interleaved, dtype):
    t, p, f, grads = inputs(rows, h, hk, d, rotated, 1 + rows % 4, dtype, seed=rows + d, weights=rows % 3 != 2)
    check(t, p, f, grads, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_more_rows_than_blocks(gpu, dtype):
    """More rows than the blocks of a launch go through at once, forward and backward."""
    t, p, f, grads = inputs(70003, 1, 1, 16, 16, 2, dtype, seed=1)
    check(t, p, f, grads)
    t, p, f, grads = inputs(20011, 3, 1, 64, 48, 3, dtype, seed=2)
    check(t, p, f, grads, interleaved=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_layouts(gpu, dtype):
    """Slices of a packed row, an odd beginning, broadcast and turned heads, gradients of one number, one weight alone."""
    g = torch.Generator().manual_seed(3)
    t, p, f, grads = inputs(40, 4, 2, 24, 24, 3, dtype, seed=4)
    packed = normal(g, 40, 8 * 24 + 3, dtype=dtype)
    for at in (0, 1):
        sliced = {**t, "q": packed[:, at:at + 96].unflatten(1, (4, 24)), "k": packed[:, at + 96:at + 144].unflatten(1, (2, 24))}
        check(sliced, p, f, grads)
        check(sliced, p, f, grads, interleaved=True)
    check({**t, "q": normal(g, 4, 40, 24, dtype=dtype).transpose(0, 1)}, p, f, grads)
    check({**t, "q": normal(g, 40, 24, 4, dtype=dtype).transpose(1, 2)}, p, f, grads)
    check({**t, "q": t["q"][:1].expand(40, 4, 24), "k": t["k"][:, :1].expand(40, 2, 24)}, p, f, grads)
    check(t, p, f, [grads[0].new_ones(1, 1, 1).expand(40, 4, 24), grads[1].transpose(0, 1).contiguous().transpose(0, 1)])
    check({n: v for n, v in t.items() if n != "k_weight"}, p, f, grads)
    check({**t, "q_weight": normal(g, 48, dtype=dtype)[::2]}, p.t().contiguous().t(), f[:, ::2], grads)
    check({**t, "q": torch._neg_view(t["q"])}, p, f, grads)


@pytest.mark.parametrize("kind", [torch.float32, torch.float64, torch.int32, torch.int64], ids=str)
def test_far_positions(gpu, kind):
    """Places of a long sequence, whose angles float32 would lose: as exact as near ones."""
    t, _, _, grads = inputs(50, 2, 1, 32, 32, 1, torch.float32, seed=5)
    g = torch.Generator().manual_seed(6)
    far = (torch.randint(0, 1 << 24, (50,), generator=g) * 64 + 5).to(kind).to("cuda:0")
    f = 10000.0 ** (-torch.arange(16, device="cuda:0") / 16)
    check(t, far, f, grads)
    check(t, torch.stack([far, -far], dim=1), torch.stack([f, 3 * f]), grads, interleaved=True)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(gpu, interleaved):
    t, p, f, grads = inputs(6, 3, 2, 20, 14, 3, torch.float32, seed=7)
    _, got = step(t, p, f, grads, interleaved=interleaved)
    f64 = {n: v.double().cpu() for n, v in t.items()}

    def loss(t):
        total = 0.0
        for name, grad in zip("qk", grads):
            near, _ = rotate_heads(t[name], p, f, t[name + "_weight"], interleaved=interleaved, dtype=torch.float32)
            total += float((near.v * grad.double().cpu().numpy()).sum())
        return total

    g = torch.Generator().manual_seed(8)
    for i, name in enumerate(("q", "k")):
        _, wanted = rotate_heads(t[name], p, f, t[name + "_weight"], interleaved=interleaved, grad=grads[i])
        for n, near in ((name, wanted["x"]), (name + "_weight", wanted["weight"])):
            v = torch.randn(f64[n].shape, generator=g).sign().double()
            slope = slope_by_differences(loss, f64, n, v)
            along = float((got[n].double().cpu() * v).sum())
            assert abs(slope - along) <= float(near.e.sum()) + 2.0 ** -20 * float(np.abs(near.v).sum()), n


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_infinities_and_nan_stay_in_their_heads(gpu, dtype):
    t, p, f, grads = inputs(20, 3, 2, 40, 20, 2, dtype, seed=9)
    clean_y, clean = step(t, p, f, grads)
    for bad in (float("nan"), float("inf")):
        x = t["q"].clone()
        x[3, 1, 5] = bad
        y, got = step({**t, "q": x}, p, f, grads)
        keep = torch.ones(20, 3, dtype=torch.bool)
        keep[3, 1] = False
        assert torch.equal(y[0][keep], clean_y[0][keep]) and torch.equal(got["q"][keep], clean["q"][keep])
        assert torch.equal(y[1], clean_y[1]) and torch.equal(got["k"], clean["k"]) and not torch.isfinite(got["q"][3, 1]).all()
    p2 = p.clone()
    p2[7] = float("nan")
    y, _ = step(t, p2, f, grads)
    keep = torch.arange(20) != 7
    assert torch.equal(y[0][keep], clean_y[0][keep]) and torch.isnan(y[0][7, :, :20]).all() and torch.equal(y[0][7, :, 20:], clean_y[0][7, :, 20:])
    zero = {**t, "q": torch.zeros_like(t["q"])}
    check(zero, p, f, grads)


def test_only_what_is_asked_for(gpu):
    t, p, f, grads = inputs(90, 4, 2, 32, 32, 3, torch.bfloat16, seed=10)
    _, all_grads = step(t, p, f, grads)
    for names in (["q"], ["k"], ["q_weight"], ["k_weight", "q"], ["k", "q_weight"]):
        leaves = {n: v.detach().requires_grad_(n in names) for n, v in t.items()}
        for n, got in zip(names, torch.autograd.grad(call(leaves, p, f), [leaves[n] for n in names], grads)):
            assert torch.equal(got, all_grads[n]), n
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    got = torch.autograd.grad(call(leaves, p, f)[1], list(leaves.values()), grads[1], allow_unused=True)
    assert torch.equal(got[1], all_grads["k"]) and torch.equal(got[3], all_grads["k_weight"]) and not got[0].any() and not got[2].any()


def test_no_rows(gpu):
    t, p, f, grads = inputs(0, 4, 2, 32, 32, 3, torch.float16)
    y, got = step(t, p, f, grads)
    assert y[0].shape == (0, 4, 32) and got["k"].shape == (0, 2, 32)
    assert torch.equal(got["q_weight"], torch.zeros(32, dtype=torch.float16, device="cuda:0"))


def test_refusals(gpu):
    t, p, f, grads = inputs(5, 4, 2, 32, 32, 3, torch.float32)
    for change, text in [({"q": t["q"][0]}, "3-D"), ({"k": t["k"][:4]}, "same rows"), ({"k": t["k"][..., :31]}, "same rows"), ({"k": t["k"].half()}, "scalar type"),
                         ({"k": t["k"].cpu()}, "CUDA tensor"), ({"q_weight": t["q_weight"][:31]}, "shape"), ({"q": t["q"].double()}, "float32, float16"),
                         ({"q": torch.zeros(5, 1, 257, device=gpu), "k": torch.zeros(5, 1, 257, device=gpu), "q_weight": None, "k_weight": None}, "dim must be <= 256")]:
        with pytest.raises(RuntimeError, match=text):
            call({**t, **change}, p, f)
    for positions, frequencies, text in [(p[:4], f, "positions must have"), (p, f[:2], "frequencies must have"), (p[:, 0], f, "frequencies must have"),
                                         (p.half(), f, "positions must be"), (p, f.double(), "scalar type"), (p.cpu(), f, "positions must be"),
                                         (p, torch.zeros(3, 17, device=gpu), "more than a head"), (torch.zeros(5, 5, device=gpu), torch.zeros(5, 16, device=gpu), "axes"),
                                         (p.clone().requires_grad_(), f, "no gradient of positions")]:
        with pytest.raises(RuntimeError, match=text):
            call(t, positions, frequencies)
    q = t["q"].clone().requires_grad_()
    y = call({**t, "q": q}, p, f)[0]
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(y.sum(), q, create_graph=True)
    with pytest.raises(TypeError):
        svox.rotate_heads(None, t["k"], p, f)


def test_a_captured_step_follows_its_inputs(gpu):
    t, p, f, grads = inputs(500, 4, 2, 32, 32, 3, torch.bfloat16, seed=11)
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}

    def run():
        y = call(leaves, p, f)
        return [*y, *torch.autograd.grad(y, list(leaves.values()), grads)]

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            for v in leaves.values():
                v.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(i)))
            p.add_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))
