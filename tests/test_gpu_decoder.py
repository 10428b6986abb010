"""Layer norm and the gated feed-forward block against their definitions in 64 bits (decoder_reference.py, whose bounds are derived
from where the operators round), at the sizes, layouts and numbers where kernels like these go wrong."""
import numpy as np
import pytest
import torch

import svox_amd as svox
from decoder_reference import gated_ffn, layer_norm, slope_by_differences

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
name_of = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def normal(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32, device="cuda:0"):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(device)


def ffn_inputs(rows, d, h, o, dtype, seed=0, bias=True, residual=True, device="cuda:0"):
    g = torch.Generator().manual_seed(seed)
    t = {"x": normal(g, rows, d, dtype=dtype, device=device), "w_gate": normal(g, h, d, scale=d ** -0.5, dtype=dtype, device=device),
         "w_up": normal(g, h, d, scale=d ** -0.5, dtype=dtype, device=device),
         "w_down": normal(g, o, h, scale=h ** -0.5, dtype=dtype, device=device)}
    if bias:
        t.update(b_gate=normal(g, h, scale=0.3, dtype=dtype, device=device), b_up=normal(g, h, scale=0.3, dtype=dtype, device=device),
                 b_down=normal(g, o, scale=0.3, dtype=dtype, device=device))
    if residual:
        t["residual"] = normal(g, rows, o, dtype=dtype, device=device)
    return t, normal(g, rows, o, dtype=dtype, device=device)


def ffn(t, act):
    return svox.gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], t.get("b_gate"), t.get("b_up"), t.get("b_down"),
                          residual=t.get("residual"), activation=act)


def ffn_step(t, act, grad):
    t = {n: v.detach().requires_grad_() for n, v in t.items()}
    y = ffn(t, act)
    return y, dict(zip(t, torch.autograd.grad(y, list(t.values()), grad)))


def check_ffn(t, act, grad):
    want, wanted = gated_ffn(t, act, grad)
    with torch.no_grad():
        want.holds(ffn(t, act).reshape(want.v.shape), "y without gradients")
    y, grads = ffn_step(t, act, grad)
    want.holds(y.reshape(want.v.shape), "y")
    for n, g in grads.items():
        assert g.shape == t[n].shape and g.dtype == t[n].dtype
        wanted[n].holds(g.reshape(wanted[n].v.shape), f"gradient of {n}")


# rows from one to more than a tile, sizes on both sides of 8, 16, 32, 64 and 128
SIZES = [(1, 1, 1, 1), (2, 3, 5, 7), (1, 64, 128, 64), (5, 8, 16, 8), (16, 24, 40, 12), (17, 33, 31, 9), (63, 49, 97, 28), (64, 64, 64, 64),
         (65, 65, 65, 65), (128, 128, 256, 128), (130, 76, 203, 49), (257, 130, 120, 200), (300, 256, 512, 256), (1000, 32, 128, 28),
         (1025, 16, 40, 4), (2050, 64, 264, 49), (33, 520, 300, 136), (700, 200, 72, 520)]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", SIZES)
def test_ffn_sizes(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows + d)
    check_ffn(t, "silu", grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 48, 63, 64])
@pytest.mark.parametrize("d,h,o", [(31, 33, 17), (32, 32, 16), (100, 257, 3), (256, 1024, 256), (1000, 515, 130)])
def test_ffn_few_rows(gpu, rows, d, h, o, dtype):
    t, _ = ffn_inputs(rows, d, h, o, dtype, seed=rows * d)
    wide = normal(torch.Generator().manual_seed(1), rows, d + 3, dtype=dtype)
    for x in (t["x"], wide[:, 1:d + 1]):
        want, _ = gated_ffn({**t, "x": x}, "silu")
        want.holds(ffn({**t, "x": x}, "silu"))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(1, 33, 31, 17), (7, 100, 257, 3), (16, 32, 32, 32), (33, 31, 130, 65), (64, 256, 96, 40), (65, 64, 72, 24),
                                        (200, 50, 60, 70), (500, 128, 40, 16)])
def test_ffn_few_rows_gradients(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows * d)
    g = torch.Generator().manual_seed(1)
    check_ffn({**t, "x": normal(g, rows, d + 3, dtype=dtype)[:, 1:d + 1]}, "gelu", normal(g, rows, o + 5, dtype=dtype)[:, 3:o + 3])


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(2049, 130, 140, 150), (3000, 264, 72, 40), (2100, 24, 40, 200), (2500, 150, 33, 129), (2060, 512, 136, 512)])
def test_ffn_products_of_whole_matrices(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=h)
    check_ffn(t, "silu", grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows", [65, 127, 128, 300, 1111, 2049])
@pytest.mark.parametrize("d,h,o", [(1, 1, 1), (31, 33, 28), (32, 32, 32), (33, 64, 49), (64, 100, 64), (65, 31, 76), (128, 300, 128), (127, 96, 4),
                                   (28, 160, 120)])
def test_ffn_narrow_layers(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows + h)
    wide = normal(torch.Generator().manual_seed(1), rows, d + 5, dtype=dtype)
    check_ffn({**t, "x": wide[:, 2:d + 2]}, "silu", grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("rows,d,h,o", [(9, 40, 72, 24), (300, 48, 96, 49), (520, 264, 160, 264)])
def test_ffn_activations(gpu, rows, d, h, o, act, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=3, bias=act in ("silu", "relu"), residual=act in ("gelu", "relu"))
    check_ffn(t, act, grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,dim", [(3, 8), (200, 64), (200, 300)])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_ffn_gradients_against_differences(gpu, rows, dim, act, dtype):
    """The kernels' gradients along one direction for every tensor, against differences of the definition in 64 bits."""
    t, grad = ffn_inputs(rows, dim, 2 * dim, dim, dtype, seed=5)
    _, grads = ffn_step(t, act, grad)
    _, wanted = gated_ffn(t, act, grad)
    f64 = {n: v.double().cpu() for n, v in t.items()}
    c = grad.double().cpu()
    fn = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[act]

    def loss(t):
        h = fn(t["x"] @ t["w_gate"].t() + t["b_gate"]) * (t["x"] @ t["w_up"].t() + t["b_up"])
        return float(((h @ t["w_down"].t() + t["b_down"] + t["residual"]) * c).sum())

    check_slopes(loss, f64, grads, wanted)


def check_slopes(loss, f64, grads, wanted):
    g = torch.Generator().manual_seed(6)
    for n in grads:
        v = torch.randn(f64[n].shape, generator=g).sign().double()
        slope = slope_by_differences(loss, f64, n, v)
        along = float((grads[n].double().cpu() * v).sum())
        # every number of the gradient is off by its bound at most; the differences are good to 2^-20 of what they are made of
        bound = float(wanted[n].e.sum()) + 2.0 ** -20 * float(np.abs(wanted[n].v).sum())
        assert abs(slope - along) <= bound, (n, slope, along, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_ffn_layouts(gpu, dtype):
    """Rows of records, rows an odd stride apart, broadcast and turned inputs, three dimensions, a gradient that is one number."""
    g = torch.Generator().manual_seed(1)
    t, grad = ffn_inputs(70, 24, 40, 24, dtype, seed=2)
    wide = normal(g, 70, 37, dtype=dtype)
    check_ffn({**t, "x": wide[:, :24]}, "silu", grad)
    check_ffn({**t, "x": wide[:, 5:29], "residual": wide[:, 13:37]}, "silu", grad)
    check_ffn({**t, "x": wide[::2, 1:25], "residual": t["residual"][::2]}, "silu", grad[:35])
    check_ffn({**t, "x": normal(g, 24, 70, dtype=dtype).t()}, "silu", grad)
    check_ffn({**t, "x": wide[:1, :24].expand(70, 24)}, "silu", grad)
    check_ffn({**t, "w_gate": t["w_gate"].t().contiguous().t(), "b_up": wide[0, ::2][:1].expand(40)}, "silu", grad)
    check_ffn(t, "silu", grad.new_ones(1, 1).expand(70, 24))
    cube = {**t, "x": normal(g, 5, 7, 2, 24, dtype=dtype), "residual": normal(g, 5, 7, 2, 24, dtype=dtype)}
    check_ffn(cube, "silu", normal(g, 5, 7, 2, 24, dtype=dtype))
    check_ffn({**cube, "x": normal(g, 7, 5, 2, 24, dtype=dtype).transpose(0, 1)}, "silu", normal(g, 5, 7, 2, 24, dtype=dtype))
    one = {**t, "x": t["x"][0], "residual": t["residual"][0]}
    check_ffn(one, "silu", grad[0])
    padded = torch.zeros(40 * 24 + 3, dtype=dtype, device="cuda:0")     # a weight that does not begin at 16 bytes
    padded[3:] = t["w_up"].reshape(-1)
    check_ffn({**t, "w_up": padded[3:].view(40, 24)}, "silu", grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(3, 16, 24, 8), (200, 40, 64, 24), (200, 300, 136, 264)])
def test_ffn_infinities_and_nan_stay_in_their_rows(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=4)
    clean_y, clean = ffn_step(t, "silu", grad)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x, dy = t["x"].clone(), grad.clone()
        x[1, 0] = bad
        y, grads = ffn_step({**t, "x": x}, "silu", grad)
        keep = torch.arange(rows, device="cuda:0") != 1
        assert torch.equal(y[keep], clean_y[keep]) and torch.equal(grads["x"][keep], clean["x"][keep])
        assert not torch.isfinite(y[1]).any()
        assert torch.equal(grads["w_down"].isfinite().all(), torch.tensor(False, device="cuda:0"))
        dy[1, 0] = bad
        y, grads = ffn_step(t, "silu", dy)
        assert torch.equal(y, clean_y) and torch.equal(grads["x"][keep], clean["x"][keep]) and not torch.isfinite(grads["x"][1]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_ffn_large_arguments_of_the_activation(gpu, act, dtype):
    """Gates up to hundreds in size, both signs, where exp overflows."""
    t, grad = ffn_inputs(66, 32, 48, 16, dtype, seed=8)
    t["x"] = t["x"] * 100
    t["w_up"] = t["w_up"] * 0.01
    check_ffn(t, act, grad)


def test_ffn_only_what_is_asked_for(gpu):
    t, grad = ffn_inputs(150, 40, 72, 24, torch.bfloat16, seed=9)
    _, all_grads = ffn_step(t, "silu", grad)
    for names in (["x"], ["w_gate"], ["w_up", "b_up"], ["w_down"], ["b_gate"], ["b_down"], ["b_up", "x"], ["residual"]):
        leaves = {n: v.detach().requires_grad_(n in names) for n, v in t.items()}
        got = torch.autograd.grad(ffn(leaves, "silu"), [leaves[n] for n in names], grad)
        for n, g in zip(names, got):
            assert torch.equal(g, all_grads[n]), n


def test_no_rows(gpu):
    for dtype in DTYPES:
        t, grad = ffn_inputs(0, 24, 40, 24, dtype)
        y, grads = ffn_step(t, "silu", grad)
        assert y.shape == (0, 24) and grads["x"].shape == (0, 24)
        assert all(float(grads[n].abs().sum()) == 0 for n in ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"))
        x = torch.empty(2, 0, 24, dtype=dtype, device="cuda:0", requires_grad=True)
        w = torch.ones(24, dtype=dtype, device="cuda:0", requires_grad=True)
        y = svox.layer_norm(x, w)
        gx, gw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
        assert y.shape == gx.shape == (2, 0, 24) and float(gw.abs().sum()) == 0


# ---- layer norm
# enough of tiles of 256 x 256 and 256 x 128 for every product and every gradient, whole numbers of nothing; laid out and in place
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(32700, 266, 500, 510), (32600, 520, 504, 264)])
def test_ffn_on_large_tiles(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows)
    check_ffn(t, "silu", grad)


# float32 tiles that fill the card once, 64 of the reduction at a time
@pytest.mark.parametrize("rows,d,h,o", [(5000, 250, 130, 250), (2300, 200, 440, 520), (2570, 65, 500, 400)])
def test_ffn_on_deep_tiles(gpu, rows, d, h, o):
    t, grad = ffn_inputs(rows, d, h, o, torch.float32, seed=rows)
    check_ffn(t, "gelu", grad)


# Narrow layers of many rows, whose hidden numbers stay in registers.
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,act", [(12290, "silu"), (16385, "gelu"), (12289, "relu"), (12303, "sigmoid")])
@pytest.mark.parametrize("d,h,o", [(1, 1, 1), (31, 33, 28), (32, 32, 32), (33, 64, 49), (64, 100, 64), (65, 31, 76), (128, 300, 128), (127, 96, 4),
                                   (28, 160, 120)])
def test_ffn_narrow_layers_of_many_rows(gpu, rows, act, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows + h, bias=act != "gelu", residual=act != "relu")
    wide = normal(torch.Generator().manual_seed(1), rows, d + 5, dtype=dtype)
    check_ffn({**t, "x": wide[:, 2:d + 2]}, act, grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_ffn_layouts_of_many_rows(gpu, dtype):
    g = torch.Generator().manual_seed(1)
    rows = 8200
    t, grad = ffn_inputs(rows, 24, 40, 24, dtype, seed=2)
    wide = normal(g, 2 * rows, 37, dtype=dtype)
    check_ffn({**t, "x": wide[::2, 1:25], "residual": wide[1::2, 13:37]}, "silu", wide[1::2, 2:26])
    check_ffn({**t, "x": normal(g, 24, rows, dtype=dtype).t()}, "silu", grad)
    check_ffn({**t, "x": wide[:1, :24].expand(rows, 24)}, "silu", grad.new_ones(1, 1).expand(rows, 24))
    check_ffn({**t, "w_gate": t["w_gate"].t().contiguous().t(), "b_up": wide[0, ::2][:1].expand(40)}, "silu", grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(8300, 40, 72, 24), (12300, 128, 40, 128), (32700, 264, 260, 264)])
def test_ffn_infinities_and_nan_among_many_rows(gpu, rows, d, h, o, dtype):
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=4)
    clean_y, clean = ffn_step(t, "silu", grad)
    keep = torch.arange(rows, device="cuda:0") != 5001
    for bad in (float("nan"), float("inf"), -float("inf")):
        x, dy = t["x"].clone(), grad.clone()
        x[5001, 0] = bad
        y, grads = ffn_step({**t, "x": x}, "silu", grad)
        assert torch.equal(y[keep], clean_y[keep]) and torch.equal(grads["x"][keep], clean["x"][keep])
        assert not torch.isfinite(y[5001]).any()
        dy[5001, 0] = bad
        y, grads = ffn_step(t, "silu", dy)
        assert torch.equal(y, clean_y) and torch.equal(grads["x"][keep], clean["x"][keep]) and not torch.isfinite(grads["x"][5001]).any()


@pytest.mark.parametrize("rows,d,h,o", [(8300, 40, 72, 24), (32700, 264, 260, 264)])
def test_ffn_only_what_is_asked_for_of_many_rows(gpu, rows, d, h, o):
    t, grad = ffn_inputs(rows, d, h, o, torch.bfloat16, seed=9)
    _, all_grads = ffn_step(t, "silu", grad)
    for names in (["x"], ["w_gate"], ["w_up", "b_up"], ["w_down"], ["b_gate"], ["b_down"], ["b_up", "x"], ["residual"]):
        leaves = {n: v.detach().requires_grad_(n in names) for n, v in t.items()}
        got = torch.autograd.grad(ffn(leaves, "silu"), [leaves[n] for n in names], grad)
        for n, g in zip(names, got):
            assert torch.equal(g, all_grads[n]), n


# Sums over many rows of what the matrix cores computed: a gradient of the hidden numbers is off by some 2^-24 of itself, up or down, and
# so is a sum of them that mostly cancel (their signs are as random); 2^-21 holds it apart from numbers that are all rounded one way,
# whose errors add up while the numbers cancel (rows^0.5 times 2^-24 at worst).
@pytest.mark.parametrize("rows,d,h,o", [(65536, 32, 64, 32), (65536, 64, 130, 64), (40000, 239, 127, 239), (20000, 130, 300, 500)])
def test_sums_over_many_rows_do_not_drift(gpu, rows, d, h, o):
    t, grad = ffn_inputs(rows, d, h, o, torch.float32, seed=h, residual=False)
    _, grads = ffn_step(t, "relu", grad)
    x, wg, wu, wd = (t[n].double() for n in ("x", "w_gate", "w_up", "w_down"))
    dh = grad.double() @ wd
    gate, up = x @ wg.t() + t["b_gate"].double(), x @ wu.t() + t["b_up"].double()
    for n, want in (("b_gate", (dh * up * (gate > 0)).sum(dim=0)), ("b_up", (dh * gate.clamp(min=0)).sum(dim=0))):
        off = (grads[n].double() - want).norm() / want.norm()
        assert off < 2.0 ** -21, (n, float(off))


def norm_step(x, weight, bias, grad, eps=1e-5):
    leaves = {n: v.detach().requires_grad_() for n, v in (("x", x), ("weight", weight), ("bias", bias)) if v is not None}
    y = svox.layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), grad)))


def check_norm(x, weight, bias, grad, eps=1e-5):
    want, wanted = layer_norm(x, weight, bias, eps, grad)
    with torch.no_grad():
        want.holds(svox.layer_norm(x, weight, bias, eps).reshape(want.v.shape), "y without gradients")
    y, grads = norm_step(x, weight, bias, grad, eps)
    want.holds(y.reshape(want.v.shape), "y")
    for n, g in grads.items():
        wanted[n].holds(g.reshape(wanted[n].v.shape), f"gradient of {n}")


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 7), (3, 8), (5, 16), (70, 17), (1000, 31), (129, 33), (64, 64), (77, 100), (33, 128), (40, 200),
                                      (21, 256), (9, 257), (300, 511), (10, 512), (6, 1000), (4, 1024), (5, 1025), (3, 2048), (7, 3000), (2, 4096),
                                      (3, 5000), (2, 8192), (2, 8200), (3, 20011)])
def test_norm_sizes(gpu, rows, dim, dtype):
    g = torch.Generator().manual_seed(rows + dim)
    x = normal(g, rows, dim, dtype=dtype) * (0.5 + torch.rand(rows, 1, generator=g).to(dtype).cuda())
    w, b, grad = normal(g, dim, shift=1.0, dtype=dtype), normal(g, dim, dtype=dtype), normal(g, rows, dim, dtype=dtype)
    check_norm(x, w, b, grad)
    if dim < 600:
        check_norm(x, None, None, grad)
        check_norm(x, w, None, grad, eps=0.1)
        check_norm(x, None, b, grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_norm_layouts(gpu, dtype):
    g = torch.Generator().manual_seed(1)
    w, b, grad = normal(g, 48, shift=1.0, dtype=dtype), normal(g, 48, dtype=dtype), normal(g, 90, 48, dtype=dtype)
    wide = normal(g, 90, 61, dtype=dtype)
    check_norm(wide[:, :48], w, b, grad)
    check_norm(wide[:, 13:], w, b, normal(g, 90, 61, dtype=dtype)[:, 3:51])
    check_norm(wide[::3, 1:49], w, b, grad[:30])
    check_norm(normal(g, 48, 90, dtype=dtype).t(), w, b, grad)
    check_norm(wide[:1, :48].expand(90, 48), w[:1].expand(48), b, grad[:1].expand(90, 48))
    check_norm(normal(g, 3, 30, 48, dtype=dtype).transpose(0, 1), w, b, normal(g, 30, 3, 48, dtype=dtype))
    check_norm(normal(g, 48, dtype=dtype), w, b, grad[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("dim", [24, 700, 9000])
def test_norm_of_special_rows(gpu, dim, dtype):
    """Rows of one value (variance 0), far from 0, with infinities and NaN; every row by itself."""
    g = torch.Generator().manual_seed(2)
    x = normal(g, 9, dim, dtype=dtype)
    x[1] = 3.0
    x[2] = 0.0
    x[3] += 1000.0
    grad, w, b = normal(g, 9, dim, dtype=dtype), normal(g, dim, shift=1.0, dtype=dtype), normal(g, dim, dtype=dtype)
    check_norm(x, w, b, grad)
    y, grads = norm_step(x, w, b, grad)
    assert torch.equal(y[1], b) and torch.equal(y[2], b)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[4, dim // 2] = bad
        y2, grads2 = norm_step(z, w, b, grad)
        keep = torch.arange(9, device="cuda:0") != 4
        assert torch.equal(y[keep], y2[keep]) and torch.equal(grads["x"][keep], grads2["x"][keep])
        assert y2[4].isnan().all() and grads2["weight"].isnan().all() and torch.equal(grads["bias"], grads2["bias"])


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_norm_gradients_against_differences(gpu, dtype):
    g = torch.Generator().manual_seed(3)
    x, w, b, c = normal(g, 40, 52, dtype=dtype), normal(g, 52, shift=1.0, dtype=dtype), normal(g, 52, dtype=dtype), normal(g, 40, 52, dtype=dtype)
    _, grads = norm_step(x, w, b, c)
    _, wanted = layer_norm(x, w, b, grad=c)
    f64 = {n: v.double().cpu() for n, v in (("x", x), ("weight", w), ("bias", b))}
    check_slopes(lambda t: float((torch.nn.functional.layer_norm(t["x"], (52,), t["weight"], t["bias"]) * c.double().cpu()).sum()), f64, grads, wanted)


# ---- both
def both(t, grad, w, b):
    y, grads = ffn_step(t, "gelu", grad)
    z, more = norm_step(t["x"], w, b, t["x"])
    return [y, z, *grads.values(), *more.values()]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_the_same_call_gives_the_same_bits(gpu, dtype):
    for rows, d, h, o in [(5000, 48, 96, 28), (3000, 264, 300, 136), (20, 64, 512, 64)]:
        t, grad = ffn_inputs(rows, d, h, o, dtype, seed=11)
        w, b = t["w_gate"][0], t["w_up"][0]
        first = both(t, grad, w, b)
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(first, both(t, grad, w, b)))


def test_on_another_stream_and_from_a_graph(gpu):
    t, grad = ffn_inputs(500, 72, 200, 40, torch.float32, seed=12)
    w, b = torch.ones(72, device="cuda:0"), torch.zeros(72, device="cuda:0")
    first = both(t, grad, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both(t, grad, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    leaves = {n: v.detach().clone().requires_grad_() for n, v in t.items()}
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ffn(leaves, "gelu"), list(leaves.values()), grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ffn(leaves, "gelu")
        grads = torch.autograd.grad(y, list(leaves.values()), grad)
    for seed in (12, 13, 14):
        t2, _ = ffn_inputs(500, 72, 200, 40, torch.float32, seed=seed)
        with torch.no_grad():
            for n in leaves:
                leaves[n].copy_(t2[n])
        graph.replay()
        want_y, want = ffn_step(t2, "gelu", grad)
        torch.cuda.synchronize()
        assert torch.equal(y, want_y) and all(torch.equal(x, want[n]) for n, x in zip(leaves, grads))


def test_matrices_of_more_than_2_31_numbers(gpu):
    rows, d = (1 << 31) // 1024 + 37, 1024
    x = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda:0").normal_(generator=torch.Generator("cuda:0").manual_seed(1))
    w, b = torch.ones(d, dtype=torch.bfloat16, device="cuda:0"), torch.zeros(d, dtype=torch.bfloat16, device="cuda:0")
    pick = torch.tensor([0, 1, rows // 2, rows - 38, rows - 2, rows - 1], device="cuda:0")
    x.requires_grad_()
    y = svox.layer_norm(x, w, b)
    (gx,) = torch.autograd.grad(y, [x], x.detach())
    want, wanted = layer_norm(x.detach()[pick], w, b, grad=x.detach()[pick])
    want.holds(y[pick])
    wanted["x"].holds(gx[pick])
    del y, gx
    g = torch.Generator().manual_seed(2)
    t = {"w_gate": normal(g, 16, d, scale=d ** -0.5, dtype=torch.bfloat16), "w_up": normal(g, 16, d, scale=d ** -0.5, dtype=torch.bfloat16),
         "w_down": normal(g, d, 16, scale=0.25, dtype=torch.bfloat16)}
    y = svox.gated_ffn(x, **t)
    (gx,) = torch.autograd.grad(y, [x], x.detach())
    want, wanted = gated_ffn({"x": x.detach()[pick], **t}, "silu", x.detach()[pick])
    want.holds(y[pick])
    wanted["x"].holds(gx[pick])


def test_gradients_cannot_be_differentiated_again(gpu):
    t, grad = ffn_inputs(4, 8, 16, 8, torch.float32)
    x = t["x"].requires_grad_()
    for y in (ffn(t, "silu"), svox.layer_norm(x)):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(y, [x], grad, create_graph=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_refusals_on_the_gpu(gpu, dtype):
    t, _ = ffn_inputs(4, 8, 16, 8, dtype)
    other = torch.float16 if dtype != torch.float16 else torch.float32
    bad = [("w_gate", t["w_gate"].to(other), "expected scalar type"), ("w_up", t["w_up"][:, :7], "must have shape"),
           ("w_down", t["w_down"].t(), "must have shape"), ("b_gate", t["b_gate"][:15], "must have shape"), ("b_up", t["b_up"].cpu(), "CUDA tensor"),
           ("b_down", t["b_down"][None], "must have shape"), ("residual", t["residual"][:3], "must have shape"),
           ("residual", t["residual"].to(other), "expected scalar type"), ("x", t["x"].double(), "float32, float16 or bfloat16"),
           ("w_gate", t["w_gate"][0], "2-D")]
    for n, v, message in bad:
        with pytest.raises(RuntimeError, match=message):
            ffn({**t, n: v}, "silu")
    with pytest.raises(ValueError, match="unknown activation"):
        ffn(t, "tanh")
    for args, message in [((t["x"], t["b_gate"]), "must have shape"), ((t["x"], t["b_down"].to(other)), "expected scalar type"),
                          ((t["x"].cpu(),), "CUDA tensor"), ((t["x"].double(),), "float32, float16 or bfloat16"),
                          ((t["x"][:, :0],), "between 1 and"), ((torch.tensor(1.0, device="cuda:0"),), "at least one dimension")]:
        with pytest.raises(RuntimeError, match=message):
            svox.layer_norm(*args)
