"""Every row counts: gradients that are sums over rows, where a row that is left out, or taken twice, shows.

A bound for a sum of a hundred thousand terms is wider than one of them.  So either all of the result's gradient but some rows is zero, and
the bound that of those rows; or the rows are alike but for their sign, and their sum is zero.
"""
import numpy as np
import pytest
import torch

import decoder_rules
import svox_amd as svox
from decoder_reference import gated_ffn, layer_norm
from test_gpu_decoder import DTYPES, ffn, ffn_inputs, ffn_step, name_of, norm_step, normal

ACTIVATIONS = ["silu", "gelu", "relu", "sigmoid"]


def some_rows(rows, seed=0):
    """The first and last rows, both sides of multiples of 16 to 256, and some anywhere: 40 at most."""
    g = torch.Generator().manual_seed(seed)
    edges = [e + s for e in (16, 32, 64, 128, 256, 4096) for s in (-1, 0)]
    ends = [rows - 1, rows - 2, rows - rows % 32, rows - rows % 32 - 1, rows - rows % 64 - 1, rows - rows % 128 - 1]
    anywhere = torch.randint(rows, (20,), generator=g).tolist()
    return sorted({r for r in [0, 1] + edges + ends + anywhere if 0 <= r < rows})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", decoder_rules.SIZES)
def test_gradients_of_some_rows_among_many(gpu, rows, d, h, o, dtype):
    act = ACTIVATIONS[(rows + d + h + o) % 4]
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows + h, residual=False)
    g = torch.Generator().manual_seed(1)
    wide, beside = normal(g, rows, d + 3, dtype=dtype), normal(g, rows, o + 5, dtype=dtype)
    t["x"], t["residual"] = wide[:, 1:d + 1], beside[:, 2:o + 2]
    pick = torch.tensor(some_rows(rows, seed=h), device=gpu)
    others = torch.ones(rows, dtype=torch.bool, device=gpu)
    others[pick] = False
    grad[others] = 0
    y, grads = ffn_step(t, act, grad)
    want, wanted = gated_ffn({**t, "x": t["x"][pick], "residual": t["residual"][pick]}, act, grad[pick])
    want.holds(y[pick], "y")
    with torch.no_grad():
        assert torch.equal(ffn(t, act), y)
    for n, found in grads.items():
        if n in ("x", "residual"):
            assert not bool(found[others].any()), n
            found = found[pick]
        wanted[n].holds(found, f"gradient of {n}")


def balanced(rows, g):
    """As many 1 as -1 in any order, and a 0 where the rows are odd."""
    signs = torch.zeros(rows)
    signs[:rows // 2], signs[rows // 2:rows // 2 * 2] = 1, -1
    return signs[torch.randperm(rows, generator=g)]


def alike(rows, d, h, o, dtype, device="cuda:0"):
    """Rows that are all the same, and weights of which dh comes out exactly, whatever the order of its terms: sums of -1, -1/2, 1/2 and 1."""
    g = torch.Generator().manual_seed(rows + h)
    few_bits = lambda *shape: torch.tensor([-1.0, -0.5, 0.5, 1.0])[torch.randint(4, shape, generator=g)].to(dtype)  # noqa: E731
    t = {"x": few_bits(1, d), "w_gate": normal(g, h, d, scale=d ** -0.5, dtype=dtype, device="cpu"),
         "w_up": normal(g, h, d, scale=d ** -0.5, dtype=dtype, device="cpu"), "w_down": few_bits(o, h), "b_gate": normal(g, h, dtype=dtype, device="cpu"),
         "b_up": normal(g, h, dtype=dtype, device="cpu"), "b_down": normal(g, o, dtype=dtype, device="cpu")}
    t = {n: v.to(device) for n, v in t.items()}
    return t, torch.sign(torch.randn(1, o, generator=g)).to(dtype).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [s for s in decoder_rules.SIZES if s[0] > 1])
def test_rows_alike_but_for_their_sign_add_up_to_nothing(gpu, rows, d, h, o, dtype):
    t, u = alike(rows, d, h, o, dtype)
    _, one = gated_ffn(t, "silu", u)
    x = t["x"].repeat(rows, 1)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        signs = balanced(rows, g)
        y, grads = ffn_step({**t, "x": x}, "silu", signs.to(gpu).to(dtype)[:, None] * u)
        assert bool((y == y[:1]).all())
        for sign in (-1, 0, 1):
            rows_of = grads["x"][(signs == sign).to(gpu)]
            assert bool((rows_of == rows_of[:1]).all()), sign
        for n in ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
            # A quarter of what one row adds.  Products and partial sums of few bits are exact in 16 bits; the sums of 24-bit numbers are off by
            # some rows / 32 roundings of a running sum of rows^0.5 terms: 2^-6 of a term for 10^5 rows.
            share = np.abs(grads[n].double().cpu().numpy()) - 0.25 * np.abs(one[n].v.reshape(grads[n].shape))
            assert (share <= 2.0 ** -20).all(), (n, float(share.max()))


# Rows on every number of lanes, and more of them than the blocks go through at once.
NORMS = [(140003, 3), (70001, 30), (40003, 60), (40003, 100), (20011, 250), (9001, 500), (9001, 1000), (9001, 2000), (2500, 4000), (2500, 8000), (2500, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,dim", NORMS)
def test_norm_gradients_of_some_rows_among_many(gpu, rows, dim, dtype):
    g = torch.Generator("cuda:0").manual_seed(dim)
    x, grad = (torch.randn(rows, dim + 1, generator=g, device=gpu).to(dtype)[:, 1:] for _ in range(2))
    w, b = (torch.randn(dim, generator=g, device=gpu).to(dtype) for _ in range(2))
    pick = torch.tensor(some_rows(rows, seed=dim), device=gpu)
    others = torch.ones(rows, dtype=torch.bool, device=gpu)
    others[pick] = False
    grad[others] = 0
    y, grads = norm_step(x, w, b, grad)
    want, wanted = layer_norm(x[pick], w, b, grad=grad[pick])
    want.holds(y[pick], "y")
    assert not bool(grads["x"][others].any())
    wanted["x"].holds(grads["x"][pick], "gradient of x")
    for n in ("weight", "bias"):
        wanted[n].holds(grads[n], f"gradient of {n}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,dim", NORMS)
def test_norm_rows_alike_but_for_their_sign_add_up_to_nothing(gpu, rows, dim, dtype):
    g = torch.Generator().manual_seed(dim)
    x, w, b, u = (normal(g, *shape, dtype=dtype) for shape in ((1, dim), (dim,), (dim,), (1, dim)))
    _, one = layer_norm(x, w, b, grad=u)
    for seed in range(3):
        signs = balanced(rows, g).to(gpu).to(dtype)
        y, grads = norm_step(x.repeat(rows, 1), w, b, signs[:, None] * u)
        assert bool((y == y[:1]).all())
        for sign in (-1, 0, 1):
            rows_of = grads["x"][signs == sign]
            assert bool((rows_of == rows_of[:1]).all()), sign
        for n in ("weight", "bias"):
            # (as above: sums in 32 bits of rows / 256 terms and more to a lane)
            assert (np.abs(grads[n].double().cpu().numpy()) <= 0.25 * np.abs(one[n].v) + 2.0 ** -20).all(), n


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("rows,d,h,o", [(98351, 17, 33, 9), (9001, 130, 300, 200)])
def test_a_row_that_is_left_out_shows(rows, d, h, o, dtype):
    """On the CPU: gradients without one of the picked rows, rounded once, lie outside the bounds of every weight and bias."""
    t, grad = ffn_inputs(rows, d, h, o, dtype, seed=rows + h, residual=False, device="cpu")
    pick = some_rows(rows, seed=h)
    t["x"], grad = t["x"][pick], grad[pick]
    _, wanted = gated_ffn(t, "silu", grad)
    for left_out in (0, len(pick) // 2, len(pick) - 1):
        some = [i for i in range(len(pick)) if i != left_out]
        _, without = gated_ffn({**t, "x": t["x"][some]}, "silu", grad[some])
        for n in ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
            with pytest.raises(AssertionError, match="outside their bound"):
                wanted[n].holds(torch.from_numpy(without[n].v).to(dtype))

