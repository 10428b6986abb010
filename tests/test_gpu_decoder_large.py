"""The leaf decoder's operators at the largest sizes they take: beyond what a launch counts in 32 bits."""
import ctypes

import pytest
import torch

import svox_amd as svox
from decoder_reference import gated_ffn
from svox_amd.csrc import decoder as D

pytestmark = pytest.mark.gpu


# Four lanes to a row in float32: 2^30 rows are as many threads as a launch cannot have.
@pytest.mark.parametrize("dtype,rows", [(torch.float32, (1 << 30) + 77), (torch.bfloat16, (1 << 31) + 77)], ids=["float32", "bfloat16"])
def test_narrow_layers_of_more_rows_than_a_launch_has_lanes_for(gpu, dtype, rows):
    g = torch.Generator("cuda:0").manual_seed(1)
    x = torch.empty(rows, 1, dtype=dtype, device=gpu).normal_(generator=g)
    residual = torch.empty(rows, 1, dtype=dtype, device=gpu).normal_(generator=g)
    t = {n: torch.full((1, 1), v, dtype=dtype, device=gpu) for n, v in (("w_gate", 0.5), ("w_up", -1.5), ("w_down", 0.75))}
    pick = torch.cat([torch.arange(at, at + 300, device=gpu) for at in (0, 64, (1 << 28) - 150, rows // 2, (1 << 30) - 300, rows - 300)])
    x.requires_grad_()
    y = svox.gated_ffn(x, **t, residual=residual)
    (gx,) = torch.autograd.grad(y, [x], residual)
    want, wanted = gated_ffn({"x": x.detach()[pick], "residual": residual[pick], **t}, "silu", residual[pick])
    want.holds(y[pick], "y")
    wanted["x"].holds(gx[pick], "gradient of x")
    # every number: the result is that of the same rows in a call of their own
    for part in range(0, rows - 77, 1 << 27):
        rows_of = slice(part, part + (1 << 27) if part + (1 << 27) < rows - 77 else rows)
        again = x.detach()[rows_of].requires_grad_()
        z = svox.gated_ffn(again, **t, residual=residual[rows_of])
        assert torch.equal(z, y[rows_of]), part
        assert torch.equal(torch.autograd.grad(z, [again], residual[rows_of])[0], gx[rows_of]), part


# Sixteen columns of the parameters' gradients to a block of 1024 lanes: 2^25 columns of both are as many as a launch cannot have.
def test_norm_gradients_of_more_columns_than_a_launch_has_lanes_for(gpu):
    dim = (1 << 25) + 9
    g = torch.Generator("cuda:0").manual_seed(2)
    x, grad = (torch.empty(2, dim, dtype=torch.bfloat16, device=gpu).normal_(generator=g) for _ in range(2))
    x.requires_grad_()
    w, b = torch.ones(dim, dtype=torch.bfloat16, device=gpu).requires_grad_(), torch.zeros(dim, dtype=torch.bfloat16, device=gpu).requires_grad_()
    dw, db = torch.autograd.grad(svox.layer_norm(x, w, b), [w, b], grad)
    assert torch.equal(db, (grad[0].float() + grad[1].float()).bfloat16())     # (two numbers have one sum)
    n = torch.nn.functional.layer_norm(x.detach().double(), (dim,))
    off = (dw.double() - (grad.double() * n).sum(dim=0)).abs()
    # a rounding to 8 bits of the sum, and n's own error: the mean and the deviation are sums of 2^17 numbers a lane
    assert bool((off <= 2.0 ** -8 * dw.double().abs() + 2.0 ** -7 * (grad.double() * n).abs().sum(dim=0) + 2.0 ** -7 * grad.double().abs().sum(dim=0)).all())


# The longest row there is, whose last step goes beyond what 32 bits count.  Numbers here and there in a row of zeros, whose sums are exact.
def test_norm_of_the_longest_row(gpu):
    dim = (1 << 31) - 1
    at = torch.tensor([0, 9, 1 << 30, dim - 2050, dim - 8, dim - 7, dim - 2, dim - 1])
    values, slopes = torch.tensor([512.0, -1024, 256, 768, -512, 1024, 640, -384]), torch.tensor([1.0, -2, 0.5, 3, 1, -1, 2, 4])
    weights, shifts = torch.tensor([1.0, 2, 3, 0.5, 1, 2, 1, 3]), torch.tensor([0.0, 1, -1, 2, 0.5, 0, -2, 1])

    def row(numbers, others=0.0):
        v = torch.full((dim,), others, dtype=torch.bfloat16, device=gpu)
        v[at.to(gpu)] = numbers.bfloat16().to(gpu)
        return v

    x, w, b, grad = row(values).requires_grad_(), row(weights, 1.0).requires_grad_(), row(shifts, 0.25).requires_grad_(), row(slopes)
    y = svox.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], grad)
    values, slopes, weights, shifts = (v.double() for v in (values, slopes, weights, shifts))
    mean = values.sum() / dim
    rstd = 1 / ((((values - mean) ** 2).sum() + (dim - len(at)) * mean ** 2) / dim + 1e-5).sqrt()
    n, dn = (values - mean) * rstd, slopes * weights
    others = -mean * rstd    # n where x is zero
    m1, m2 = dn.sum() / dim, (dn * n).sum() / dim
    want = {"y": (y, n * weights + shifts, others + 0.25), "x": (dx, rstd * (dn - m1 - n * m2), rstd * (-m1 - others * m2)),
            "weight": (dw, slopes * n, 0.0), "bias": (db, slopes, 0.0)}
    for name, (got, there, elsewhere) in want.items():
        got = got.detach()
        near = got[at.to(gpu)].double().cpu()
        # (8 bits, and sums of some ten numbers in 32)
        assert bool(((near - there).abs() <= 2.0 ** -8 * there.abs() + 1e-5).all()), (name, near, there)
        got[at.to(gpu)] = 0
        rest = torch.tensor(float(elsewhere)).bfloat16().to(gpu)
        for part in range(0, dim, 1 << 28):
            some = got[part:part + (1 << 28)]
            off = some != rest
            off[at[(at >= part) & (at < part + (1 << 28))].to(gpu) - part] = False
            # (the last of a number's 8 bits may differ)
            assert not bool(off.any()) or bool(((some[off].double() - float(elsewhere)).abs() <= 2.0 ** -8 * abs(float(elsewhere)) + 1e-12).all()), (name, part)


# The gradient of a weight of more than 2^32 numbers over no rows: zeros, and nothing beyond them.
def test_no_rows_and_a_weight_of_more_numbers_than_a_launch_has_lanes(gpu):
    hidden, dim, margin = 1 << 22, 1025, 1000
    w = torch.ones(hidden * dim + margin, dtype=torch.bfloat16, device=gpu)
    spec = D.GatedFfnC(x=16, w_gate=16, w_up=16, w_down=16, rows=0, x_stride=dim, dim=dim, hidden=hidden, out=1, dtype=D.BF16)
    grads = D.GatedFfnGradsC(w_gate=w.data_ptr())
    lib = D.load_library()
    assert lib.svox_gated_ffn_backward(ctypes.byref(spec), None, 1, ctypes.byref(grads), None, 0, None) == 0, lib.svox_decoder_last_error()
    torch.cuda.synchronize()
    assert not bool(w[:-margin].any()) and bool((w[-margin:] == 1).all())
