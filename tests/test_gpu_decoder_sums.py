"""Gradients that are sums over many rows."""
import pytest
import torch

from test_gpu_decoder import ffn_inputs, ffn_step

pytestmark = pytest.mark.gpu


# What the matrix cores round one way must not add up: 2^-21 as for the other sizes (tests/test_gpu_decoder.py).  Results of one step of
# the reduction and of several; gradients of either sign, and of one, whose running sums are as large as the sums themselves.
@pytest.mark.parametrize("rows,d,h,o", [(65536, 96, 127, 28), (131072, 80, 33, 20), (65536, 200, 64, 300), (30000, 130, 300, 500), (65536, 48, 96, 60)])
@pytest.mark.parametrize("signs", ["either", "one"])
def test_sums_of_float32_gradients_do_not_drift(gpu, rows, d, h, o, signs):
    t, grad = ffn_inputs(rows, d, h, o, torch.float32, seed=h, residual=False)
    if signs == "one":
        grad = grad.abs()
    _, grads = ffn_step(t, "relu", grad)
    x, wg, wu, wd = (t[n].double() for n in ("x", "w_gate", "w_up", "w_down"))
    dh = grad.double() @ wd
    gate, up = x @ wg.t() + t["b_gate"].double(), x @ wu.t() + t["b_up"].double()
    wanted = {"b_gate": (dh * up * (gate > 0)).sum(dim=0), "b_up": (dh * gate.clamp(min=0)).sum(dim=0), "b_down": grad.double().sum(dim=0)}
    off = {n: float((grads[n].double() - want).norm() / want.norm()) * 2.0 ** 21 for n, want in wanted.items()}
    print(off)
    assert all(v < 1 for v in off.values()), off
