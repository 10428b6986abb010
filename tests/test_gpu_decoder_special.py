"""The leaf decoder's operators on infinite numbers, at sizes that leave a part of a tile without numbers of the matrices."""
import pytest
import torch

from test_gpu_decoder import ffn_step

pytestmark = pytest.mark.gpu


# Few rows, narrow layers, whole matrices on each size of tiles; hidden units that end inside of 4, 8 and 32.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["float16", "bfloat16"])
@pytest.mark.parametrize("rows,d,h,o", [(5, 20, 13, 9), (70, 300, 13, 200), (3000, 20, 13, 9), (3000, 128, 40, 128), (98400, 33, 250, 7), (3000, 136, 43, 20),
                                        (9000, 136, 300, 200), (40000, 264, 203, 264), (40000, 264, 504, 264)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_an_infinite_number_makes_infinite_sums_and_no_nan(gpu, rows, d, h, o, act, dtype):
    """With positive numbers throughout, the result's and the gradient's row of an infinite one is infinite; the others stay as they are."""
    g = torch.Generator().manual_seed(1)
    positive = lambda *shape: (torch.rand(*shape, generator=g) * 0.1 + 0.05).to(dtype).to(gpu)  # noqa: E731
    t = {"x": positive(rows, d), "w_gate": positive(h, d), "w_up": positive(h, d), "w_down": positive(o, h)}
    grad, row = positive(rows, o), rows // 2
    clean_y, clean = ffn_step(t, act, grad)
    others = torch.arange(rows, device=gpu) != row
    x, dy = t["x"].clone(), grad.clone()
    x[row, d // 2], dy[row, o // 2] = float("inf"), float("inf")
    y, _ = ffn_step({**t, "x": x}, act, grad)
    assert bool((y[row] == float("inf")).all()) and torch.equal(y[others], clean_y[others])
    _, grads = ffn_step(t, act, dy)
    assert bool((grads["x"][row] == float("inf")).all()) and torch.equal(grads["x"][others], clean["x"][others])
