"""float32's kernels of long axes, and float16's scales of rows and keys, where masks, odd numbers and heads of many rows meet them."""
import pytest
import torch

from test_gpu_attention import check, inputs, packed, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 64, 128, 30, 50, 99])
@pytest.mark.parametrize("causal", [False, True])
def test_long_sequences_of_float32(gpu, d, causal):
    """Two sequences, rows and keys before, behind and between them, by direct loads and others."""
    x, grad = inputs(5000, 5200, 2, 1, d, torch.float32, seed=d)
    check(x, grad, torch.tensor([10, 2400, 4990], device=gpu), torch.tensor([0, 2600, 5150], device=gpu), causal=causal)


@pytest.mark.parametrize("d", [32, 64, 128, 50])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_masked_rows_hold_has_no_influence_on_long_sequences(gpu, d, bad):
    x, grad = inputs(4400, 4400, 2, 2, d, torch.float32, seed=d)
    offsets = packed([2100, 2300])
    clean_y, clean = step(x, grad, offsets, causal=True)
    for name in ("q", "k", "v", "grad"):
        broken, dy = {n: v.clone() for n, v in x.items()}, grad.clone()
        (dy if name == "grad" else broken[name])[300, :, 3] = bad
        y, grads = step(broken, dy, offsets, causal=True)
        assert torch.equal(y[2100:], clean_y[2100:]) and torch.equal(y[:300], clean_y[:300]), name
        assert all(torch.equal(grads[n][2100:], clean[n][2100:]) for n in grads), name
        assert not torch.isfinite(grads[{"grad": "v", "v": "q"}.get(name, name)][:2100]).all(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("t,h,kv_heads,d", [(3, 300, 1, 24), (5, 130, 2, 64), (70, 24, 8, 128), (190, 7, 1, 32)])
def test_heads_of_more_rows_than_a_tile_or_odd_ones(gpu, t, h, kv_heads, d, dtype):
    x, grad = inputs(t, t + 40, h, kv_heads, d, dtype, seed=h)
    check(x, grad, causal=True)
    check(x, grad, packed([t - 2, 0, 2]), packed([10, 20, t + 10]), causal=True)


@pytest.mark.parametrize("d", [32, 64, 128, 33])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 60000.0])
def test_scales_of_rows_are_their_own(gpu, d, bad):
    """A row whose gradient is huge or none, among others of the same tile: theirs keep every bit."""
    x, grad = inputs(300, 300, 2, 1, d, torch.float16, seed=d, spread=0.5)
    _, clean = step(x, grad)
    other = grad.clone()
    other[17, :, 2] = bad
    _, grads = step(x, other)
    keep = torch.arange(300) != 17
    assert torch.equal(grads["q"][keep], clean["q"][keep])
    assert not torch.equal(grads["q"][17], clean["q"][17])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_gradients_of_nothing(gpu, dtype):
    x, grad = inputs(100, 100, 2, 1, 64, dtype, seed=5)
    _, grads = step(x, torch.zeros_like(grad))
    assert not any(v.any() for v in grads.values())
    x["v"].zero_()
    y, grads = step(x, grad)
    assert not y.any() and not grads["q"].any() and not grads["k"].any()
    x["k"].zero_()
    check(x, grad, causal=True)
