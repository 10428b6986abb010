"""More sequences than half of what 32 bits count, found among one another by several kinds of search."""
import pytest
import torch

import svox_amd as svox
from test_gpu_attention import inputs, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
def test_more_than_2_to_30_sequences(gpu, causal):
    """Bit for bit what the last ones give by themselves: nearly all others are empty."""
    lengths = torch.tensor([1, 0, 0, 2, 0, 0, 0, 3, 0, 1] * 60, dtype=torch.int32)          # (some hundred places to a tile of rows)
    lengths[250], lengths[300] = 40, 150
    rows = int(lengths.sum())
    few = torch.cat([torch.zeros(1, dtype=torch.int32), lengths.cumsum(0).int()]).to(gpu)
    x, grad = inputs(rows, rows, 2, 1, 16, torch.bfloat16, seed=1)
    want_y, want = step(x, grad, few, causal=causal)
    many = torch.zeros((1 << 30) + 12345 + len(few), dtype=torch.int32, device=gpu)
    many[-len(few):] = few
    y, grads = step(x, grad, many, causal=causal)
    torch.cuda.synchronize()
    assert torch.equal(y, want_y) and all(torch.equal(grads[n], want[n]) for n in want)
