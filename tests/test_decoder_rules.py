"""The sizes the leaf decoder's kernels are tested on reach every one of them, by the rules as they are now."""
import pytest

import decoder_rules

WIDTHS = {1: (1, 2, 4), 3: (1, 2)}
TILES = {1: ("small", "medium", "large"), 3: ("small", "deep", "medium")}
WEIGHTS = {1: ("small whole", "small in parts", "medium in parts", "large whole", "large in parts"), 3: ("small in parts", "medium whole", "medium in parts")}


@pytest.mark.parametrize("planes", [1, 3], ids=["16 bits", "float32"])
def test_every_kernel_is_reached(planes, tmp_path):
    program = decoder_rules.compiled(str(tmp_path))
    kernels = decoder_rules.kernels_of(program, planes, decoder_rules.SIZES)
    assert len(kernels) == len(decoder_rules.SIZES)
    wanted = {f"weights {of}" for of in WEIGHTS[planes]}
    for at in ("forward", "gradients"):
        wanted |= {f"{at} few {tiles}" for tiles in (1, 2, 4)} | {f"{at} {of} {size}" for of in ("hidden", "result") for size in TILES[planes]}
        wanted |= {f"{at} narrow {i} {o} by {rows}" for i in WIDTHS[planes] for o in WIDTHS[planes] for rows in ((1, 2) if planes == 1 else (1,))}
    assert wanted == set().union(*kernels)
