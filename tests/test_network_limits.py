"""The largest sizes that the operators of networks over cells take are refused or accepted by the host, before anything is launched."""
import ctypes

import pytest

from svox_amd.csrc import network as N

UNSUPPORTED = -4
LAUNCH = (1 << 24) - 64          # tiles of 128 that a launch has blocks for, in whole runs for all XCDs


def spec(**kw):
    s = N.AttentionC(q=16, k=16, v=16, offsets=16, key_offsets=16, queries=5, keys=7, sequences=16, q_stride=8, q_head=8, k_stride=8, k_head=8, v_stride=8,
                     v_head=8, heads=1, kv_heads=1, dim=8, scale=0.5)
    for name, value in kw.items():
        setattr(s, name, value)
    return ctypes.byref(s)


@pytest.mark.parametrize("sequences", [16, 17, 5000])
@pytest.mark.parametrize("axis", ["queries", "keys"])
@pytest.mark.parametrize("heads", [1, 8, 63])
def test_attention_has_blocks_for_every_size_it_takes(axis, heads, sequences):
    lib = N.load_library()
    kw = dict(heads=heads, kv_heads=heads, sequences=sequences, q_stride=8 * heads, k_stride=8 * heads, v_stride=8 * heads)
    least = LAUNCH // heads * 128 + 1            # one tile more than there are blocks for
    grads = ctypes.byref(N.AttentionGradsC(out=16, lse=16, grad=16, grad_stride=8 * heads, grad_head=8, q=16, k=16, v=16))
    for size in (least, least + 127, (1 << 31) - 1025):
        if size * heads < 1 << 31 or size == least:
            assert lib.svox_attention(spec(**kw, **{axis: size}), 16, None, None, 16, 1 << 60, None) == UNSUPPORTED
            assert lib.svox_attention_backward(spec(**kw, **{axis: size}), grads, 16, 1 << 60, None) == UNSUPPORTED
    assert lib.svox_attention_workspace_bytes(spec(**kw, **{axis: least - 1}), 0) >= 0
    assert lib.svox_attention_workspace_bytes(spec(**kw, **{axis: least - 1}), 1) > 0


@pytest.mark.parametrize("heads", [1, 8])
def test_without_runs_there_are_blocks_for_a_few_more(heads):
    lib = N.load_library()
    size = (LAUNCH // heads + 1) * 128
    for sequences in (2, 15):
        for axis in ("queries", "keys"):
            assert lib.svox_attention_workspace_bytes(spec(heads=heads, kv_heads=heads, sequences=sequences, **{axis: size}), 1) > 0


def test_heads_of_keys_are_at_least_one():
    lib = N.load_library()
    s = N.RotateHeadsC(q=16, k=16, positions=16, frequencies=16, rows=4, q_stride=32, q_head=8, k_stride=16, k_head=8, heads=4, kv_heads=0, dim=8, rotated=6, axes=3, eps=1e-6)
    assert lib.svox_rotate_heads(ctypes.byref(s), 16, 16, None) == -2 and b"kv_heads" in lib.svox_network_last_error()
