"""The C ABI of the operators of networks over cells, their refusals that need no GPU, and the bounds their GPU tests compare with."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import svox_amd as svox
from network_reference import attention, clip_norm, rotate_heads
from svox_amd.csrc import network as N

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "svox_network.h")
STRUCTS = {"SvoxClipTensor": N.ClipTensorC, "SvoxRotateHeads": N.RotateHeadsC, "SvoxAttention": N.AttentionC,
           "SvoxAttentionGrads": N.AttentionGradsC}


def test_header_library_and_mirror_agree():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(svox_[a-z_]+)\s*\(", text)))
    assert sorted(N.SIGNATURES) == declared
    out = subprocess.run(["nm", "-D", "--defined-only", N.LIB_PATH], stdout=subprocess.PIPE, text=True, check=True).stdout
    assert sorted(line.split()[-1] for line in out.splitlines() if " T " in line) == declared


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f.rstrip("_")}));' for f, _ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines())
    for name, mirror in STRUCTS.items():
        assert int(got[name]) == ctypes.sizeof(mirror), name
        for f, _ in mirror._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(mirror, f).offset, f"{name}.{f}"


def with_fields(spec, kw):
    for k, v in kw.items():
        setattr(spec, k, v)
    return ctypes.byref(spec)


def test_argument_errors_of_clip_norm_come_before_anything_touches_a_device():
    lib = N.load_library()

    def table(**kw):
        t = N.ClipTensorC(from_=16, to=16, count=5, dtype=0)
        return with_fields(t, kw)

    assert lib.svox_clip_norm(table(), 1, 1.0, None, 16, 64, None) == -1
    assert lib.svox_clip_norm(None, 1, 1.0, 16, 16, 64, None) == -1
    for kw, rc in [({"count": -1}, -2), ({"dtype": 3}, -3), ({"dtype": -1}, -3), ({"from_": None}, -1), ({"to": None}, -1), ({"count": 1 << 60}, -2)]:
        assert lib.svox_clip_norm(table(**kw), 1, 1.0, 16, 16, 64, None) == rc, kw
        assert lib.svox_network_last_error()
    for most in (-1.0, math.nan):
        assert lib.svox_clip_norm(table(), 1, most, 16, 16, 64, None) == -2
    assert lib.svox_clip_norm(table(), -1, 1.0, 16, 16, 64, None) == -2
    least = lib.svox_clip_norm_workspace_bytes(table(), 1)
    assert least == 8 and lib.svox_clip_norm_workspace_bytes(table(count=0, from_=None), 1) == 0 and lib.svox_clip_norm_workspace_bytes(None, 0) == 0
    assert lib.svox_clip_norm(table(), 1, 1.0, 16, 16, least - 1, None) == -2
    assert lib.svox_clip_norm(table(), 1, 1.0, 16, 8, least, None) == -2
    assert lib.svox_clip_norm(table(), 1, 1.0, 16, None, least, None) == -1


def test_argument_errors_of_rotate_heads_come_before_anything_touches_a_device():
    lib = N.load_library()

    def spec(**kw):
        return with_fields(N.RotateHeadsC(q=16, k=16, positions=16, frequencies=16, rows=4, q_stride=32, q_head=8, k_stride=16, k_head=8, heads=4, kv_heads=2,
                                          dim=8, rotated=6, axes=3, eps=1e-6), kw)

    grad = (ctypes.c_int64 * 4)(32, 8, 16, 8)
    assert lib.svox_rotate_heads(None, 16, 16, None) == -1
    for kw, rc in [({"dtype": 3}, -3), ({"rows": -1}, -2), ({"heads": 0}, -2), ({"kv_heads": 0}, -2), ({"heads": 1 << 21}, -2), ({"dim": 0}, -2),
                   ({"dim": 257}, -4), ({"rotated": 5}, -2), ({"rotated": 10}, -2), ({"rotated": -2}, -2), ({"axes": 0}, -2), ({"axes": 5}, -2),
                   ({"position_type": 4}, -3), ({"q": None}, -1), ({"k": None}, -1), ({"positions": None}, -1), ({"frequencies": None}, -1),
                   ({"q_stride": -1}, -2), ({"k_head": -8}, -2), ({"rows": 1 << 45}, -2), ({"q_stride": 1 << 45}, -2)]:
        assert lib.svox_rotate_heads(spec(**kw), 16, 16, None) == rc, kw
        assert lib.svox_rotate_heads_backward(spec(**kw), 16, 16, grad, 16, 16, 16, 16, 16, 1 << 20, None) == rc, kw
    assert lib.svox_rotate_heads(spec(), None, 16, None) == -1
    assert lib.svox_rotate_heads(spec(rows=0, q=None, k=None, positions=None), None, None, None) == 0
    least = lib.svox_rotate_heads_workspace_bytes(spec(), 1)
    assert least > 0 and lib.svox_rotate_heads_workspace_bytes(spec(), 0) == 0
    assert lib.svox_rotate_heads_backward(spec(), 16, 16, None, 16, 16, 16, 16, 16, least, None) == -1
    assert lib.svox_rotate_heads_backward(spec(), None, 16, grad, 16, 16, 16, 16, 16, least, None) == -1
    assert lib.svox_rotate_heads_backward(spec(), 16, 16, grad, 16, 16, 16, 16, 16, least - 1, None) == -2
    assert lib.svox_rotate_heads_backward(spec(), 16, 16, grad, None, None, None, None, None, 0, None) == 0


def test_argument_errors_of_attention_come_before_anything_touches_a_device():
    lib = N.load_library()

    def spec(**kw):
        return with_fields(N.AttentionC(q=16, k=16, v=16, queries=5, keys=7, sequences=1, q_stride=32, q_head=8, k_stride=16, k_head=8, v_stride=16, v_head=8,
                                        heads=4, kv_heads=2, dim=8, scale=0.5), kw)

    def grads(**kw):
        return with_fields(N.AttentionGradsC(out=16, lse=16, grad=16, grad_stride=32, grad_head=8, q=16, k=16, v=16), kw)

    assert lib.svox_attention(None, 16, None, None, 16, 1 << 20, None) == -1
    for kw, rc in [({"dtype": 3}, -3), ({"queries": -1}, -2), ({"keys": -1}, -2), ({"heads": 0}, -2), ({"kv_heads": 0}, -2), ({"heads": 5}, -2), ({"dim": 0}, -2),
                   ({"dim": 129}, -4), ({"scale": 0.0}, -2), ({"scale": -1.0}, -2), ({"scale": math.nan}, -2), ({"scale": math.inf}, -2), ({"sequences": 0}, -2),
                   ({"sequences": 2}, -1), ({"key_offsets": 16}, -1), ({"offsets": 16}, -2), ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1),
                   ({"queries": 1 << 30, "offsets": 16, "key_offsets": 16}, -4), ({"keys": 1 << 31}, -4), ({"heads": 1 << 20, "queries": 1 << 11}, -4),
                   ({"q_stride": -1}, -2), ({"v_head": -8}, -2), ({"k_stride": 1 << 45}, -2)]:
        assert lib.svox_attention(spec(**kw), 16, None, None, 16, 1 << 40, None) == rc, kw
        assert lib.svox_attention_backward(spec(**kw), grads(), 16, 1 << 40, None) == rc, kw
        assert lib.svox_network_last_error()
    assert lib.svox_attention(spec(), None, None, None, 16, 1 << 20, None) == -1
    assert lib.svox_attention(spec(queries=0, q=None), None, None, None, None, 0, None) == 0
    long = spec(keys=100000)
    least = lib.svox_attention_workspace_bytes(long, 0)
    assert least > 0 and lib.svox_attention_workspace_bytes(spec(), 0) == 0
    assert lib.svox_attention(long, 16, None, None, None, least, None) == -1
    assert lib.svox_attention(long, 16, None, None, 16, least - 1, None) == -2
    assert lib.svox_attention(long, 16, None, None, 8, least, None) == -2
    least = lib.svox_attention_workspace_bytes(spec(), 1)
    assert least > 0
    assert lib.svox_attention_backward(spec(), None, 16, least, None) == -1
    for kw, rc in [({"grad": None}, -1), ({"out": None}, -1), ({"lse": None}, -1), ({"grad_stride": -1}, -2)]:
        assert lib.svox_attention_backward(spec(), grads(**kw), 16, least, None) == rc, kw
    assert lib.svox_attention_backward(spec(), grads(), 16, least - 1, None) == -2
    assert lib.svox_attention_backward(spec(), grads(q=None, k=None, v=None), None, 0, None) == 0


CALLS = {"rotate_heads": lambda x: svox.rotate_heads(x, x, torch.zeros(3), torch.zeros(4))[0], "clip_norm": lambda x: svox.clip_norm([x], 1.0)[0],
         "attention": lambda x: svox.attention(x, x, x)}


@pytest.mark.parametrize("name", list(CALLS))
def test_there_is_no_cpu_path_and_no_tracing(name):
    call, x = CALLS[name], torch.ones(3, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        call(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(x)


def test_what_is_no_tensor():
    x = torch.zeros(3, 2, 8)
    for call in (lambda: svox.attention(None, x, x), lambda: svox.attention(x, x, x, [0, 3]), lambda: svox.rotate_heads(x, x, [0, 1, 2], x), lambda: svox.clip_norm([1.0], 1.0),
                 lambda: svox.attention(x, x, x, scale="1")):
        with pytest.raises(TypeError):
            call()


def test_gradients_that_are_not_there():
    p = torch.zeros(3, requires_grad=True)
    assert svox.clip_grad_norm([p], 1.0) == 0 and svox.clip_grad_norm(p, 1.0) == 0 and svox.clip_grad_norm([], 1.0) == 0
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        svox.clip_grad_norm(p, 1.0)


def sees_a_mistake(near, got):
    """The bound holds for `got`, and not where its numbers are out of place."""
    near.holds(got)
    off = got.detach().clone().reshape(-1)
    off[0] += max(1.0, float(off.abs().max()))
    with pytest.raises(AssertionError):
        near.holds(off.reshape(got.shape))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_bounds_hold_for_torch_and_see_a_mistake(dtype, interleaved):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(30, 3, 24, generator=g).to(dtype), (1 + 0.2 * torch.randn(24, generator=g)).to(dtype)
    grad, p, f = torch.randn(30, 3, 24, generator=g).to(dtype), torch.rand(30, 2, generator=g) * 9, torch.rand(2, 10, generator=g)
    xx, ww = x.float().requires_grad_(), w.float().requires_grad_()
    n = xx * torch.rsqrt((xx * xx).mean(-1, keepdim=True) + 1e-6) * ww
    angle = (p.double() @ f.double())[:, None]
    c, s = angle.cos().float(), angle.sin().float()
    a, b = (n[..., :20:2], n[..., 1:20:2]) if interleaved else (n[..., :10], n[..., 10:20])
    turned = [a * c - b * s, b * c + a * s]
    y = torch.cat([torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1), n[..., 20:]], -1)
    dx, dw = torch.autograd.grad(y, (xx, ww), grad.float())
    want, wanted = rotate_heads(x, p, f, w, interleaved=interleaved, grad=grad)
    sees_a_mistake(want, y.to(dtype))
    sees_a_mistake(wanted["x"], dx.to(dtype))
    sees_a_mistake(wanted["weight"], dw.to(dtype))
    norm = torch.linalg.vector_norm(x.double()).float()
    near, (scaled,) = clip_norm([x], 2.0)
    sees_a_mistake(near, norm)
    sees_a_mistake(scaled, (x.float() * (2.0 / norm)).to(dtype))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_bounds_of_attention_hold_for_torch_and_see_a_mistake(dtype, causal):
    g = torch.Generator().manual_seed(1)
    q, k, v, grad = (torch.randn(*s, generator=g).to(dtype) for s in ((20, 4, 24), (30, 2, 24), (30, 2, 24), (20, 4, 24)))
    want, wanted = attention(q, k, v, [0, 12, 20], [0, 9, 30], causal=causal, grad=grad)
    f = [x.float().requires_grad_() for x in (q, k, v)]
    parts = []
    for q0, q1, k0, k1 in ((0, 12, 0, 9), (12, 20, 9, 30)):
        qq, kk, vv = (x.transpose(0, 1) for x in (f[0][q0:q1], f[1][k0:k1].repeat_interleave(2, 1), f[2][k0:k1].repeat_interleave(2, 1)))
        s = qq @ kk.transpose(1, 2) * 24 ** -0.5
        hidden = (torch.arange(k1 - k0) - torch.arange(q1 - q0)[:, None] > (k1 - k0) - (q1 - q0)) & causal
        empty = hidden.all(1, keepdim=True)
        p = torch.softmax(s.masked_fill(hidden & ~empty, float("-inf")), -1).masked_fill(empty, 0.0)
        parts.append((p @ vv).transpose(0, 1))
    y = torch.cat(parts)
    sees_a_mistake(want, y.to(dtype))
    for name, got in zip("qkv", torch.autograd.grad(y, f, grad.float())):
        sees_a_mistake(wanted[name], got.to(dtype))


def test_a_decoder_with_heads_is_a_module_like_others(tmp_path):
    plain = svox.LeafDecoder(24, 4)
    assert not any("attend" in n or "frequencies" in n for n in plain.state_dict())
    decoder = svox.LeafDecoder(24, 4, depth=2, heads=4, kv_heads=2)
    assert [tuple(p.shape) for p in decoder.attends[1].parameters()] == [(48, 24), (24, 24), (6,), (6,), (24,), (24,)]
    assert "frequencies" not in decoder.state_dict() and set(plain.state_dict()) < set(decoder.state_dict())
    torch.save(decoder.state_dict(), tmp_path / "decoder.pt")
    other = svox.LeafDecoder(24, 4, depth=2, heads=4, kv_heads=2)
    other.load_state_dict(torch.load(tmp_path / "decoder.pt", weights_only=True))
    frequencies = decoder.frequencies.view(torch.float32)
    assert frequencies.shape == (3, 3) and torch.equal(frequencies, torch.eye(3) * 2 * math.pi)
    assert torch.equal(decoder.half().frequencies.view(torch.float32), frequencies) and decoder.attends[0].w_qkv.dtype == torch.float16
    wide = svox.LeafDecoder(64, 4, heads=1).frequencies.view(torch.float32)
    assert wide.shape == (3, 32) and wide.max() == wide[1, 31] == torch.tensor(2 * math.pi * 256) and (wide != 0).sum() == 32
    for kw in ({"heads": 5}, {"heads": 4, "kv_heads": 3}, {"heads": -1}, {"heads": 4, "kv_heads": 0}, {"heads": 4, "window": 0}):
        with pytest.raises(ValueError):
            svox.LeafDecoder(24, 4, **kw)
    with pytest.raises(ValueError, match="positions"):
        decoder(torch.zeros(5, 24))
