"""The C ABI of the leaf decoder's operators, their refusals that need no GPU, and the bounds its GPU tests compare with."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import svox_amd as svox
from decoder_reference import gated_ffn, layer_norm
from svox_amd.csrc import decoder as D

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "svox_decoder.h")


def test_header_library_and_mirror_agree():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(svox_[a-z_]+)\s*\(", text)))
    assert sorted(D.SIGNATURES) == declared
    out = subprocess.run(["nm", "-D", "--defined-only", D.LIB_PATH], stdout=subprocess.PIPE, text=True, check=True).stdout
    assert sorted(line.split()[-1] for line in out.splitlines() if " T " in line) == declared


def test_struct_layouts_match_the_c_compiler(tmp_path):
    structs = {"SvoxLayerNorm": D.LayerNormC, "SvoxGatedFfn": D.GatedFfnC, "SvoxGatedFfnGrads": D.GatedFfnGradsC}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, mirror in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines())
    for name, mirror in structs.items():
        assert int(got[name]) == ctypes.sizeof(mirror), name
        for f, _ in mirror._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(mirror, f).offset, f"{name}.{f}"


def test_argument_errors_come_before_anything_touches_a_device():
    lib = D.load_library()

    def norm(**kw):
        s = D.LayerNormC(x=16, weight=16, bias=16, rows=4, x_stride=8, dim=8, dtype=0, eps=1e-5)
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    def ffn(**kw):
        s = D.GatedFfnC(x=16, w_gate=16, w_up=16, w_down=16, rows=4, x_stride=8, dim=8, hidden=16, out=8)
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    ref = ctypes.byref
    assert lib.svox_layer_norm(None, None, None, None) == -1
    for kw, rc in [({"dtype": 3}, -3), ({"dtype": -1}, -3), ({"rows": -1}, -2), ({"dim": 0}, -2), ({"x_stride": 7}, -2), ({"x": None}, -1),
                   ({"rows": 1 << 60, "x_stride": 1 << 20}, -2), ({}, -1)]:
        assert lib.svox_layer_norm(ref(norm(**kw)), None, None, None) == rc, kw
        assert lib.svox_decoder_last_error()
    assert lib.svox_layer_norm(ref(norm(rows=0)), None, None, None) == 0
    assert lib.svox_layer_norm_backward(ref(norm()), None, 16, 8, 16, None, None, None, 0, None) == -1
    assert lib.svox_layer_norm_backward(ref(norm()), 16, 16, 7, 16, None, None, None, 0, None) == -2
    least = lib.svox_layer_norm_workspace_bytes(ref(norm()), 1)
    assert least > 0 and lib.svox_layer_norm_workspace_bytes(ref(norm()), 0) == 0
    assert lib.svox_layer_norm_backward(ref(norm()), 16, 16, 8, 16, 16, 16, 16, least - 1, None) == -2
    assert lib.svox_layer_norm_backward(ref(norm()), 16, 16, 8, 16, 16, 16, 8, least, None) == -2
    assert lib.svox_layer_norm_backward(ref(norm()), 16, 16, 8, 16, 16, 16, None, least, None) == -1
    for kw, rc in [({"dtype": 3}, -3), ({"rows": -1}, -2), ({"hidden": 0}, -2), ({"out": 0}, -2), ({"dim": 0}, -2), ({"activation": 4}, -4),
                   ({"w_up": None}, -1), ({"residual": 16, "residual_stride": 7}, -2), ({"x_stride": 3}, -2), ({"rows": 1 << 45}, -2), ({}, -1)]:
        assert lib.svox_gated_ffn(ref(ffn(**kw)), None, None, 0, None) == rc, kw
    assert lib.svox_gated_ffn(ref(ffn(rows=0)), None, None, 0, None) == 0
    least = lib.svox_gated_ffn_workspace_bytes(ref(ffn()), 1)
    assert least > 0 and lib.svox_gated_ffn_workspace_bytes(ref(ffn(rows=0)), 1) == 0
    grads = D.GatedFfnGradsC(x=16)
    assert lib.svox_gated_ffn_backward(ref(ffn()), 16, 8, None, 16, least, None) == -1
    assert lib.svox_gated_ffn_backward(ref(ffn()), 16, 7, ref(grads), 16, least, None) == -2
    assert lib.svox_gated_ffn_backward(ref(ffn()), 16, 8, ref(grads), 16, least - 1, None) == -2


def test_there_is_no_cpu_path():
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        svox.layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        svox.gated_ffn(x, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))
    with pytest.raises(TypeError):
        svox.layer_norm(None)


def test_leaf_decoder_is_a_module_like_others(tmp_path):
    decoder = svox.LeafDecoder(12, 28, hidden=40, depth=2, activation="gelu")
    assert [tuple(p.shape) for p in decoder.ffns[2].parameters()] == [(40, 12), (40, 12), (28, 40), (40,), (40,), (28,)]
    assert len(decoder.norms) == len(decoder.ffns) == 3 and all(p.requires_grad for p in decoder.parameters())
    torch.save(decoder.state_dict(), tmp_path / "decoder.pt")
    other = svox.LeafDecoder(12, 28, hidden=40, depth=2)
    other.load_state_dict(torch.load(tmp_path / "decoder.pt", weights_only=True))
    assert all(torch.equal(a, b) for a, b in zip(decoder.parameters(), other.parameters()))
    assert svox.LeafDecoder(16, 4).ffns[0].w_gate.shape == (64, 16)
    with pytest.raises(ValueError, match="unknown activation"):
        svox.LeafDecoder(12, 4, activation="tanh")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        decoder(torch.zeros(5, 12))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_bounds_hold_for_torch_and_see_a_mistake(dtype):
    """torch's own float32 result, rounded once, lies within the reference's bounds; one with numbers of a column out of place does not."""
    g = torch.Generator().manual_seed(0)
    of = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).to(dtype)  # noqa: E731
    t = {"x": of(40, 24), "w_gate": of(40, 24, scale=0.2), "w_up": of(40, 24, scale=0.2), "w_down": of(24, 40, scale=0.16), "b_gate": of(40),
         "b_up": of(40), "b_down": of(24), "residual": of(40, 24)}
    grad = of(40, 24)
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}
    for name, fn in act.items():
        f = {n: v.float().requires_grad_() for n, v in t.items()}
        y = (fn(f["x"] @ f["w_gate"].t() + f["b_gate"]) * (f["x"] @ f["w_up"].t() + f["b_up"])) @ f["w_down"].t() + f["b_down"] + f["residual"]
        grads = dict(zip(f, torch.autograd.grad(y, list(f.values()), grad.float())))
        want, wanted = gated_ffn(t, name, grad)
        wrong(want, y.to(dtype))
        for n in grads:
            wrong(wanted[n], grads[n].to(dtype))
    w, b = of(24), of(24)
    f = [v.float().requires_grad_() for v in (t["x"], w, b)]
    y = torch.nn.functional.layer_norm(f[0], (24,), f[1], f[2])
    want, wanted = layer_norm(t["x"], w, b, grad=grad)
    wrong(want, y.to(dtype))
    for n, v in zip(("x", "weight", "bias"), torch.autograd.grad(y, f, grad.float())):
        wrong(wanted[n], v.to(dtype))


def wrong(near, got):
    near.holds(got)
    off = got.detach().clone()
    off[..., 0] = torch.roll(off[..., 0], 1) if off.dim() > 1 else off[..., 0] + 4.0
    with pytest.raises(AssertionError):
        near.holds(off)
