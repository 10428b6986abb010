"""What the operators of a leaf decoder are measured on: layer norm and the gated feed-forward block, the two that a
small network is made of which turns the features kept in the leaves of a tree into the records a renderer reads.

A pass is one call of `svox_amd.layer_norm` or `svox_amd.gated_ffn` (forward), or the call and its gradients through
autograd (step).  The sizes are those such networks have: rows from one queried point to the cells of a 64^3 grid,
features and records of the sizes tree records have (28 of SH9, 49 of SH16, 76 of SH25) and of powers of two, widths up to
a thousand features with four hidden units for each.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # the features of one queried point: a call's latency
        {"name": "norm_point", "op": "layer_norm", "pass": "forward", "dtype": "bfloat16", "rows": 1, "dim": 256, "affine": True, "extra": 0},
        # every cell of a 64^3 grid of features, before it is decoded
        {"name": "norm_leaves", "op": "layer_norm", "pass": "forward", "dtype": "bfloat16", "rows": 262144, "dim": 128, "affine": True, "extra": 0},
        # training on the colour features of SH16 records where they lie, the density left out of every row
        {"name": "norm_step_records", "op": "layer_norm", "pass": "step", "dtype": "float32", "rows": 100003, "dim": 48, "affine": True, "extra": 1},
        # training a wide network
        {"name": "norm_step_wide", "op": "layer_norm", "pass": "step", "dtype": "bfloat16", "rows": 65536, "dim": 1024, "affine": True, "extra": 0},
        # one queried point through a block of a wide network, as a viewer's probe asks for it
        {"name": "ffn_point", "op": "gated_ffn", "pass": "forward", "dtype": "bfloat16", "rows": 1, "dim": 512, "hidden": 2048, "out": 512,
         "activation": "silu", "bias": True, "residual": True},
        # a handful of queried points, half precision
        {"name": "ffn_points", "op": "gated_ffn", "pass": "forward", "dtype": "float16", "rows": 37, "dim": 256, "hidden": 1024, "out": 256,
         "activation": "gelu", "bias": True, "residual": True},
        # writing a 64^3 grid of SH16 records from 64 features a leaf
        {"name": "ffn_leaves", "op": "gated_ffn", "pass": "forward", "dtype": "bfloat16", "rows": 262144, "dim": 64, "hidden": 256, "out": 49,
         "activation": "silu", "bias": True, "residual": False},
        # the same in single precision, the type of the trees, for SH9 records from 32 features
        {"name": "ffn_leaves_f32", "op": "gated_ffn", "pass": "forward", "dtype": "float32", "rows": 65537, "dim": 32, "hidden": 128, "out": 28,
         "activation": "silu", "bias": True, "residual": False},
        # a training step of a block of a decoder on a batch of leaves
        {"name": "ffn_step_leaves", "op": "gated_ffn", "pass": "step", "dtype": "bfloat16", "rows": 131072, "dim": 64, "hidden": 256, "out": 64,
         "activation": "silu", "bias": True, "residual": True},
        # a training step with sizes that divide by nothing: SH25 records in, SH16 records out
        {"name": "ffn_step_odd", "op": "gated_ffn", "pass": "step", "dtype": "float16", "rows": 10007, "dim": 76, "hidden": 203, "out": 49,
         "activation": "gelu", "bias": True, "residual": False},
        # a training step in single precision
        {"name": "ffn_step_f32", "op": "gated_ffn", "pass": "step", "dtype": "float32", "rows": 8192, "dim": 256, "hidden": 1024, "out": 256,
         "activation": "silu", "bias": True, "residual": True},
        # the largest training step: a wide block
        {"name": "ffn_step_wide", "op": "gated_ffn", "pass": "step", "dtype": "bfloat16", "rows": 16384, "dim": 1024, "hidden": 4096, "out": 1024,
         "activation": "silu", "bias": True, "residual": True},
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = {"op": rng.choice(["layer_norm", "gated_ffn", "gated_ffn"]), "pass": rng.choice(["forward", "step"]),
            "dtype": rng.choice(["float32", "bfloat16", "float16"]), "rows": _size(rng, 1, 262144)}

    def width(low, high):   # half of them whole multiples of 16, the others as they fall
        n = _size(rng, low, high)
        return max(16, n // 16 * 16) if rng.random() < 0.5 else n

    case["dim"] = width(16, 1024)
    if case["op"] == "layer_norm":
        case["affine"], case["extra"] = rng.random() < 0.8, rng.choice([0, 0, 0, 1])
    else:
        case["hidden"] = width(32, 4096)
        case["residual"] = rng.random() < 0.5
        case["out"] = case["dim"] if case["residual"] else width(4, 1024)
        case["activation"], case["bias"] = rng.choice(["silu", "gelu", "relu", "sigmoid"]), rng.random() < 0.7
    most = {x["name"]: work(x) for x in listed()}["ffn_step_wide" if case["op"] == "gated_ffn" else "norm_step_wide"]
    # (single precision costs some six times the matrix work of half precision here)
    dear = 6.0 if case["op"] == "gated_ffn" and case["dtype"] == "float32" else 1.0
    share = max(work(case)["flops"] * dear / most["flops"], work(case)["bytes"] / most["bytes"])
    if share > 1:
        case["rows"] = max(1, int(case["rows"] / (1.05 * share)))
    return case


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    n, d, step = case["rows"], case["dim"], case["pass"] == "step"
    if case["op"] == "layer_norm":
        affine = 2 * d if case["affine"] else 0
        values = 2 * n * d + affine              # x and the parameters in, y out
        if step:
            values += 2 * n * d + affine         # grad_output in; the gradients of x and of the parameters out
        return {"bytes": size * values, "flops": (8 + (14 if step else 0)) * n * d}
    h, o = case["hidden"], case["out"]
    weights = 2 * h * d + h * o + ((2 * h + o) if case["bias"] else 0)
    values = n * d + weights + n * o + (n * o if case["residual"] else 0)
    if step:
        values += n * o + n * d + weights        # grad_output in; the gradients of x and of the parameters out
    return {"bytes": size * values, "flops": (3 if step else 1) * 2 * n * (2 * h * d + h * o)}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    step = case["pass"] == "step"

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale + shift).to(dtype)

    n, d = case["rows"], case["dim"]
    if case["op"] == "layer_norm":
        # features whose mean and spread differ from row to row, as a network's residual stream has them
        records = torch.randn(n, d + case["extra"], generator=g, device=DEVICE)
        records = records * (0.5 + torch.rand(n, 1, generator=g, device=DEVICE)) + 0.3 * torch.randn(n, 1, generator=g, device=DEVICE)
        inputs = {"x": records.to(dtype)[:, :d]}
        if case["affine"]:
            inputs["weight"], inputs["bias"] = normal(d, scale=0.1, shift=1.0), normal(d, scale=0.1)
        grad = normal(n, d) if step else None
    else:
        h, o = case["hidden"], case["out"]
        inputs = {"x": normal(n, d), "w_gate": normal(h, d, scale=d ** -0.5), "w_up": normal(h, d, scale=d ** -0.5),
                  "w_down": normal(o, h, scale=h ** -0.5)}
        if case["bias"]:
            inputs.update(b_gate=normal(h, scale=0.1), b_up=normal(h, scale=0.1), b_down=normal(o, scale=0.1))
        if case["residual"]:
            inputs["residual"] = normal(n, o)
        grad = normal(n, o) if step else None
    if step:
        inputs = {name: x.detach().requires_grad_() for name, x in inputs.items()}
    return {"case": dict(case), "inputs": inputs, "grad": grad}


def run(state):
    if own:
        return _call(state)
    with torch.no_grad():
        return (_plain_norm if state["case"]["op"] == "layer_norm" else _plain_ffn)(state)


# ---- the framework's operators
def _call(state):
    import svox_amd as svox
    case, inputs, grad = state["case"], state["inputs"], state["grad"]
    if case["op"] == "layer_norm":
        y = svox.layer_norm(inputs["x"], inputs.get("weight"), inputs.get("bias"))
    else:
        y = svox.gated_ffn(inputs["x"], inputs["w_gate"], inputs["w_up"], inputs["w_down"], inputs.get("b_gate"), inputs.get("b_up"),
                           inputs.get("b_down"), residual=inputs.get("residual"), activation=case["activation"])
    if grad is None:
        return {"y": y}
    names = list(inputs)
    grads = torch.autograd.grad(y, [inputs[name] for name in names], grad)
    return {"y": y.detach(), "grads": dict(zip(names, grads))}


# ---- their plain forms: 32 bits, rounded once
def _plain_norm(state):
    inputs, grad = state["inputs"], state["grad"]
    dtype = inputs["x"].dtype
    x = inputs["x"].float()
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + 1e-5)
    normal = centred * rstd
    affine = "weight" in inputs
    y = normal * inputs["weight"].float() + inputs["bias"].float() if affine else normal
    if grad is None:
        return {"y": y.to(dtype)}
    dy = grad.float()
    dn = dy * inputs["weight"].float() if affine else dy
    dx = rstd * (dn - dn.mean(dim=1, keepdim=True) - normal * (dn * normal).mean(dim=1, keepdim=True))
    grads = {"x": dx.to(dtype)}
    if affine:
        grads.update(weight=(dy * normal).sum(dim=0).to(dtype), bias=dy.sum(dim=0).to(dtype))
    return {"y": y.to(dtype), "grads": grads}


def _activation(name, g):
    """act(g) and its derivative"""
    if name == "relu":
        positive = (g > 0).float()
        return g * positive, positive
    if name == "gelu":
        below = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return s, s * (1.0 - s)
    return g * s, s * (1.0 + g * (1.0 - s))


def _plain_ffn(state):
    inputs, grad, case = state["inputs"], state["grad"], state["case"]
    dtype = inputs["x"].dtype
    x, w_gate, w_up, w_down = (inputs[name].float() for name in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ w_gate.t(), x @ w_up.t()
    if case["bias"]:
        gate, up = gate + inputs["b_gate"].float(), up + inputs["b_up"].float()
    act, slope = _activation(case["activation"], gate)
    hidden = act * up
    y = hidden @ w_down.t()
    if case["bias"]:
        y = y + inputs["b_down"].float()
    if case["residual"]:
        y = y + inputs["residual"].float()
    if grad is None:
        return {"y": y.to(dtype)}
    dy = grad.float()
    dhidden = dy @ w_down
    dgate, dup = dhidden * up * slope, dhidden * act
    grads = {"x": dgate @ w_gate + dup @ w_up, "w_gate": dgate.t() @ x, "w_up": dup.t() @ x, "w_down": dy.t() @ hidden}
    if case["bias"]:
        grads.update(b_gate=dgate.sum(dim=0), b_up=dup.sum(dim=0), b_down=dy.sum(dim=0))
    if case["residual"]:
        grads["residual"] = dy
    return {"y": y.to(dtype), "grads": {name: g.to(dtype) for name, g in grads.items()}}


# ---- in 64 bits, from the definitions; the gradients by differentiation
def exact(case, seed):
    state = prepare(case, seed)
    leaves = {name: x.detach().double().requires_grad_() for name, x in state["inputs"].items()}
    x = leaves["x"]
    if case["op"] == "layer_norm":
        mean = x.sum(dim=1, keepdim=True) / case["dim"]
        variance = (x - mean).pow(2).sum(dim=1, keepdim=True) / case["dim"]
        y = (x - mean) / torch.sqrt(variance + 1e-5)
        if case["affine"]:
            y = y * leaves["weight"] + leaves["bias"]
    else:
        gate, up = torch.matmul(x, leaves["w_gate"].t()), torch.matmul(x, leaves["w_up"].t())
        if case["bias"]:
            gate, up = gate + leaves["b_gate"], up + leaves["b_up"]
        act = {"silu": lambda g: g * torch.sigmoid(g), "gelu": lambda g: g * torch.special.ndtr(g), "relu": torch.relu, "sigmoid": torch.sigmoid}
        y = torch.matmul(act[case["activation"]](gate) * up, leaves["w_down"].t())
        if case["bias"]:
            y = y + leaves["b_down"]
        if case["residual"]:
            y = y + leaves["residual"]
    if state["grad"] is None:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, list(leaves.values()), state["grad"].double())
    return {"y": y.detach(), "grads": dict(zip(leaves, grads))}
