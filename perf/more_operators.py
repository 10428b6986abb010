"""What the operators of networks over the cells of a tree are measured on: attention within packed sequences of cells, norms of
queries and keys with the rotation by their positions, and the norm of many gradients with its clipping.

A pass is one call of `svox_amd.attention`, `svox_amd.rotate_heads` or `svox_amd.clip_norm` (forward), or the call and its
gradients through autograd (step).  The sizes are those of a leaf decoder's networks: sequences are windows of consecutive cells
(a cell is a token, eight to a node), from one queried point to the cells of a 64^3 grid, features of 64 to 1024 numbers in heads of
16 to 128; gradients are those of a decoder's weights and of a tree's records (28 numbers of SH9, 49 of SH16).
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one queried point that looks at the cells of a coarse tree: a call of few rows over a long axis
        {"name": "attend_point", "op": "attention", "pass": "forward", "dtype": "bfloat16", "layout": "even", "sequences": 1, "queries": 1, "keys": 32775,
         "heads": 8, "kv_heads": 2, "dim": 64, "causal": False, "mix": 0},
        # every cell of a 64^3 grid within windows of 512 consecutive ones, as a picture's tree is decoded
        {"name": "attend_windows", "op": "attention", "pass": "forward", "dtype": "bfloat16", "layout": "even", "sequences": 512, "queries": 262144,
         "keys": 262144, "heads": 4, "kv_heads": 4, "dim": 32, "causal": False, "mix": 0},
        # a training step in single precision, a decoder's own type, in windows of 64 cells
        {"name": "attend_step_f32", "op": "attention", "pass": "step", "dtype": "float32", "layout": "even", "sequences": 512, "queries": 32768,
         "keys": 32768, "heads": 4, "kv_heads": 4, "dim": 16, "causal": False, "mix": 0},
        # a training step on trees of many sizes packed one after another, their cells generated one by one, grouped heads
        {"name": "attend_step_packed", "op": "attention", "pass": "step", "dtype": "float16", "layout": "ragged", "sequences": 61, "queries": 30011,
         "keys": 30011, "heads": 8, "kv_heads": 2, "dim": 64, "causal": True, "mix": 5},
        # the largest training step: one long sequence, wide heads
        {"name": "attend_step_long", "op": "attention", "pass": "step", "dtype": "bfloat16", "layout": "even", "sequences": 1, "queries": 16384,
         "keys": 16384, "heads": 8, "kv_heads": 8, "dim": 128, "causal": True, "mix": 0},
        # one queried point: a call's latency
        {"name": "rotate_point", "op": "rotate_heads", "pass": "forward", "dtype": "bfloat16", "rows": 1, "heads": 8, "kv_heads": 2, "dim": 64,
         "rotated": 64, "axes": 3, "interleaved": False, "weights": True},
        # every cell of a 64^3 grid by its centre, heads that share keys
        {"name": "rotate_leaves", "op": "rotate_heads", "pass": "forward", "dtype": "bfloat16", "rows": 262144, "heads": 8, "kv_heads": 2, "dim": 32,
         "rotated": 32, "axes": 3, "interleaved": False, "weights": True},
        # a training step in single precision, sizes that divide by little, a part of each head left unrotated
        {"name": "rotate_step_f32", "op": "rotate_heads", "pass": "step", "dtype": "float32", "rows": 10007, "heads": 6, "kv_heads": 3, "dim": 44,
         "rotated": 30, "axes": 3, "interleaved": True, "weights": True},
        # the largest: a training step of wide layers, cells by their place in the sequence
        {"name": "rotate_step_wide", "op": "rotate_heads", "pass": "step", "dtype": "bfloat16", "rows": 131072, "heads": 8, "kv_heads": 4, "dim": 128,
         "rotated": 128, "axes": 1, "interleaved": False, "weights": True},
        # the weights of a small decoder: a call of many small tensors
        {"name": "clip_decoder", "op": "clip_norm", "pass": "forward", "dtype": "float32", "depth": 2, "dim": 64, "hidden": 256, "record": 49, "leaves": 0, "over": 3.0},
        # the weights of a wide decoder in half precision and the features of a 32^3 grid
        {"name": "clip_features", "op": "clip_norm", "pass": "forward", "dtype": "bfloat16", "depth": 3, "dim": 512, "hidden": 2048, "record": 76, "leaves": 32768,
         "over": 1.7},
        # the records of a large tree with a decoder's weights, in single precision
        {"name": "clip_tree", "op": "clip_norm", "pass": "forward", "dtype": "float32", "depth": 1, "dim": 28, "hidden": 112, "record": 28, "leaves": 4000003, "over": 40.0},
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotate_heads", "clip_norm"])
    case = {"op": op, "pass": "forward" if op == "clip_norm" else rng.choice(["forward", "step"]), "dtype": rng.choice(["float32", "bfloat16", "float16"])}
    if op == "clip_norm":
        case.update(depth=rng.randint(1, 6), dim=_size(rng, 16, 512), record=rng.choice([4, 28, 49, 76]), leaves=rng.choice([0, _size(rng, 100, 4000000)]),
                    over=rng.choice([0.5, 1.3, 8.0]))
        case["hidden"] = 4 * case["dim"]
    else:
        case["kv_heads"] = rng.choice([1, 1, 2, 3, 4, 8])
        case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 8])
        case["dim"] = rng.choice([16, 32, 64, 128, rng.randint(8, 128)])
        while case["heads"] * case["dim"] > 1024:
            case["heads"], case["kv_heads"] = case["heads"] // case["kv_heads"], 1
            if case["heads"] * case["dim"] > 1024:
                case["heads"] = 4
    if op == "rotate_heads":
        case.update(rows=_size(rng, 1, 262144), axes=rng.choice([1, 2, 3]), interleaved=rng.random() < 0.4, weights=rng.random() < 0.8)
        case["rotated"] = case["dim"] // 2 * 2 if rng.random() < 0.7 else 2 * rng.randint(1, case["dim"] // 2)
    if op == "attention":
        kind = rng.choice(["windows", "windows", "ragged", "ragged", "few"])
        case.update(layout="even" if kind == "windows" else "ragged", causal=rng.random() < 0.5, mix=rng.randint(1, 1000000))
        if kind == "windows":
            length, case["sequences"] = _size(rng, 8, 1024), _size(rng, 1, 512)
            case["queries"] = case["keys"] = length * case["sequences"]
        elif kind == "ragged":
            case["sequences"] = _size(rng, 1, 200)
            case["queries"] = case["keys"] = _size(rng, max(64, case["sequences"]), 32768)
        else:                # a few queries a sequence, over many keys
            case["sequences"] = _size(rng, 1, 32)
            case["queries"], case["keys"] = case["sequences"] * rng.choice([1, 1, 2, 7, 20]), _size(rng, 1000, 262144)
    most = {x["name"]: work(x) for x in listed()}[{"attention": "attend_step_long", "rotate_heads": "rotate_step_wide", "clip_norm": "clip_tree"}[op]]
    # (single precision costs some ten times the matrix work of half precision here)
    dear = 10.0 if op == "attention" and case["dtype"] == "float32" else 1.0
    while True:
        w = work(case)
        share = max(w["flops"] * dear / most["flops"], w["bytes"] / most["bytes"])
        if share <= 1:
            return case
        if op == "rotate_heads":
            case["rows"] = max(1, int(case["rows"] / (1.05 * share)))
        elif op == "clip_norm":
            case["leaves"] = int(case["leaves"] / (1.05 * share))
        elif case["sequences"] > 1 and case["layout"] == "even":
            length, case["sequences"] = case["keys"] // case["sequences"], max(1, int(case["sequences"] / (1.05 * share)))
            case["queries"] = case["keys"] = length * case["sequences"]
        else:
            same = case["queries"] == case["keys"]
            case["keys"] = max(1, int(0.7 * case["keys"]))
            case["queries"] = case["keys"] if same else case["queries"]
            case["sequences"] = min(case["sequences"], case["queries"])


def _lengths(total, case, seed):
    """`total` cells in as many sequences as the case has: alike, or from very short to long"""
    n = case["sequences"]
    if case["layout"] == "even":
        return [total // n] * n
    rng = random.Random(seed)
    weights = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(n)]
    ends = [0]
    for w in weights:
        ends.append(ends[-1] + w)
    ends = [int(total * e / ends[-1]) for e in ends[:-1]] + [total]
    return [b - a for a, b in zip(ends, ends[1:])]


def _both_lengths(case):
    keys = _lengths(case["keys"], case, case["mix"])
    if case["queries"] == case["keys"]:
        return keys, keys
    return [case["queries"] // case["sequences"]] * case["sequences"], keys


def _clip_shapes(case):
    d, h, o = case["dim"], case["hidden"], case["record"]
    shapes = []
    for block in range(case["depth"] + 1):
        out = d if block < case["depth"] else o
        shapes += [(d,), (d,), (h, d), (h, d), (out, h), (h,), (h,), (out,)]
    if case["leaves"]:
        shapes.append((case["leaves"], d))
    return shapes


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    step = case["pass"] == "step"
    if case["op"] == "clip_norm":
        n = sum(math.prod(s) for s in _clip_shapes(case))
        return {"bytes": 2 * size * n, "flops": 3 * n}
    if case["op"] == "rotate_heads":
        n, heads, d = case["rows"], case["heads"] + case["kv_heads"], case["dim"]
        parameters = 2 * d if case["weights"] else 0
        # heads and the gradient of the result in, the result and the heads' gradients out
        values = (4 if step else 2) * n * heads * d + (2 if step else 1) * parameters
        return {"bytes": size * values + 4 * n * case["axes"], "flops": (24 if step else 8) * n * heads * d}
    q_lengths, k_lengths = _both_lengths(case)
    pairs = 0
    for a, b in zip(q_lengths, k_lengths):
        if not case["causal"]:
            pairs += a * b
        else:                # query i of a sees keys up to i + b - a
            first = max(0, a - b)
            low, high = first + 1 + b - a, b
            pairs += (low + high) * (a - first) // 2
    wide, narrow = case["queries"] * case["heads"] * case["dim"], case["keys"] * case["kv_heads"] * case["dim"]
    values = 2 * wide + 2 * narrow                                # q, k, v in, the result out
    if step:
        values += 2 * wide + 2 * narrow                           # its gradient in, those of q, k and v out
    return {"bytes": size * values, "flops": (14 if step else 4) * pairs * case["heads"] * case["dim"]}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    step = case["pass"] == "step"

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale + shift).to(dtype)

    if case["op"] == "clip_norm":
        # gradients of tensors whose sizes differ as those of biases, weights and features do
        scales = [10.0 ** -(i % 4) for i in range(len(_clip_shapes(case)))]
        tensors = [normal(*s, scale=scale) for s, scale in zip(_clip_shapes(case), scales)]
        # a bound that the norm exceeds `over` times (or does not, where that is below one); in expectation: the values' own spread
        expected = math.sqrt(sum(math.prod(s) * scale * scale for s, scale in zip(_clip_shapes(case), scales)))
        return {"case": dict(case), "tensors": tensors, "max_norm": expected / case["over"]}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate_heads":
        n = case["rows"]
        # queries, keys and values of a row side by side, as one product leaves them
        packed = normal(n, (h + 2 * hk) * d, scale=1.5)
        inputs = {"q": packed[:, :h * d].unflatten(1, (h, d)), "k": packed[:, h * d:(h + hk) * d].unflatten(1, (hk, d))}
        if case["weights"]:
            inputs["q_weight"], inputs["k_weight"] = normal(d, scale=0.1, shift=1.0), normal(d, scale=0.1, shift=1.0)
        pairs = case["rotated"] // 2
        if case["axes"] == 1:                 # places in a sequence, as far as a tree of a million cells has them
            positions = torch.randint(0, 1 << 20, (n, 1), generator=g, device=DEVICE).float()
            frequencies = 10000.0 ** (-torch.arange(pairs, device=DEVICE, dtype=torch.float32) / pairs)[None]
        else:                                 # centres of cells, each axis on a part of the pairs
            positions = torch.rand(n, case["axes"], generator=g, device=DEVICE)
            which = torch.arange(pairs, device=DEVICE)
            waves = 2 * math.pi * 2.0 ** (8.0 * (which // case["axes"]) / max(1, pairs // case["axes"]))
            frequencies = torch.where(which % case["axes"] == torch.arange(case["axes"], device=DEVICE)[:, None], waves, torch.zeros_like(waves)).float()
        state = {"positions": positions, "frequencies": frequencies.contiguous()}
        grads = [normal(n, h, d), normal(n, hk, d)] if step else None
    else:
        tq, tk = case["queries"], case["keys"]
        # queries and keys of unit norm times a weight, rotated: entries near a normal distribution's
        inputs = {"q": normal(tq, h, d), "k": normal(tk, hk, d), "v": normal(tk, hk, d)}
        q_lengths, k_lengths = _both_lengths(case)
        state = {"q_lengths": q_lengths, "k_lengths": k_lengths}
        for name, lengths in (("offsets", q_lengths), ("key_offsets", k_lengths)):
            state[name] = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEVICE)
        grads = [normal(tq, h, d)] if step else None
    if step:
        inputs = {name: x.detach().requires_grad_() for name, x in inputs.items()}
    return {"case": dict(case), "inputs": inputs, "grads": grads, **state}


def run(state):
    if own:
        return _call(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "rotate_heads": _plain_rotate, "clip_norm": _plain_clip}[state["case"]["op"]](state)


# ---- the framework's operators
def _call(state):
    import svox_amd as svox
    case = state["case"]
    if case["op"] == "clip_norm":
        norm, tensors = svox.clip_norm(state["tensors"], state["max_norm"])
        return {"norm": norm, "tensors": list(tensors)}
    inputs = state["inputs"]
    if case["op"] == "attention":
        same = state["q_lengths"] is state["k_lengths"]
        out = [svox.attention(inputs["q"], inputs["k"], inputs["v"], state["offsets"], None if same else state["key_offsets"], causal=case["causal"])]
    else:
        out = list(svox.rotate_heads(inputs["q"], inputs["k"], state["positions"], state["frequencies"], inputs.get("q_weight"), inputs.get("k_weight"),
                                     interleaved=case["interleaved"]))
    if state["grads"] is None:
        return {"out": out}
    grads = torch.autograd.grad(out, list(inputs.values()), state["grads"])
    return {"out": [y.detach() for y in out], "grads": dict(zip(inputs, grads))}


# ---- their plain forms: 32 bits, rounded once
def _plain_clip(state):
    total = torch.zeros((), dtype=torch.float64, device=DEVICE)
    for x in state["tensors"]:
        total = total + (x.float() * x.float()).sum(dtype=torch.float64)     # (a long sum)
    norm = total.sqrt()
    factor = torch.where(norm > state["max_norm"], state["max_norm"] / norm, torch.ones_like(norm)).float()
    return {"norm": norm.float(), "tensors": [(x.float() * factor).to(x.dtype) for x in state["tensors"]]}


def _turn(x, cos, sin, rotated, interleaved):
    first, second = (x[..., :rotated:2], x[..., 1:rotated:2]) if interleaved else (x[..., :rotated // 2], x[..., rotated // 2:rotated])
    a, b = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., rotated:]], dim=-1)


def _plain_rotate(state):
    case, inputs = state["case"], state["inputs"]
    dtype = inputs["q"].dtype
    angles = state["positions"].double() @ state["frequencies"].double()     # (64 bits: far positions)
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]
    out, grads = [], {}
    for i, name in enumerate(("q", "k")):
        x = inputs[name].float()
        r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6)
        w = inputs[name + "_weight"].float() if case["weights"] else None
        n = x * r
        out.append(_turn(n if w is None else n * w, cos, sin, case["rotated"], case["interleaved"]).to(dtype))
        if state["grads"] is not None:
            dy = _turn(state["grads"][i].float(), cos, -sin, case["rotated"], case["interleaved"])
            if w is not None:
                grads[name + "_weight"] = (dy * n).sum(dim=(0, 1)).to(dtype)
                dy = dy * w
            grads[name] = (r * (dy - n * (dy * n).mean(dim=-1, keepdim=True))).to(dtype)
    return {"out": out} if state["grads"] is None else {"out": out, "grads": {name: grads[name] for name in inputs}}


def _plain_attention(state):
    case, inputs = state["case"], state["inputs"]
    dtype = inputs["q"].dtype
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group, scale = h // hk, d ** -0.5
    q, k, v = (inputs[name].float() for name in ("q", "k", "v"))
    step = state["grads"] is not None
    dy = state["grads"][0].float() if step else None
    y = torch.empty_like(q)
    if step:
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q_lengths, k_lengths = state["q_lengths"], state["k_lengths"]
    at, q0, k0 = 0, 0, 0
    while at < len(q_lengths):
        a, b = q_lengths[at], k_lengths[at]
        # neighbours of the same lengths together, as far as their scores fit
        n = 1
        while at + n < len(q_lengths) and (q_lengths[at + n], k_lengths[at + n]) == (a, b) and (n + 1) * h * a * b <= 1 << 28:
            n += 1
        if a > 0 and b > 0:
            keys = lambda x: x[k0:k0 + n * b].view(n, b, hk, d).permute(0, 2, 1, 3).contiguous()                       # noqa: E731
            kk, vv = keys(k), keys(v)                                                                                  # (n, hk, b, d)
            rows = max(1, min(a, (1 << 28) // (n * h * b)))                                                            # of a sequence at a time
            for r in range(0, a, rows):
                c = min(rows, a - r)
                pick = lambda x: x[q0:q0 + n * a].view(n, a, hk, group, d)[:, r:r + c].permute(0, 2, 3, 1, 4).reshape(n, hk, group * c, d)   # noqa: E731
                seen = min(b, max(0, r + c + b - a)) if case["causal"] else b
                qq = pick(q)
                s = (qq @ kk[:, :, :seen].transpose(2, 3)) * scale
                if case["causal"]:
                    hidden = torch.arange(seen, device=DEVICE) > (torch.arange(r, r + c, device=DEVICE) + (b - a))[:, None]
                    s = s.masked_fill(hidden.repeat(group, 1), -math.inf)
                    s = s - s.amax(dim=-1, keepdim=True).clamp_min(-1e30) if seen else s                               # (a row may see nothing)
                else:
                    s = s - s.amax(dim=-1, keepdim=True)
                p = s.exp()
                total = p.sum(dim=-1, keepdim=True)
                p = p / torch.where(total > 0, total, torch.ones_like(total))
                o = p @ vv[:, :, :seen]
                put = lambda to, x: to[q0:q0 + n * a].view(n, a, hk, group, d)[:, r:r + c].copy_(x.view(n, hk, group, c, d).permute(0, 3, 1, 2, 4))   # noqa: E731
                put(y, o)
                if step:
                    do = pick(dy)
                    ds = p * (do @ vv[:, :, :seen].transpose(2, 3) - (do * o).sum(dim=-1, keepdim=True)) * scale
                    put(dq, ds @ kk[:, :, :seen])
                    dk[k0:k0 + n * b].view(n, b, hk, d)[:, :seen] += (ds.transpose(2, 3) @ qq).permute(0, 2, 1, 3)
                    dv[k0:k0 + n * b].view(n, b, hk, d)[:, :seen] += (p.transpose(2, 3) @ do).permute(0, 2, 1, 3)
        else:                # nothing to see
            y[q0:q0 + n * a] = 0
            if step:
                dq[q0:q0 + n * a] = 0
        at, q0, k0 = at + n, q0 + n * a, k0 + n * b
    out = {"out": [y.to(dtype)]}
    if step:
        out["grads"] = {"q": dq.to(dtype), "k": dk.to(dtype), "v": dv.to(dtype)}
    return out


# ---- in 64 bits, from the definitions; the gradients by differentiation
def exact(case, seed):
    if case["op"] == "attention" and (case["sequences"] * case["kv_heads"] > 8000 or work(case)["flops"] > 3e13):
        return None
    state = prepare(case, seed)
    if case["op"] == "clip_norm":
        norm = torch.cat([torch.linalg.vector_norm(x.double())[None] for x in state["tensors"]]).pow(2).sum().sqrt()
        factor = min(1.0, state["max_norm"] / float(norm))
        return {"norm": norm, "tensors": [x.double() * factor for x in state["tensors"]]}
    leaves = {name: x.detach().double().requires_grad_(state["grads"] is not None) for name, x in state["inputs"].items()}
    if case["op"] == "rotate_heads":
        out = []
        for name in ("q", "k"):
            x = leaves[name]
            n = x / torch.sqrt(x.pow(2).sum(dim=-1, keepdim=True) / case["dim"] + 1e-6)
            if case["weights"]:
                n = n * leaves[name + "_weight"]
            rotated, pairs = case["rotated"], case["rotated"] // 2
            angle = sum(state["positions"].double()[:, i, None] * state["frequencies"].double()[i] for i in range(case["axes"]))[:, None]
            j = torch.arange(pairs, device=DEVICE)
            first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + pairs)
            turned = torch.complex(n[..., first], n[..., second]) * torch.polar(torch.ones_like(angle), angle)
            place = torch.argsort(torch.cat([first, second, torch.arange(rotated, case["dim"], device=DEVICE)]))
            out.append(torch.cat([turned.real, turned.imag, n[..., rotated:]], dim=-1)[..., place])
        if state["grads"] is None:
            return {"out": out}
        grads = torch.autograd.grad(out, list(leaves.values()), [x.double() for x in state["grads"]])
        return {"out": [y.detach() for y in out], "grads": dict(zip(leaves, grads))}
    h, hk, d, step = case["heads"], case["kv_heads"], case["dim"], state["grads"] is not None
    group = h // hk
    y = torch.zeros(case["queries"], h, d, dtype=torch.float64, device=DEVICE)
    grads = {name: torch.zeros_like(x) for name, x in leaves.items()}
    q0 = k0 = 0
    for a, b in zip(state["q_lengths"], state["k_lengths"]):
        for head in range(hk):
            if a == 0 or b == 0:
                continue
            part = {"q": (slice(q0, q0 + a), slice(head * group, (head + 1) * group)), "k": (slice(k0, k0 + b), head), "v": (slice(k0, k0 + b), head)}
            for one in range(group):          # (a head at a time: the scores of a long sequence are large)
                where = {**part, "q": (slice(q0, q0 + a), head * group + one)}
                mine = {name: leaves[name].detach()[where[name]].clone().requires_grad_(step) for name in leaves}
                s = torch.mm(mine["q"], mine["k"].t().contiguous()) / math.sqrt(d)
                empty = torch.zeros(a, 1, dtype=torch.bool, device=DEVICE)
                if case["causal"]:
                    i, j = torch.arange(a, device=DEVICE)[:, None], torch.arange(b, device=DEVICE)[None]
                    hidden = j - i > b - a
                    empty = hidden.all(dim=1, keepdim=True)
                    s = s.masked_fill(hidden & ~empty, -math.inf)
                o = torch.mm(torch.softmax(s, dim=1).masked_fill(empty, 0.0), mine["v"])
                y[where["q"]] = o.detach()
                if step:
                    for name, x in zip(mine, torch.autograd.grad(o, list(mine.values()), state["grads"][0][where["q"]].double())):
                        grads[name][where[name]] += x
        q0, k0 = q0 + a, k0 + b
    return {"out": [y], "grads": grads} if step else {"out": [y]}
