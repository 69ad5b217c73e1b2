"""The linear operators around deformable attention, as measurable cases over their real ranges.

* ``linear``   fused_linear: ``act(x W^T + b) + residual``, the projections and feed-forward of the
               layers around the attention;
* ``grouped``  grouped_linear: the same with weights of its own for each group of consecutive rows
               (the levels of a volume pyramid, or experts), groups of ragged sizes.

A case is a dict of plain values.  ``train``: forward and backward, the gradients of every input
returned beside the output; otherwise the forward alone.  ``act``: "none", "relu", "gelu" (erf),
"gelu_tanh" or "silu".  ``residual``: a residual is added in the epilogue.  ``pad``: x is the first
``k`` columns of rows that are ``pad`` elements longer (a split of a wider projection).  Grouped
cases give ``levels`` (the rows of each group) or ``groups`` and ``rows`` (sizes then follow the
seed, as a router's do: some large, some empty), and ``batch`` items that share the group table.

With ``own`` false an operator is computed by elementary operations in 32 bits, rounded once at the
end.  The sizes of groups are known on the host there; grouped_linear reads them on the device.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _linear(name, rows, k, n, dtype, train, act="none", residual=False, pad=0):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train,
            "act": act, "residual": residual, "pad": pad}


def _grouped(name, k, n, dtype, train, levels="", groups=0, rows=0, batch=1, act="none", residual=False):
    return {"name": name, "kind": "grouped", "k": k, "n": n, "dtype": dtype, "train": train, "levels": levels,
            "groups": groups, "rows": rows, "batch": batch, "act": act, "residual": residual}


def listed():
    return [
        # one query through an output projection: latency
        _linear("query_bf16_infer", 1, 256, 256, "bf16", False, residual=True),
        # a batch of eight rows through a wide layer: the weights' bytes count
        _linear("wide_rows_bf16_infer", 8, 4096, 4096, "bf16", False, act="silu"),
        # a decoder's feed-forward for 2 x 200 object queries
        _linear("decoder_fp16_infer", 400, 256, 1024, "fp16", False, act="gelu"),
        # an encoder layer's output projection and residual over a volume at strides 16 and 32
        _linear("output_bf16_train", 73728, 256, 256, "bf16", True, residual=True),
        # the first half of that layer's feed-forward
        _linear("ffn_bf16_train", 73728, 256, 1024, "bf16", True, act="gelu"),
        # the largest volume (strides 8, 16 and 32) through a feed-forward at inference
        _linear("ffn_large_fp16_infer", 598016, 256, 1024, "fp16", False, act="relu"),
        # odd sizes in full precision, x a part of wider rows
        _linear("ragged_fp32_train", 10013, 250, 333, "fp32", True, act="silu", residual=True, pad=7),
        # a product bound by the matrix units, as wide heads have it
        _linear("square_bf16_infer", 4096, 4096, 4096, "bf16", False, act="gelu_tanh", residual=True),
        # a projection with weights per level over the largest volume's three levels
        _grouped("levels_bf16_train", 256, 256, "bf16", True, levels="524288,65536,8192"),
        # the same over a tiny crop in full precision: launches and host time count
        _grouped("levels_tiny_fp32_train", 256, 256, "fp32", True, levels="512,64"),
        # experts of a feed-forward in training, ragged, some empty
        _grouped("experts_fp16_train", 512, 1024, "fp16", True, groups=64, rows=16411, act="gelu"),
        # a few rows over many experts: most groups hold one row, two or none
        _grouped("experts_few_bf16_infer", 1024, 2048, "bf16", False, groups=64, rows=96, act="silu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row length: half of them multiples of 32, the rest as they come."""
    w = _log_int(rng, lo, hi)
    return max(32, w // 32 * 32) if rng.random() < 0.5 else w


def draw(rng):
    kind = rng.choice(["linear", "linear", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    act = rng.choice(ACTS)
    if train and dtype == "fp32" and act == "relu":
        act = "silu"   # relu's derivative jumps at 0: which side a rounded sum falls on is no fp32 result
    residual = rng.random() < 0.4
    k, n = _width(rng, 24, 4096), _width(rng, 24, 4096)
    # below the largest listed passes: their products, and their rows' bytes
    most = 1.5e11 * (0.33 if train else 1.0) * (0.5 if dtype == "fp32" else 1.0)
    rows = min(_log_int(rng, 1, 590000), int(most / (k * n)), int(3e8 * (0.5 if train else 1.0) / (k + 2 * n)))
    rows = max(1, rows)
    if kind == "linear":
        case = _linear("", rows, k, n, dtype, train, act, residual, pad=rng.choice([0, 0, 0, 8, 5]))
    elif rng.random() < 0.5:
        batch = rng.choice([1, 1, 2])
        per = max(3, rows // batch)
        sizes, left = [], per
        for _ in range(rng.choice([1, 2, 3])):   # levels, each about an eighth of the one before
            sizes.append(max(1, left - left // 8))
            left //= 8
        case = _grouped("", k, n, dtype, train, levels=",".join(str(s) for s in sizes), batch=batch, act=act,
                        residual=residual)
    else:
        groups = _log_int(rng, 4, 96)
        while groups * k * n > 1.5e8:
            groups = max(1, groups // 2)
        case = _grouped("", k, n, dtype, train, groups=groups, rows=rows, act=act, residual=residual)
    del case["name"]
    return case


# ---------------------------------------------------------------------------- inputs


def _group_sizes(case, seed):
    """Rows of each group of one batch item."""
    if case["levels"]:
        return [int(s) for s in case["levels"].split(",")]
    rng = random.Random(1000003 * seed + case["rows"])
    weights = [0.0 if rng.random() < 0.1 else math.exp(rng.gauss(0.0, 0.6)) for _ in range(case["groups"])]
    if sum(weights) == 0.0:
        weights[0] = 1.0
    sizes = [0] * case["groups"]
    if case["rows"] <= 4096:
        for g in rng.choices(range(case["groups"]), weights=weights, k=case["rows"]):
            sizes[g] += 1
        return sizes
    total = sum(weights)
    sizes = [int(case["rows"] * w / total) for w in weights]
    sizes[max(range(len(weights)), key=lambda g: weights[g])] += case["rows"] - sum(sizes)
    return sizes


def _host_inputs(case, seed):
    """The case's tensors on the GPU, in its type: x, weight, bias, residual, grad_output."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dt)

    k, n = case["k"], case["n"]
    if case["kind"] == "linear":
        lead, groups, sizes = (case["rows"],), (), None
        x = normal((case["rows"], k + case["pad"]))[:, :k]
    else:
        sizes = _group_sizes(case, seed)
        rows = sum(sizes)
        lead = (case["batch"], rows) if case["batch"] > 1 else (rows,)
        groups = (len(sizes),)
        x = normal((*lead, k))
    weight = normal((*groups, n, k), 1.0 / math.sqrt(k))
    bias = normal((*groups, n), 0.1)
    residual = normal((*lead, n)) if case["residual"] else None
    grad = normal((*lead, n)) if case["train"] else None
    return x, weight, bias, residual, grad, sizes


def prepare(case, seed):
    x, weight, bias, residual, grad, sizes = _host_inputs(case, seed)
    state = {"case": case, "x": x, "weight": weight, "bias": bias, "residual": residual, "grad": grad, "sizes": sizes}
    if sizes is not None:
        dev = x.device
        bounds = [0]
        for s in sizes:
            bounds.append(bounds[-1] + s)
        state["group_start"] = torch.tensor(bounds, dtype=torch.int64, device=dev)
        longest = max(sizes)
        # many groups: one batched product over groups padded to the longest, where that is not
        # mostly padding
        if len(sizes) > 8 and case["batch"] == 1 and len(sizes) * longest <= max(6 * bounds[-1], 16 * len(sizes)):
            slot = torch.cat([torch.arange(s) + g * longest for g, s in enumerate(sizes)])
            state["slot"], state["slots"] = slot.to(dev), (len(sizes), longest)
    if case["train"]:
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name] = state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------- plain form


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    """act'(z)."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t() + s["bias"].float()
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    if not case["train"]:
        return y.to(dt)
    dz = s["grad"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(z, case["act"])
    out = {"y": y.to(dt), "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt), "db": dz.sum(0).to(dt)}
    if case["residual"]:
        out["dr"] = s["grad"]
    return out


def _products(a, bs, sizes):
    """Each group's rows of a [..., S, K] times its matrix of bs [E, K, N]."""
    return torch.cat([p @ b for p, b in zip(a.split(sizes, dim=-2), bs)], dim=-2)


def _padded(a, s):
    """a's rows, group by group, in [E, longest, ...] with zeros behind each group's last."""
    e, longest = s["slots"]
    p = a.new_zeros(e * longest, a.shape[-1])
    p[s["slot"]] = a
    return p.view(e, longest, a.shape[-1])


def _plain_grouped(s):
    case, sizes = s["case"], s["sizes"]
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    wt = w.transpose(1, 2)
    bias = s["bias"].float().repeat_interleave(torch.diff(s["group_start"]), dim=0, output_size=x.shape[-2])
    padded = "slot" in s
    if padded:
        xp = _padded(x, s)
        z = torch.bmm(xp, wt).flatten(0, 1)[s["slot"]] + bias
    else:
        z = _products(x, wt, sizes) + bias
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    if not case["train"]:
        return y.to(dt)
    dz = s["grad"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(z, case["act"])
    if padded:
        dp = _padded(dz, s)
        dx = torch.bmm(dp, w).flatten(0, 1)[s["slot"]]
        dw, db = torch.bmm(dp.transpose(1, 2), xp), dp.sum(1)
    else:
        dx = _products(dz, w, sizes)
        parts = [(d.flatten(0, -2), p.flatten(0, -2)) for d, p in zip(dz.split(sizes, dim=-2), x.split(sizes, dim=-2))]
        dw = torch.stack([d.t() @ p for d, p in parts])
        db = torch.stack([d.sum(0) for d, _ in parts])
    out = {"y": y.to(dt), "dx": dx.to(dt), "dw": dw.to(dt), "db": db.to(dt)}
    if case["residual"]:
        out["dr"] = s["grad"]
    return out


# ---------------------------------------------------------------------------- one pass


def _own(s):
    from ops3d_amd.linear import fused_linear, grouped_linear

    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["kind"] == "linear":
        y = fused_linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"])
    else:
        y = grouped_linear(s["x"], s["weight"], s["group_start"], s["bias"], activation=act, residual=s["residual"])
    if not case["train"]:
        return y
    names = ["x", "weight", "bias"] + (["residual"] if case["residual"] else [])
    grads = torch.autograd.grad(y, [s[name] for name in names], s["grad"])
    return {"y": y.detach(), **dict(zip(("dx", "dw", "db", "dr"), grads))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["kind"] == "linear" else _plain_grouped(state)


# ---------------------------------------------------------------------------- what a pass needs


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    k, n = case["k"], case["n"]
    if case["kind"] == "linear":
        rows, groups, used = case["rows"], 1, 1
    else:
        sizes = _group_sizes(case, 0)
        rows, groups, used = case["batch"] * sum(sizes), len(sizes), sum(s > 0 for s in sizes)
    elements = rows * k + used * (n * k + n) + rows * n * (2 if case["residual"] else 1)   # x, W, b, r in; y out
    if case["train"]:
        # grad_output in; grad x, W, b out (grad r is grad_output)
        elements += rows * n + rows * k + groups * (n * k + n)
    return {"bytes": e * elements, "flops": 2.0 * rows * n * k * (3 if case["train"] else 1)}


# ---------------------------------------------------------------------------- the definition in 64 bits


def _reference_act(z, act):
    f = torch.nn.functional
    return {"none": lambda t: t, "relu": f.relu, "gelu": f.gelu, "silu": f.silu,
            "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](z)


def exact(case, seed):
    x, weight, bias, residual, grad, sizes = _host_inputs(case, seed)
    leaf = [None if t is None else t.double().requires_grad_(case["train"]) for t in (x, weight, bias, residual)]
    x, weight, bias, residual = leaf
    if sizes is None:
        z = torch.addmm(bias, x, weight.t())
    else:
        z = torch.cat([torch.nn.functional.linear(x.narrow(-2, sum(sizes[:g]), size), weight[g], bias[g])
                       for g, size in enumerate(sizes)], dim=-2)
    y = _reference_act(z, case["act"])
    if residual is not None:
        y = y + residual
    if not case["train"]:
        return y
    grads = torch.autograd.grad(y, [t for t in leaf if t is not None], grad.double())
    return {"y": y.detach(), **dict(zip(("dx", "dw", "db", "dr"), grads))}
