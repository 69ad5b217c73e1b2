"""Attention over all tokens, layer norm and rotary positions, as measurable cases over their real ranges.

* ``attention``  packed_attention: softmax(q k^T scale) v with grouped heads, causal or not, over items of a
                 batch with lengths of their own or over sequences packed one behind another;
* ``norm``       layer_norm: over the last axis, with weight and bias;
* ``rotary``     rotary_positions: pairs of channels turned by the token's position along one of several
                 axes (depth, height and width of a volume, or time, height and width).

A case is a dict of plain values.  ``train``: forward and backward, the gradients of every input
returned beside the output; otherwise the forward alone.

Attention: ``form`` "batch" has ``items`` of ``nq`` queries and ``nk`` keys; with ``ragged`` the items use
fewer of them (a cache filled to different lengths, padded queries).  "packed" splits ``nq`` query rows
into ``items`` sequences, whose sizes follow the seed; ``cross`` does the same with ``nk`` key rows,
otherwise the keys are the queries' tokens.  q, k and v are parts of one projection's rows where
they have the same tokens, k and v of one buffer otherwise.

With ``own`` false an operator is computed by elementary operations in 32 bits (angles in 64), rounded
once at the end.  The lengths are known on the host there; packed_attention reads them on the device.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


def _attention(name, form, items, nq, nk, heads, kv_heads, dim, dtype, train, causal=False, ragged=False, cross=False):
    return {"name": name, "kind": "attention", "form": form, "items": items, "nq": nq, "nk": nk, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train, "causal": causal, "ragged": ragged,
            "cross": cross}


def _norm(name, rows, width, dtype, train, pad=0):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "train": train, "pad": pad}


def _rotary(name, items, tokens, heads, dim, sections, layout, dtype, train, pad=0):
    return {"name": name, "kind": "rotary", "items": items, "tokens": tokens, "heads": heads, "dim": dim,
            "sections": sections, "layout": layout, "dtype": dtype, "train": train, "pad": pad}


def listed():
    return [
        # one new token for each of eight requests, over caches filled to different lengths
        _attention("decode_bf16_infer", "batch", 8, 1, 8192, 32, 8, 128, "bf16", False, ragged=True),
        # 2 x 200 object queries among themselves: latency
        _attention("objects_fp16_infer", "batch", 2, 200, 200, 8, 8, 32, "fp16", False),
        # the same queries over every token of a volume's three levels
        _attention("volume_cross_bf16_infer", "batch", 2, 200, 37376, 8, 8, 32, "bf16", False),
        # a volume's finest level among itself at inference
        _attention("volume_bf16_infer", "batch", 1, 32768, 32768, 8, 8, 32, "bf16", False),
        # an encoder layer's attention over a packed set of crops of different sizes
        _attention("crops_bf16_train", "packed", 7, 16411, 16411, 8, 8, 32, "bf16", True),
        # whole prompts of different lengths, causal, with grouped heads
        _attention("prompts_bf16_train", "packed", 5, 8192, 8192, 16, 4, 128, "bf16", True, causal=True),
        # odd sizes in full precision, queries and keys of different lengths
        _attention("ragged_fp32_train", "packed", 6, 1013, 2029, 6, 2, 36, "fp32", True, causal=True, cross=True),
        # the norms of an encoder layer over a volume at strides 16 and 32
        _norm("volume_norm_bf16_train", 73728, 256, "bf16", True),
        # the same over 2 x 200 object queries at inference: latency
        _norm("objects_norm_fp16_infer", 400, 256, "fp16", False),
        # odd and wide rows in full precision, part of wider rows
        _norm("wide_norm_fp32_train", 2053, 4101, "fp32", True, pad=3),
        # queries' and keys' heads of that encoder layer, positions along three axes
        _rotary("volume_rotary_bf16_train", 1, 73728, 16, 32, "5,5,6", "halves", "bf16", True),
        # wide heads of a few frames' tokens, part of a projection's rows
        _rotary("frames_rotary_fp16_infer", 2, 1551, 20, 128, "16,24,24", "pairs", "fp16", False, pad=256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "norm", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5])
        dim = rng.choice([32, 32, 64, 128, rng.randint(4, 128)])
        form = rng.choice(["batch", "packed"])
        causal, cross = rng.random() < 0.4, rng.random() < 0.4
        # below the largest listed passes: their products, and their logits
        most = 2.5e11 * (0.3 if train else 1.0) * (0.15 if dtype == "fp32" else 1.0)
        pairs = min(most / (4 * heads * dim), 4e9 * (0.3 if train else 1.0) / heads)
        if form == "batch":
            items = _log_int(rng, 1, 16)
            nq = 1 if not train and rng.random() < 0.4 else _log_int(rng, 1, 30000)
            nk = nq if nq > 1 and not cross else _log_int(rng, 1, 60000)
            nk = max(1, min(nk, int(1e8 / (items * kv_heads * dim))))
            while items * nq * nk > pairs or items * nq * heads * dim > 1.2e8:
                nq, nk = max(1, nq * 3 // 4), max(1, nk * 3 // 4) if nk * 2 > nq else nk
            case = _attention("", "batch", items, nq, nk, heads, kv_heads, dim, dtype, train, causal, rng.random() < 0.5, cross)
        else:
            items = _log_int(rng, 1, 40)
            nq = _log_int(rng, 1, 20000)
            nk = _log_int(rng, 1, 20000) if cross else nq
            while nq * nk > pairs:   # as though one sequence held nearly all
                nq, nk = max(1, nq * 3 // 4), max(1, nk * 3 // 4)
            case = _attention("", "packed", items, nq, nk, heads, kv_heads, dim, dtype, train, causal, False, cross)
    elif kind == "norm":
        width = _log_int(rng, 16, 12000)
        if rng.random() < 0.5:
            width = max(16, width // 32 * 32)
        rows = max(1, min(_log_int(rng, 1, 300000), int(4e7 * (0.5 if train else 1.0) / width)))
        case = _norm("", rows, width, dtype, train, rng.choice([0, 0, 8, 5]))
    else:
        dim = rng.choice([32, 64, 128, rng.randint(6, 128)])
        axes = rng.choice([1, 2, 3, 3])
        left, sections = dim // 2, []
        for a in range(axes):
            n = left // (axes - a) if rng.random() < 0.7 else rng.randint(0, left // (axes - a))
            sections.append(n)
            left -= n
        heads = rng.choice([1, 2, 5, 8, 16, 40])
        items = rng.choice([1, 1, 2, 5])
        tokens = max(1, min(_log_int(rng, 1, 80000), int(6e7 * (0.5 if train else 1.0) / (items * heads * dim))))
        case = _rotary("", items, tokens, heads, dim, ",".join(str(s) for s in sections), rng.choice(["halves", "pairs"]),
                       dtype, train, rng.choice([0, 0, 64, 7]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------- inputs


def _lengths(case, seed):
    """Queries and keys of each item or sequence."""
    rng = random.Random(1000003 * seed + 7 * case["nq"] + case["nk"])
    items, nq, nk = case["items"], case["nq"], case["nk"]
    if case["form"] == "batch":
        if not case["ragged"]:
            return [nq] * items, [nk] * items
        ql = [nq] * items if nq == 1 else [rng.randint(0, nq) for _ in range(items)]
        same = nq == nk and not case["cross"]
        return ql, list(ql) if same else [rng.randint(nk // 4, nk) for _ in range(items)]

    def split(rows):
        weights = [0.0 if rng.random() < 0.08 else math.exp(rng.gauss(0.0, 0.8)) for _ in range(items)]
        if sum(weights) == 0.0:
            weights[0] = 1.0
        total = sum(weights)
        sizes = [int(rows * w / total) for w in weights]
        sizes[max(range(items), key=lambda i: weights[i])] += rows - sum(sizes)
        return sizes

    ql = split(nq)
    return ql, split(nk) if case["cross"] else list(ql)


def _inputs(case, seed):
    """The case's tensors on the GPU, in its type."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dt)

    if case["kind"] == "attention":
        h, hk, d, nq, nk = (case[n] for n in ("heads", "kv_heads", "dim", "nq", "nk"))
        lead = (case["items"],) if case["form"] == "batch" else ()
        if nq == nk and not case["cross"] and nq > 1:
            rows = normal((*lead, nq, h + 2 * hk, d))
            q, k, v = rows.split([h, hk, hk], dim=-2)
        else:
            q = normal((*lead, nq, h, d))
            k, v = normal((*lead, nk, 2 * hk, d)).split([hk, hk], dim=-2)
        grad = normal((*lead, nq, h, d)) if case["train"] else None
        return {"q": q, "k": k, "v": v, "grad": grad}
    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        # activations' rows have means and scales of their own
        x = torch.randn(rows, width + case["pad"], generator=gen, device=dev)
        x = x * (0.5 + torch.rand(rows, 1, generator=gen, device=dev)) + torch.randn(rows, 1, generator=gen, device=dev)
        return {"x": x.to(dt)[:, :width], "weight": normal((width,), 0.2) + 1, "bias": normal((width,), 0.2),
                "grad": normal((rows, width)) if case["train"] else None}
    items, tokens, heads, dim = (case[n] for n in ("items", "tokens", "heads", "dim"))
    axes = len(case["sections"].split(","))
    x = normal((items, tokens, heads * dim + case["pad"]))[..., :heads * dim].unflatten(-1, (heads, dim))
    # voxels of a large stitched volume, or frames and pixels: whole and half steps
    extent = torch.tensor([4096.0, 512.0, 2048.0][:axes], device=dev)
    positions = torch.floor(torch.rand(items, tokens, axes, generator=gen, device=dev) * extent) + 0.5
    return {"x": x, "positions": positions, "grad": normal((items, tokens, heads, dim)) if case["train"] else None}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["kind"] == "attention":
        dev = state["q"].device
        state["lengths"] = ql, kl = _lengths(case, seed)
        if case["form"] == "packed":
            for name, sizes in (("q_start", ql), ("k_start", kl)):
                bounds = [0]
                for s in sizes:
                    bounds.append(bounds[-1] + s)
                state[name] = torch.tensor(bounds, dtype=torch.int64, device=dev)
        elif case["ragged"]:
            state["q_len"] = torch.tensor(ql, dtype=torch.int64, device=dev)
            state["k_len"] = torch.tensor(kl, dtype=torch.int64, device=dev)
        leaves = ("q", "k", "v")
    else:
        leaves = ("x", "weight", "bias") if case["kind"] == "norm" else ("x",)
    if case["train"]:
        for name in leaves:
            state[name] = state[name].detach().requires_grad_(True)
    return state


def _sections(case):
    return tuple(int(n) for n in case["sections"].split(","))


# ---------------------------------------------------------------------------- plain form


def _plain_rows(q, k, v, ql, kl, causal, grad):
    """Attention of items [B, N, H, D] whose lengths are ql, kl; in 32 bits, some query rows at a time.
    Returns the output and the gradients of q, k and v."""
    b, nq, h, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    g, scale = h // hk, 1.0 / math.sqrt(d)
    kt = k.float().permute(0, 2, 3, 1).contiguous()   # [B, Hk, D, Nk]
    vh = v.float().transpose(1, 2).contiguous()       # [B, Hk, Nk, D]
    full = min(kl) == nk and min(ql) == nq
    if causal or not full:
        lens_q, lens_k = (torch.tensor(n, device=q.device).view(b, 1, 1, 1, 1) for n in (ql, kl))
        col = torch.arange(nk, device=q.device)
    out = torch.empty(b, nq, h, d, device=q.device)
    dq = dk = dv = None
    if grad is not None:
        dq = torch.empty_like(out)
        kh, vt = kt.transpose(2, 3).contiguous(), vh.transpose(2, 3).contiguous()
        dk, dv = torch.zeros_like(vh), torch.zeros_like(vh)
    step = max(1, min(nq, (1 << 28) // max(1, b * h * nk)))
    for r0 in range(0, nq, step):
        n = min(step, nq - r0)

        def rows(t):   # [B, Hk, G * n, D]
            return t[:, r0:r0 + n].float().unflatten(2, (hk, g)).permute(0, 2, 3, 1, 4).reshape(b, hk, g * n, d)

        def back(t):   # [B, n, H, D]
            return t.view(b, hk, g, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)

        qh = rows(q)
        s = ((qh @ kt) * scale).view(b, hk, g, n, nk)
        if causal or not full:
            at = torch.arange(r0, r0 + n, device=q.device).view(n, 1)
            seen = (col < lens_k) & (at < lens_q)
            if causal:
                seen = seen & (col <= at + lens_k - lens_q)
            s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = (p / torch.where(total == 0, 1.0, total)).view(b, hk, g * n, nk)
        o = p @ vh
        out[:, r0:r0 + n] = back(o)
        if grad is not None:
            do = rows(grad)
            dv += p.transpose(2, 3) @ do
            ds = p * (do @ vt - (do * o).sum(-1, keepdim=True)) * scale
            dq[:, r0:r0 + n] = back(ds @ kh)
            dk += ds.transpose(2, 3) @ qh
    if grad is None:
        return out, None, None, None
    return out, dq, dk.transpose(1, 2), dv.transpose(1, 2)


def _plain_attention(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    q, k, v, grad = s["q"], s["k"], s["v"], s["grad"]
    ql, kl = s["lengths"]
    if case["form"] == "batch":
        parts = _plain_rows(q, k, v, ql, kl, case["causal"], grad)
    else:
        parts = [torch.zeros(t.shape, device=t.device) for t in ((q, q, k, v) if case["train"] else (q,))]
        q0 = k0 = 0
        for nq, nk in zip(ql, kl):
            if nq and nk:
                at = [slice(q0, q0 + nq), slice(q0, q0 + nq), slice(k0, k0 + nk), slice(k0, k0 + nk)]
                got = _plain_rows(q[None, at[0]], k[None, at[2]], v[None, at[2]], [nq], [nk], case["causal"],
                                  None if grad is None else grad[None, at[0]])
                for whole, rows, part in zip(parts, at, got):
                    whole[rows] = part[0]
            q0, k0 = q0 + nq, k0 + nk
    if not case["train"]:
        return parts[0].to(dt)
    return {name: t.to(dt) for name, t in zip(("y", "dq", "dk", "dv"), parts)}


def _plain_norm(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    centred = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    n = centred * r
    y = (n * w + s["bias"].float()).to(dt)
    if not case["train"]:
        return y
    g = s["grad"].float()
    gw = g * w
    dx = r * (gw - gw.mean(-1, keepdim=True) - n * (gw * n).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dw": (g * n).sum(0).to(dt), "db": g.sum(0).to(dt)}


def _turn(x, cos, sin, layout, pairs):
    """Pairs of channels of x [..., H, D] turned by the angles whose cosines and sines are given."""
    a, b = (x[..., :pairs], x[..., pairs:2 * pairs]) if layout == "halves" else (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([u, w], -1) if layout == "halves" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _plain_rotary(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    sections = _sections(case)
    dev = s["x"].device
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=dev, dtype=torch.int64)
    freq = torch.tensor([THETA ** (-i / n) for n in sections for i in range(n)], device=dev, dtype=torch.float64)
    angle = s["positions"].double()[..., axis] * freq   # [B, S, P]
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    y = _turn(s["x"].float(), cos, sin, case["layout"], sum(sections)).to(dt)
    if not case["train"]:
        return y
    return {"y": y, "dx": _turn(s["grad"].float(), cos, -sin, case["layout"], sum(sections)).to(dt)}


# ---------------------------------------------------------------------------- one pass


def _own(s):
    case = s["case"]
    if case["kind"] == "attention":
        from ops3d_amd.attention import packed_attention

        y = packed_attention(s["q"], s["k"], s["v"], q_start=s.get("q_start"), k_start=s.get("k_start"),
                             q_len=s.get("q_len"), k_len=s.get("k_len"), causal=case["causal"])
        names = ("q", "k", "v")
    elif case["kind"] == "norm":
        from ops3d_amd.norm import layer_norm

        y = layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
        names = ("x", "weight", "bias")
    else:
        from ops3d_amd.rotary import rotary_positions

        y = rotary_positions(s["x"], s["positions"], _sections(case), theta=THETA, layout=case["layout"])
        names = ("x",)
    if not case["train"]:
        return y
    grads = torch.autograd.grad(y, [s[name] for name in names], s["grad"])
    keys = {"attention": ("dq", "dk", "dv"), "norm": ("dx", "dw", "db"), "rotary": ("dx",)}[case["kind"]]
    return {"y": y.detach(), **dict(zip(keys, grads))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "rotary": _plain_rotary}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------- what a pass needs


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["kind"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        ql, kl = _lengths(case, 0)
        pairs = 0   # of a query and a key that it sees
        for nq, nk in zip(ql, kl):
            if not case["causal"]:
                pairs += nq * nk
            else:   # query i sees i + 1 + nk - nq keys
                first = max(0, nq - nk)
                pairs += (nq - first) * nk - (nq - first) * (nq - first - 1) // 2
        rows = case["nq"] * (case["items"] if case["form"] == "batch" else 1)   # of the output, all of it written
        elements = sum(ql) * h * d + 2 * sum(kl) * hk * d + rows * h * d        # q, k, v in; y out
        if train:   # grad_output in; grad q, k, v out
            keys = case["nk"] * (case["items"] if case["form"] == "batch" else 1)
            elements += sum(ql) * h * d + rows * h * d + 2 * keys * hk * d
        return {"bytes": e * elements, "flops": (14.0 if train else 4.0) * pairs * h * d}
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        elements = 2 * n + 2 * case["width"] + (2 * n + 2 * case["width"] if train else 0)
        return {"bytes": e * elements, "flops": (20.0 if train else 8.0) * n}
    n = case["items"] * case["tokens"] * case["heads"] * case["dim"]
    axes = len(_sections(case))
    return {"bytes": e * n * (4 if train else 2) + 4 * axes * case["items"] * case["tokens"],
            "flops": (6.0 if train else 3.0) * n}


# ---------------------------------------------------------------------------- the definition in 64 bits


def _exact_sequence(q, k, v, causal, grad):
    """One sequence [N, H, D], head by head, some queries at a time, in 64 bits by autograd."""
    nq, h, d = q.shape
    nk, hk = k.shape[:2]
    out = torch.zeros(nq, h, d, dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)] if grad is not None else None
    if nq == 0 or nk == 0:
        return out, grads
    step = max(1, (1 << 26) // nk)
    for head in range(h):
        kk, vv = (t[:, head * hk // h].double() for t in (k, v))
        for r0 in range(0, nq, step):
            leaves = [q[r0:r0 + step, head].double(), kk, vv]
            leaves = [t.detach().requires_grad_(grad is not None) for t in leaves]
            logits = torch.mm(leaves[0], leaves[1].t()).div(math.sqrt(d))
            if causal:
                last = torch.arange(r0, min(nq, r0 + step), device=q.device) + (nk - nq)   # each query's last key
                hidden = torch.arange(nk, device=q.device)[None] > last[:, None]
                empty = (last < 0)[:, None]
                logits = logits.masked_fill(hidden & ~empty, -math.inf)
                probs = torch.softmax(logits, -1).masked_fill(empty, 0.0)
            else:
                probs = torch.softmax(logits, -1)
            y = torch.mm(probs, leaves[2])
            out[r0:r0 + step, head] = y.detach()
            if grad is not None:
                dq, dk, dv = torch.autograd.grad(y, leaves, grad[r0:r0 + step, head].double())
                grads[0][r0:r0 + step, head] = dq
                grads[1][:, head * hk // h] += dk
                grads[2][:, head * hk // h] += dv
    return out, grads


def _exact_attention(case, seed, t):
    ql, kl = _lengths(case, seed)
    q, k, v, grad = t["q"], t["k"], t["v"], t["grad"]
    wide = torch.float64
    y = torch.zeros(q.shape, dtype=wide, device=q.device)
    grads = [torch.zeros(a.shape, dtype=wide, device=a.device) for a in (q, k, v)] if grad is not None else None
    for i, (nq, nk) in enumerate(zip(ql, kl)):
        if case["form"] == "batch":
            at_q, at_k = (i, slice(0, nq)), (i, slice(0, nk))
        else:
            at_q, at_k = slice(sum(ql[:i]), sum(ql[:i + 1])), slice(sum(kl[:i]), sum(kl[:i + 1]))
        out, parts = _exact_sequence(q[at_q], k[at_k], v[at_k], case["causal"], None if grad is None else grad[at_q])
        y[at_q] = out
        if grads is not None:
            for whole, at, part in zip(grads, (at_q, at_k, at_k), parts):
                whole[at] = part
    return y if grads is None else {"y": y, **dict(zip(("dq", "dk", "dv"), grads))}


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, seed, t)
    if case["kind"] == "norm":
        leaves = [t[n].double().requires_grad_(case["train"]) for n in ("x", "weight", "bias")]
        y = torch.nn.functional.layer_norm(leaves[0], (case["width"],), leaves[1], leaves[2], 1e-5)
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, leaves, t["grad"].double())
        return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), grads))}
    # a pair as a complex number, times exp(i angle)
    sections = _sections(case)
    parts = [t["positions"][..., a:a + 1].double() * torch.exp(
        torch.arange(n, device=t["x"].device, dtype=torch.float64) * (-math.log(THETA) / max(n, 1)))
        for a, n in enumerate(sections)]
    angle = torch.cat(parts, -1)[:, :, None, :]
    pairs = sum(sections)

    def turn(x, sign):
        x = x.double()
        first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if case["layout"] == "halves" else (
            slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), sign * angle)
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if not case["train"]:
        return turn(t["x"], 1.0)
    return {"y": turn(t["x"], 1.0), "dx": turn(t["grad"], -1.0)}
