"""Calls of the linear operators that their use brings along, beside the sizes and types of test_linear.py
(whose helpers and float64 restatement are used here)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import linear as ref
from ops3d_amd import FlashDeformAttn3D, _extension, fused_linear, grouped_linear
from test_linear import DTYPES, gpu, log, make, grouped_case


# act' far out, small beside 1: z, and act's names
SATURATED = [("silu", -10.0), ("silu", -12.0), ("silu", -6.0), ("gelu", -3.5), ("gelu", -4.0), ("gelu_tanh", -3.5),
             ("gelu_tanh", -4.0), ("silu", -1.5), ("gelu", -1.0), ("gelu", 0.25), ("gelu", 3.0)]


@gpu
@pytest.mark.parametrize("rows", [40, 2000])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("activation,z", SATURATED)
def test_saturated_units_keep_their_gradients(gpu_device, activation, z, dtype, rows):
    """Units that share a saturated z: their act' is held relative to its size, so the gradients' errors,
    which add up over the rows, stay within the roundings."""
    dt = DTYPES[dtype]
    log(f"[case] saturated {activation} {z} {dtype} {rows}")
    x = torch.ones(rows, 32, dtype=dt, device="cuda").requires_grad_(True)
    w = torch.zeros(40, 32, dtype=dt, device="cuda").requires_grad_(True)
    b = torch.full((40,), z, dtype=dt, device="cuda").requires_grad_(True)
    u = torch.full((rows, 40), 16.0, dtype=dt, device="cuda")
    y = fused_linear(x, w, b, activation)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), u)
    d = ref.act(torch.tensor(z, dtype=torch.float64), activation)[1].item()
    # act' evaluated to 2^-14 of itself out here (the error function's polynomial is off by 6e-4 of its tail,
    # which is at most 1 / z^2 of act'), held to 2^-11; dz and the result rounded by half a step each, and a
    # sum of equal fp32 terms of up to 2000 2^-24
    rel = 2.0 ** -14 + 2.0 ** -11 + 2 * torch.finfo(dt).eps / 2 + 2000 * 2.0 ** -24
    want = rows * 16.0 * d
    for name, got in (("db", db), ("dw", dw)):
        err = (got.double() / want - 1).abs().max().item()
        assert err <= rel, f"{name}: off by {err:.2e} of {want:.3e}"
    assert not dx.any()


def bindings():
    """The extension module's operators and those of the binding without it, under one signature."""
    C = _extension._C
    bare = type(C)(C._lib, C.__file__)
    return {"module": C.linear, "ctypes": lambda *a: type(C).linear(bare, *a)}


@gpu
@pytest.mark.parametrize("binding", ["module", "ctypes"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("batch,N,start", [(0, 24, [10, 60, 150]), (2, 7, [10, 60, 60, 150]), (3, 1, [-5, 90, 40, 170]),
                                           (2, 40, [0, 30, 200]), (0, 130, [200, 200, 200]), (0, 16, [5, 100])])
def test_residual_gradient_of_rows_in_no_group(gpu_device, batch, N, start, dtype, binding):
    """y is 0 in rows of no group whatever the residual holds, so the residual's gradient is 0 there."""
    S, K, E = 200, 16, {2: 2, 3: 2, 4: 3}[len(start)]
    log(f"[case] residual gradient {batch} {N} {start} {dtype} {binding}")
    gen = torch.Generator(device="cuda").manual_seed(31)
    lead = (batch, S) if batch else (S,)
    dt = DTYPES[dtype]
    x, w, r, u = (make(gen, s, dt) for s in ((*lead, K), (E, N, K), (*lead, N), (*lead, N)))
    inside = (ref.group_of_rows(S, start, E) >= 0).cuda()[:, None]
    u = torch.where(inside, u, torch.full_like(u, float("nan")))
    table = torch.tensor(start, device="cuda")
    op = bindings()[binding]
    want = torch.where(inside, u, torch.zeros_like(u))
    for leaves in ((r,), (x, w, r)):
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        y = op(*(leaves[:2] if len(leaves) == 3 else (x, w)), None, leaves[-1], table, 0)
        assert torch.equal(torch.autograd.grad(y, leaves, u)[-1], want)
    # rows in a wider matrix, one row for all, another order of the axes
    for v in (torch.cat([u, u], -1)[..., :N], u[..., :1, :].nan_to_num(1.0).expand(*lead, N),
              u.transpose(-1, -2).contiguous().transpose(-1, -2)):
        rl = r.detach().requires_grad_(True)
        (dr,) = torch.autograd.grad(op(x, w, None, rl, table, 0), rl, v)
        assert torch.equal(dr, torch.where(inside, v, torch.zeros_like(v)))


@gpu
def test_residual_gradient_captured(gpu_device):
    """The same in a graph, replayed with other groups between eager calls."""
    gen = torch.Generator(device="cuda").manual_seed(32)
    x, w, r, u = (make(gen, s, torch.bfloat16) for s in ((300, 32), (2, 48, 32), (300, 48), (300, 48)))
    start = torch.tensor([10, 60, 150], device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    log("[case] residual gradient captured")

    def step():
        return torch.autograd.grad(grouped_linear(x, w, start, None, "silu", r), leaves, u)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for table in ([10, 60, 150], [0, 0, 300], [299, 299, 300], [0, 0, 0]):
        start.copy_(torch.tensor(table))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(outs, want))
        row = torch.arange(300, device="cuda")[:, None]
        assert torch.equal(outs[2], torch.where((row >= table[0]) & (row < table[2]), u, torch.zeros_like(u)))


def test_keep_rows_refusals():
    if _extension._C is None:
        pytest.skip("library not built")
    lib, p = _extension._C._lib, ctypes.c_void_p(256)   # a stand-in: refused before any launch

    def call(src=p, ld=8, start=p, count=2, dst=p, dtype=2, batch=1, rows=4, groups=2, features=8):
        return lib.ops3d_linear_keep_rows(src, ld, start, count, dst, dtype, batch, rows, groups, features, None)

    for text, kw in (("unsupported dtype", dict(dtype=9)), ("rows", dict(rows=-1)), ("out_features", dict(features=0)),
                     ("groups must be", dict(groups=0)), ("negative", dict(ld=-1)), ("NULL", dict(start=None)),
                     ("NULL", dict(src=None)), ("NULL", dict(dst=None)), ("must have", dict(count=4)),
                     ("8-byte", dict(start=ctypes.c_void_p(260))), ("element size", dict(dst=ctypes.c_void_p(257)))):
        assert call(**kw) == 1 and text in lib.ops3d_fda_last_error().decode(), (text, lib.ops3d_fda_last_error())
    assert call(src=None, dst=None, rows=0) == 0
    with pytest.raises(RuntimeError, match="CPU"):
        _extension._C.linear_keep_rows(torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64), 2)

@gpu
@pytest.mark.parametrize("wide", [torch.float32, torch.float64])
def test_autocast_residual_of_rows_in_no_group(gpu_device, wide):
    """Under autocast a wider residual is added outside the product: rows of no group stay 0 all the same."""
    gen = torch.Generator(device="cuda").manual_seed(33)
    x, w, r, u = (make(gen, s, torch.float32) for s in ((2, 50, 32), (2, 24, 32), (2, 50, 24), (2, 50, 24)))
    r, u = r.to(wide), u.to(wide)
    start = torch.tensor([7, 20, 41], device="cuda")
    rl = r.requires_grad_(True)
    log(f"[case] autocast, rows of no group {wide}")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = grouped_linear(x, w, start, None, "gelu", rl)
        row = grouped_linear(x, w, start, None, "gelu", rl[0, 0])   # added outside, it may be broadcast
    plain = grouped_linear(x.bfloat16(), w.bfloat16(), start, None, "gelu")
    inside = (ref.group_of_rows(50, [7, 20, 41], 2) >= 0).cuda()[:, None]
    assert y.dtype == wide
    assert torch.equal(y, torch.where(inside, plain + r, torch.zeros_like(r)))
    assert torch.equal(row, torch.where(inside, plain + r[0, 0], torch.zeros_like(r)))
    assert torch.equal(torch.autograd.grad(y, rl, u)[0], torch.where(inside, u, torch.zeros_like(u)))


@gpu
@pytest.mark.parametrize("binding", ["module", "ctypes"])
@pytest.mark.parametrize("act", [0, 2])
def test_gradient_penalty_raises(gpu_device, act, binding):
    """A gradient that depends on something that requires one raises when it is differentiated, also where
    grad_output is a plain tensor: a penalty on it must not be dropped."""
    gen = torch.Generator(device="cuda").manual_seed(34)
    op = bindings()[binding]
    log(f"[case] penalty {act} {binding}")

    def leaves(*wanted):
        sizes = {"x": (20, 16), "w": (24, 16), "b": (24,), "r": (20, 24)}
        return [make(gen, s, torch.float32).requires_grad_(k in wanted) for k, s in sizes.items()]

    x, w, b, r = leaves("x", "w", "b", "r")
    for wanted in (x, w, b):
        y = op(x, w, b, r, None, act)
        (g,) = torch.autograd.grad(y.sum(), wanted, create_graph=True)
        if wanted is b and not act:
            assert not g.requires_grad      # a sum of grad_output alone
            continue
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (y.sum() + g.pow(2).sum()).backward()
    # a weight without a gradient and no activation: x's gradient is a constant, and the penalty's is 0
    x, w, b, r = leaves("x")
    y = op(x, w, b, r, None, act)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    if not act:
        assert not g.requires_grad
        (y.sum() + g.pow(2).sum()).backward()
        assert torch.equal(x.grad, g)
    else:
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (y.sum() + g.pow(2).sum()).backward()
    # the residual's gradient is grad_output itself, as often as wanted
    x, w, b, r = leaves("r")
    u = make(gen, (20, 24), torch.float32).requires_grad_(True)
    (g,) = torch.autograd.grad(op(x, w, b, r, None, act), r, u, create_graph=True)
    assert torch.equal(torch.autograd.grad(g.pow(2).sum(), u)[0], 2 * u)
    start = torch.tensor([3, 9, 17], device="cuda")
    y = op(x, torch.stack([w, w]), torch.stack([b, b]), r, start, act)
    (g,) = torch.autograd.grad(y, r, u, create_graph=True)
    inside = (ref.group_of_rows(20, [3, 9, 17], 2) >= 0).cuda()[:, None]
    assert torch.equal(torch.autograd.grad(g.pow(2).sum(), u)[0], torch.where(inside, 2 * u, torch.zeros_like(u)))


@gpu
def test_many_items_of_many_groups(gpu_device):
    """More groups than an item has rows: no more tiles than rows, and no launch of 2^32 threads."""
    S, E = 128, 1024
    log("[case] 64 items of 1024 groups")
    grouped_case(S, [i // 8 for i in range(E)], E, 32, 4096, torch.bfloat16, "silu", batch=64)


@gpu
def test_grids_beyond_one_launch(gpu_device):
    """2^32 threads and more, in several launches: products of one term, which are exact."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    bf = torch.bfloat16
    with torch.no_grad():
        log("[case] 17 groups of one row, 2^24 columns")
        E, N = 17, 1 << 24
        x, w = make(gen, (E, 1), bf), make(gen, (E, N, 1), bf)
        y = grouped_linear(x, w, torch.arange(E, device="cuda"))
        for e in range(E):
            assert torch.equal(y[e], (x[e].float() * w[e, :, 0].float()).to(bf))
        del x, w, y
    log("[case] 1.1e9 rows of one feature")
    rows = 1_100_000_000
    x = (torch.arange(rows, dtype=torch.int32, device="cuda") % 251).to(bf)[:, None].requires_grad_(True)
    w = torch.full((1, 1), -2.0, dtype=bf, device="cuda")
    y = fused_linear(x, w)
    assert torch.equal(y, x.detach() * -2)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(dx, y.detach())
    del x, y, dx
    log("[case] 4096 groups, three with a row, 262208 features")
    E, K = 4096, 262208
    w = torch.zeros(E, 1, K, dtype=bf, device="cuda").requires_grad_(True)
    x, u = make(gen, (5, K), bf), make(gen, (5, 1), bf)
    table = torch.tensor([0] + [1] * 2000 + [2] * 2094 + [3, 4], device="cuda")   # rows 0, 1, 2 and 3 each in a group
    assert table.numel() == E + 1
    (dw,) = torch.autograd.grad(grouped_linear(x, w, table), w, u)
    full = {int((table[1:] > r).nonzero()[0, 0]): r for r in range(4)}
    for e, r in full.items():
        assert torch.equal(dw[e, 0], (u[r].float() * x[r].float()).to(bf))
    empty = torch.ones(E, dtype=torch.bool, device="cuda")
    empty[list(full)] = False
    assert not dw[empty].any()


def test_too_many_tiles_are_refused():
    if _extension._C is None:
        pytest.skip("library not built")
    lib, p = _extension._C._lib, ctypes.c_void_p(256)   # a stand-in: refused before any launch
    many = 1 << 24
    assert lib.ops3d_linear_forward(p, 8, p, None, None, 0, None, 0, p, None, None, 0, 2, 0, 1, many, 1, many, 8, None) == 1
    assert b"2^31 tiles" in lib.ops3d_fda_last_error()
    assert lib.ops3d_linear_backward(p, many, p, None, 0, None, p, 8, p, None, None, p, 1 << 62, 2, 1, many, 1, 8, many,
                                     None) == 1
    assert b"gradient: 2^31 tiles" in lib.ops3d_fda_last_error()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("wants", [False, True])
def test_forward_mode_is_refused(which, wants, device):
    """A tensor with a tangent is refused, with gradients wanted or not: y would come without one."""
    fw = torch.autograd.forward_ad
    t = {"x": torch.ones(5, 8), "weight": torch.ones(4, 8), "bias": torch.ones(4), "residual": torch.ones(5, 4)}
    t = {k: v.to(device).requires_grad_(wants) for k, v in t.items()}
    if _extension._C is None:
        pytest.skip("library not built")
    with fw.dual_level():
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        for f in bindings().values():
            for grad in (torch.enable_grad(), torch.no_grad()):
                with grad, pytest.raises(RuntimeError, match="forward-mode"):
                    f(t["x"], t["weight"], t["bias"], t["residual"], None, 0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            fused_linear(**t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            grouped_linear(t["x"], t["weight"][None], torch.zeros(1, dtype=torch.int64, device=device),
                           t["bias"][None], None, t["residual"])


@gpu
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_transforms_are_refused(gpu_device, which):
    """torch.func and vmap wrap tensors without memory of their own: every argument raises."""
    t = {"x": torch.ones(5, 8), "weight": torch.ones(4, 8), "bias": torch.ones(4), "residual": torch.ones(5, 4)}
    t = {k: v.cuda() for k, v in t.items()}
    log(f"[case] transforms of {which}")

    def f(v):
        return fused_linear(**{**t, which: v})

    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: f(v).sum())(t[which])
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (t[which],), (t[which],))
    with pytest.raises(RuntimeError):
        torch.vmap(f)(torch.stack([t[which]] * 3))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("wants", [False, True])
def test_tracing_is_refused(wants, device):
    """A trace would record the output's allocation without the kernels that fill it."""
    if _extension._C is None:
        pytest.skip("library not built")
    x, w = torch.ones(5, 8, device=device), torch.ones(4, 8, device=device).requires_grad_(wants)
    start = torch.zeros(1, dtype=torch.int64, device=device)
    calls = [lambda t, w: fused_linear(t, w), lambda t, w: grouped_linear(t, w[None], start)]
    calls += [lambda t, w, f=f: f(t, w, None, None, None, 0) for f in bindings().values()]
    for call in calls:
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x, w), check_trace=False)


@gpu
def test_module_residual_goes_through_output_proj(gpu_device):
    """With a residual, output_proj's hooks run and what stands in its place is called, as without one."""
    from ops3d_amd.workloads import level_meta

    torch.manual_seed(0)
    st, lsi = level_meta(((4, 4, 8), (2, 2, 4)), gpu_device)
    m = FlashDeformAttn3D(32, 4, 2, 4).to(gpu_device)
    q, v = torch.randn(2, 9, 32, device=gpu_device), torch.randn(2, 144, 32, device=gpu_device)
    refp, res = torch.rand(2, 9, 1, 3, device=gpu_device), torch.randn(2, 9, 32, device=gpu_device)
    args = (q, refp, v, st, lsi)
    log("[case] module residual")

    def check(want):
        # one product of 32 terms, in another order: 2 * 33 * 2^-24 of a sum of |terms| below 2^6, twice
        torch.testing.assert_close(m(*args, residual=res), want, rtol=0, atol=2 * 66 * 2.0 ** -24 * 64)

    with torch.no_grad():
        check(m(*args) + res)
        seen = []
        for hook in (m.output_proj.register_forward_hook(lambda mod, i, o: seen.append(o.clone())),
                     m.output_proj.register_forward_hook(lambda mod, i, o: 2 * o),
                     m.output_proj.register_forward_pre_hook(lambda mod, i: (i[0] * 3,))):
            check(m(*args) + res)
            hook.remove()
        assert len(seen) == 2 and torch.equal(seen[0], seen[1])
        plain = m.output_proj
        m.output_proj = torch.nn.Sequential(plain, torch.nn.Tanh())
        check(m(*args) + res)
        m.output_proj = plain
        torch.nn.utils.parametrizations.weight_norm(m.output_proj)
        m.output_proj.parametrizations.weight.original0.mul_(2)
        check(m(*args) + res)
    seen = []
    m.output_proj = torch.nn.Linear(32, 32).to(gpu_device)
    hook = m.output_proj.register_full_backward_hook(lambda mod, gi, go: seen.append(go[0]))
    m(*args, residual=res).sum().backward()
    assert len(seen) == 1
    hook.remove()


@gpu
def test_autocast_leaves_float64(gpu_device):
    """As torch's, autocast casts no float64: refused as without it, not cut to 16 bits."""
    x, w = torch.ones(5, 8, dtype=torch.float64, device="cuda"), torch.ones(4, 8, dtype=torch.float64, device="cuda")
    log("[case] autocast float64")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(ValueError, match="unsupported"):
            fused_linear(x, w)
        with pytest.raises(ValueError, match="dtype differs"):
            fused_linear(x.float(), w)
        y = fused_linear(x.float(), w.float(), None, None, torch.ones(5, 4, dtype=torch.float64, device="cuda"))
    assert y.dtype == torch.float64 and torch.equal(y, torch.full_like(y, 9.0))


def test_workspace_of_the_wanted_gradients():
    if _extension._C is None:
        pytest.skip("library not built")
    lib = _extension._C._lib
    of, every = lib.ops3d_linear_backward_workspace_bytes_for, lib.ops3d_linear_backward_workspace_bytes
    X, W, B = 1, 2, 4
    for case in ((2, 1, 73728, 1, 1024, 256, 0), (2, 1, 598016, 3, 256, 256, 1), (0, 1, 1, 1, 1856, 3301, 0),
                 (1, 64, 512, 16, 1024, 1024, 1), (2, 2, 4096, 64, 256, 256, 1)):
        for act in (0, 1):
            assert of(*case, act, X | W | B) == every(*case, act)
            assert all(of(*case, act, w) <= every(*case, act) for w in range(8))
            assert of(*case, act, 0) == 0 and of(*case, act, 8) == 0
    rows, N, K = 73728, 1024, 256
    case, dz = (2, 1, rows, 1, N, K, 0), rows * N * 2
    assert of(*case, 1, X) == 0                       # neither dz nor partial sums
    assert of(*case, 0, X | B) == of(*case, 0, B) and 0 < of(*case, 0, B) < 2 << 20
    assert of(*case, 1, B) == dz + of(*case, 0, B)
    assert of(*case, 1, W) == dz + of(*case, 0, W)
    assert of(*case, 0, W) + of(*case, 0, B) == of(*case, 0, W | B)
    assert of(2, 1, 1, 1, 3301, 1856, 0, 0, X) > 0    # a long sum in parts


@gpu
@pytest.mark.parametrize("asked", [False, True])
@pytest.mark.parametrize("binding", ["module", "ctypes"])
def test_memory_of_the_wanted_gradients(gpu_device, asked, binding):
    """x's gradient alone takes its own memory and no dz or partial sums: with the other inputs frozen, or
    (the module's node) with a backward pass that asks for nothing else."""
    if asked and binding == "ctypes":
        pytest.skip("a Function in Python is not told what a pass asks for")
    rows, N, K, bf = 73728, 1024, 256, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(51)
    log(f"[case] memory {asked} {binding}")
    x, w, b, u = (make(gen, s, bf) for s in ((rows, K), (N, K), (N,), (rows, N)))
    x.requires_grad_(True)
    for t in (w, b):
        t.requires_grad_(asked)
    y = bindings()[binding](x, w, b, None, None, 2)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    (dx,) = torch.autograd.grad(y, x, u)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < rows * K * 2 + (4 << 20)
    y = bindings()[binding](x, w.detach().requires_grad_(True), b.detach().requires_grad_(True), None, None, 2)
    assert torch.equal(torch.autograd.grad(y, x, u)[0], dx)


@gpu
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_each_gradient_asked_for_alone(gpu_device, bias, grouped):
    """A pass that asks for one gradient or some gets what a pass for all gets."""
    gen = torch.Generator(device="cuda").manual_seed(52)
    log(f"[case] asked alone {bias} {grouped}")
    E = (3,) if grouped else ()
    t = [make(gen, s, torch.bfloat16).requires_grad_(True) for s in ((700, 64), (*E, 40, 64), (700, 40))]
    b = make(gen, (*E, 40), torch.bfloat16).requires_grad_(True) if bias else None
    u, table = make(gen, (700, 40), torch.bfloat16), torch.tensor([5, 100, 400, 650], device="cuda")
    for act in (0, 4):
        y = _extension._C.linear(t[0], t[1], b, t[2], table if grouped else None, act)
        leaves = t + ([b] if bias else [])
        every = torch.autograd.grad(y, leaves, u, retain_graph=True)
        for pick in ([0], [1], [2], [0, 2], [1, 2], [0, 1], *([[3], [2, 3], [0, 3], [1, 3]] if bias else [])):
            got = torch.autograd.grad(y, [leaves[i] for i in pick], u, retain_graph=True)
            assert all(torch.equal(g, every[i]) for g, i in zip(got, pick)), pick


# Rows in thousands: a worst-case bound of their sums is wider than the sums themselves.  With small whole
# numbers every fp32 sum is exact (below 2^24), in any order, so results are the exact ones rounded once.
LONG = [("bf16", 40000, 256, 256, None), ("fp16", 20011, 100, 520, "relu"), ("fp32", 20011, 90, 130, "relu"),
        ("bf16", 65607, 256, 504, "relu"), ("fp16", 70001, 128, 512, None), ("bf16", 66001, 512, 128, None),
        ("fp16", 140001, 256, 256, None), ("bf16", 140033, 256, 256, "relu"), ("bf16", 9000, 24, 40, "relu"),
        ("fp32", 30000, 256, 256, None), ("bf16", 73728, 250, 333, "relu")]


def whole(gen, shape, dtype, device="cuda"):
    return torch.randint(-2, 3, shape, generator=gen, device=device).to(dtype)


def exact_step(x, w, b, r, u, activation, group):
    """y and the gradients of x, w and b in 64 bits; group: of each row, -1 for none."""
    x, w, b, r, u = (t.double() for t in (x, w, b, r, u))
    y, dx, dw, db = torch.zeros_like(r), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for g in range(w.shape[0]):
        at = (group == g).nonzero().flatten().to(x.device)
        z, a = ref.act(x[at] @ w[g].t() + b[g], activation)[0], u[at]
        y[at] = z + r[at]
        if activation:
            a = a * (z > 0)
        dx[at], dw[g], db[g] = a @ w[g], a.t() @ x[at], a.sum(0)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def exact_case(start, lead, E, K, N, dtype, activation):
    dt = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(61)
    x, w, b, r, u = (whole(gen, s, dt) for s in ((*lead, K), (E, N, K), (E, N), (*lead, N), (*lead, N)))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    if start is None:
        group = torch.zeros(lead[0], dtype=torch.int64)
        y = fused_linear(x, w[0], b[0], activation, r)
    else:
        group = ref.group_of_rows(lead[-1], start, E).repeat(lead[0] if len(lead) > 1 else 1)
        y = grouped_linear(x, w, torch.tensor(start, device="cuda"), b, activation, r)
    got = dict(zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, leaves, u))))
    flat = [t.detach().reshape(-1, t.shape[-1]) for t in (x, r, u)]
    want = exact_step(flat[0], w.detach(), b.detach(), flat[1], flat[2], activation, group)
    for name, e in want.items():
        assert e.abs().max() < 60000, name       # fits fp16
        assert torch.equal(got[name].detach().reshape(e.shape), e.to(dt)), name


@gpu
@pytest.mark.parametrize("dtype,rows,K,N,activation", LONG)
def test_long_sums_exact(gpu_device, dtype, rows, K, N, activation):
    log(f"[case] exact {rows}x{K}->{N} {dtype} {activation}")
    exact_case(None, (rows,), 1, K, N, dtype, activation)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("K,N", [(256, 256), (128, 512), (256, 504), (250, 129)])
def test_grouped_long_sums_exact(gpu_device, K, N, dtype):
    """Long groups of two items, a last stage that ends inside, a short group, rows of none."""
    log(f"[case] exact grouped {K}->{N} {dtype}")
    exact_case([70, 100, 60000, 99990], (2, 100003), 3, K, N, dtype, None)
    exact_case([0, 34990, 39400], (40011,), 3, K, N, dtype, "relu")


def test_exact_sums_show_a_lost_stage():
    """The rounded gradient tells a sum without one stage of 64 rows, or without the rows behind the last
    whole one, from the whole sum, and so it tells zeros."""
    for dtype, rows, _, _, activation in [*LONG, ("bf16", 119800, 0, 0, None), ("fp16", 69980, 0, 0, "relu")]:
        gen = torch.Generator().manual_seed(62)
        dt = DTYPES[dtype]
        x, u = (whole(gen, (rows, 16), torch.float64, "cpu") for _ in range(2))
        if activation:
            u = u * (torch.rand(u.shape, generator=gen) < 0.5)
        dw, db = (u.t() @ x).to(dt), u.sum(0).to(dt)
        last = rows - (rows % 64 or 64)
        for a in (0, rows // 128 * 64, last):
            b = min(a + 64, rows)
            assert ((u.t() @ x - u[a:b].t() @ x[a:b]).to(dt) != dw).sum() > 64     # of 256
            assert ((u.sum(0) - u[a:b].sum(0)).to(dt) != db).any()
        assert (dw != 0).sum() > 200
