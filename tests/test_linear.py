"""The linear operators (fused_linear, grouped_linear) against their float64 restatement
(oracle/linear.py) within componentwise bounds derived there, their refusals, and the module that
calls them.  CPU: the restatement itself, refusals, sizes.  GPU: everything that computes."""
from __future__ import annotations

import ctypes
import sys

import pytest
import torch

from oracle import linear as ref
from ops3d_amd import FlashDeformAttn3D, FlashDeformAttnFromOffsets, GroupedLinear, _extension, fused_linear, grouped_linear
from ops3d_amd.linear import ACTIVATIONS
from ops3d_amd.workloads import level_meta

gpu = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def log(text):
    print(text, flush=True)
    sys.stdout.flush()


def make(gen, shape, dtype, scale=1.0, device="cuda"):
    return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)


def check(name, got, want, where=None):
    value, bound = want
    got = got.double().reshape(value.shape)
    assert torch.isfinite(got).all() or not torch.isfinite(value).all(), f"{name}: not finite"
    over = (got - value).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{name}: {int((over > 0).sum())}/{over.numel()} outside the bound, by at most {worst:.3e}"


def flat(t):
    return None if t is None else t.detach().reshape(-1, t.shape[-1])


def compare(x, weight, bias, residual, activation, group, outs, grad=None):
    """outs: y, or y and the gradients dx, dw, db."""
    w = weight if weight.dim() == 3 else weight[None]
    b = None if bias is None else bias.reshape(w.shape[0], -1)
    want = ref.run(flat(x), w.detach(), None if b is None else b.detach(), flat(residual), activation, group, flat(grad))
    for name, got in outs.items():
        if got is not None:
            check(name, got.detach(), want[name])


def linear_case(rows, K, N, dtype, activation=None, with_bias=True, with_residual=False, train=True, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x, w = make(gen, (rows, K), dtype), make(gen, (N, K), dtype, K ** -0.5)
    b = make(gen, (N,), dtype, 0.3) if with_bias else None
    r = make(gen, (rows, N), dtype) if with_residual else None
    u = make(gen, (rows, N), dtype)
    leaves = [t.requires_grad_(train) for t in (x, w, b, r) if t is not None]
    y = fused_linear(x, w, b, activation, r)
    outs = {"y": y}
    if train:
        grads = list(torch.autograd.grad(y, leaves, u))
        outs["dx"], outs["dw"] = grads[0], grads[1]
        if with_bias:
            outs["db"] = grads[2]
        if with_residual:
            assert torch.equal(grads[-1], u)
    assert y.dtype == dtype and y.shape == (rows, N)
    compare(x, w, b, r, activation, torch.zeros(rows, dtype=torch.int64), outs, u)


def grouped_case(S, start, groups, K, N, dtype, activation=None, batch=0, with_bias=True, with_residual=False, train=True,
                 seed=0):
    """batch 0: x [S, K]; otherwise [batch, S, K]."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lead = (batch, S) if batch else (S,)
    x, w = make(gen, (*lead, K), dtype), make(gen, (groups, N, K), dtype, K ** -0.5)
    b = make(gen, (groups, N), dtype, 0.3) if with_bias else None
    r = make(gen, (*lead, N), dtype) if with_residual else None
    u = make(gen, (*lead, N), dtype)
    group = ref.group_of_rows(S, start, groups).repeat(max(batch, 1))
    leaves = [t.requires_grad_(train) for t in (x, w, b, r) if t is not None]
    y = grouped_linear(x, w, torch.tensor(start, dtype=torch.int64, device="cuda"), b, activation, r)
    outs = {"y": y}
    if train:
        grads = list(torch.autograd.grad(y, leaves, u))
        outs["dx"], outs["dw"] = grads[0], grads[1]
        if with_bias:
            outs["db"] = grads[2]
    assert y.shape == (*lead, N)
    compare(x, w, b, r, activation, group, outs, u)
    outside = (group < 0).to(y.device)
    assert not flat(y)[outside].any()
    if train:
        assert not flat(outs["dx"])[outside].any()


# ---------------------------------------------------------------------------- CPU


@pytest.mark.parametrize("activation", list(ACTIVATIONS))
def test_restatement_against_torch_and_differences(activation):
    """oracle/linear.py against torch.nn.functional and central differences, in float64."""
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(9, 5, generator=gen).double(), torch.randn(2, 4, 5, generator=gen).double()
    b, r, u = (torch.randn(s, generator=gen).double() for s in ((2, 4), (9, 4), (9, 4)))
    group = ref.group_of_rows(9, [1, 4], 2)
    assert group.tolist() == [-1, 0, 0, 0, 1, 1, 1, 1, 1]
    assert ref.group_of_rows(9, [-3, 7, 5, 40], 3).tolist() == [0] * 7 + [2] * 2
    out = ref.run(x.float(), w.float(), b.float(), r.float(), activation, group, u.float())

    def f(x, w, b):
        z = torch.stack([torch.nn.functional.linear(x[i], w[g], b[g]) if (g := group[i]) >= 0 else torch.zeros(4).double()
                         for i in range(9)])
        fn = {None: lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
              "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[activation]
        return (fn(z) + r.float().double()) * (group >= 0)[:, None]

    args = [t.float().double() for t in (x, w, b)]
    torch.testing.assert_close(out["y"][0], f(*args), rtol=1e-12, atol=1e-12)
    for i, name in enumerate(("dx", "dw", "db")):
        d = torch.randn(args[i].shape, generator=gen).double()
        h = 1e-6
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + h * d, args[i] - h * d
        slope = ((f(*plus) - f(*minus)) / (2 * h) * u.float().double()).sum()
        # differences of step h: h^2 |f'''| and 2^-53 |f| / h, both below 1e-8 here
        torch.testing.assert_close((out[name][0] * d).sum(), slope, rtol=1e-7, atol=1e-7)


def test_python_refusals_on_the_cpu():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="activation must be one of"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="activation must be one of"):
        fused_linear(x, w, activation=["relu"])
    with pytest.raises(ValueError, match="group_start"):
        grouped_linear(x, w[None], None)
    if _extension._C is None:
        pytest.skip("library not built")
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        fused_linear(x, w)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        grouped_linear(x, w[None], torch.zeros(1, dtype=torch.int64))


@pytest.fixture(scope="module")
def lib():
    if _extension._C is None:
        pytest.skip("library not built")
    return _extension._C._lib


def _forward(lib, ptr=None, **kw):
    a = dict(x=ptr, ldx=8, w=ptr, b=None, r=None, ldr=0, start=None, count=0, y=ptr, ag=None, dtype=2, act=0, batch=1,
             rows=4, groups=1, N=8, K=8)
    a.update(kw)
    return lib.ops3d_linear_forward(a["x"], a["ldx"], a["w"], a["b"], a["r"], a["ldr"], a["start"], a["count"], a["y"],
                                    a["ag"], None, 0, a["dtype"], a["act"], a["batch"], a["rows"], a["groups"], a["N"],
                                    a["K"], None)


def _backward(lib, ptr=None, **kw):
    a = dict(x=ptr, ldx=8, w=ptr, start=None, count=0, ag=None, u=ptr, ldu=8, gx=ptr, gw=ptr, gb=ptr, ws=None, ws_bytes=0,
             dtype=2, batch=1, rows=4, groups=1, N=8, K=8)
    a.update(kw)
    return lib.ops3d_linear_backward(a["x"], a["ldx"], a["w"], a["start"], a["count"], a["ag"], a["u"], a["ldu"], a["gx"],
                                     a["gw"], a["gb"], a["ws"], a["ws_bytes"], a["dtype"], a["batch"], a["rows"],
                                     a["groups"], a["N"], a["K"], None)


def test_c_refusals_before_device_work(lib):
    p = ctypes.c_void_p(256)   # a stand-in: every call here is refused before any launch

    def refused(call, text, **kw):
        assert call(lib, p, **kw) == 1
        assert text in lib.ops3d_fda_last_error().decode(), lib.ops3d_fda_last_error()

    for call in (_forward, _backward):
        refused(call, "unsupported dtype code 7", dtype=7)
        refused(call, "rows", rows=-1)
        refused(call, "rows", batch=-1)
        refused(call, "rows", batch=1 << 16, rows=1 << 16)
        refused(call, "out_features", N=0)
        refused(call, "out_features", K=(1 << 24) + 1)
        refused(call, "groups must be in 1..4096", groups=0)
        refused(call, "groups must be in 1..4096", groups=4097, start=p, count=4097)
        refused(call, "group_start is NULL", groups=2)
        refused(call, "group_start must have", groups=2, start=p, count=4)
        refused(call, "8-byte aligned", groups=2, start=ctypes.c_void_p(260), count=2)
        refused(call, "too many groups", groups=4096, start=p, count=4096, batch=1 << 20, rows=1)
        refused(call, "must not be negative", ldx=-1)
        refused(call, "NULL", w=None)
        refused(call, "aligned to their element size", w=ctypes.c_void_p(257))
    refused(_forward, "unknown activation 5", act=5)
    refused(_forward, "act_grad must be NULL", ag=p)
    refused(_forward, "NULL", y=None)
    refused(_backward, "NULL", x=None)
    refused(_backward, "NULL", u=None)
    need = lib.ops3d_linear_backward_workspace_bytes(2, 1, 100000, 1, 256, 256, 0, 0)
    assert need > 0 and need % 256 == 0
    refused(_backward, "workspace too small", rows=100000, N=256, K=256)
    refused(_backward, "workspace too small", rows=100000, N=256, K=256, ws=p, ws_bytes=need - 1)
    refused(_backward, "256-byte aligned", rows=100000, N=256, K=256, ws=ctypes.c_void_p(264), ws_bytes=need)
    # nothing to do: no pointer is touched
    assert _forward(lib, rows=0) == 0 and _forward(lib, batch=0) == 0


def test_workspace_sizes(lib):
    def f(*args, act=0):
        return lib.ops3d_linear_backward_workspace_bytes(*args, act)

    assert f(2, 1, 4, 1, 8, 8, 0, act=1) == 256            # dz
    assert f(2, 1, 4, 1, 8, 8, 0) == 0                     # one chunk: results are written at once
    assert f(2, 1, 0, 1, 8, 8, 0) == 0 and f(9, 1, 4, 1, 8, 8, 0) == 0 and f(2, 1, 4, 2, 8, 8, 0) == 0
    assert f(2, 1, 16384, 64, 1024, 512, 1) == 0           # as many groups as chunks are wanted
    assert f(2, 2, 4096, 64, 256, 256, 1) > 0              # two items share the groups' gradients
    # the partial sums of a training step stay small beside its tensors
    assert f(2, 1, 598016, 1, 256, 256, 0) < 64 << 20


def test_workspace_of_many_items(lib):
    """Partial sums follow the blocks that fill the device, not items times groups."""
    f = lib.ops3d_linear_backward_workspace_bytes
    assert f(2, 64, 512, 128, 4096, 1024, 1, 0) == 0
    assert f(2, 64, 512, 16, 1024, 1024, 1, 0) < 512 << 20
    assert f(0, 1000, 50, 4, 256, 256, 1, 0) < 64 << 20
    # 4096 groups and a million rows: below the weights' own gradients, held in fp32
    assert f(1, 512, 2048, 4096, 256, 256, 1, 0) <= 4096 * 256 * 256 * 4


def test_module_signatures_cpu():
    m = FlashDeformAttn3D(32, 4, 2, 4, level_value_proj=True)
    assert isinstance(m.value_proj, GroupedLinear) and m.value_proj.weight.shape == (2, 32, 32)
    assert sorted(k for k in m.state_dict() if k.startswith("value_proj")) == ["value_proj.bias", "value_proj.weight"]
    plain = FlashDeformAttn3D(32, 4, 2, 4)
    assert isinstance(plain.value_proj, torch.nn.Linear)
    assert GroupedLinear(3, 4, 5, bias=False).bias is None


# ---------------------------------------------------------------------------- GPU: plain product


SHAPES = [(1, 1, 1), (1, 256, 256), (2, 7, 3), (7, 40, 130), (15, 33, 17), (16, 64, 64), (17, 8, 16), (31, 250, 129),
          (33, 2048, 40), (50, 2500, 70), (64, 129, 65), (65, 64, 64), (127, 250, 333), (129, 63, 200), (400, 256, 1024),
          (1000, 72, 8)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,K,N", SHAPES)
def test_linear_sizes(gpu_device, rows, K, N, dtype):
    log(f"[case] linear {rows}x{K}->{N} {dtype}")
    act = list(ACTIVATIONS)[(rows + K + N) % 5]
    linear_case(rows, K, N, DTYPES[dtype], act, with_bias=rows % 2 == 0 or N > 16, with_residual=K % 2 == 0)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("activation", list(ACTIVATIONS))
@pytest.mark.parametrize("rows", [9, 300])
def test_linear_activations(gpu_device, rows, activation, dtype):
    log(f"[case] linear {rows}x96->80 {activation} {dtype}")
    linear_case(rows, 96, 80, DTYPES[dtype], activation, with_residual=True)


@gpu
@pytest.mark.parametrize("dtype,rows,K,N", [("bf16", 40000, 256, 256), ("fp16", 20011, 100, 520), ("fp32", 20011, 90, 130),
                                            ("bf16", 1024, 2048, 2048), ("fp32", 1030, 1000, 1030),
                                            ("bf16", 9000, 24, 40)])
def test_linear_large(gpu_device, dtype, rows, K, N):
    """The larger tiles, chunks of rows that are joined, and their edges."""
    log(f"[case] linear large {rows}x{K}->{N} {dtype}")
    linear_case(rows, K, N, DTYPES[dtype], "silu", with_residual=True)
    linear_case(rows, K, N, DTYPES[dtype], None)


@gpu
@pytest.mark.parametrize("dtype,rows,K,N,act", [("bf16", 65607, 256, 504, "relu"), ("fp16", 70001, 128, 512, None),
                                                ("bf16", 66001, 512, 128, None), ("fp16", 140001, 256, 256, None),
                                                ("bf16", 140033, 256, 256, "silu")])
def test_linear_many_rows(gpu_device, dtype, rows, K, N, act):
    """Short sums over many rows, of the forward and of the input gradient; last tiles and slices that overlap."""
    log(f"[case] linear many rows {rows}x{K}->{N} {dtype} {act}")
    linear_case(rows, K, N, DTYPES[dtype], act, with_residual=True)
    linear_case(rows, K, N, DTYPES[dtype], act, train=False, seed=1)


@gpu
@pytest.mark.parametrize("K,N,act", [(256, 1024, "relu"), (1024, 256, None), (128, 1016, None)])
def test_grouped_many_rows(gpu_device, K, N, act):
    """The same in groups: rows of none, a group shorter than a tile, two items."""
    log(f"[case] grouped many rows {K}->{N} {act}")
    grouped_case(100003, [70, 100, 60000, 99990], 3, K, N, torch.bfloat16, act, batch=2, with_residual=True)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,K,N", [(1, 1856, 3301), (70, 3000, 100), (130, 1111, 72), (300, 640, 1100), (65, 129, 2000)])
def test_linear_long_sums(gpu_device, rows, K, N, dtype):
    """Sums that are cut into parts, of the forward or of the input gradient, and joined."""
    log(f"[case] linear long sums {rows}x{K}->{N} {dtype}")
    linear_case(rows, K, N, DTYPES[dtype], "gelu", with_residual=True)
    linear_case(rows, K, N, DTYPES[dtype], None, with_bias=False)


@gpu
@pytest.mark.parametrize("want", ["x", "w", "b", "r", "xb"])
def test_linear_some_gradients(gpu_device, want):
    """Only the gradients that are asked for, each as it is with the others."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    t = {"x": make(gen, (70, 48), torch.float32), "w": make(gen, (56, 48), torch.float32), "b": make(gen, (56,), torch.float32),
         "r": make(gen, (70, 56), torch.float32)}
    u = make(gen, (70, 56), torch.float32)
    log(f"[case] gradients of {want}")
    full = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    every = dict(zip(full, torch.autograd.grad(fused_linear(full["x"], full["w"], full["b"], "gelu", full["r"]),
                                               list(full.values()), u)))
    some = {k: v.clone().requires_grad_(k in want) for k, v in t.items()}
    got = torch.autograd.grad(fused_linear(some["x"], some["w"], some["b"], "gelu", some["r"]),
                              [some[k] for k in want], u)
    for k, g in zip(want, got):
        assert torch.equal(g, every[k]), k


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [5, 90])
def test_linear_strides(gpu_device, rows, dtype):
    """Parts of wider rows at odd offsets, extra axes, a transposed weight, expanded and negated tensors."""
    dt = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(5)
    log(f"[case] strides {rows} {dtype}")
    wide = make(gen, (rows, 100), dt)
    w, b, r = make(gen, (24, 33), dt, 0.2), make(gen, (24,), dt), make(gen, (rows, 60), dt)
    x, res = wide[:, 5:38], r[:, 3:27]
    base = fused_linear(x.contiguous(), w, b, "silu", res.contiguous())
    compare(x, w, b, res, "silu", torch.zeros(rows, dtype=torch.int64), {"y": base})
    assert torch.equal(fused_linear(x, w, b, "silu", res), base)
    assert torch.equal(fused_linear(x, w.t().contiguous().t(), b, "silu", res), base)
    assert torch.equal(fused_linear(torch._neg_view(-x), torch._neg_view(-w), torch._neg_view(-b), "silu",
                                    torch._neg_view(-res)), base)
    assert torch.equal(fused_linear(x.t().contiguous().t(), w, b, "silu", res), base)
    assert torch.equal(fused_linear(x.reshape(1, rows, 1, 33), w, b, "silu", res[None, :, None]), base[None, :, None])
    one = fused_linear(x[:1].expand(rows, 33), w, b, "silu", res[:1].expand(rows, 24))
    assert torch.equal(one, base[:1].expand(rows, 24))
    alone = fused_linear(x[0], w, b, "silu", res[0])
    assert alone.shape == (24,)
    compare(x[:1], w, b, res[:1], "silu", torch.zeros(1, dtype=torch.int64), {"y": alone})
    # an expanded gradient (of a sum) and a strided one
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = fused_linear(xl, wl, b, "silu")
    u = make(gen, (1, 24), dt).expand(rows, 24)
    for g in (u, make(gen, (rows, 24, 2), dt)[..., 0]):
        got = torch.autograd.grad(y, (xl, wl), g, retain_graph=True)
        want = torch.autograd.grad(y, (xl, wl), g.contiguous(), retain_graph=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_linear_shared_and_broadcast_inputs(gpu_device):
    """One tensor as x and residual, an expanded residual, a weight used twice: gradients add up."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w = make(gen, (40, 32), torch.float32).requires_grad_(True), make(gen, (32, 32), torch.float32, 0.2).requires_grad_(True)
    r = make(gen, (1, 32), torch.float32).requires_grad_(True)
    u = make(gen, (40, 32), torch.float32)
    log("[case] shared inputs")
    y = fused_linear(fused_linear(x, w, None, "gelu", x), w, None, None, r.expand(40, 32))
    got = torch.autograd.grad(y, (x, w, r), u)
    xd, wd, rd = (t.detach().double().requires_grad_(True) for t in (x, w, r))
    h = torch.nn.functional.gelu(xd @ wd.t()) + xd
    want = torch.autograd.grad(h @ wd.t() + rd, (xd, wd, rd), u.double())
    for g, e in zip(got, want):
        # fp32 sums of up to 64 terms in two layers, values of order 10: 2^-24 * 64 * 4 of the largest
        assert (g.double() - e).abs().max() <= 2.0 ** -24 * 256 * e.abs().max()


@gpu
@pytest.mark.parametrize("rows", [0, 1])
def test_linear_no_rows(gpu_device, rows):
    x = torch.zeros(rows, 8, device="cuda", requires_grad=True)
    w, b = (torch.ones(s, device="cuda", requires_grad=True) for s in ((4, 8), (4,)))
    log(f"[case] {rows} rows")
    y = fused_linear(x, w, b, "relu")
    grads = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == (rows, 4) and grads[0].shape == (rows, 8)
    assert torch.equal(grads[1], torch.zeros(4, 8, device="cuda"))
    assert torch.equal(grads[2], torch.full((4,), float(rows), device="cuda"))
    assert fused_linear(x.detach()[None].expand(3, rows, 8), w, b).shape == (3, rows, 4)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [20, 200])
def test_linear_nan_and_infinity(gpu_device, rows, dtype):
    """A row's NaN or infinity stays in its row of y and dx; NaN gradients are kept behind activations."""
    dt = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(7)
    x, w = make(gen, (rows, 40), dt), make(gen, (24, 40), dt, 0.2)
    x[3, 7], x[9, 0] = float("nan"), float("inf")
    log(f"[case] nan rows {rows} {dtype}")
    for act in ACTIVATIONS:
        xl = x.detach().requires_grad_(True)
        y = fused_linear(xl, w, None, act)
        clean = fused_linear(torch.where(torch.isfinite(x), x, torch.zeros_like(x)), w, None, act)
        keep = [i for i in range(rows) if i not in (3, 9)]
        assert torch.equal(y[keep], clean[keep])
        assert torch.isnan(y[3]).all()
        assert not torch.isfinite(y[9]).all()
        (dx,) = torch.autograd.grad(y, xl, torch.ones_like(y))
        assert torch.isfinite(dx[keep]).all()
        if act not in (None, "relu"):
            assert torch.isnan(dx[3]).all()
    big = torch.full((4, 8), 300.0, dtype=dt, device="cuda")
    y = fused_linear(big, big)
    assert torch.equal(y, torch.full((4, 4), 8 * 300.0 * 300.0, device="cuda").to(dt))   # fp16: infinity


@gpu
def test_linear_extreme_activations(gpu_device):
    """Activations and their derivatives far from zero: the limits, no NaN."""
    z = torch.tensor([-1e30, -3e4, -100.0, -20.0, 20.0, 100.0, 3e4, 1e30], device="cuda")
    eye = torch.ones(1, 1, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        for act in ("relu", "gelu", "gelu_tanh", "silu"):
            log(f"[case] extremes {act} {dt}")
            x = z.to(dt)[:, None].requires_grad_(True)
            y = fused_linear(x, eye.to(dt), None, act)
            (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
            torch.testing.assert_close(y, torch.where(x > 0, x, torch.zeros_like(x)), rtol=0, atol=1e-6)
            torch.testing.assert_close(dx, (x > 0).to(dt), rtol=0, atol=1e-6)
            top = torch.tensor([[float("inf")], [float("nan")]], dtype=dt, device="cuda")
            y = fused_linear(top, eye.to(dt), None, act)
            assert torch.isposinf(y[0]).all() and torch.isnan(y[1]).all()


@gpu
def test_linear_offsets_over_32_bits(gpu_device):
    """More than 2^31 elements of x and y: rows at the far end."""
    rows, K, N = (1 << 23) + 77, 264, 256
    log("[case] 2^31 elements")
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(8)
    w = make(gen, (N, K), torch.bfloat16, K ** -0.5)
    tail = 500
    x[-tail:] = make(gen, (tail, K), torch.bfloat16)
    assert x.numel() > 1 << 31
    with torch.no_grad():
        y = fused_linear(x, w, None, "gelu")
        near = fused_linear(x[-tail:], w, None, "gelu")
    check("y", y[-tail:], ref.run(x[-tail:], w[None], None, None, "gelu", torch.zeros(tail, dtype=torch.int64))["y"])
    assert not y[: 1 << 20].any()
    assert near.shape == (tail, N)
    del y
    u = torch.zeros(rows, N, dtype=torch.bfloat16, device="cuda")
    u[-tail:] = make(gen, (tail, N), torch.bfloat16)
    wl = w.detach().requires_grad_(True)
    xl = x.requires_grad_(True)
    dx, dw = torch.autograd.grad(fused_linear(xl, wl), (xl, wl), u)
    want = ref.run(x.detach()[-tail:], w[None], None, None, None, torch.zeros(tail, dtype=torch.int64), u[-tail:])
    check("dx", dx[-tail:], want["dx"])
    check("dw", dw[None], want["dw"])
    assert not dx[: 1 << 20].any()


# ---------------------------------------------------------------------------- GPU: groups


GROUPS = [
    # S, group_start, groups, batch
    (1, [0], 1, 0),
    (20, [0, 3, 3, 17], 4, 0),                      # an empty group, the last to the end
    (20, [2, 3, 9, 12], 3, 0),                      # rows of no group on both sides
    (300, [0, 100, 100, 250, 250], 4, 2),           # E + 1 entries, an empty group, rows behind the last, two items
    (600, [0, 512], 2, 3),                          # levels
    (700, [-5, 130, 90, 10000, 650], 5, 2),         # not monotone, out of range
    (50, [50, 50, 50], 2, 2),                       # no group has a row
    (900, [i * 9 for i in range(101)], 100, 0),     # more than 64 groups, one ragged tile each
    (900, [min(i * i // 10, 880) for i in range(130)], 130, 2),
    (40000, [0, 34990, 39400], 3, 0),
    (30000, [100, 25000, 25001, 29999], 3, 2),
    (150, [3, 70, 70, 149], 3, 2),                  # with 1500 features: sums in parts
    (9, [0, 2, 2, 7], 4, 700),                      # chunks of several items
    (70, [2, 68, 69], 3, 400),                      # the same, a group of more rows than a chunk's, rows of no group
    (33, [i // 2 for i in range(60)], 60, 150),
]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_grouped_sizes(gpu_device, case, dtype):
    S, start, groups, batch = GROUPS[case]
    K, N = (1500, 900) if case == 11 else [(40, 24), (64, 64), (33, 70), (136, 129)][case % 4]
    act = list(ACTIVATIONS)[case % 5]
    log(f"[case] grouped {case}: {S} rows, {groups} groups, batch {batch}, {K}->{N} {act} {dtype}")
    grouped_case(S, start, groups, K, N, DTYPES[dtype], act, batch, with_bias=case != 5, with_residual=case % 2 == 0)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K,N", [(512, 512), (515, 513)])
def test_grouped_many_items(gpu_device, K, N, dtype):
    """Weights' gradients in wide tiles, a chunk taking the same rows of several items."""
    log(f"[case] grouped many items {K}->{N} {dtype}")
    start = [0, 1, 1, 2, 3, 5, 8, 13, 21, 30, 31, 32, 33, 34, 35, 36, 37, 40, 50, 55]
    grouped_case(60, start, 20, K, N, DTYPES[dtype], "silu", batch=40)


@gpu
@pytest.mark.parametrize("K,N,act", [(515, 1001, None), (1001, 515, "gelu"), (1024, 1032, "relu")])
def test_grouped_large(gpu_device, K, N, act):
    """The widest tiles in groups that end inside them, unaligned and aligned."""
    log(f"[case] grouped large {K}->{N} {act}")
    grouped_case(12300, [3, 700, 6007], 3, K, N, torch.bfloat16, act, batch=2, with_residual=True)


@gpu
def test_linear_leading_axes(gpu_device):
    """One row without a leading axis and rows under three give the same bits as a matrix."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    x, w, b = make(gen, (2, 3, 4, 40), torch.float16), make(gen, (24, 40), torch.float16, 0.2), make(gen, (24,), torch.float16)
    r, u = make(gen, (2, 3, 4, 24), torch.float16), make(gen, (2, 3, 4, 24), torch.float16)
    log("[case] linear leading axes")

    def step(x, r, u):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y = fused_linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
        return (y.detach(), *torch.autograd.grad(y, leaves, u))

    want, four = step(x.reshape(24, 40), r.reshape(24, 24), u.reshape(24, 24)), step(x, r, u)
    assert four[0].shape == (2, 3, 4, 24) and four[1].shape == x.shape
    assert all(torch.equal(a.reshape(e.shape), e) for a, e in zip(four, want))
    one, row = step(x[0, 0, 0], r[0, 0, 0], u[0, 0, 0]), step(x[0, 0, :1], r[0, 0, :1], u[0, 0, :1])
    assert one[0].shape == (24,) and one[1].shape == (40,)
    assert all(torch.equal(a.reshape(e.shape), e) for a, e in zip(one, row))


@gpu
@pytest.mark.parametrize("dtype,rows,K,N,act", [("bf16", 4100, 1096, 3336, "silu"), ("fp16", 12290, 1024, 1032, None),
                                                ("bf16", 4097, 2056, 4096, "gelu")])
def test_linear_wide_long(gpu_device, dtype, rows, K, N, act):
    """Wide tiles of long sums: rows, columns and a stage that end inside them."""
    log(f"[case] linear wide {rows}x{K}->{N} {dtype} {act}")
    linear_case(rows, K, N, DTYPES[dtype], act, with_residual=True)


@gpu
def test_grouped_equals_plain(gpu_device):
    """One group of all rows gives the plain product's bits; equal weights give one product's rows."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    x, w, b = make(gen, (500, 64), torch.bfloat16), make(gen, (96, 64), torch.bfloat16, 0.1), make(gen, (96,), torch.bfloat16)
    start = torch.tensor([0, 77, 77, 300], device="cuda")
    log("[case] grouped equals plain")
    y = fused_linear(x, w, b, "gelu")
    assert torch.equal(grouped_linear(x, w[None], start[:1], b[None], "gelu"), y)
    assert torch.equal(grouped_linear(x, w.expand(4, 96, 64), start, b.expand(4, 96), "gelu"), y)


@gpu
def test_grouped_rows_outside_are_not_read(gpu_device):
    """NaN in rows of no group reach no output."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    x, w = make(gen, (200, 32), torch.float32), make(gen, (2, 48, 32), torch.float32)
    u, r = make(gen, (200, 48), torch.float32), make(gen, (200, 48), torch.float32)
    for t in (x, u, r):
        t[:10], t[150:] = float("nan"), float("nan")
    start = torch.tensor([10, 60, 150], device="cuda")
    log("[case] NaN outside")
    for act in (None, "silu"):
        xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = grouped_linear(xl, wl, start, None, act, r)
        dx, dw = torch.autograd.grad(y, (xl, wl), u)
        for t in (y, dx, dw):
            assert torch.isfinite(t).all()
        assert not y[:10].any() and not y[150:].any() and not dx[:10].any() and not dx[150:].any()


@gpu
def test_grouped_no_rows(gpu_device):
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w, b = (torch.ones(s, device="cuda", requires_grad=True) for s in ((3, 4, 8), (3, 4)))
    log("[case] grouped, no rows")
    for lead in ((0,), (2, 0), (0, 5)):
        xl = torch.zeros(*lead, 8, device="cuda", requires_grad=True)
        y = grouped_linear(xl, w, torch.zeros(3, dtype=torch.int64, device="cuda"), b)
        grads = torch.autograd.grad(y, (xl, w, b), torch.ones_like(y))
        assert y.shape == (*lead, 4) and grads[0].shape == xl.shape
        assert not grads[1].any() and not grads[2].any()


# ---------------------------------------------------------------------------- GPU: how it is called


@gpu
def test_refusals(gpu_device):
    x, w, b = torch.zeros(6, 8, device="cuda"), torch.zeros(4, 8, device="cuda"), torch.zeros(4, device="cuda")
    start = torch.zeros(1, dtype=torch.int64, device="cuda")
    log("[case] refusals")

    def refused(error, text, f, *args, **kw):
        with pytest.raises(error, match=text):
            f(*args, **kw)

    refused(ValueError, "features", fused_linear, x[:, :7], w)
    refused(ValueError, "weight must be", fused_linear, x, w[None])
    refused(ValueError, "weight must be", grouped_linear, x, w, start)
    refused(ValueError, "bias must be", fused_linear, x, w, b[:3])
    refused(ValueError, "bias must be", grouped_linear, x, w[None], start, b)
    refused(ValueError, "residual must have", fused_linear, x, w, b, None, b)
    refused(ValueError, "dtype differs", fused_linear, x, w.half())
    refused(ValueError, "dtype differs", fused_linear, x, w, b.bfloat16())
    refused(ValueError, "unsupported", fused_linear, x.double(), w.double())
    refused(RuntimeError, "CPU", fused_linear, x, w.cpu())
    refused(RuntimeError, "CPU", grouped_linear, x, w[None], start.cpu())
    refused(ValueError, "int64", grouped_linear, x, w[None], start.int())
    refused(ValueError, "int64", grouped_linear, x, w[None], start[None])
    refused(ValueError, "int64", grouped_linear, x, w.expand(2, 4, 8), torch.zeros(4, dtype=torch.int64, device="cuda")[::2])
    refused(ValueError, "entries", grouped_linear, x, w[None], torch.zeros(3, dtype=torch.int64, device="cuda"))
    refused(ValueError, "x must be", grouped_linear, x[None, None], w[None], start)
    refused(ValueError, "out_features", fused_linear, x[:, :0], w[:, :0])
    refused(ValueError, "out_features", fused_linear, x, w[:0])
    refused(ValueError, "groups must be", grouped_linear, x, w.expand(5000, 4, 8), torch.zeros(5000, dtype=torch.int64, device="cuda"))
    refused(ValueError, "dense", fused_linear, x.to_sparse(), w)
    y = fused_linear(x.requires_grad_(True), w)
    u = torch.ones_like(y, requires_grad=True)
    (g,) = torch.autograd.grad(y, x, u, create_graph=True)
    refused(RuntimeError, "differentiate twice", g.sum().backward)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ctypes_binding_gives_the_same(gpu_device, dtype):
    """The binding without the extension module: the same bits."""
    C, N = _extension._C, type(_extension._C)
    bare = N(C._lib, C.__file__)   # without the extension module's functions
    gen = torch.Generator(device="cuda").manual_seed(13)
    dt = DTYPES[dtype]
    x, w, b = make(gen, (2, 300, 40), dt), make(gen, (3, 24, 40), dt), make(gen, (3, 24), dt)
    r, u = make(gen, (2, 300, 24), dt), make(gen, (2, 300, 24), dt)
    start = torch.tensor([5, 100, 120], device="cuda")
    log(f"[case] ctypes {dtype}")
    for args in ((x, w, b, r, start), (x, w[0], b[0], r, None)):
        got, want = N.linear_forward(C, *args, 2, True), C.linear_forward(*args, 2, True)
        assert torch.equal(got[0], want[0])
        if args[4] is None:
            assert torch.equal(got[1], want[1])
        back = (x, args[1], args[4], want[1], u, 40, 3 if args[4] is not None else 0, True, True)
        for g, e in zip(N.linear_backward(C, *back), C.linear_backward(*back)):
            assert torch.equal(g, e)
        grads = []
        for f in (C.linear, lambda *a: N.linear(bare, *a)):
            leaves = [t.detach().requires_grad_(True) for t in args[:4]]
            y = f(*leaves, args[4], 2)
            assert torch.equal(y, want[0])
            grads.append(torch.autograd.grad(y, leaves, u.clone().requires_grad_(True), create_graph=True))
            with pytest.raises(RuntimeError, match="differentiate twice"):
                grads[-1][0].sum().backward()
        for a, e in zip(*grads):
            assert torch.equal(a, e)


@gpu
def test_repeatable_and_two_streams(gpu_device):
    """The same bits every time, also from two streams at once and on a stream other than the tensors' own."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    x, w, u = make(gen, (20000, 128), torch.bfloat16), make(gen, (3, 192, 128), torch.bfloat16, 0.1), make(gen, (20000, 192), torch.bfloat16)
    start = torch.tensor([0, 15000, 19000], device="cuda")
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)

    def step():
        y = grouped_linear(xl, wl, start, None, "gelu")
        return (y.detach(), *torch.autograd.grad(y, (xl, wl), u))

    log("[case] streams")
    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@gpu
def test_captured_and_replayed(gpu_device):
    """Forward and backward in a graph, replayed with new inputs (and other groups) between eager calls."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    x, w, b = make(gen, (2000, 64), torch.bfloat16), make(gen, (3, 96, 64), torch.bfloat16, 0.1), make(gen, (3, 96), torch.bfloat16)
    u, r, start = make(gen, (2000, 96), torch.bfloat16), make(gen, (2000, 96), torch.bfloat16), torch.tensor([0, 900, 1500], device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]

    def step():
        y = grouped_linear(x, w, start, b, "silu", r)
        return (y.detach(), *torch.autograd.grad(y, leaves, u))

    log("[case] capture")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    with torch.no_grad():
        for i in range(4):
            for t in (x, w, u, r):
                t.copy_(make(gen, t.shape, t.dtype))
            start.copy_(torch.tensor([[0, 900, 1500], [10, 10, 1999], [0, 0, 0], [1999, 2000, 2000]][i]))
            g.replay()
            torch.cuda.synchronize()
            with torch.enable_grad():
                want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(outs, want)), i


@gpu
@pytest.mark.parametrize("activation", list(ACTIVATIONS))
def test_gradients_against_differences(gpu_device, activation):
    """Directional derivatives of the fp32 operator: central differences of step h are off by
    h^2 / 6 |f'''| and by the sums' rounding over h."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    x, w, b = make(gen, (60, 20), torch.float32), make(gen, (2, 12, 20), torch.float32, 0.2), make(gen, (2, 12), torch.float32)
    u, start = make(gen, (60, 12), torch.float32), torch.tensor([0, 35], device="cuda")
    log(f"[case] differences {activation}")

    def f(args):
        with torch.no_grad():
            return (grouped_linear(args[0], args[1], start, args[2], activation).double() * u.double()).sum()

    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(grouped_linear(x, w, start, b, activation), leaves, u)
    own = ref.run(x.detach(), w.detach(), b.detach(), None, activation, ref.group_of_rows(60, [0, 35], 2), u)
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        d = make(gen, leaves[i].shape, torch.float32)
        plus, minus = [t.detach() for t in leaves], [t.detach() for t in leaves]
        plus[i], minus[i] = plus[i] + h * d, minus[i] - h * d
        slope = (f(plus) - f(minus)) / (2 * h)
        dz = (f_z(plus, start) - f_z(minus, start)).abs() / (2 * h)      # |z'| per output
        # |f'''| <= 3 for the smooth activations; relu: outputs whose z changes sign within the step
        # give anything from 0 to |z'|
        if activation == "relu":
            jump = (f_z(plus, start) * f_z(minus, start) <= 0) & (dz > 0)
            bound = (u.double().abs() * dz * jump).sum()
        else:
            bound = 0 if activation is None else (u.double().abs() * 3 * dz ** 3).sum() * h * h / 6
        size = (u.double().abs() * (f_z([t.abs() for t in plus], start) + 1)).sum()
        bound = bound + 2 * 24 * 2.0 ** -24 * size / h + (own[("dx", "dw", "db")[i]][1] * d.abs()).sum()
        assert abs((g.double() * d.double()).sum() - slope) <= bound, i


def f_z(args, start):
    """z of the two groups in 64 bits."""
    x, w, b = (t.double() for t in args)
    cut = int(start[1])
    return torch.cat([x[:cut] @ w[0].t() + b[0], x[cut:] @ w[1].t() + b[1]])


@gpu
def test_autocast(gpu_device):
    """As torch's linear under autocast: the product in the autocast type; a wider residual keeps its own."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    x, w, b, r = (make(gen, s, torch.float32) for s in ((50, 32), (24, 32), (24,), (50, 24)))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    log("[case] autocast")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = fused_linear(x, w, b, "gelu")
        y2 = fused_linear(x, w, b, "gelu", r)
        y3 = fused_linear(x, w, b, "gelu", r.bfloat16())
    want = fused_linear(x.bfloat16(), w.bfloat16(), b.bfloat16(), "gelu")
    assert y.dtype == torch.bfloat16 and torch.equal(y, want)
    assert y2.dtype == torch.float32 and torch.equal(y2, want + r)
    assert y3.dtype == torch.bfloat16
    grads = torch.autograd.grad(y2.sum(), leaves)
    assert all(g.dtype == torch.float32 for g in grads)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_layer(gpu_device, dtype):
    """An encoder layer as it is used: attention with a projection per level and the residual in the
    output projection, then a feed-forward of two fused layers; output and (fp32, where both layers
    sample at the same bits of the same projection) gradients against torch's linear layers in fp32."""
    dt = DTYPES[dtype]
    torch.manual_seed(0)
    shapes, C, G, L, K, B = ((4, 8, 16), (2, 4, 8)), 64, 4, 2, 4, 2
    st, lsi = level_meta(shapes, gpu_device)
    S = sum(d * h * w for d, h, w in shapes)
    log(f"[case] layer {dtype}")
    m = FlashDeformAttn3D(C, G, L, K, level_value_proj=True).to(gpu_device)
    with torch.no_grad():
        m.value_proj.bias.normal_(0, 0.1)
        m.sampling.weight.normal_(0, 0.02)
    w1, b1, w2, b2 = (torch.randn(s, device=gpu_device) * 0.1 for s in ((4 * C, C), (4 * C,), (C, 4 * C), (C,)))
    x = torch.randn(B, S, C, device=gpu_device)
    refp = torch.rand(B, S, 1, 3, device=gpu_device)
    u = torch.randn(B, S, C, device=gpu_device)
    # the parameters as the type holds them, in both layers
    with torch.no_grad():
        for t in (*m.parameters(), w1, b1, w2, b2, x, u):
            t.copy_(t.to(dt).float())

    def layer(fused):
        cast = (lambda t: t.detach().to(dt).requires_grad_(True)) if fused else (lambda t: t.detach().clone().requires_grad_(True))
        p = {k: cast(v) for k, v in m.named_parameters()}
        f = {k: cast(v) for k, v in (("w1", w1), ("b1", b1), ("w2", w2), ("b2", b2), ("x", x))}
        xs = f["x"]
        if fused:
            h = torch.func.functional_call(m, p, (xs, refp, xs, st, lsi), {"residual": xs})
            y = fused_linear(fused_linear(h, f["w1"], f["b1"], "gelu"), f["w2"], f["b2"], residual=h)
        else:
            lin = torch.nn.functional.linear
            cut = int(lsi[1])
            v = torch.cat([lin(xs[:, :cut], p["value_proj.weight"][0], p["value_proj.bias"][0]),
                           lin(xs[:, cut:], p["value_proj.weight"][1], p["value_proj.bias"][1])], 1)
            oa = lin(xs, p["sampling.weight"], p["sampling.bias"])
            a = FlashDeformAttnFromOffsets.apply(v.view(B, S, G, C // G), st, lsi, oa.view(B, S, G, -1), refp, 64, K)
            h = lin(a, p["output_proj.weight"], p["output_proj.bias"]) + xs
            y = lin(torch.nn.functional.gelu(lin(h, f["w1"], f["b1"])), f["w2"], f["b2"]) + h
        leaves = {**p, **f}
        return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), u.to(y.dtype))))

    y, grads = layer(True)
    want, gwant = layer(False)
    # norm-wise: fp32 differs by its sums' order over five products; bf16 by up to 2^-8 at each of a
    # dozen steps, and by sampling positions (of up to 4 voxels: off by 2^-7) times a voxel's value
    # difference.  Gradients of positions jump between voxels: no bf16 tolerance for them.
    tol = 1e-5 if dtype == "fp32" else 3e-2
    for name, a, e in [("y", y, want)] + [(k, grads[k], gwant[k]) for k in gwant if dtype == "fp32"]:
        err = (a.detach().double() - e.detach().double()).norm() / e.detach().double().norm()
        assert err <= (tol if not name.startswith("sampling") else 4 * tol), f"{name}: {err:.2e}"
