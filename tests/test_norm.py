"""layer_norm against its float64 restatement (oracle/norm.py) within componentwise bounds derived there,
and its refusals.  CPU: the restatement itself, refusals, sizes.  GPU: everything that computes."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import norm as ref
from ops3d_amd import _extension, layer_norm

gpu = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def make(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale + shift).to(dtype)


def check(name, got, want):
    value, bound = want
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - value).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{name}: {int((over > 0).sum())}/{over.numel()} outside the bound, by at most {worst:.3e}"


def compare(x, w, b, u, eps=1e-5, norm=layer_norm):
    """Forward and backward of x [..., C], all gradients."""
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xl, wl, bl = next(it), next(it) if w is not None else None, next(it) if b is not None else None
    y = norm(xl, wl, bl, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, u)
    C = x.shape[-1]
    vector = (w if w is not None else b).dtype if w is not None or b is not None else None
    want = ref.run(x.reshape(-1, C), w, b, eps, u.reshape(-1, C), vector_dtype=vector)
    check("y", y, want["y"])
    for name, t, g in zip(("dx", *(n for n, v in (("dw", w), ("db", b)) if v is not None)), leaves, grads):
        assert g.dtype == t.dtype
        check(name, g, want[name])
    with torch.no_grad():   # the form without statistics
        assert torch.equal(norm(x, w, b, eps), y)
    return y, grads


# ---------------------------------------------------------------------------- CPU


def test_restatement_against_torch_and_differences():
    gen = torch.Generator().manual_seed(0)
    x, w, b, u = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((5, 7), (7,), (7,), (5, 7)))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (7,), leaves[1], leaves[2], 1e-3)
    grads = torch.autograd.grad(y, leaves, u)
    got = ref.run(x, w, b, 1e-3, u, dtype=torch.float32, vector_dtype=torch.float32)
    for name, want in zip(("y", "dx", "dw", "db"), (y, *grads)):
        assert torch.allclose(got[name][0], want, rtol=1e-12, atol=1e-12)
    step = 1e-6
    for i, j in ((0, 0), (3, 5)):
        d = torch.zeros_like(x)
        d[i, j] = step
        up, down = (ref.run(x + s * d, w, b, 1e-3, dtype=torch.float32)["y"][0] for s in (1, -1))
        assert abs(((up - down) * u).sum() / (2 * step) - got["dx"][0][i, j]) < 1e-6


def test_refusals_on_the_cpu():
    x = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="CPU"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="CPU"):
        layer_norm(x.requires_grad_(), torch.ones(4), torch.zeros(4))


@pytest.fixture(scope="module")
def lib():
    import os

    if not os.path.exists(_extension.LIB_PATH):
        pytest.skip("libops3d_fda.so not built")
    return _extension.load_library()


def test_c_refusals_before_device_work(lib):
    def forward(x=16, ld=4, w=16, b=16, y=16, stats=None, dtype=0, wdtype=0, rows=3, width=4, eps=1e-5):
        return lib.ops3d_layer_norm_forward(x, ld, w, b, y, stats, dtype, wdtype, rows, width, eps, None)

    for bad in ({"dtype": 3}, {"dtype": 1, "wdtype": 2}, {"rows": -1}, {"rows": 2 ** 41}, {"width": 0}, {"width": 2 ** 24 + 1},
                {"ld": -1}, {"eps": -1.0}, {"eps": float("nan")}, {"eps": float("inf")}, {"x": None}, {"y": None}, {"x": 18},
                {"w": 17}, {"stats": 18}):
        assert forward(**bad) == 1, bad
        assert lib.ops3d_fda_last_error()
    assert forward(rows=0) == 0

    def backward(x=16, w=16, stats=16, g=16, gx=16, gw=256, gb=256, ws=256, n=None, rows=3, width=4):
        need = lib.ops3d_layer_norm_backward_workspace_bytes(0, rows, width, int(gw is not None), int(gb is not None))
        return lib.ops3d_layer_norm_backward(x, 4, w, stats, g, 4, gx, gw, gb, ws, need if n is None else n, 0, 0, rows, width, None)

    for bad in ({"x": None}, {"stats": None}, {"g": None}, {"ws": None}, {"n": 8}, {"ws": 264}, {"gx": 17}, {"width": 0}):
        assert backward(**bad) == 1, bad
    assert backward(gx=None, gw=None, gb=None) == 0


def test_workspace_sizes(lib):
    def size(*a):
        return lib.ops3d_layer_norm_backward_workspace_bytes(*a)

    assert size(0, 0, 16, 1, 1) == 0 and size(0, 10, 16, 0, 0) == 0 and size(5, 10, 16, 1, 1) == 0
    one = size(2, 73728, 256, 1, 0)
    assert one == size(2, 73728, 256, 0, 1) == 512 * 256 * 4 and size(2, 73728, 256, 1, 1) == 2 * one


# ---------------------------------------------------------------------------- GPU

# widths of every plan: lanes, waves, blocks, longer than a block holds; odd ones and ends inside chunks
WIDTHS = [1, 2, 3, 7, 8, 9, 31, 64, 65, 100, 128, 129, 250, 256, 257, 511, 512, 515, 768, 1000, 1024, 1025, 2048, 2051, 4096,
          4101, 6000, 8192, 8193, 16390, 20011]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(gpu_device, width, dtype):
    gen = torch.Generator(device="cuda").manual_seed(width)
    dt = DTYPES[dtype]
    rows = 37 if width > 600 else 301
    compare(make(gen, (rows, width), dt, 1.3, 0.4), make(gen, (width,), dt, 0.3, 1.0), make(gen, (width,), dt, 0.3),
            make(gen, (rows, width), dt))


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,width", [(1, 256), (2, 24), (5000, 40), (70001, 256), (20003, 1000), (3001, 4101)])
def test_rows(gpu_device, rows, width, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    dt = DTYPES[dtype]
    compare(make(gen, (rows, width), dt), make(gen, (width,), dt, 0.3, 1.0), make(gen, (width,), dt), make(gen, (rows, width), dt))


@gpu
@pytest.mark.parametrize("which", ["none", "weight", "bias", "both"])
@pytest.mark.parametrize("dtype,vector", [("bf16", "fp32"), ("fp16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32")])
@pytest.mark.parametrize("width", [72, 9000])
def test_vectors(gpu_device, width, dtype, vector, which):
    gen = torch.Generator(device="cuda").manual_seed(3)
    dt, vt = DTYPES[dtype], DTYPES[vector]
    w = make(gen, (width,), vt, 0.3, 1.0) if which in ("weight", "both") else None
    b = make(gen, (width,), vt) if which in ("bias", "both") else None
    compare(make(gen, (2, 11, width), dt), w, b, make(gen, (2, 11, width), dt), eps=1e-3)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("width", [33, 256, 3001])
def test_strides(gpu_device, width, dtype):
    """Parts of wider rows, rows a row apart, repeated rows, transposed and unaligned ones."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    dt = DTYPES[dtype]
    w, b = make(gen, (width,), dt), make(gen, (width,), dt)
    wide = make(gen, (40, width + 5), dt)
    u = make(gen, (20, width), dt)
    for x in (wide[:20, 3:width + 3], wide[::2, :width], wide[:1, 1:width + 1].expand(20, width), make(gen, (width, 20), dt).t()):
        compare(x, w, b, u)
        compare(u, w, b, x)   # gradients with those strides
    strided = make(gen, (2 * width,), dt)[::2]
    compare(u, strided, strided.flip(0), u)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_far_from_zero_and_flat_rows(gpu_device, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    dt = DTYPES[dtype]
    for width in (100, 256, 5000):
        x = make(gen, (30, width), torch.float32)
        x[:10] += 2000.0
        x[10:15] = 3.0         # flat: variance 0
        x[15:20] = 0.0
        x[20:25] *= 1e-4       # below eps
        compare(x.to(dt), make(gen, (width,), dt), make(gen, (width,), dt), make(gen, (30, width), dt))
        if dtype == "fp32":
            compare(x, None, None, make(gen, (30, width), dt), eps=1e-12)


@gpu
def test_not_finite_rows_stay_their_own(gpu_device):
    x = torch.randn(40, 300, device="cuda")
    x[3, 7], x[9, 2] = float("nan"), float("inf")
    y = layer_norm(x)
    bad = ~torch.isfinite(y).all(-1)
    assert bad.nonzero().flatten().tolist() == [3, 9]


@gpu
def test_no_rows(gpu_device):
    for width in (16, 9001):
        x = torch.zeros(0, width, device="cuda", requires_grad=True)
        w, b = torch.ones(width, device="cuda", requires_grad=True), torch.zeros(width, device="cuda", requires_grad=True)
        y = layer_norm(x, w, b)
        gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
        assert y.shape == gx.shape == (0, width) and not gw.any() and not gb.any()
    assert layer_norm(torch.zeros(3, 0, 4, device="cuda")).shape == (3, 0, 4)
    one = torch.randn(300, device="cuda")   # a single row without leading axes
    check("y", layer_norm(one), ref.run(one[None], None, None, 1e-5)["y"])


@gpu
@pytest.mark.parametrize("want", ["x", "w", "b", "wb", "xw", "xb"])
@pytest.mark.parametrize("width", [200, 9000])
def test_some_gradients(gpu_device, width, want):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w, b, u = (make(gen, s, torch.bfloat16) for s in ((50, width), (width,), (width,), (50, width)))
    leaves = {"x": x, "w": w, "b": b}
    for name in want:
        leaves[name].requires_grad_(True)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, [leaves[n] for n in want], u, retain_graph=True)
    full = ref.run(x.detach(), w.detach(), b.detach(), 1e-5, u)
    for name, g in zip(want, grads):
        check("d" + name, g, full["d" + name])
        alone, = torch.autograd.grad(y, [leaves[name]], u, retain_graph=True)   # asked for by itself
        assert torch.equal(alone, g)


@gpu
def test_gradients_against_differences(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(7)
    x, w, b, u = (torch.randn(s, generator=gen, device="cuda") for s in ((6, 50), (50,), (50,), (6, 50)))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(x, w, b), leaves, u)
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        v = torch.randn(leaf.shape, generator=gen, device="cuda")
        step = 2.0 ** -7
        at = [t.detach() for t in leaves]
        sides = []
        for sign in (1, -1):
            moved = list(at)
            moved[i] = at[i] + sign * step * v
            sides.append((layer_norm(*moved).double() * u.double()).sum())
        slope = (sides[0] - sides[1]) / (2 * step)
        exact = (g.double() * v.double()).sum()
        # third derivatives times step^2 / 6 (some tens in sum), and rounding of y over the step
        assert abs(slope - exact) < 2e-3 * (1 + abs(exact)), i


@gpu
def test_offsets_over_32_bits(gpu_device):
    width, rows = 8192, 2 ** 18 + 3
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, width, device="cuda").to(x)
    y = layer_norm(x.requires_grad_(True))
    u = torch.zeros_like(y)
    u[-2:] = 1 + x[-2:].detach()
    gx, = torch.autograd.grad(y, x, u)
    want = ref.run(x[-2:].detach(), None, None, 1e-5, u[-2:])
    check("y", y[-2:], want["y"])
    check("dx", gx[-2:], want["dx"])
    assert not y[:5].any() and not gx[:5].any()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ctypes_binding_gives_the_same(gpu_device, dtype):
    native = _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)
    gen = torch.Generator(device="cuda").manual_seed(8)
    dt = DTYPES[dtype]
    for vt in {dt, torch.float32}:
        x, u = make(gen, (90, 130), dt), make(gen, (90, 130), dt)
        w, b = make(gen, (130,), vt), make(gen, (130,), vt)
        one = compare(x, w, b, u)
        two = compare(x, w, b, u, norm=native.layer_norm)
        assert torch.equal(one[0], two[0]) and all(torch.equal(a, c) for a, c in zip(one[1], two[1]))
    with pytest.raises(ValueError, match="weight must be"):
        native.layer_norm(x, w[:5], None, 1e-5)


@gpu
def test_repeatable_and_two_streams(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w, b, u = (make(gen, s, torch.bfloat16).requires_grad_(True) for s in ((20000, 256), (256,), (256,), (20000, 256)))

    def step():
        y = layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], u.detach())]

    first = step()
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, c) for a, c in zip(first, out))


@gpu
def test_captured_and_replayed(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(10)
    x, w, b, u = (make(gen, s, torch.bfloat16) for s in ((3000, 256), (256,), (256,), (3000, 256)))

    def step(xs):
        leaves = [t.detach().requires_grad_(True) for t in (xs, w, b)]
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, u)]

    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for seed in range(3):
        new = make(torch.Generator(device="cuda").manual_seed(seed), x.shape, x.dtype)
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, c) for a, c in zip(got, step(new)))


@gpu
def test_refusals(gpu_device):
    x = torch.randn(4, 6, device="cuda")
    w = torch.ones(6, device="cuda")
    for args, error in (((x.double(), None, None), ValueError), ((x, w.half(), None), ValueError), ((x, w[:5], None), ValueError),
                        ((x, w.cpu(), None), RuntimeError), ((x.half(), w.half(), w), ValueError), ((x, w[None], None), ValueError),
                        ((x[0, 0], None, None), ValueError), ((x[:, :0], None, None), ValueError), ((x, w, None, -1.0), ValueError),
                        ((x, w, None, float("nan")), ValueError), ((x.to_sparse(), None, None), ValueError)):
        with pytest.raises(error):
            layer_norm(*args)


@gpu
@pytest.mark.parametrize("binding", ["module", "ctypes"])
def test_differentiated_twice_raises(gpu_device, binding):
    norm = layer_norm if binding == "module" else _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH).layer_norm
    x = torch.randn(4, 6, device="cuda", requires_grad=True)
    y = norm(x, None, None, 1e-5)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@gpu
def test_forward_mode_tracing_and_transforms_are_refused(gpu_device):
    x = torch.randn(4, 6, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(dual)
    with pytest.raises(RuntimeError):
        torch.jit.trace(layer_norm, (x,), check_trace=False)
    with pytest.raises(Exception):
        torch.func.vmap(layer_norm)(x)


@gpu
def test_autocast_keeps_the_type(gpu_device):
    x, w = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16), torch.randn(64, device="cuda")
    with torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(layer_norm(x, w), layer_norm(x, w)) and layer_norm(x, w).dtype == torch.bfloat16
