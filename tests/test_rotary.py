"""rotary_positions against its float64 restatement (oracle/rotary.py) within componentwise bounds derived
there, and its refusals.  CPU: the restatement itself, refusals.  GPU: everything that computes."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import rotary as ref
from ops3d_amd import _extension, axial_frequencies, rotary_positions

gpu = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def make(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=gen.device).to(dtype)


def check(name, got, want):
    value, bound = want
    over = (got.detach().double() - value).abs() - bound
    assert torch.isfinite(got).all()
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{name}: {int((over > 0).sum())}/{over.numel()} outside the bound, by at most {worst:.3e}"


def compare(x, positions, sections, layout="halves", u=None, turn=rotary_positions, **kw):
    leaf = x.detach().requires_grad_(True)
    y = turn(leaf, positions, sections, layout=layout, **kw)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    sec = (sections,) if isinstance(sections, int) else sections
    freq = kw.get("frequencies") or axial_frequencies(sec, kw.get("theta", 10000.0))
    u = torch.randn_like(y) if u is None else u
    g, = torch.autograd.grad(y, leaf, u)
    check("y", y, ref.run(x, positions, sec, freq, layout))
    check("dx", g, ref.run(u, positions, sec, freq, layout, inverse=True))
    return y, g


# ---------------------------------------------------------------------------- CPU


def test_restatement_turns_and_depends_on_distances():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(4, 3, 10, generator=gen, dtype=torch.float64).float()
    pos = torch.randint(0, 50, (4, 2), generator=gen)
    sections, freq = (2, 3), axial_frequencies((2, 3))
    for layout in ("halves", "pairs"):
        y, _ = ref.run(x, pos, sections, freq, layout)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
        back, _ = ref.run(y.float(), pos, sections, freq, layout, inverse=True)
        assert torch.allclose(back, x.double(), atol=1e-5)
        shifted, _ = ref.run(x, pos + 7, sections, freq, layout)   # products depend on differences
        assert torch.allclose(y[0] @ y[1].t(), shifted[0] @ shifted[1].t(), atol=1e-9)
    # one axis, one pair, by hand
    one, _ = ref.run(torch.tensor([[[1.0, 0.0, 5.0]]]), torch.tensor([[0.5]]), (1,), (math.pi,), "halves")
    assert torch.allclose(one, torch.tensor([[[0.0, 1.0, 5.0]]], dtype=torch.float64), atol=1e-15)


def test_frequencies():
    assert axial_frequencies((2, 0, 1), 100.0) == (1.0, 100.0 ** -0.5, 1.0)
    assert axial_frequencies(2, 16.0) == (1.0, 0.25)


def test_refusals_on_the_cpu():
    x, pos = torch.zeros(3, 2, 8), torch.zeros(3, 2)
    for args, kw in (((x, pos, (2, 3)), {}), ((x, pos, (2,)), {}), ((x, pos, (-1, 2)), {}), ((x, pos, ()), {}), ((x, pos, (1.5, 1)), {}),
                     ((x, pos, (1, 1)), {"layout": "thirds"}), ((x, pos, (1, 1)), {"theta": 0.0}), ((x, pos, (1, 1)), {"theta": math.inf}),
                     ((x, pos, (1, 1)), {"frequencies": [1.0]})):
        with pytest.raises(ValueError):
            rotary_positions(*args, **kw)
    with pytest.raises(RuntimeError, match="CPU"):
        rotary_positions(x, pos, (1, 1))


def test_c_refusals_before_device_work():
    import os

    if not os.path.exists(_extension.LIB_PATH):
        pytest.skip("libops3d_fda.so not built")
    lib = _extension.load_library()
    strides = (ctypes.c_int64 * 3)(0, 8, 8)

    def call(x=16, xs=strides, pos=16, ptype=0, freq=(1.0, 0.5), axis=(0, 1), pairs=2, axes=2, layout=0, y=16, ys=strides, dtype=0,
             items=1, tokens=3, heads=1, dim=8):
        return lib.ops3d_rotary(x, xs, pos, ptype, 0, (ctypes.c_double * 2)(*freq) if freq else None, (ctypes.c_int * 2)(*axis) if axis else None,
                                pairs, axes, layout, 0, y, ys, dtype, items, tokens, heads, dim, None)

    for bad in ({"dtype": 5}, {"ptype": 2}, {"layout": 2}, {"items": -1}, {"items": 65536}, {"tokens": -1}, {"tokens": 2 ** 31}, {"heads": -1},
                {"heads": 65537}, {"dim": 0}, {"dim": 3}, {"heads": 60000, "dim": 60000}, {"axes": 0}, {"axes": 9}, {"pairs": -1}, {"pairs": 129, "dim": 512},
                {"freq": None}, {"axis": None}, {"axis": (0, 2)}, {"axis": (-1, 0)}, {"freq": (math.nan, 1.0)}, {"freq": (math.inf, 1.0)},
                {"x": None}, {"y": None}, {"pos": None}, {"xs": None}, {"ys": None}, {"x": 18}, {"pos": 18}, {"pos": 20, "ptype": 1}):
        assert call(**bad) == 1, bad
        assert lib.ops3d_fda_last_error()
    assert call(tokens=0) == call(items=0) == call(heads=0) == 0


# ---------------------------------------------------------------------------- GPU

CASES = [   # tokens, heads, dim, sections
    (1, 1, 2, (1,)), (3, 2, 32, (5, 5, 6)), (100, 8, 32, (8, 8)), (77, 3, 36, (6, 6, 6)), (50, 5, 64, (16, 8, 8)), (40, 4, 128, (16, 24, 24)),
    (33, 2, 128, (8, 8, 8)), (29, 7, 7, (1, 2)), (20, 1, 300, (40, 40, 40)), (9, 2, 256, (128,)), (500, 16, 32, (0, 7, 4)), (5, 3, 16, (0, 0))]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_sizes(gpu_device, case, layout, dtype):
    tokens, heads, dim, sections = CASES[case]
    gen = torch.Generator(device="cuda").manual_seed(case)
    for lead, plead in (((), ()), ((3,), ()), ((3,), (3,))):
        x = make(gen, (*lead, tokens, heads, dim), DTYPES[dtype])
        pos = torch.randint(0, 5000, (*plead, tokens, len(sections)), generator=gen, device="cuda")
        compare(x, pos, sections, layout)
        compare(x, pos.float() + 0.5, sections, layout, theta=500.0)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_large(gpu_device, dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = make(gen, (70001, 16, 32), DTYPES[dtype])
    pos = torch.randint(0, 4096, (70001, 3), generator=gen, device="cuda")
    compare(x, pos, (5, 5, 6))
    compare(make(gen, (3, 40, 130), DTYPES[dtype]), pos[:3], (20, 20, 20), "pairs")


@gpu
def test_far_positions(gpu_device):
    """Angles of 10^9 turns keep their fraction; negative ones and fractions too."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = make(gen, (200, 2, 16), torch.float32)
    pos = torch.randint(-2 ** 33, 2 ** 33, (200, 2), generator=gen, device="cuda")
    compare(x, pos, (4, 4), theta=3.0)
    compare(x, (torch.rand(200, 2, generator=gen, device="cuda") - 0.5) * 1e7, (4, 4))
    compare(x, pos.clamp(-9, 9), (4, 4), frequencies=[0.0, -1.0, 1e-3, 7.5, 2.0, -0.25, 1.0, 3.0])


@gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strides(gpu_device, dtype, layout):
    """Parts of a projection's rows, unaligned ones, heads before tokens, repeated and strided channels."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    dt = DTYPES[dtype]
    pos = torch.randint(0, 100, (20, 3), generator=gen, device="cuda")
    rows = make(gen, (2, 20, 9, 32), dt)
    for x in (rows[:, :, :5], rows[:, :, 1::2], rows[..., 1:27], rows[..., :2, :].expand(2, 20, 2, 32), rows[:, :1, :4].expand(2, 20, 4, 32),
              rows.transpose(1, 2).contiguous().transpose(1, 2), rows[..., ::2], make(gen, (2, 20 * 9 * 32 + 3), dt)[:, 3:].view(2, 20, 9, 32)):
        compare(x, pos, (3, 2, 2), layout)
        y = make(gen, x.shape, dt)
        compare(y, pos[None].expand(2, 20, 3), (3, 2, 2), layout, u=x)
    compare(rows, pos.t().contiguous().t(), (3, 2, 2), layout)


@gpu
def test_empty(gpu_device):
    for shape in ((0, 4, 8), (2, 0, 4, 8), (0, 3, 4, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = rotary_positions(x, torch.zeros(shape[-3], 1, device="cuda"), 2)
        g, = torch.autograd.grad(y, x, torch.zeros_like(y))
        assert y.shape == g.shape == shape


@gpu
def test_offsets_over_32_bits(gpu_device):
    x = torch.zeros(2, 2 ** 20 + 1, 16, 80, dtype=torch.float16, device="cuda")   # 2.7e9 elements
    x[1, -1] = torch.randn(16, 80, device="cuda").to(x)
    pos = torch.full((2 ** 20 + 1, 2), 5, device="cuda")
    y = rotary_positions(x, pos, (20, 20))
    check("y", y[1, -1:], ref.run(x[1, -1:], pos[-1:], (20, 20), axial_frequencies((20, 20)), "halves"))
    assert not y[0, :3].any()


@gpu
def test_ctypes_binding_gives_the_same(gpu_device):
    native = _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, pos = make(gen, (2, 30, 4, 24), torch.bfloat16), torch.randint(0, 99, (2, 30, 2), generator=gen, device="cuda")
    u = make(gen, x.shape, x.dtype)

    def other(x, positions, sections, layout):
        from ops3d_amd.rotary import LAYOUTS, _pairs

        return native.rotary(x, positions, *_pairs(sections, 10000.0), LAYOUTS[layout])

    for layout in ("halves", "pairs"):
        for p in (pos, pos.float()):
            one, two = compare(x, p, (4, 6), layout, u), compare(x, p, (4, 6), layout, u, turn=other)
            assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@gpu
def test_differentiated_twice(gpu_device):
    """The gradient is linear in the output's: its own gradient is the turn again."""
    x = torch.randn(5, 2, 8, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda")[:, None]
    y = rotary_positions(x, pos, 4)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)   # 2 x
    assert torch.allclose(g, 2 * x, atol=1e-5)
    gg, = torch.autograd.grad(g.square().sum(), x)
    assert torch.allclose(gg, 8 * x, atol=1e-4)


@gpu
def test_captured_and_replayed_and_two_streams(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, pos = make(gen, (900, 8, 32), torch.bfloat16), torch.randint(0, 99, (900, 3), generator=gen, device="cuda")

    def step(xs, ps):
        leaf = xs.detach().requires_grad_(True)
        y = rotary_positions(leaf, ps, (5, 5, 6))
        return [y.detach(), *torch.autograd.grad(y, leaf, xs)]

    sx, sp = x.clone(), pos.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(sx, sp)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step(x, pos)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(sx, sp)
    for seed in range(3):
        new = torch.Generator(device="cuda").manual_seed(seed)
        sx.copy_(make(new, x.shape, x.dtype))
        sp.copy_(torch.randint(0, 999, pos.shape, generator=new, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step(sx, sp)))


@gpu
def test_refusals(gpu_device):
    x, pos = torch.randn(4, 2, 8, device="cuda"), torch.zeros(4, 2, device="cuda")
    for args, error in (((x.double(), pos), ValueError), ((x, pos.half()), ValueError), ((x, pos.double()), ValueError), ((x, pos.int()), ValueError),
                        ((x, pos.cpu()), RuntimeError), ((x, pos[:3]), ValueError), ((x, pos[None]), ValueError), ((x[0], pos), ValueError),
                        ((x[None], pos[None].expand(2, 4, 2)), ValueError), ((x, pos.clone().requires_grad_()), ValueError), ((x, pos[0]), ValueError),
                        ((x.to_sparse(), pos), ValueError)):
        with pytest.raises(error):
            rotary_positions(*args, (2, 2))
    with pytest.raises(ValueError):
        rotary_positions(torch.randn(4, 2, 300, device="cuda"), pos, (65, 64))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotary_positions(torch.autograd.forward_ad.make_dual(x, x), pos, (2, 2))
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda t: rotary_positions(t, pos, (2, 2)), (x,), check_trace=False)
    with pytest.raises(Exception):
        torch.func.vmap(lambda t: rotary_positions(t, pos, (2, 2)))(x[None])


@gpu
@pytest.mark.parametrize("binding", ["module", "ctypes"])
def test_more_items_than_a_call_takes(gpu_device, binding):
    """Windows of a volume as a batch: more than the 65535 items that the C entry takes at once."""
    native = _extension._C if binding == "module" else _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)

    def turn(x, positions, sections, layout):
        from ops3d_amd.rotary import LAYOUTS, _pairs

        return native.rotary(x, positions, *_pairs(sections, 10000.0), LAYOUTS[layout])

    gen = torch.Generator(device="cuda").manual_seed(7)
    x = make(gen, (140000, 3, 9), torch.bfloat16)[:, :, :8].unflatten(-1, (1, 8))
    compare(x, torch.randint(0, 99, (3, 2), generator=gen, device="cuda"), (2, 1), turn=turn)
    compare(x, torch.randint(0, 99, (140000, 3, 2), generator=gen, device="cuda"), (2, 2), "pairs", turn=turn)
