"""packed_attention against its float64 restatement (oracle/attention.py) within componentwise bounds
derived there, and its refusals.  CPU: the restatement itself, refusals, sizes.  GPU: everything that
computes."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from oracle import attention as ref
from ops3d_amd import _extension, packed_attention

gpu = pytest.mark.gpu
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("y", "dq", "dk", "dv")


def make(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(dtype)


def check(name, got, want):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - value).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{name}: {int((over > 0).sum())}/{over.numel()} outside the bound, by at most {worst:.3e}"


def table(x):
    return None if x is None else torch.tensor(x, dtype=torch.int64, device="cuda")


def compare(q, k, v, causal=False, scale=None, q_start=None, k_start=None, q_len=None, k_len=None, u=None, attend=packed_attention,
            train=True):
    """Forward and backward; the forms with and without statistics agree."""
    kw = {"q_start": table(q_start), "k_start": table(k_start), "q_len": table(q_len), "k_len": table(k_len), "causal": causal}
    if scale is not None:
        kw["scale"] = scale
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v)]
    y = attend(*leaves, **kw)
    assert y.shape == q.shape and y.dtype == q.dtype and y.is_contiguous()
    outs = [y.detach()]
    if train:
        u = torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(99), device="cuda").to(q.dtype) if u is None else u
        outs += torch.autograd.grad(y, leaves, u)
        with torch.no_grad():
            assert torch.equal(attend(q, k, v, **kw), y)
    scale = scale or q.shape[-1] ** -0.5
    if q_start is not None:
        want = ref.packed(q, k, v, q_start, q_start if k_start is None else k_start, causal, scale, u if train else None)
    elif q.dim() == 3:
        want = ref.packed(q, k, v, [0, q.shape[0]], [0, k.shape[0]], causal, scale, u if train else None)
    else:
        want = ref.items(q, k, v, q_len, k_len, causal, scale, u if train else None)
    for name, got in zip(NAMES, outs):
        check(name, got, want[name])
    return outs


def case(dtype, nq, nk, H, Hk, D, causal=False, lead=(), seed=0, logits=1.0, **kw):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[dtype]
    return compare(make(gen, (*lead, nq, H, D), dt, logits), make(gen, (*lead, nk, Hk, D), dt), make(gen, (*lead, nk, Hk, D), dt), causal, **kw)


# ---------------------------------------------------------------------------- CPU


@pytest.mark.parametrize("causal", [False, True])
def test_restatement_against_torch_and_differences(causal):
    gen = torch.Generator().manual_seed(0)
    q, k, v, u = (torch.randn(s, generator=gen) for s in ((5, 4, 6), (7, 2, 6), (7, 2, 6), (5, 4, 6)))
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(2, dim=1) for t in leaves[1:])
    mask = torch.ones(5, 7, dtype=torch.bool).tril(2) if causal else None
    y = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1)[None] for t in (leaves[0], kk, vv)), attn_mask=mask, scale=0.3)
    y = y[0].transpose(0, 1)
    grads = torch.autograd.grad(y, leaves, u.double())
    got = ref.sequence(q, k, v, causal, 0.3, u)
    for name, want in zip(NAMES, (y, *grads)):
        assert torch.allclose(got[name][0], want, rtol=1e-12, atol=1e-12), name
    step = 1e-3   # a second opinion on a gradient: differences
    d = torch.zeros_like(k)
    d[1, 1, 2] = step
    up, down = (ref.sequence(q, k + s * d, v, causal, 0.3)["y"][0] for s in (1, -1))
    assert abs(((up - down) * u).sum() / (2 * step) - got["dk"][0][1, 1, 2]) < 1e-4


def test_restatement_of_sequences():
    assert ref.bounds_of([-3, 4, 2, 9], 6) == [0, 4, 4, 6]
    q = torch.randn(6, 1, 2)
    out = ref.packed(q, q, q, [1, 3, 3, 5], [1, 3, 3, 5], True, 1.0, q)
    assert not out["y"][0][[0, 5]].any() and not out["dq"][0][[0, 5]].any() and torch.equal(out["y"][0][1], q[1].double())
    # more queries than keys: the first see none
    out = ref.sequence(q, q[:4], q[:4], True, 1.0)
    assert not out["y"][0][:2].any() and torch.equal(out["y"][0][2], q[0].double())


def test_refusals_on_the_cpu():
    x = torch.zeros(3, 2, 4)
    with pytest.raises(RuntimeError, match="CPU"):
        packed_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CPU"):
        packed_attention(x.requires_grad_(), x, x)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(x, x, x, scale=scale)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_extension.LIB_PATH):
        pytest.skip("libops3d_fda.so not built")
    return _extension.load_library()


def problem(**kw):
    p = _extension._AttentionProblem()
    for name, value in {"q_rows": 5, "k_rows": 7, "items": 2, "heads": 4, "kv_heads": 2, "dim": 8, "scale": 1.0, **kw}.items():
        setattr(p, name, value)
    return p


def test_c_refusals_before_device_work(lib):
    def tensor(data=16, item=0, token=8, head=8):
        return _extension._AttentionTensor(data, item, token, head)

    def forward(p, q=tensor(), k=tensor(), v=tensor(), o=tensor(), rest=None, lse=None, ws=None, n=0):
        return lib.ops3d_attention_forward(p, q, k, v, o, rest, lse, ws, n, None)

    packed = {"q_start": 16, "k_start": 16, "items": 1, "sequences": 3, "q_start_count": 4, "k_start_count": 3}
    bad = [{"dtype": 3}, {"heads": 3}, {"heads": 0}, {"kv_heads": 0}, {"dim": 0}, {"dim": 129}, {"scale": 0.0}, {"scale": -1.0},
           {"scale": math.nan}, {"scale": math.inf}, {"q_rows": -1}, {"k_rows": -1}, {"q_rows": 2 ** 31}, {"q_rows": 2 ** 30}, {"k_rows": 2 ** 31},
           {"items": -1}, {"items": 2 ** 25}, {"q_start": 16}, {"k_start": 16}, {"q_len": 12}, {**packed, "items": 2}, {**packed, "q_len": 16},
           {**packed, "sequences": 0}, {**packed, "sequences": 65537}, {**packed, "q_start_count": 5}, {**packed, "k_start_count": 2},
           {**packed, "k_start": 20}, {"items": 2 ** 20, "kv_heads": 128, "heads": 128, "q_rows": 2 ** 16}]
    for kw in bad:
        assert forward(problem(**kw), ws=256, n=2 ** 60) == 1, kw
        assert lib.ops3d_fda_last_error()
    for kw in ({"q": tensor(None)}, {"k": tensor(None)}, {"v": tensor(18)}, {"o": tensor(None)}, {"q": None}, {"lse": 18}, {"rest": 19, "p": problem(dtype=1)}, {"q": tensor(token=-1)}):
        assert forward(**{"p": problem(), **kw}) == 1, kw
    assert lib.ops3d_attention_forward(None, None, None, None, None, None, None, None, 0, None) == 1
    assert forward(problem(items=0)) == forward(problem(q_rows=0)) == 0
    few = problem(q_rows=1, k_rows=100000, items=1)
    need = lib.ops3d_attention_forward_workspace_bytes(few)
    assert need > 0
    assert forward(few, ws=None, n=need) == forward(few, ws=256, n=need - 1) == forward(few, ws=264, n=need) == 1

    def backward(p, q=tensor(), k=tensor(), v=tensor(), o=tensor(), rest=None, lse=16, g=tensor(), gq=tensor(), gk=tensor(), gv=tensor(), ws=256, n=None):
        n = lib.ops3d_attention_backward_workspace_bytes(p) if n is None else n
        return lib.ops3d_attention_backward(p, q, k, v, o, rest, lse, g, gq, gk, gv, ws, n, None)

    for kw in ({"lse": None}, {"lse": 18}, {"gk": None}, {"gv": None}, {"g": None}, {"o": tensor(None)}, {"ws": None}, {"n": 16}, {"gq": tensor(17)}):
        assert backward(problem(), **kw) == 1, kw
    assert backward(problem(dim=200)) == 1
    assert backward(problem(), gq=None, gk=None, gv=None) == 0
    assert backward(problem(items=0)) == 0


def test_workspace_sizes(lib):
    size = lib.ops3d_attention_forward_workspace_bytes
    assert size(problem(dim=200)) == size(problem(items=0)) == size(problem(q_rows=0)) == 0
    assert size(problem(q_rows=20000, k_rows=20000, heads=8, kv_heads=8)) == 0   # blocks enough
    back = lib.ops3d_attention_backward_workspace_bytes
    assert back(problem(dim=200)) == back(problem(items=0)) == 0
    assert back(problem()) >= 2 * 4 * 5 * 4


# ---------------------------------------------------------------------------- GPU

DIMS = [1, 4, 7, 16, 31, 32, 33, 36, 48, 64, 72, 80, 96, 100, 127, 128]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim", DIMS)
def test_dims(gpu_device, dim, dtype):
    case(dtype, 70, 130, 4, 2, dim, causal=True, seed=dim)
    case(dtype, 9, 40, 2, 2, dim, seed=dim)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (1, 300), (300, 1), (15, 16), (16, 17), (17, 15), (63, 65), (64, 64), (128, 128),
                                   (129, 127), (200, 200), (257, 511), (500, 90), (333, 1000)])
def test_lengths(gpu_device, nq, nk, causal, dtype):
    case(dtype, nq, nk, 2, 1, 32, causal, seed=nq)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 8), (3, 3), (8, 1), (10, 2), (7, 1), (12, 4), (40, 8), (33, 1)])
def test_grouped_heads(gpu_device, H, Hk, dtype):
    for nq, nk in ((1, 70), (3, 300), (100, 100)):
        case(dtype, nq, nk, H, Hk, 40, causal=True, seed=H)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("nq,nk,H,Hk", [(1300, 1300, 8, 8), (2100, 900, 8, 4), (3, 9000, 4, 2), (9000, 3, 4, 2), (40, 5000, 2, 2), (5000, 40, 2, 2)])
def test_large(gpu_device, nq, nk, H, Hk, dim, dtype):
    """Every tiling, and parts of long sides joined."""
    case(dtype, nq, nk, H, Hk, dim, causal=nq > nk and nk > 40, seed=1)


SEQUENCES = [   # q rows, q_start, k rows, k_start (None: the queries')
    (10, [0, 10], 10, None), (300, [0, 100, 101, 101, 290, 300], 300, None), (300, [5, 100, 290], 300, None), (50, [0, 0, 0, 50, 50], 50, None),
    (70, [-4, 80, 30, 200], 70, None), (200, [0, 1, 33, 150, 200], 400, [0, 130, 130, 131, 400]), (400, [0, 130, 130, 131, 390], 90, [3, 4, 33, 60, 80]),
    (40, [20, 20], 40, [3, 30]), (64, [40, 10, 5], 64, [40, 64, 64]), (150, list(range(0, 151)), 150, None),
    (1000, [0, 300, 301, 700, 1000], 1000, None)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("at", range(len(SEQUENCES)))
def test_packed_sequences(gpu_device, at, causal, dtype):
    nq, q_start, nk, k_start = SEQUENCES[at]
    outs = case(dtype, nq, nk, 4, 2, 24, causal, seed=at, q_start=q_start, k_start=k_start)
    bounds = ref.bounds_of(q_start, nq)
    for t in outs[:2]:
        assert not t[:bounds[0]].any() and not t[bounds[-1]:].any()


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_many_sequences(gpu_device, dtype):
    gen = torch.Generator().manual_seed(3)
    sizes = torch.randint(0, 4, (3000,), generator=gen)
    sizes[100] = 700
    start = [0] + sizes.cumsum(0).tolist()
    rows = start[-1]
    other = [0] + sizes.flip(0).cumsum(0).tolist()
    case(dtype, rows + 3, rows + 3, 2, 1, 16, True, q_start=start)
    case(dtype, rows, rows, 1, 1, 32, False, q_start=start, k_start=other)
    odd = list(start)
    odd[7], odd[300], odd[2000] = rows + 900, -5, 3   # the largest so far counts, held to the rows
    case(dtype, rows, rows, 2, 2, 32, False, q_start=[5] + odd[1:], k_start=other)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("sequences,rows", [(63, 900), (64, 900), (65, 900), (66, 3000), (130, 20000), (1022, 5000), (1023, 5000), (4097, 4200)])
def test_sequences_found_and_looked_up(gpu_device, sequences, rows, dtype):
    """Around the numbers of sequences where blocks stop finding their own, and where a thread gets more of them."""
    gen = torch.Generator().manual_seed(sequences)
    start = [2] + sorted(torch.randint(2, rows - 3, (sequences - 1,), generator=gen).tolist()) + [rows - 3]
    case(dtype, rows, rows, 2, 1, 32, sequences % 2 == 0, q_start=start)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk,q_len,k_len", [
    (1, 600, None, [600, 1, 0, 77]), (1, 40, [1, 0, 1, 1], [40, 40, 0, 3]), (50, 90, [50, 0, 7, 33], [90, 20, 0, 64]), (50, 90, None, [91, -3, 5, 10 ** 12]),
    (200, 200, [200, 120, 1, 65], None), (3, 3000, None, [3000, 5, 0, 1700])])
def test_items_with_lengths(gpu_device, nq, nk, q_len, k_len, causal, dtype):
    case(dtype, nq, nk, 4, 2, 32, causal, lead=(4,), q_len=q_len, k_len=k_len)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_that_do_not_count_are_not_read(gpu_device, dtype):
    """NaN in rows of no sequence, behind an item's length, and in the output's places there."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    dt = DTYPES[dtype]
    for nq, nk, ql, kl in ((100, 130, 70, 33), (1, 700, 1, 650), (700, 30, 650, 17)):
        for causal in (False, True):
            q, k, v, u = (make(gen, s, dt) for s in ((nq, 4, 32), (nk, 2, 32), (nk, 2, 32), (nq, 4, 32)))
            for t, n in ((q, ql), (k, kl), (v, kl), (u, ql)):
                t[n:] = float("nan")
            args = {"q_len": table([ql]), "k_len": table([kl])}, {"q_start": table([0, ql]), "k_start": table([0, kl])}
            for kw in args:
                leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
                y = packed_attention(*leaves, causal=causal, **kw)
                outs = [y.detach(), *torch.autograd.grad(y, leaves, u)]
                want = ref.packed(q, k, v, [0, ql], [0, kl], causal, 32 ** -0.5, u)
                for name, got in zip(NAMES, outs):
                    check(name, got, want[name])


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_extreme_logits(gpu_device, dtype):
    """Large and growing logits (the reference is raised again and again), equal ones, tiny and large scales."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    dt = DTYPES[dtype]
    case(dtype, 100, 700, 2, 2, 32, seed=6, logits=12.0)
    q, k, v = (make(gen, (n, 1, 32), dt) for n in (90, 1000, 1000))
    k = (torch.linspace(-9, 9, 1000, device="cuda")[:, None, None] * torch.ones(1, 1, 32, device="cuda")).to(dt)
    compare(torch.ones_like(q), k, v)                      # each key above those before it
    compare(-torch.ones_like(q), k, v)                     # below
    compare(q, torch.zeros_like(k), v)
    compare(q, k, v, scale=1e-6)
    compare(q, q, q, scale=20.0, causal=True)


@gpu
def test_not_finite_values_reach_those_that_see_them(gpu_device):
    q, k, v = torch.randn(40, 2, 32, device="cuda"), torch.randn(60, 2, 32, device="cuda"), torch.randn(60, 2, 32, device="cuda")
    for t, row in ((q, 3), (k, 5), (v, 5)):
        bad = [x.clone() for x in (q, k, v)]
        at = [x is t for x in (q, k, v)].index(True)
        bad[at][row, 1, 0] = float("nan")
        y = packed_attention(*bad)
        assert torch.isfinite(y[:, 0]).all()
        if at == 0:
            assert y[3, 1].isnan().all() and torch.isfinite(y[[0, 2, 4, 39], 1]).all()
        elif at == 1:
            assert y[:, 1].isnan().all()
        else:
            assert y[:, 1, 0].isnan().all() and torch.isfinite(y[:, 1, 1:]).all()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,H,Hk,D", [(150, 150, 4, 2, 32), (150, 170, 2, 2, 36), (700, 700, 2, 1, 64), (300, 300, 2, 2, 128), (2100, 2100, 8, 8, 32),
                                          (4200, 4200, 8, 8, 32), (2300, 2300, 16, 4, 128), (3, 5000, 2, 1, 64)])
def test_hidden_values_that_are_not_finite(gpu_device, nq, nk, H, Hk, D, dtype):
    """Causal: NaN and infinities in keys and values reach no query before them, and in queries and output gradients
    no key behind them, in the same tile or another."""
    gen = torch.Generator(device="cuda").manual_seed(nq)
    dt = DTYPES[dtype]
    q, k, v, u = (make(gen, s, dt) for s in ((nq, H, D), (nk, Hk, D), (nk, Hk, D), (nq, H, D)))
    want = ref.sequence(q, k, v, True, D ** -0.5, u)
    off = nk - nq
    late, early = max(off + 1, nk - 60), nq // 3   # a key, and a query, counted among their own
    for bad in (float("nan"), float("inf"), -float("inf")):
        kk, vv = k.clone(), v.clone()
        kk[late, 0, D // 2], vv[late, :, 0], vv[late + (late + 1 < nk), 0, D - 1] = bad, bad, bad
        leaves = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
        y = packed_attention(*leaves, causal=True)
        gq, _, _ = torch.autograd.grad(y, leaves, u)
        clean = slice(0, late - off)   # the queries before the key
        for name, got in (("y", y), ("dq", gq)):
            check(name, got[clean], tuple(t[clean] for t in want[name]))
        assert not torch.isfinite(y[late - off:, :, 0]).any()
        qq, uu = q.clone(), u.clone()
        qq[early, 0, 0], uu[early, :, D - 1] = bad, bad
        leaves = [t.detach().requires_grad_(True) for t in (qq, k, v)]
        y = packed_attention(*leaves, causal=True)
        _, gk, gv = torch.autograd.grad(y, leaves, uu)
        clean = slice(early + off + 1, nk)   # the keys that the query does not see
        for name, got in (("dk", gk), ("dv", gv)):
            check(name, got[clean], tuple(t[clean] for t in want[name]))
        assert not torch.isfinite(gv[:early + off + 1, :, D - 1]).any()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk", [(5, 1), (5, 70), (9000, 70), (40000, 70), (3, 5001)])
def test_infinity_in_the_last_value(gpu_device, nq, nk, dtype):
    """The last row stands in for those behind it in its tile, whose weight is 0: an infinity there stays one."""
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q, k, v = (make(gen, s, DTYPES[dtype]) for s in ((nq, 2, 32), (nk, 2, 32), (nk, 2, 32)))
    value, bound = ref.sequence(q, k, v, False, 32 ** -0.5)["y"]
    v[-1, 0, 3], v[-1, 1, 4] = math.inf, -math.inf
    y = packed_attention(q, k, v)
    assert (y[:, 0, 3] == math.inf).all() and (y[:, 1, 4] == -math.inf).all()
    keep = torch.isfinite(y)
    assert keep.sum() == y.numel() - 2 * nq
    check("y", y[keep], (value[keep], bound[keep]))


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("dim", [32, 36])
def test_strides(gpu_device, dim, dtype):
    """Parts of one projection, unaligned rows, heads before tokens, shared and strided ones, and gradients so."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    dt = DTYPES[dtype]
    B, N, H = 2, 150, 4
    rows = make(gen, (B, N, 3 * H * dim + 1), dt)
    for part in (rows[..., :-1], rows[..., 1:]):
        q, k, v = part.unflatten(-1, (3 * H, dim)).split(H, dim=2)
        compare(q, k, v, causal=True)
        compare(q, k, v, u=v)
        compare(q[0], k[0, :77], v[0, :77])
    x = make(gen, (B, H, N, dim), dt).transpose(1, 2)
    compare(x, x.flip(1), x, causal=True, u=x)
    shared = make(gen, (1, N, 1, dim), dt).expand(B, N, H, dim)
    y = make(gen, (B, N, H, dim), dt)
    compare(y, shared, y)
    compare(shared, y, shared, u=shared)
    wide = make(gen, (B, N, H, 2 * dim), dt)[..., ::2]
    compare(wide, y, wide, u=wide)


@gpu
@pytest.mark.parametrize("want", ["q", "k", "v", "qk", "kv", "qv"])
def test_some_gradients(gpu_device, want):
    gen = torch.Generator(device="cuda").manual_seed(8)
    for nq, nk in ((150, 150), (2, 4000), (4000, 2)):
        q, k, v, u = (make(gen, s, torch.bfloat16) for s in ((nq, 4, 32), (nk, 2, 32), (nk, 2, 32), (nq, 4, 32)))
        leaves = {"q": q, "k": k, "v": v}
        full = compare(q, k, v, u=u)
        for name in want:
            leaves[name].requires_grad_(True)
        y = packed_attention(q, k, v)
        grads = torch.autograd.grad(y, [leaves[n] for n in want], u, retain_graph=True)
        for name, g in zip(want, grads):
            assert torch.equal(g, full["yqkv".index(name)])
            alone, = torch.autograd.grad(y, [leaves[name]], u, retain_graph=True)
            assert torch.equal(alone, g)


@gpu
def test_empty(gpu_device):
    for q_shape, k_shape in (((0, 2, 8), (5, 2, 8)), ((5, 2, 8), (0, 2, 8)), ((0, 2, 8), (0, 2, 8)), ((0, 3, 2, 8), (0, 3, 1, 8)),
                             ((2, 0, 2, 8), (2, 3, 1, 8)), ((2, 3, 2, 8), (2, 0, 1, 8))):
        q, k, v = (torch.randn(s, device="cuda", requires_grad=True) for s in (q_shape, k_shape, k_shape))
        y = packed_attention(q, k, v, causal=True)
        grads = torch.autograd.grad(y, [q, k, v], torch.ones_like(y))
        assert y.shape == q_shape and not y.any()
        for t, g in zip((q, k, v), grads):
            assert g.shape == t.shape and not g.any()


@gpu
def test_offsets_over_32_bits(gpu_device):
    """A cache of more than 2^31 elements: its last item and its last rows."""
    rows, H, D = 2 ** 18, 33, 128
    k = torch.zeros(2, rows, H, D, dtype=torch.bfloat16, device="cuda")   # 2.2e9 elements
    gen = torch.Generator(device="cuda").manual_seed(9)
    k[1, -40:] = make(gen, (40, H, D), torch.bfloat16)
    q = make(gen, (2, 3, H, D), torch.bfloat16, 3.0)
    y = packed_attention(q, k, k)
    part = torch.cat([torch.zeros(1000, H, D, dtype=k.dtype, device="cuda"), k[1, -1000:]])
    last = packed_attention(q[1], k[1, -500:], k[1, -500:], causal=True)
    check("causal", last, ref.sequence(q[1], k[1, -500:], k[1, -500:], True, D ** -0.5)["y"])
    # all keys but 40 are 0: a logit of 0 each
    s = torch.einsum("qhd,khd->qhk", q[1].double(), k[1, -40:].double()) * D ** -0.5
    total = torch.exp(s).sum(-1) + (rows - 40)
    want = torch.einsum("qhk,khd->qhd", torch.exp(s), k[1, -40:].double()) / total[..., None]
    bound = torch.einsum("qhk,khd->qhd", torch.exp(s), k[1, -40:].double().abs()) / total[..., None] * (2.0 ** -8 + 2.0 ** -9 + (rows / 4 + 40) * ref.U)
    check("y", y[1], (want, bound + 2.0 ** -9 * want.abs() + 1e-30))
    assert not y[0].any()
    del part


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ctypes_binding_gives_the_same(gpu_device, dtype):
    native = _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)

    def other(q, k, v, q_start, k_start, q_len, k_len, causal, scale=None):
        k_start = q_start if k_start is None else k_start
        return native.attention(q, k, v, q_start, k_start, q_len, k_len, causal, scale or q.shape[-1] ** -0.5)

    gen = torch.Generator(device="cuda").manual_seed(10)
    dt = DTYPES[dtype]
    q, k, v, u = (make(gen, s, dt) for s in ((2, 90, 4, 40), (2, 130, 2, 40), (2, 130, 2, 40), (2, 90, 4, 40)))
    for kw in ({"causal": True}, {"k_len": [130, 3], "q_len": [0, 90]}):
        one, two = compare(q, k, v, u=u, **kw), compare(q, k, v, u=u, attend=other, **kw)
        assert all(torch.equal(a, b) for a, b in zip(one, two))
    kw = {"q_start": [0, 30, 80], "k_start": [4, 50, 130]}
    one, two = compare(q[0], k[0], v[0], u=u[0], **kw), compare(q[0], k[0], v[0], u=u[0], attend=other, **kw)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    with pytest.raises(ValueError, match="go together"):
        native.attention(q[0], k[0], v[0], table([0, 90]), None, None, None, False, 1.0)


@gpu
def test_repeatable_and_two_streams(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(11)
    big = [make(gen, s, torch.bfloat16).requires_grad_(True) for s in ((900, 8, 32), (900, 4, 32), (900, 4, 32))]
    few = [make(gen, s, torch.bfloat16).requires_grad_(True) for s in ((2, 8, 64), (20000, 4, 64), (20000, 4, 64))]

    def step(leaves):
        y = packed_attention(*leaves, causal=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]

    first = [step(big), step(few)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([step(big), step(few)])
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(first, out):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("few", [False, True])
def test_captured_and_replayed(gpu_device, few):
    """Replays see new values, new starts and new lengths."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    shapes = ((3, 2, 8, 32), (3, 6000, 4, 32)) if few else ((500, 8, 32), (500, 4, 32))
    q, k, v = make(gen, shapes[0], torch.bfloat16), make(gen, shapes[1], torch.bfloat16), make(gen, shapes[1], torch.bfloat16)
    where = table([6000, 40, 0]) if few else table([0, 100, 100, 500])

    def step(q, k, v, where):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = packed_attention(*leaves, **({"k_len": where} if few else {"q_start": where}), causal=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, q)]

    static = [t.clone() for t in (q, k, v, where)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    tables = ([5, 6000, 3000], [0, 1, 2], [6000, 6000, 6000]) if few else ([3, 10, 300, 410], [0, 0, 500, 500], [0, 250, 260, 500])
    for seed, new in enumerate(tables):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for t in static[:3]:
            t.copy_(make(gen, t.shape, t.dtype))
        static[3].copy_(table(new))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step(*static)))


@gpu
def test_gradients_against_differences(gpu_device):
    gen = torch.Generator(device="cuda").manual_seed(13)
    at = [torch.randn(s, generator=gen, device="cuda") for s in ((12, 4, 8), (20, 2, 8), (20, 2, 8))]
    u = torch.randn(12, 4, 8, generator=gen, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in at]
    grads = torch.autograd.grad(packed_attention(*leaves, causal=True), leaves, u)
    for i, g in enumerate(grads):
        d = torch.randn(g.shape, generator=gen, device="cuda")
        d = d / d.norm()
        step = 2.0 ** -6
        sides = []
        for sign in (1, -1):
            moved = list(at)
            moved[i] = at[i] + sign * step * d
            sides.append((packed_attention(*moved, causal=True).double() * u.double()).sum())
        slope = (sides[0] - sides[1]) / (2 * step)
        exact = (g.double() * d.double()).sum()
        # a unit direction: third derivatives of a few units times step^2 / 6, rounding of y over the step
        assert abs(slope - exact) < 2e-3 * (1 + abs(exact)), i


@gpu
def test_refusals(gpu_device):
    q, k = torch.randn(6, 4, 8, device="cuda"), torch.randn(9, 2, 8, device="cuda")
    start, lens = table([0, 3, 6]), table([3])

    def bad(error, *args, **kw):
        with pytest.raises(error):
            packed_attention(*args, **kw)

    bad(ValueError, q.double(), k.double(), k.double())
    bad(ValueError, q, k.half(), k)
    bad(ValueError, q, k, k[:8])
    bad(ValueError, q, k[..., :4], k[..., :4])
    bad(ValueError, q[:, :3], k, k)                 # 3 heads over 2
    bad(ValueError, q, k[:, :0], k[:, :0])
    bad(ValueError, q[0], k[0], k[0])
    bad(ValueError, q[None], k, k)
    bad(ValueError, q[None], k[None].expand(2, 9, 2, 8), k[None].expand(2, 9, 2, 8))
    bad(RuntimeError, q, k.cpu(), k)
    bad(RuntimeError, q, k, k, k_len=lens.cpu())
    bad(ValueError, q, k, k, k_len=lens.int())
    bad(ValueError, q, k, k, k_len=table([1, 2]))
    bad(ValueError, q, k, k, k_start=start)
    bad(ValueError, q, k, k, q_start=start, k_start=table([0, 9]))
    bad(ValueError, q, k, k, q_start=table([0]))
    bad(ValueError, q, k, k, q_start=start, k_len=lens)
    bad(ValueError, q[None], k[None], k[None], q_start=start)
    bad(ValueError, q, k, k, q_start=start[None])
    bad(ValueError, q, k, k, q_start=table([0, 1, 3, 3, 6, 6])[::2], k_start=start)
    bad(ValueError, *(torch.zeros(3, 1, 129, device="cuda") for _ in range(3)))
    bad(ValueError, q.to_sparse(), k, k)


@gpu
@pytest.mark.parametrize("binding", ["module", "ctypes"])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_differentiated_twice_raises(gpu_device, binding, which):
    native = _extension._C if binding == "module" else _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)
    x = [torch.randn(4, 2, 8, device="cuda", requires_grad=True) for _ in range(3)]
    y = native.attention(*x, None, None, None, None, False, 0.3)
    g, = torch.autograd.grad(y.sum(), x[which], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()


@gpu
def test_forward_mode_tracing_and_transforms_are_refused(gpu_device):
    x = torch.randn(4, 2, 8, device="cuda")
    for at in range(3):
        with torch.autograd.forward_ad.dual_level():
            args = [x] * 3
            args[at] = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="forward-mode"):
                packed_attention(*args)
    with pytest.raises(RuntimeError):
        torch.jit.trace(packed_attention, (x, x, x), check_trace=False)
    with pytest.raises(Exception):
        torch.func.vmap(packed_attention)(x[None], x[None], x[None])


@gpu
def test_autocast(gpu_device):
    x = torch.randn(50, 2, 32, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = packed_attention(x, x.half(), x.bfloat16())
        with pytest.raises(ValueError):
            packed_attention(x.double(), x, x)
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, packed_attention(x.bfloat16(), x.half().bfloat16(), x.bfloat16()))
