"""packed_attention where inputs are not finite, rows do not count, sums are cut into parts, numbers are small
or large for their type, and calls are many: against oracle/attention.py, or against the definition where a
result is not finite."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as ref
from ops3d_amd import _extension, packed_attention
from test_attention import DTYPES, check, gpu, make, table


def inputs(dtype, nq, nk, H, Hk, D, lead=(), seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [make(gen, (*lead, *s), DTYPES[dtype]) for s in ((nq, H, D), (nk, Hk, D), (nk, Hk, D), (nq, H, D))]


def step(q, k, v, u, **kw):
    """[y, dq, dk, dv]"""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = packed_attention(*leaves, **kw)
    return [y.detach(), *torch.autograd.grad(y, leaves, u)]


def parts(dtype, nq, nk, H, Hk, D, items=1, causal=False, sequences=0):
    """Whether the forward of this problem is cut into parts: its workspace holds them (and, of more than 64
    sequences, the table of tiles)."""
    p = _extension._AttentionProblem()
    for name, value in {"q_rows": nq, "k_rows": nk, "items": items, "heads": H, "kv_heads": Hk, "dim": D, "scale": 1.0, "causal": causal,
                        "dtype": list(DTYPES).index(dtype), "sequences": sequences}.items():
        setattr(p, name, value)
    if sequences:
        p.q_start = p.k_start = 256
        p.q_start_count = p.k_start_count = sequences + 1
    return _extension.load_library().ops3d_attention_forward_workspace_bytes(p) > 0


IN_PARTS = [(1, 8192, 4, 1, 64, False), (3, 5000, 2, 2, 32, False), (200, 9000, 8, 8, 32, False), (4200, 4200, 8, 8, 32, True), (3, 5000, 2, 1, 128, True)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,H,Hk,D,causal", IN_PARTS)
def test_nan_reaches_queries_whose_keys_are_cut_into_parts(gpu_device, nq, nk, H, Hk, D, causal, dtype):
    """A part whose logits are all NaN has no largest one, and counts all the same."""
    assert parts(dtype, nq, nk, H, Hk, D, causal=causal)
    q, k, v, u = inputs(dtype, nq, nk, H, Hk, D, seed=nq)
    want = ref.sequence(q, k, v, causal, D ** -0.5, u)
    other = slice(H // Hk, H) if Hk > 1 else slice(0, 0)   # query heads of other key heads than the first
    bad = q.clone()
    bad[nq // 2, 0, 1] = math.nan
    y, dq, _, _ = step(bad, k, v, u, causal=causal)
    keep = torch.ones(nq, H, dtype=torch.bool, device="cuda")
    keep[nq // 2, 0] = False
    assert y[nq // 2, 0].isnan().all() and dq[nq // 2, 0].isnan().all()
    for name, got in (("y", y), ("dq", dq)):
        check(name, got[keep], tuple(t[keep] for t in want[name]))
    for keys in (slice(0, nk), slice(0, nk - nk // 3), slice(nk // 3, nk), slice(128, 1024)):
        bad = k.clone()
        bad[keys, 0, D - 1] = math.nan
        y, dq, dk, dv = step(q, bad, v, u, causal=causal)
        first = max(0, keys.start - (nk - nq)) if causal else 0   # the first query that sees one of them
        assert y[first:, :H // Hk].isnan().all() and dq[first:, :H // Hk].isnan().all()
        assert dk[keys, 0].isnan().all() and dv[keys, 0].isnan().all()
        for name, got in (("y", y), ("dq", dq)):
            check(name, got[:first], tuple(t[:first] for t in want[name]))
            check(name, got[:, other], tuple(t[:, other] for t in want[name]))
        with torch.no_grad():
            assert torch.equal(packed_attention(q, bad, v, causal=causal).isnan(), y.isnan())


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nq,nk,H,Hk,D", [(3, 5000, 2, 1, 64), (5, 4000, 4, 4, 128), (70, 6000, 4, 2, 32), (70, 90, 4, 2, 32)])
def test_gradients_of_rows_that_do_not_count(gpu_device, nq, nk, H, Hk, D, value, dtype):
    """Zeros, also beside keys and values that are not finite, in parts or not."""
    q, k, v, u = inputs(dtype, nq, nk, H, Hk, D, lead=(2,), seed=nq)
    k[0, 7, 0, 0], v[0, nk - 1, Hk - 1, 1], k[1, nk // 2, 0, 0], v[1, 5, 0, 1] = value, value, value, value
    lens = [nq - 1, nq // 3]
    q_len = table(lens)
    y, dq, _, _ = step(q, k, v, u, q_len=q_len)
    for i, n in enumerate(lens):
        assert not y[i, n:].any() and not dq[i, n:].any()
    y, dq, _, _ = step(q[0], k[0], v[0], u[0], q_start=table([1, lens[0]]), k_start=table([0, nk]))
    for t in (y, dq):
        assert not t[:1].any() and not t[lens[0]:].any()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,H,Hk,D", [(1, 70, 2, 2, 32), (5, 70, 2, 2, 32), (70, 70, 4, 2, 32), (9000, 70, 2, 2, 32), (333, 8000, 6, 2, 64), (70, 300, 2, 2, 128),
                                          (70, 300, 2, 2, 36), (5000, 20000, 6, 2, 32)])
def test_infinity_in_the_last_output_gradient(gpu_device, nq, nk, H, Hk, D, dtype):
    """Rows behind the last one in its tile have no weight: an infinity in the last one stays one in the values'
    gradients, and the other channels know nothing of it."""
    q, k, v, u = inputs(dtype, nq, nk, H, Hk, D, seed=nq)
    value, bound = ref.sequence(q, k, v, False, D ** -0.5, u)["dv"]
    u[-1, H // Hk - 1, 3], u[-1, H - 1, 4] = math.inf, -math.inf
    _, _, _, dv = step(q, k, v, u)
    assert (dv[:, 0, 3] == math.inf).all() and (dv[:, Hk - 1, 4] == -math.inf).all()
    keep = torch.isfinite(dv)
    assert keep.sum() == dv.numel() - 2 * nk
    check("dv", dv[keep], (value[keep], bound[keep]))


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,H,Hk,D", [(1, 70, 2, 2, 32), (5, 70, 2, 1, 36), (70, 300, 6, 2, 64), (70, 300, 2, 2, 128), (9000, 70, 2, 2, 32), (333, 5000, 2, 2, 33)])
def test_keys_whose_logits_are_all_minus_infinity(gpu_device, nq, nk, H, Hk, D, dtype):
    """Such keys have no weight, and gradients of 0: rows behind the last query, zeros or not, are no queries of theirs."""
    q, k, v, u = inputs(dtype, nq, nk, H, Hk, D, seed=nq)
    q[..., 0] = q[..., 0].abs() + 0.5
    gone = [0, nk // 2, nk - 1]
    k[gone, :, 0] = -math.inf
    y, dq, dk, dv = step(q, k, v, u)
    left = torch.ones(nk, dtype=torch.bool, device="cuda")
    left[gone] = False
    want = ref.sequence(q, k[left], v[left], False, D ** -0.5, u)
    assert not dk[gone].any() and not dv[gone].any()
    check("y", y, want["y"])
    check("dq", dq[..., 1:], tuple(t[..., 1:] for t in want["dq"]))   # 0 times the infinity in the first channel
    check("dk", dk[left], want["dk"])
    check("dv", dv[left], want["dv"])


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,H,Hk,D", [(5, 9, 2, 1, 32), (70, 150, 4, 2, 36), (1, 600, 2, 1, 64), (1, 8192, 4, 1, 64), (200, 9000, 8, 8, 32), (2600, 2600, 8, 8, 32)])
def test_logits_that_are_all_minus_infinity(gpu_device, nq, nk, H, Hk, D, dtype):
    """Softmax of them is NaN, as their keys are: a query is only 0 where it sees no key."""
    q, k, v, u = inputs(dtype, nq, nk, H, Hk, D, seed=nk)
    q[..., 0] = 1
    k[:, 0, 0] = -math.inf
    y, dq, dk, dv = step(q, k, v, u)
    own = slice(0, H // Hk)   # the first key head's queries
    for t in (y[:, own], dq[:, own], dk[:, 0], dv[:, 0]):
        assert t.isnan().all()
    assert torch.isfinite(y[:, H // Hk:]).all() and torch.isfinite(dq[:, H // Hk:]).all()
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v).isnan(), y.isnan())


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,H,Hk,D", [(90, 2, 1, 32), (700, 2, 2, 64), (4200, 8, 8, 32), (2300, 8, 2, 128)])
def test_one_logit_of_minus_infinity(gpu_device, n, H, Hk, D, dtype):
    """Causal: the first key has it.  The first query sees no other and gives NaN, the rest as without that key; queries
    before the keys see none and give 0."""
    q, k, v, u = inputs(dtype, n, n, H, Hk, D, seed=n)
    q[..., 0] = 1
    bad = k.clone()
    bad[0, :, 0] = -math.inf
    y, dq, dk, dv = step(q, bad, v, u, causal=True)
    assert y[0].isnan().all() and dq[0].isnan().all() and dk[0].isnan().all() and dv[0].isnan().all()
    want = ref.sequence(q[1:], k[1:], v[1:], True, D ** -0.5, u[1:])
    check("y", y[1:], want["y"])
    check("dq", dq[1:, :, 1:], tuple(t[..., 1:] for t in want["dq"]))   # 0 times the infinity in the first channel
    check("dk", dk[1:], want["dk"])
    check("dv", dv[1:], want["dv"])
    y, dq, dk, dv = step(q, k[:n // 2], v[:n // 2], u, causal=True)
    first = n - n // 2
    assert not y[:first].any() and not dq[:first].any() and y[first:].any(-1).all()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nk", [9, 300, 5000])
def test_infinite_outputs_and_their_gradients(gpu_device, nk, dtype):
    """An infinite value makes the output's product with its gradient infinite, and the other keys' gradients with it."""
    q, k, v, u = inputs(dtype, 1, nk, 1, 1, 32, seed=nk)
    v[4, 0, 2] = math.inf
    y, dq, dk, dv = step(q, k, v, u)
    assert y[0, 0, 2] == math.inf and torch.isfinite(y).sum() == 31
    others = torch.arange(nk, device="cuda") != 4
    sign = -torch.sign(u[0, 0, 2]) * torch.sign(q[0])   # logits' gradients are P (dP - delta)
    assert torch.equal(dk[others], (sign * math.inf)[None].expand(nk - 1, 1, 32))
    assert dk[4].isnan().all() and dq.isnan().all() and torch.isfinite(dv).all()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("nq,nk,D,causal", [(1, 20, 32, False), (5, 90, 33, False), (70, 70, 32, True), (300, 400, 64, True), (300, 300, 128, True), (5, 5000, 32, True)])
def test_infinite_gradients_beside_finite_ones(gpu_device, nq, nk, D, causal, dtype):
    """One head of one query has an infinite output gradient, that of the first key's logit is minus infinity: the key's
    gradient is an infinity of the query's sign, whatever the other rows of the tile are, hidden ones among them."""
    q, k, v, u = inputs(dtype, nq, nk, 2, 1, D, seed=nq)
    row = nq // 2
    last = nk - nq + row if causal else nk - 1   # the last key that it sees
    v[:, 0, 1] = v[:, 0, 1].abs() + 0.25
    v[0, 0, 1] = -0.01
    u[row, 1, 1] = math.inf
    _, dq, dk, dv = step(q, k, v, u, causal=causal)
    assert torch.equal(dk[0, 0], -torch.sign(q[row, 1]) * math.inf)
    assert dk[1:last + 1].isnan().all() and torch.isfinite(dk[last + 1:]).all()
    assert (dv[:last + 1, 0, 1] == math.inf).all() and torch.isfinite(dv[last + 1:]).all() and torch.isfinite(dv[:, 0, 2:]).all()
    assert dq[row, 1].isnan().all() and torch.isfinite(dq).sum() == dq.numel() - D


@gpu
@pytest.mark.parametrize("nq,nk,H,Hk,D,causal", [(50, 6000, 2, 1, 32, False), (700, 700, 4, 2, 64, True), (6000, 50, 2, 2, 32, False), (300, 300, 2, 1, 128, False),
                                                 (300, 400, 3, 1, 36, True), (9000, 9000, 8, 8, 32, True), (1, 8192, 8, 2, 128, False)])
@pytest.mark.parametrize("size", [1e-4, 1.0, 2000.0])
def test_fp16_gradients_of_small_and_large_ones(gpu_device, size, nq, nk, H, Hk, D, causal):
    """Logits' gradients are held in fp16 times a power of two of their query's or key's own."""
    q, k, v, u = inputs("fp16", nq, nk, H, Hk, D, seed=nq)
    if size > 1:   # products of v and grad_out pass fp16, what is made of them does not
        q, k, v = q * 0.01, k * 0.01, v * 100
    u = (u.float() * size).half()
    want = ref.sequence(q, k, v, causal, D ** -0.5, u)
    for name, got in zip(("y", "dq", "dk", "dv"), step(q, k, v, u, causal=causal)):
        value, bound = want[name]
        fits = value.abs() + bound < 65504
        assert fits.float().mean() > 0.9, name
        check(name, got[fits], (value[fits], bound[fits]))


@gpu
def test_fp16_gradients_that_grow_along_the_sum(gpu_device):
    """Each query's and each key's largest comes last, or first, over many powers of two; zeros first."""
    q, k, v, u = inputs("fp16", 600, 700, 2, 1, 32, seed=3)
    for flip in (False, True):
        up = torch.exp2(torch.linspace(-20, 9, 600, device="cuda"))[:, None, None]
        down = torch.exp2(torch.linspace(-14, 5, 700, device="cuda"))[:, None, None]
        if flip:
            up, down = up.flip(0), down.flip(0)
        uu, vv = (u * up).half(), (v * down).half()
        uu[:40] = 0
        want = ref.sequence(q, k, vv, False, 32 ** -0.5, uu)
        for name, got in zip(("y", "dq", "dk", "dv"), step(q, k, vv, uu)):
            check(name, got, want[name])


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,D", [(70, 33), (200, 36), (700, 64), (300, 128)])
def test_infinite_gradients_again_and_again(gpu_device, n, D, dtype):
    """Of several queries far apart: the sums, infinities by then, are scaled no further."""
    q, k, v, u = inputs(dtype, n, n, 1, 1, D, seed=n)
    q = q.abs() + 0.25
    v[:, 0, 1] = v[:, 0, 1].abs() + 0.25
    v[0, 0, 1] = -0.01
    rows = [2, n // 2, n - 1]
    u[rows, 0, 1] = math.inf
    _, dq, dk, dv = step(q, k, v, u)
    assert (dk[0] == -math.inf).all() and dk[1:].isnan().all()
    assert (dv[:, 0, 1] == math.inf).all() and torch.isfinite(dv).sum() == dv.numel() - n
    assert dq[rows].isnan().all() and torch.isfinite(dq).sum() == dq.numel() - 3 * D


@gpu
def test_more_blocks_than_one_launch_has(gpu_device):
    """2^24 blocks of 256 threads and some: items of one token, whose result is the value."""
    items = (1 << 21) + 5
    gen = torch.Generator(device="cuda").manual_seed(17)
    q, k, v, u = (torch.randint(-3, 4, (items, 1, 8, 8), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16) for _ in range(4))
    y, dq, dk, dv = step(q, k, v, u)
    assert torch.equal(y, v) and torch.equal(dv, u) and not dq.any() and not dk.any()


def wide(dtype, rows, runs, H, Hk):
    """Blocks of 128 columns of queries, and of keys: from 512 on attention_capi.hip takes these tiles."""
    return [-(-rows * g // 128) * runs * Hk for g in (H // Hk, 1)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,group", [(32, 1), (32, 3), (36, 1), (64, 4), (128, 1), (128, 3)])
def test_tiles_of_128_columns(gpu_device, dim, group, causal, dtype):
    """Many items of more than 128 tokens, with lengths and without."""
    items, n, Hk = 32, 150, 8
    assert min(wide(dtype, n, items, group * Hk, Hk)) >= 512
    q, k, v, u = inputs(dtype, n, n, group * Hk, Hk, dim, lead=(items,), seed=dim)
    for lens in (None, [(41 * i) % (n + 1) for i in range(items)]):
        got = step(q, k, v, u, causal=causal, q_len=table(lens), k_len=table(lens))
        want = ref.items(q, k, v, lens, lens, causal, dim ** -0.5, u)
        for name, t in zip(("y", "dq", "dk", "dv"), got):
            check(name, t, want[name])


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sequences,dim,group,cross", [(40, 32, 3, True), (40, 64, 4, False), (40, 128, 1, True), (70, 32, 1, False), (70, 128, 1, True)])
def test_packed_tiles_of_128_columns(gpu_device, sequences, dim, group, cross, causal, dtype):
    """Sequences in the order of what they see, and looked up in a table."""
    Hk, rows = 8, sequences * 150
    assert min(wide(dtype, 150, sequences, group * Hk, Hk)) >= 512
    gen = torch.Generator().manual_seed(dim)

    def starts():
        return [3] + sorted(torch.randint(3, rows - 5, (sequences - 1,), generator=gen).tolist()) + [rows - 5]

    q_start = starts()
    k_start = starts() if cross else q_start
    q, k, v, u = inputs(dtype, rows, rows, group * Hk, Hk, dim, seed=dim)
    got = step(q, k, v, u, causal=causal, q_start=table(q_start), k_start=table(k_start))
    want = ref.packed(q, k, v, q_start, k_start, causal, dim ** -0.5, u)
    for name, t in zip(("y", "dq", "dk", "dv"), got):
        check(name, t, want[name])


@gpu
@pytest.mark.parametrize("sequences", [5, 70])
def test_c_starts_without_the_last_end(gpu_device, sequences):
    """From C: with `sequences` entries the last sequence ends with the rows."""
    rows, H, D = 900, 2, 32
    gen = torch.Generator().manual_seed(sequences)
    start = [0] + sorted(torch.randint(0, rows, (sequences - 1,), generator=gen).tolist())
    q, k, v, u = inputs("bf16", rows, rows, H, H, D)
    native = _extension._NativeFDA(_extension.load_library(), _extension.LIB_PATH)
    outs = []
    for count in (sequences, sequences + 1):
        at = table(start + [rows])[:count].clone()
        p = native._attention_problem(q, k, v, table(start + [rows]), table(start + [rows]), None, None, True, 0.2)
        assert p.sequences == sequences
        p.q_start = p.k_start = at.data_ptr()
        p.q_start_count = p.k_start_count = count
        y, dq, dk, dv = (torch.full_like(q, math.nan) for _ in range(4))
        lse, n = torch.empty(1, H, rows, device="cuda"), native._lib.ops3d_attention_forward_workspace_bytes(p)
        m = native._lib.ops3d_attention_backward_workspace_bytes(p)
        ws = torch.empty(max(n, m, 1), dtype=torch.uint8, device="cuda")
        tq, tk, tv, ty, tu, tgq, tgk, tgv = (native._attention_tensor(t) for t in (q, k, v, y, u, dq, dk, dv))
        stream = torch.cuda.current_stream().cuda_stream
        assert native._lib.ops3d_attention_forward(p, tq, tk, tv, ty, None, lse.data_ptr(), ws.data_ptr(), n, stream) == 0
        assert native._lib.ops3d_attention_backward(p, tq, tk, tv, ty, None, lse.data_ptr(), tu, tgq, tgk, tgv, ws.data_ptr(), m, stream) == 0
        torch.cuda.synchronize()
        outs.append((y, dq, dk, dv))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(outs[0][0], packed_attention(q, k, v, q_start=table(start + [rows]), causal=True, scale=0.2))
