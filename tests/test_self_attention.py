"""SelfAttention3D: norm, projection, rotary positions, attention and output projection as they are used together,
against the same layer in plain float64 operations."""
from __future__ import annotations

import math

import pytest
import torch

from ops3d_amd import (SelfAttention3D, axial_frequencies, fused_linear, layer_norm, packed_attention, rotary_positions)

gpu = pytest.mark.gpu


def plain(m, x, positions, spans):
    """The layer on x [S, C] in float64, for the sequences [a, b) of spans; x for rows of none is itself plus the bias."""
    p = {n: t.double() for n, t in m.named_parameters()}
    H, Hk, D = m.num_heads, m.num_kv_heads, m.head_dim
    n = torch.nn.functional.layer_norm(x, (m.embed_dim,), p["norm.weight"], p["norm.bias"], m.norm.eps)
    rows = (n @ p["qkv.weight"].t() + p["qkv.bias"]).unflatten(-1, (H + 2 * Hk, D))
    if sum(m.sections):
        P = sum(m.sections)
        axis = [a for a, k in enumerate(m.sections) for _ in range(k)]
        angle = (positions.double()[:, axis] * torch.tensor(axial_frequencies(m.sections, m.theta), dtype=torch.float64, device=x.device))[:, None]
        a, b, rest = rows[:, :H + Hk, :P], rows[:, :H + Hk, P:2 * P], rows[:, :H + Hk, 2 * P:]
        turned = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), rest], -1)
        rows = torch.cat([turned, rows[:, H + Hk:]], 1)
    out = torch.zeros(len(x), H, D, dtype=torch.float64, device=x.device)
    pieces = []
    for a, b in spans:
        q, k, v = (t.transpose(0, 1) for t in rows[a:b].split([H, Hk, Hk], 1))
        k, v = (t.repeat_interleave(H // Hk, 0) for t in (k, v))
        s = q @ k.transpose(1, 2) / math.sqrt(D)
        if m.causal:
            s = s.masked_fill(torch.ones(b - a, b - a, device=x.device, dtype=torch.bool).triu(1), -math.inf)
        pieces.append((a, b, (torch.softmax(s, -1) @ v).transpose(0, 1)))
    for a, b, t in pieces:
        out = torch.cat([out[:a], t, out[b:]])
    return out.flatten(1) @ p["output_proj.weight"].t() + p["output_proj.bias"] + x


def layer(dtype=torch.float32, **kw):
    torch.manual_seed(0)
    m = SelfAttention3D(**{"embed_dim": 128, "num_heads": 4, "num_kv_heads": 2, **kw}).cuda()
    with torch.no_grad():
        for t in m.parameters():
            t.add_(0.05 * torch.randn_like(t))
    return m.to(dtype)


def test_constructor():
    m = SelfAttention3D(96, 3)
    assert m.sections == (5, 5, 6) and m.qkv.out_features == 3 * 96 and m.num_kv_heads == 3
    for kw in ({"num_heads": 7}, {"num_heads": 8, "num_kv_heads": 3}, {"num_kv_heads": 0}, {"sections": (10, 10, 10)}):
        with pytest.raises(ValueError):
            SelfAttention3D(256, **kw) if "num_heads" in kw else SelfAttention3D(256, 8, **kw)


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sections", [None, (3, 4), ()])
def test_against_plain_operations(gpu_device, causal, sections):
    """fp32: five steps of sums of at most 512 products, each off by 512 2^-24 of its terms' size at worst, and
    conditioned by a factor of a few: 1e-3 of the largest value bounds the values, and their gradients, twice as
    many steps."""
    m = layer(causal=causal, sections=sections)
    gen = torch.Generator(device="cuda").manual_seed(1)
    S, axes = 217, len(m.sections) or 1
    x = torch.randn(S, 128, generator=gen, device="cuda", requires_grad=True)
    u = torch.randn(S, 128, generator=gen, device="cuda")
    pos = torch.randint(0, 64, (S, axes), generator=gen, device="cuda")
    start = torch.tensor([0, 40, 40, 150, 210], device="cuda")
    y = m(x, pos, start=start)
    leaves = [x, *m.parameters()]
    grads = torch.autograd.grad(y, leaves, u)
    wide = SelfAttention3D(128, 4, 2, sections=m.sections, causal=causal).cuda().double()
    wide.load_state_dict({k: t.double() for k, t in m.state_dict().items()})
    xd = x.detach().double().requires_grad_(True)
    want = plain(wide, xd, pos, [(0, 40), (40, 150), (150, 210)])
    exact = torch.autograd.grad(want, [xd, *wide.parameters()], u.double())
    for name, a, b in zip(["y", "x", *(n for n, _ in m.named_parameters())], (y, *grads), (want, *exact)):
        assert (a.double() - b).abs().max() <= 1e-3 * b.abs().max(), name


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_is_its_operators(gpu_device, dtype):
    """A batch with lengths, bit by bit; an item alone gives what it gives in the batch."""
    m = layer(dtype)
    x = torch.randn(3, 70, 128, device="cuda").to(dtype)
    pos = torch.randint(0, 32, (70, 3), device="cuda")
    lengths = torch.tensor([70, 33, 0], device="cuda")
    with torch.no_grad():
        y = m(x, pos, lengths=lengths)
        n = layer_norm(x, m.norm.weight, m.norm.bias)
        rows = fused_linear(n, m.qkv.weight, m.qkv.bias).view(3, 70, 8, 32)
        qk = rotary_positions(rows[:, :, :6], pos, m.sections)
        o = packed_attention(qk[:, :, :4], qk[:, :, 4:], rows[:, :, 6:], q_len=lengths, k_len=lengths).flatten(2)
        assert torch.equal(y, fused_linear(o, m.output_proj.weight, m.output_proj.bias, residual=x))
        assert not o[1, 33:].any() and not o[2].any()


@gpu
def test_hooks_and_replacements_are_called(gpu_device):
    m = layer()
    x, pos = torch.randn(20, 128, device="cuda"), torch.zeros(20, 3, device="cuda")
    seen = []
    want = m(x, pos)
    for sub in (m.qkv, m.output_proj):
        sub.register_forward_hook(lambda *a: seen.append(1))
    assert torch.allclose(m(x, pos), want, atol=1e-4) and len(seen) == 2
    with pytest.raises(ValueError, match="positions"):
        m(x)


@gpu
def test_training_step_captured(gpu_device):
    """Forward and backward in a graph, replayed on new values and new sequences, against the eager step."""
    m = layer(torch.bfloat16, causal=True)
    params = list(m.parameters())
    x = torch.randn(300, 128, device="cuda").bfloat16()
    pos = torch.randint(0, 32, (300, 3), device="cuda")
    start = torch.tensor([0, 100, 300], device="cuda")

    def step(x, start):
        leaf = x.detach().requires_grad_(True)
        y = m(leaf, pos, start=start)
        return [y.detach(), *torch.autograd.grad(y, [leaf, *params], x)]

    sx, ss = x.clone(), start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, ss)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(sx, ss)
    for seed, bounds in enumerate(([0, 10, 300], [5, 5, 290], [0, 150, 300])):
        sx.copy_(torch.randn(300, 128, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        ss.copy_(torch.tensor(bounds))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step(sx, ss)))


@gpu
def test_autocast_keeps_norm_in_32_bits(gpu_device):
    m = layer()
    x, pos = torch.randn(50, 128, device="cuda"), torch.randint(0, 9, (50, 3), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, pos)
    assert y.dtype == torch.float32   # the residual's
    assert (y - m(x, pos)).abs().max() < 0.1
