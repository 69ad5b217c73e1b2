"""Multi-scale deformable attention over 3-D volumes, built on the offset-mode op.

The caller of the reference's op computes the sampling locations (reference points + offsets
scaled per level), the attention logits, and concatenates them into ``sampling_loc_attn``
(reference tests/test_flash_deform_attn.py:30-37); its backward splits the gradient again.
``FlashDeformAttn3D`` produces the packed planar layout with ONE linear projection of the query
(for each head: the L*K (x,y,z) offsets in voxels of their level, then the L*K logits) and hands
it to ``FlashDeformAttnFromOffsets``, which forms the locations inside the kernels: no add,
divide, cat or split pass on either side of the op.  With ``level_value_proj`` the values of each
level have a projection of their own (``GroupedLinear`` over the flattened levels), and a ``residual``
given to the forward is added in the output projection's epilogue.

``SelfAttention3D`` is the layer beside it in which every token sees all others: object queries among
themselves, the tokens of a coarse level, or crops of different sizes packed one behind another.
"""
from __future__ import annotations

import math

import torch
from torch import nn

from .attention import packed_attention
from .flash_deform_attn import FlashDeformAttnFromOffsets
from .linear import fused_linear, grouped_linear
from .norm import layer_norm
from .rotary import rotary_positions


class GroupedLinear(nn.Module):
    """A linear layer with weights of its own for each of ``groups`` groups of consecutive rows.

    forward(x [S, in] or [B, S, in], group_start int64 [groups] or [groups + 1], residual=None) -> the
    same with ``out_features`` (see ``grouped_linear``; a level_start_index is a group_start)."""

    def __init__(self, groups: int, in_features: int, out_features: int, bias: bool = True, activation=None):
        super().__init__()
        self.groups, self.in_features, self.out_features, self.activation = groups, in_features, out_features, activation
        self.weight = nn.Parameter(torch.empty(groups, out_features, in_features))
        self.bias = nn.Parameter(torch.empty(groups, out_features)) if bias else None
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        for w in self.weight:
            nn.init.xavier_uniform_(w)
        if self.bias is not None:
            nn.init.zeros_(self.bias)

    def forward(self, x, group_start, residual=None):
        return grouped_linear(x, self.weight, group_start, self.bias, self.activation, residual)


def _plain_linear(m: nn.Module) -> bool:
    """Whether calling m is torch's linear product of its weight and bias and nothing else: no subclass
    (a parametrisation is one), no forward of its own, no hooks, no tensor subclasses (quantised weights)."""
    own = type(m) is nn.Linear and "forward" not in vars(m)
    hooks = any(getattr(m, name, None) for name in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks",
                                                    "_backward_pre_hooks"))
    return own and not hooks and not nn.modules.module._has_any_global_hook() and all(
        p is None or type(p) in (torch.Tensor, nn.Parameter) for p in (m.weight, m.bias))


class FlashDeformAttn3D(nn.Module):
    """value_proj -> deformable attention (FlashDeformAttnFromOffsets) -> output_proj.

    forward(query [B,Q,C], reference_points [B,Q,1 or L,3] float32 in [0,1], value [B,S,C],
    spatial_shapes [L,3] int64 (D,H,W), level_start_index [L] int64, residual [B,Q,C] or None) ->
    [B,Q,C], the residual added to output_proj's result (in its epilogue, where output_proj is a plain
    nn.Linear without hooks).  level_value_proj: value_proj
    has a weight and bias of its own for each level.
    """

    def __init__(self, embed_dim: int = 256, num_heads: int = 8, num_levels: int = 4, num_points: int = 4,
                 im2col_step: int = 64, level_value_proj: bool = False):
        super().__init__()
        if embed_dim % num_heads:
            raise ValueError(f"embed_dim ({embed_dim}) must be divisible by num_heads ({num_heads})")
        self.embed_dim, self.num_heads = embed_dim, num_heads
        self.num_levels, self.num_points = num_levels, num_points
        self.head_dim = embed_dim // num_heads
        self.im2col_step = im2col_step
        self.packed = 4 * num_levels * num_points   # per head: 3*L*K offsets, then L*K logits
        self.level_value_proj = level_value_proj
        self.value_proj = (GroupedLinear(num_levels, embed_dim, embed_dim) if level_value_proj
                           else nn.Linear(embed_dim, embed_dim))
        self.sampling = nn.Linear(embed_dim, num_heads * self.packed)
        self.output_proj = nn.Linear(embed_dim, embed_dim)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        if self.level_value_proj:
            self.value_proj.reset_parameters()
        else:
            nn.init.xavier_uniform_(self.value_proj.weight)
            nn.init.zeros_(self.value_proj.bias)
        nn.init.xavier_uniform_(self.output_proj.weight)
        nn.init.zeros_(self.output_proj.bias)
        # offsets start on a ring of directions per head, point k at k+1 voxels; logits at 0
        nn.init.zeros_(self.sampling.weight)
        G, L, K = self.num_heads, self.num_levels, self.num_points
        bias = torch.zeros(G, self.packed)
        golden = math.pi * (3.0 - math.sqrt(5.0))   # spread G directions over the sphere
        for g in range(G):
            zc = 1.0 - 2.0 * (g + 0.5) / G
            r = math.sqrt(max(0.0, 1.0 - zc * zc))
            d = torch.tensor([r * math.cos(golden * g), r * math.sin(golden * g), zc])
            d = d / d.abs().max()
            for l in range(L):
                for k in range(K):
                    s = l * K + k
                    bias[g, 3 * s: 3 * s + 3] = d * (k + 1)
        self.sampling.bias.copy_(bias.flatten())

    def forward(self, query, reference_points, value, spatial_shapes, level_start_index, residual=None):
        B, Q, C = query.shape
        S = value.shape[1]
        v = self.value_proj(value, level_start_index) if self.level_value_proj else self.value_proj(value)
        v = v.view(B, S, self.num_heads, self.head_dim)
        oa = self.sampling(query).view(B, Q, self.num_heads, self.packed)   # packed planar, as produced
        out = FlashDeformAttnFromOffsets.apply(v, spatial_shapes, level_start_index, oa,
                                               reference_points.to(torch.float32), self.im2col_step, self.num_points)
        if residual is None:
            return self.output_proj(out)
        if _plain_linear(self.output_proj):
            return fused_linear(out, self.output_proj.weight, self.output_proj.bias, residual=residual)
        return self.output_proj(out) + residual


class LayerNorm(nn.Module):
    """layer_norm over the last axis with a weight and a bias.  Kept in float32 beside 16-bit inputs, they get
    float32 gradients, and no input is cast."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.width, self.eps = width, eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class SelfAttention3D(nn.Module):
    """norm -> qkv -> rotary positions of queries and keys -> attention over all tokens -> output_proj, and x added.

    forward(x [B,S,C] or [S,C], positions [S,A] or [B,S,A] (float32 or int64), start, lengths) -> x's shape:
    x + output_proj(attention).  start [E + 1] int64 on x's device: the rows of x [S,C] are E packed
    sequences (see ``packed_attention``).  lengths [B] int64: how many rows of each item of x [B,S,C] count;
    the others see nothing and are seen by none.

    num_kv_heads key and value heads are shared by num_heads query heads.  sections: how many channel pairs
    of a head turn along each of the A axes; by default head_dim / 2 over three axes (depth, height, width), as
    evenly as they go, None of them with an empty tuple (positions are then not looked at).  The residual is
    added in output_proj's epilogue, where that is a plain nn.Linear without hooks.
    """

    def __init__(self, embed_dim: int = 256, num_heads: int = 8, num_kv_heads: int | None = None, sections=None,
                 theta: float = 10000.0, causal: bool = False, eps: float = 1e-5):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dim % num_heads:
            raise ValueError(f"embed_dim ({embed_dim}) must be divisible by num_heads ({num_heads})")
        if num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads})")
        self.embed_dim, self.num_heads, self.num_kv_heads = embed_dim, num_heads, num_kv_heads
        self.head_dim = embed_dim // num_heads
        pairs = self.head_dim // 2
        self.sections = tuple((pairs + a) // 3 for a in range(3)) if sections is None else tuple(sections)
        if sum(self.sections) > pairs:
            raise ValueError(f"sections {self.sections} do not fit heads of {self.head_dim} channels")
        self.theta, self.causal = theta, causal
        self.norm = LayerNorm(embed_dim, eps)
        self.qkv = nn.Linear(embed_dim, (num_heads + 2 * num_kv_heads) * self.head_dim)
        self.output_proj = nn.Linear(embed_dim, embed_dim)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        for m in (self.qkv, self.output_proj):
            nn.init.xavier_uniform_(m.weight)
            nn.init.zeros_(m.bias)

    def forward(self, x, positions=None, start=None, lengths=None):
        H, Hk = self.num_heads, self.num_kv_heads
        y = self.norm(x)
        y = fused_linear(y, self.qkv.weight, self.qkv.bias) if _plain_linear(self.qkv) else self.qkv(y)
        qk, v = y.unflatten(-1, (H + 2 * Hk, self.head_dim)).split([H + Hk, Hk], dim=-2)
        if self.sections:
            if positions is None:
                raise ValueError("positions are needed for the sections")
            qk = rotary_positions(qk, positions, self.sections, self.theta)
        q, k = qk.split([H, Hk], dim=-2)
        out = packed_attention(q, k, v, q_start=start, q_len=lengths, k_len=lengths, causal=self.causal).flatten(-2)
        if _plain_linear(self.output_proj):
            return fused_linear(out, self.output_proj.weight, self.output_proj.bias, residual=x)
        return self.output_proj(out) + x
