"""Cross attention to an encoder's states of another length, forward and backward as HIP kernels (csrc/cross_attention_*.hip, C ABI
include/rlipv2_attention.h; workspaces and the autograd node: csrc/torch_operators.cpp).

`cross_attention` is the operator, `CrossAttention` the module around it.  It takes what the fixed-size core of the ALIF fusion
(`alif.AlifAttentionFunction`) does not: any lengths from one query or key on, heads of 8 to 256 elements, heads that share a key
head, padding that really masks, float32, strided operands.  `RLIPv2_BiMultiHeadAttention` runs both directions of the fusion
through it with `alif.cross_attention_core` switched on (reference models/fuse_helper.py:395-462)."""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, roofline

_DTYPES = (torch.float32, torch.bfloat16)


def cross_attention(query, key, value, key_padding_mask=None, key_lengths=None, scale=None, keep=None, keep_scale=1.0):
    """softmax(scale query key^T) value over the keys that count, [B, Lq, H, D].

    query [B, Lq, H, D], key / value [B, Lk, Hk, D]: bfloat16 or float32, all of one type, on one GPU; H a multiple of Hk (query
    head h reads key head h // (H // Hk)), D a multiple of 8 up to 256.  Any strides: operands whose heads are not contiguous or
    whose rows are not 16-byte aligned are copied first.  A key / value of batch stride 0 (`expand`) is read in place.
    key_padding_mask [B, Lk] bool: True marks keys that do not count (as `NestedTensor.mask`); key_lengths [B] int32: only the
    first ones count.  Both may be given.  Masked keys and values are never multiplied with (a NaN there stays there) and get
    zero gradients; a query without any key gives zeros.
    scale: 1e-30 to 1e30, 1 / sqrt(D) by default.  keep [B, H, Lq, Lk] bool or uint8: dropout mask of the probabilities, kept ones are
    multiplied by `keep_scale`.
    Sums, maxima and gradients are accumulated in float32; calls are repeatable bit for bit.  bfloat16 rounds the probabilities, and in
    the backward pass of calls of more than 2^24 of them (batch and heads included) or with `keep` also dS, for the products with them:
    errors of 1.1 (result) and 1.4 times (those gradients) a rounded exact value's; smaller calls' gradients are at 1.0.  Differentiable (once, in
    reverse mode) in query, key and value; capturable in a HIP graph."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"cross_attention: {name} must be a [batch, tokens, heads, head size] tensor")
    if query.dtype not in _DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError(f"cross_attention: query, key and value must all be bfloat16 or all float32 (got {query.dtype}, {key.dtype}, "
                        f"{value.dtype})")
    B, Lq, H, D = query.shape
    Lk, Hk = key.shape[1], key.shape[2]
    if key.shape != value.shape or key.shape[0] != B or key.shape[3] != D:
        raise ValueError(f"cross_attention: key and value must be [{B}, Lk, Hk, {D}] (got {tuple(key.shape)}, {tuple(value.shape)})")
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"cross_attention: {H} query heads cannot share {Hk} key heads")
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"cross_attention: the head size must be a multiple of 8 up to 256 (got {D})")
    if scale is None:
        scale = D ** -0.5
    scale, keep_scale = float(scale), float(keep_scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"cross_attention: scale must lie between 1e-30 and 1e30 (got {scale})")
    if key_padding_mask is not None:
        if key_padding_mask.dtype != torch.bool or key_padding_mask.shape != (B, Lk):
            raise ValueError(f"cross_attention: key_padding_mask must be a bool tensor [{B}, {Lk}], True where a key does not count")
        if key_padding_mask.stride(1) != 1:
            key_padding_mask = key_padding_mask.contiguous()
    if key_lengths is not None:
        if key_lengths.dtype != torch.int32 or key_lengths.shape != (B,):
            raise ValueError(f"cross_attention: key_lengths must be an int32 tensor [{B}]")
        key_lengths = key_lengths.contiguous()
    if keep is not None:
        if keep.dtype not in (torch.bool, torch.uint8) or keep.shape != (B, H, Lq, Lk):
            raise ValueError(f"cross_attention: keep must be a bool or uint8 tensor [{B}, {H}, {Lq}, {Lk}]")
        keep = keep.contiguous()
    device = query.device
    for name, t in (("key", key), ("value", value), ("key_padding_mask", key_padding_mask), ("key_lengths", key_lengths), ("keep", keep)):
        if t is not None and t.device != device:
            raise RuntimeError(f"cross_attention: {name} must be on the query's device")
    if not query.is_cuda:
        raise RuntimeError("Not implemented on the CPU")
    out = _lib.operators().cross_attention(query, key, value, key_padding_mask, key_lengths, keep, scale, keep_scale)
    if roofline.active:
        # (the backward node is C++ and reports nothing: its operands are added here, where it will run)
        moved = roofline.tensor_bytes(query, key, value, key_padding_mask, key_lengths, keep, out)
        again = roofline.tensor_bytes(query, key, value, out) if out.requires_grad else 0
        roofline.add(moved + (moved + again if again else 0), (14 if again else 4) * B * H * Lq * Lk * D)
    return out


class CrossAttention(nn.Module):
    """Multi-head attention of queries [B, Lq, embed_dim] to an encoder's states [B, Lk, states_dim] of another length.

    `project_states(states)` gives the key and value heads; a server that asks one image or text again and again keeps them and
    passes them as `projected`, which leaves the query projection, one kernel and the output projection per call.  `num_kv_heads`:
    key heads shared by groups of query heads."""

    def __init__(self, embed_dim, num_heads, states_dim=None, num_kv_heads=None, head_dim=None, dropout=0.0, bias=True):
        super().__init__()
        self.num_heads = num_heads
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        self.head_dim = embed_dim // num_heads if head_dim is None else head_dim
        if num_heads % self.num_kv_heads:
            raise ValueError(f"{num_heads} query heads cannot share {self.num_kv_heads} key heads")
        if head_dim is None and self.head_dim * num_heads != embed_dim:
            raise ValueError(f"embed_dim {embed_dim} is not divisible by num_heads {num_heads}")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"dropout must be at least 0 and below 1 (got {dropout})")
        states_dim = embed_dim if states_dim is None else states_dim
        self.dropout = dropout
        self.q_proj = nn.Linear(embed_dim, num_heads * self.head_dim, bias=bias)
        self.k_proj = nn.Linear(states_dim, self.num_kv_heads * self.head_dim, bias=bias)
        self.v_proj = nn.Linear(states_dim, self.num_kv_heads * self.head_dim, bias=bias)
        self.out_proj = nn.Linear(num_heads * self.head_dim, embed_dim, bias=bias)
        for lin in (self.q_proj, self.k_proj, self.v_proj, self.out_proj):
            nn.init.xavier_uniform_(lin.weight)
            if lin.bias is not None:
                nn.init.zeros_(lin.bias)

    def project_states(self, states, states_pos=None):
        """(key, value) heads [B, Lk, num_kv_heads, head_dim] of encoder states; `states_pos` is added for the keys only"""
        B, T, _ = states.shape
        k = self.k_proj(states if states_pos is None else states + states_pos)
        return (k.view(B, T, self.num_kv_heads, self.head_dim), self.v_proj(states).view(B, T, self.num_kv_heads, self.head_dim))

    def forward(self, query, states=None, query_pos=None, states_pos=None, key_padding_mask=None, key_lengths=None, projected=None):
        if (states is None) == (projected is None):
            raise ValueError("CrossAttention: give either states or projected (from project_states)")
        key, value = self.project_states(states, states_pos) if projected is None else projected
        B, T, _ = query.shape
        q = self.q_proj(query if query_pos is None else query + query_pos).view(B, T, self.num_heads, self.head_dim)
        keep = None
        if self.training and self.dropout > 0.0:
            keep = torch.rand((B, self.num_heads, T, key.shape[1]), device=query.device) >= self.dropout
        out = cross_attention(q, key, value, key_padding_mask=key_padding_mask, key_lengths=key_lengths, keep=keep,
                              keep_scale=1.0 / (1.0 - self.dropout) if keep is not None else 1.0)
        return self.out_proj(out.reshape(B, T, self.num_heads * self.head_dim))
