"""Attention of the encoder layer on the library's kernels (eve_attn_fwd / eve_attn_bwd; the reference's explicit
`softmax(q.float() @ k.float().T) @ v`, models/multiway_transformer.py:112-128): one pass over the keys forward, the
probabilities recomputed backward, a key mask, heads that share keys and values.  No CPU fallback.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import ops


def _check(q: Tensor, Nk: int, Hkv: int, key_mask: Optional[Tensor], scale: Optional[float], on: bool):
    """-> (key_mask, scale) as the kernels take them; q [.., H, D] with the batch in front.  Shapes first, then the device."""
    B, H, D = q.shape[0], q.shape[-2], q.shape[-1]
    if max(*q.shape, Nk, Hkv) >= 1 << 31:  # the C calls' sizes are 32-bit
        raise ValueError(f"eve_amd.attention: sizes {tuple(q.shape)}, {Nk} keys of {Hkv} heads (2^31 and more are not supported)")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"eve_amd.attention: {H} query heads cannot share {Hkv} key/value heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"eve_amd.attention: head width {D} (a multiple of 8 up to 128 is supported)")
    scale = D ** -0.5 if scale is None else float(scale)
    if not ops.ATTN_SCALES[0] <= scale <= ops.ATTN_SCALES[1]:
        raise ValueError(f"eve_amd.attention: scale {scale} (must lie between 2^-100 and 2^100)")
    if key_mask is not None:
        if key_mask.shape != (B, Nk):
            raise ValueError(f"eve_amd.attention: `key_mask` has shape {tuple(key_mask.shape)}, the keys need {(B, Nk)}")
        if key_mask.device != q.device:
            raise RuntimeError(f"eve_amd.attention: `key_mask` is on {key_mask.device}, the queries on {q.device}")
        key_mask = key_mask.bool().contiguous()
    if not on:
        raise RuntimeError(f"eve_amd.attention runs on one MI355X (queries on {q.device}); no CPU fallback")
    return key_mask, scale


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale):  # type: ignore[override]
        q, k, v = ops.attn_readable(q), ops.attn_readable(k), ops.attn_readable(v)
        need = any(ctx.needs_input_grad[:3])
        out, lse = ops.attn_fwd(q, k, v, key_mask, scale, want_lse=need)
        if need:
            ctx.save_for_backward(q, k, v, key_mask, out, lse)
            ctx.scale = scale
        return out

    @staticmethod
    @ops.once_differentiable
    def backward(ctx, dout):  # type: ignore[override]
        q, k, v, key_mask, out, lse = ctx.saved_tensors
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        ops.attn_bwd(ops.attn_dense(dout), q, k, v, key_mask, out, lse, ctx.scale, dq, dk, dv)
        return dq, dk, dv, None, None


class _SelfAttentionFn(torch.autograd.Function):
    """The three parts of one [B, N, 3, H, D] product, read where they lie; their gradient in one tensor of that shape."""

    @staticmethod
    def forward(ctx, qkv, key_mask, scale):  # type: ignore[override]
        qkv = ops.attn_readable(qkv)
        need = ctx.needs_input_grad[0]
        out, lse = ops.attn_qkv_fwd(qkv, key_mask, scale, want_lse=need)
        if need:
            ctx.save_for_backward(qkv, key_mask, out, lse)
            ctx.scale = scale
        return out

    @staticmethod
    @ops.once_differentiable
    def backward(ctx, dout):  # type: ignore[override]
        qkv, key_mask, out, lse = ctx.saved_tensors
        dqkv = qkv.new_empty(qkv.shape)
        ops.attn_qkv_bwd(ops.attn_dense(dout), qkv, key_mask, out, lse, ctx.scale, dqkv)
        return dqkv, None, None


def attention(q: Tensor, k: Tensor, v: Tensor, key_mask: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """softmax(scale q k^T) v over the keys that `key_mask` leaves, differentiable in q, k and v.

    q [B, Nq, H, D]; k, v [B, Nk, Hkv, D], float32 or bfloat16, at any strides (read in place where the last dimension is
    contiguous and rows start on 16-byte boundaries, else copied); H a multiple of Hkv: head h reads key head h // (H // Hkv).
    D is a multiple of 8 up to 128.  key_mask [B, Nk]: nonzero = visible.  scale: D ** -0.5 unless given, from 2^-100 to 2^100.
    -> [B, Nq, H, D].  A sample without a visible key gives zeros and passes no gradient (a row whose
    visible scores are all -inf is NaN, as the formula has it); masked keys and values may hold
    anything, NaN included.  Scores and sums are float32; results do not depend on the order of execution."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 4:
            raise ValueError(f"eve_amd.attention: `{n}` must be [B, N, heads, width], got {tuple(t.shape)}")
    ops._dt(q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"eve_amd.attention: q, k and v have types {q.dtype}, {k.dtype}, {v.dtype}: one is needed")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"eve_amd.attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not belong together")
    on = q.is_cuda and k.device == q.device and v.device == q.device
    key_mask, scale = _check(q, k.shape[1], k.shape[2], key_mask, scale, on)
    if ops._tracks(q, k, v):
        return _AttentionFn.apply(q, k, v, key_mask, scale)
    return ops.attn_fwd(ops.attn_readable(q), ops.attn_readable(k), ops.attn_readable(v), key_mask, scale, want_lse=False)[0]


def self_attention(qkv: Tensor, key_mask: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """`attention` over the three parts of one product qkv [B, N, 3, H, D] -> [B, N, H, D]; the gradient comes in qkv's shape."""
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"eve_amd.self_attention: `qkv` must be [B, N, 3, heads, width], got {tuple(qkv.shape)}")
    ops._dt(qkv)
    key_mask, scale = _check(qkv, qkv.shape[1], qkv.shape[3], key_mask, scale, qkv.is_cuda)
    if ops._tracks(qkv):
        return _SelfAttentionFn.apply(qkv, key_mask, scale)
    return ops.attn_qkv_fwd(ops.attn_readable(qkv), key_mask, scale, want_lse=False)[0]
