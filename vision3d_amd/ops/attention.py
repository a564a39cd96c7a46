"""Softmax attention of the transformer layers over packs: inside every sequence (cloud) of a pack, and of new tokens
against a cache of keys and values.  The reference's layers pad a pack to a batch, mask, and materialise the (N, M) scores
of every head; here the scores live in registers, sequences of any lengths lie one behind the other, and the lengths stay
on the device (no synchronisation).
"""
from typing import Optional

import torch
from torch import Tensor

from .. import ext
from ._autograd import recorded


def _require_cuda(name, q, k, v):
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError(f"{name}: CUDA tensors required (no CPU fallback in vision3d_amd)")


def _rows(t: Tensor, group: int) -> Tensor:
    """The strides that the kernels take: any but the last dimension's, which is 1, as long as a tile's rows (129 at most, of
    ``group`` heads: the queries of one key head, or 0 for keys) lie within 32-bit byte offsets; other inputs are copied."""
    shape = t.shape
    if len(shape) < 3 or t.is_contiguous() or t.numel() == 0:
        return t
    row, head, unit = t.stride()[-3:]
    rows, heads, dim = shape[-3:]
    row, head = 0 if rows == 1 else row, 0 if heads == 1 else head
    near = 129 * row + group * head + dim < 1 << 29
    return t if unit == 1 and (row == 0 or row >= dim) and near else t.contiguous()


def _operands(q: Tensor, k: Tensor, v: Tensor):
    if q.is_contiguous() and k.is_contiguous() and v.is_contiguous():
        return q, k, v
    group = q.shape[-2] // max(k.shape[-2], 1) if q.dim() > 1 and k.dim() > 1 else 1
    return _rows(q, group), _rows(k, 0), _rows(v, 0)


def _lengths(lengths: Tensor, like: Tensor) -> Tensor:
    """The reference's loops take the lengths on either side and in any integer type; the kernels int64 on the device."""
    if lengths.dtype != torch.long or not lengths.is_cuda or lengths.get_device() != like.get_device():
        lengths = lengths.to(device=like.device, dtype=torch.long)
    return lengths.contiguous()


def _scale(scale, dim):
    return float(dim) ** -0.5 if scale is None else float(scale)


class _AttentionPack(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lengths, s_lengths, scale, causal):
        q, k, v = _operands(q, k, v)
        out = q.new_empty(q.shape)
        lse = q.new_empty(q.shape[:2], dtype=torch.float32)
        # 16-bit outputs: the backward's grad . out needs what the rounding took from them
        rest = None if q.dtype == torch.float32 else torch.empty_like(out)
        ext.attention_pack_forward(q, k, v, q_lengths, s_lengths, out, lse, scale, causal, rest)
        ctx.save_for_backward(q, k, v, out, rest, lse, q_lengths, s_lengths)
        ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, rest, lse, q_lengths, s_lengths = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq = q.new_empty(q.shape) if need_q else None
        dk, dv = (k.new_empty(k.shape), v.new_empty(v.shape)) if need_k or need_v else (None, None)
        ext._attention_pack_backward(grad.contiguous(), q, k, v, out, lse, q_lengths, s_lengths, dq, dk, dv, ctx.scale,
                                     ctx.causal, rest)
        return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


def attention_pack_mode(q_feats: Tensor, k_feats: Tensor, v_feats: Tensor, q_lengths: Tensor,
                        s_lengths: Optional[Tensor] = None, scale: Optional[float] = None, causal: bool = False) -> Tensor:
    """q_feats (N, H, D), k_feats and v_feats (M, KV, D), lengths (B,) -> (N, H, D): per sequence and head the softmax over
    ``scale * q . k`` (``scale`` = D ** -0.5 if None) of its keys, applied to its values.

    H is a multiple of KV: query head h reads key head ``h // (H // KV)``.  ``s_lengths`` None: the keys are the queries'
    sequences (self-attention).  ``causal``: query i of a sequence sees the keys j <= i + (s_length - q_length), so the last
    query sees them all.  A query without keys yields zeros and has no gradient; what a query does not see does not reach
    it, infinities and NaN included (in the forward).  Rows behind the last sequence come out as zeros.  fp32, fp16 or bf16,
    D from 8 (fp32: 4) to 256; the inputs may be views of one projection (only the last dimension has to be contiguous).
    Gradients of the tensors that ask for them; no second and no forward-mode derivative.
    """
    _require_cuda("attention_pack_mode", q_feats, k_feats, v_feats)
    q_lengths = _lengths(q_lengths, q_feats)
    s_lengths = q_lengths if s_lengths is None else _lengths(s_lengths, q_feats)
    scale = _scale(scale, q_feats.shape[-1])
    if recorded(q_feats, k_feats, v_feats):
        return _AttentionPack.apply(q_feats, k_feats, v_feats, q_lengths, s_lengths, scale, causal)
    out = q_feats.new_empty(q_feats.shape)
    ext.attention_pack_forward(*_operands(q_feats, k_feats, v_feats), q_lengths, s_lengths, out, None, scale, causal)
    return out


def cached_attention(q_feats: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor,
                     scale: Optional[float] = None) -> Tensor:
    """q_feats (B, T, H, D) = the newest T tokens of B sequences, k_cache and v_cache (B, C, KV, D), lengths (B,) = filled
    rows of each cache, the new tokens' among them -> (B, T, H, D).

    Token t sees the rows j <= lengths[b] - T + t; rows past a length are never read (they may hold anything).  The serving
    form of ``attention_pack_mode(..., causal=True)``: no gradient, the keys are divided over the whole GPU however few the
    sequences are.  Only the last dimension of each tensor has to be contiguous.
    """
    _require_cuda("cached_attention", q_feats, k_cache, v_cache)
    if recorded(q_feats, k_cache, v_cache):
        raise RuntimeError("cached_attention: no gradient; call it under torch.no_grad() or use attention_pack_mode")
    q, k, v = _operands(q_feats, k_cache, v_cache)
    if q.dim() == 4 and q.shape[1] > 1 and q.shape[0] > 1 and q.stride(0) != q.shape[1] * q.stride(1):
        q = q.contiguous()
    out = q.new_empty(q.shape)
    ext.cached_attention(q, k, v, _lengths(lengths, q), out, _scale(scale, q.shape[-1]))
    return out
