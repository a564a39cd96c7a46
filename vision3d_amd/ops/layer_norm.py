"""Layer normalisation of feature rows, the norm of the transformer layers over packs (the reference's layers call
``torch.nn.LayerNorm``; a post-norm layer adds the residual first: here the sum is formed inside the kernel).

One kernel forward; backward recomputes the sum and the normalised rows from the inputs and the saved statistics, so
nothing of the input's size is kept besides the inputs themselves.  The gradients of the weight and the bias are added in
a fixed order (no atomics).
"""
from typing import Optional

import torch
from torch import Tensor

from .. import ext
from ._autograd import recorded


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feats, weight, bias, eps, residual):
        out = torch.empty_like(feats)
        stats = feats.new_empty((2, feats.shape[0]), dtype=torch.float32)
        ext.layer_norm_forward(feats, residual, weight, bias, out, stats, eps)
        ctx.save_for_backward(feats, weight, residual, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        feats, weight, residual, stats = ctx.saved_tensors
        need_feats, need_weight, need_bias, _, need_residual = ctx.needs_input_grad
        grad_feats = torch.empty_like(feats) if need_feats or need_residual else None
        grad_weight = torch.empty_like(weight) if need_weight else None
        grad_bias = feats.new_empty(feats.shape[1:], dtype=ctx.bias_dtype) if need_bias else None
        if feats.shape[0] == 0:  # no rows: the column sums are empty
            for t in (grad_weight, grad_bias):
                if t is not None:
                    t.zero_()
        else:
            ext._layer_norm_backward(grad.contiguous(), feats, residual, weight, stats, grad_feats, grad_weight, grad_bias)
        return grad_feats if need_feats else None, grad_weight, grad_bias, None, grad_feats if need_residual else None


def layer_norm(feats: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               residual: Optional[Tensor] = None) -> Tensor:
    """feats (*, C) (+ residual of the same shape), weight / bias (C,) -> (*, C): every row normalised to mean 0 and
    variance 1 (biased, + eps), scaled and shifted.

    fp32, fp16 or bf16 features; weight and bias both in the features' type or both in fp32.  Statistics and sums are fp32;
    the output has the features' type.  At most 16384 channels (8192 in fp32).  Gradients flow to all four tensors; no second
    and no forward-mode derivative.
    """
    for t in (feats, weight, bias, residual):
        if t is not None and not t.is_cuda:
            raise RuntimeError("layer_norm: CUDA tensors required (no CPU fallback in vision3d_amd)")
    if feats.dim() < 1:
        raise RuntimeError("layer_norm: feats must have a channel dimension")
    if residual is not None and residual.shape != feats.shape:
        raise RuntimeError("layer_norm: residual must have the shape of feats")
    if feats.dim() != 2:
        channels = feats.shape[-1]
        rows = feats.reshape(-1, channels)
        return layer_norm(rows, weight, bias, eps, None if residual is None else residual.reshape(-1, channels)).view(
            feats.shape)
    feats = feats.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    if recorded(feats, weight, bias, residual):
        return _LayerNorm.apply(feats, weight, bias, eps, residual)
    out = torch.empty_like(feats)
    ext.layer_norm_forward(feats, residual, weight, bias, out, None, eps)
    return out
