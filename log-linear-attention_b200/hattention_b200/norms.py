"""Layer norm, the row norm in front of a mixer, beside the l2norm and the gated norm that the mixers use themselves.  (No counterpart in
the reference.)"""
from typing import Optional

import torch

from . import _lib


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x, with gradients for all three.  Rows have up to 2^30 values.

    x is bf16 or fp32 and y has its type; weight and bias (N,) have one type, x's or fp32.  Statistics and the sums over rows of the
    parameters' gradients are fp32, and those sums are taken in an order that the sizes alone decide: the same call gives the same bits."""
    y = _lib.host().layer_norm(x, weight, bias, eps)
    if y is not None:
        return y
    if x.ndim < 1 or x.shape[-1] < 1 or (x.numel() > 0 and x.shape[-1] > 2 ** 30):
        raise ValueError("rows of at least one value, and at most 2^30")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"x is bfloat16 or float32; got {x.dtype}")
    for p in (weight, bias):
        if p is not None:
            if p.dtype not in (x.dtype, torch.float32) or (weight is not None and p.dtype != weight.dtype):
                raise TypeError("weight and bias have one type, x's or float32")
            if p.shape != x.shape[-1:]:
                raise ValueError(f"weight and bias have the shape {tuple(x.shape[-1:])}; got {tuple(p.shape)}")
    if not x.is_cuda or any(p is not None and p.device != x.device for p in (weight, bias)):
        raise RuntimeError("the norm kernels need CUDA tensors of one device (there is no CPU path)")
    if x.numel() > 0:
        raise NotImplementedError("layer_norm has no forward-mode derivative, and takes at most 2^31 - 1 rows")
    y = x if weight is None else x * weight
    return (y if bias is None else y + bias).to(x.dtype).clone()
