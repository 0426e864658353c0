"""Gated linear recurrence of independent channels, h_t = exp(g_t) h_{t-1} + x_t: a layer of a hybrid stack beside the log-linear
ones, whose level states decay in the same way.  (No counterpart in the reference.)"""
from typing import Optional, Tuple

import torch

from . import _lib


def _check(x: torch.Tensor, g: torch.Tensor, state: Optional[torch.Tensor], ndim: int) -> None:
    """Raises for what the kernels do not take."""
    if x.ndim != ndim or g.shape != x.shape:
        raise ValueError(f"x and g have {ndim} dimensions and one shape; got {tuple(x.shape)} and {tuple(g.shape)}")
    if x.numel() > 0 and max(x.shape) >= 2 ** 31:
        raise ValueError(f"sizes are below 2^31; got {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32) or g.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"x is bfloat16 or float32, g of x's type or float32; got {x.dtype} and {g.dtype}")
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError("states are kept in fp32")
        if state.shape != (x.shape[0], x.shape[-1]):
            raise ValueError(f"the state has the shape {(x.shape[0], x.shape[-1])}; got {tuple(state.shape)}")
    if not x.is_cuda or g.device != x.device or (state is not None and state.device != x.device):
        raise RuntimeError("the recurrence kernels need CUDA tensors of one device (there is no CPU path)")


def gated_recurrence(x: torch.Tensor, g: torch.Tensor, initial_state: Optional[torch.Tensor] = None,
                     output_final_state: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """o_t = h_t = exp(g_t) h_{t-1} + x_t for x (B,T,D) and log decays g (B,T,D); returns (o, h_T or None), with gradients for
    x, g and the initial state.

    x is bf16 or fp32 and o has its type; g has x's type or is fp32; states are (B,D) fp32, an absent one is zeros.  All sums are fp32.
    exp(g) is exact to 2^-22 of itself for fp32 x; for bf16 x to |g| 2^-24 more, and 0 below 2^-126.
    g <= 0, as log decays are; -inf starts a channel anew at that token, so that packed sequences stay apart.  (Above 0 the products of
    exp(g) over 512 tokens have to stay finite.)  Sequences of different lengths are padded with x = 0 and g = 0: the state behind the padding is the one at the
    sequence's end, and where the padding's outputs have no gradient, the sequence's own tokens have those that they have without it.  T is any size up to 2^30, D any, B ceil(D / 32) below 2^31; even D moves two channels a load."""
    r = _lib.host().gated_recurrence(x, g, initial_state, output_final_state)
    if r is not None:
        return r
    _check(x, g, initial_state, 3)
    if x.numel() > 0:
        raise NotImplementedError("gated_recurrence has no forward-mode derivative")
    h = initial_state if initial_state is not None else x.new_zeros((x.shape[0], x.shape[2]), dtype=torch.float32)
    return x + g.to(x.dtype), h.clone() if output_final_state else None


def gated_recurrence_step(state: torch.Tensor, x: torch.Tensor, g: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token: x, g (B,D) -> (o (B,D), state).  `state` (B,D) fp32, contiguous, is advanced in place.  One launch that reads no host
    values, so it can be captured into a CUDA graph and replayed."""
    o = _lib.host().gated_recurrence_step(state, x, g)
    if o is not None:
        return o, state
    _check(x, g, state, 2)
    if not state.is_contiguous() or state.data_ptr() % 16 != 0:
        raise ValueError("the state is advanced in place: it has to be contiguous and to start at a 16-byte boundary")
    if x.numel() > 0:
        raise NotImplementedError("gated_recurrence_step has no forward-mode derivative")
    return torch.empty_like(x), state
