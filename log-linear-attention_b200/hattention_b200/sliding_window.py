"""Softmax attention over a sliding window with sinks: query t sees the tokens s <= t with t - s < window or s < sinks.  The exact-attention
layer of a hybrid stack; like the log-linear layers it decodes from a state of fixed size.  (No counterpart in the reference.)"""
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib


class WindowState(NamedTuple):
    """What a sequence needs to go on: k, v (B, sinks + window, G, K) bf16 and the tokens seen, lengths (B,G) int64 on the device (the same
    number for every head of a sequence: each head's part of a step counts for itself).  Token t is in slot t if t < sinks, else in slot
    sinks + (t - sinks) % window.  A step changes the tensors in place; sequences may be of different lengths."""
    k: torch.Tensor
    v: torch.Tensor
    lengths: torch.Tensor
    window: int
    sinks: int

    @classmethod
    def empty(cls, B: int, G: int, K: int, window: int, sinks: int = 0, device="cuda") -> "WindowState":
        """The state before the first token."""
        k = torch.zeros(B, sinks + window, G, K, dtype=torch.bfloat16, device=device)
        return cls(k, torch.zeros_like(k), torch.zeros(B, G, dtype=torch.int64, device=device), window, sinks)


def _check(q, k, v, window: int, sinks: int, scale: float, ndim: int) -> None:
    """Raises for what the kernels do not take."""
    if window < 1 or sinks < 0 or max(window, sinks) > 2 ** 29:
        raise ValueError(f"window >= 1 and sinks >= 0, both at most 2^29; got {window} and {sinks}")
    if not (0.0 < scale < 3.4e38):
        raise ValueError(f"the scale is positive and finite; got {scale}")
    if q.ndim != ndim or k.ndim != ndim or k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q (.., H, K), k and v (.., G, K) with {ndim} dimensions; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[-2] < 1 or q.shape[-2] < 1 or q.shape[-2] % k.shape[-2] != 0:
        raise ValueError(f"{q.shape[-2]} query heads over {k.shape[-2]} heads of k and v")
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise NotImplementedError("the window kernels take bfloat16")
    if q.shape[-1] not in (64, 128):
        raise NotImplementedError("heads are 64 or 128 wide")
    if not (q.is_cuda and q.device == k.device == v.device):
        raise RuntimeError("the window kernels need CUDA tensors of one device (there is no CPU path)")


def _scale(scale: Optional[float], K: int) -> float:
    return scale if scale is not None else 1.0 / math.sqrt(K) if K > 0 else 1.0


def sliding_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                             scale: Optional[float] = None) -> torch.Tensor:
    """o (B,T,H,K) = softmax attention of q (B,T,H,K) over k, v (B,T,G,K), H a multiple of G, each query over the last `window` tokens,
    itself among them, and the first `sinks`; with gradients.  bf16, K = 64 or 128, any T up to 2^24, B and H up to 65535; scale K^-0.5 unless it is given.
    A window of T or more is plain causal attention.

    Scores, statistics and sums are fp32; weights, and the scores' gradients, are rounded to bf16 for the matrix products, so that outputs and gradients are
    off by about the square root of two of what their own rounding makes, 2.4e-3 in norm.  Sequences of up to 64 tokens, where sums are of few products, keep 16 bits of both.

    Values of tokens that a query does not see reach it as 0 times themselves where they share a tile with ones that it sees: a batch
    padded behind its sequences is fine, as long as the padding is finite."""
    scale = _scale(scale, q.shape[-1])
    o = _lib.host().sliding_window_attention(q, k, v, window, sinks, scale, _lib.CHECK_STATUS)
    if o is not None:
        return o
    _check(q, k, v, window, sinks, scale, 4)
    if q.numel() > 0:
        raise NotImplementedError("sliding_window_attention has no forward-mode derivative, and takes at most 2^24 tokens")
    return q + 0 * (k.sum() + v.sum())


def sliding_window_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, scale: Optional[float] = None,
                           lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, WindowState]:
    """Outputs for prompts and the state to continue from.  With `lengths` (B,) int64 on the device, sequence b has lengths[b] tokens (0 to T)
    and finite padding behind them, whose outputs say nothing.  Rounded as sliding_window_attention is."""
    scale = _scale(scale, q.shape[-1])
    r = _lib.host().sliding_window_prefill(q, k, v, window, sinks, scale, lengths, _lib.CHECK_STATUS)
    if r is not None:
        return r[0], WindowState(r[1], r[2], r[3], window, sinks)
    _check(q, k, v, window, sinks, scale, 4)
    if lengths is not None and (lengths.dtype != torch.int64 or lengths.shape != q.shape[:1] or lengths.device != q.device):
        raise TypeError("lengths is an int64 tensor (B,) on q's device")
    if q.numel() > 0:
        raise NotImplementedError("sliding_window_prefill takes at most 2^24 tokens of at most 65535 sequences")
    return q.detach().clone(), WindowState.empty(q.shape[0], k.shape[2], q.shape[3], window, sinks, q.device)


def sliding_window_step(state: WindowState, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        scale: Optional[float] = None) -> Tuple[torch.Tensor, WindowState]:
    """One token of every sequence: q (B,H,K), k, v (B,G,K) -> (o (B,H,K), state).  The token's k and v take the place of the one that leaves
    the window.  One launch that reads no host values, so it can be captured into a CUDA graph and replayed.  Weights keep 16 bits in its product with v: outputs are off by
    their own rounding alone."""
    scale = _scale(scale, q.shape[-1])
    o = _lib.host().sliding_window_step(q, k, v, state.k, state.v, state.lengths, state.window, state.sinks, scale)
    if o is not None:
        return o, state
    _check(q, k, v, state.window, state.sinks, scale, 3)
    B, G, K = k.shape
    for c in (state.k, state.v):
        if c.shape != (B, state.sinks + state.window, G, K) or c.dtype != torch.bfloat16 or c.device != q.device:
            raise ValueError(f"the state holds bfloat16 {(B, state.sinks + state.window, G, K)} on q's device; got {c.dtype} {tuple(c.shape)}")
        if not c.is_contiguous() or c.data_ptr() % 16 != 0:
            raise ValueError("the state is advanced in place: it has to be contiguous and to start at 16-byte boundaries")
    if q.numel() > 0 and state.k.data_ptr() == state.v.data_ptr():
        raise ValueError("the state's k and v are one tensor")
    if state.lengths.shape != (B, G) or state.lengths.dtype != torch.int64 or state.lengths.device != q.device or not state.lengths.is_contiguous():
        raise ValueError("the state's lengths are a contiguous int64 tensor (B,G) on q's device")
    if q.numel() > 0:
        raise NotImplementedError("sliding_window_step has no forward-mode derivative")
    return torch.empty_like(q), state
