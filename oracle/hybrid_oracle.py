"""The operators of hybrid stacks from their definitions, in 64 bits on whatever device the operands are on; differentiable.
Test infrastructure only."""
import math

import torch


def gated_recurrence(x, g, h0=None):
    """h_t = exp(g_t) h_{t-1} + x_t, a token at a time: x, g (B,T,D), h0 (B,D) -> (o (B,T,D), h_T)."""
    x, a = x.double(), g.double().exp()
    h = h0.double() if h0 is not None else torch.zeros_like(x[:, 0])
    o = []
    for t in range(x.shape[1]):
        h = a[:, t] * h + x[:, t]
        o.append(h)
    return torch.stack(o, 1), h


def seen(T, window, sinks, device):
    """(T,T): whether query t sees token s."""
    t, s = torch.arange(T, device=device)[:, None], torch.arange(T, device=device)[None]
    return (s <= t) & ((t - s < window) | (s < sinks))


def window_probabilities(q, k, window, sinks, scale=None):
    """(B,H,T,T) softmax of the scaled scores over the tokens that a query sees."""
    q, k = q.double(), k.double().repeat_interleave(q.shape[2] // k.shape[2], 2)
    S = torch.einsum("bthk,bshk->bhts", q, k) * (scale if scale is not None else 1.0 / math.sqrt(q.shape[-1]))
    return S.masked_fill(~seen(q.shape[1], window, sinks, q.device), -math.inf).softmax(-1)


def sliding_window_attention(q, k, v, window, sinks=0, scale=None):
    P = window_probabilities(q, k, window, sinks, scale)
    return torch.einsum("bhts,bshk->bthk", P, v.double().repeat_interleave(q.shape[2] // v.shape[2], 2))


def window_slots(k, n, window, sinks):
    """The slots (sinks + window, ..) of a sequence k (T, ..) after its first n tokens, filled a token at a time."""
    out = torch.zeros((sinks + window,) + k.shape[1:], dtype=k.dtype, device=k.device)
    for t in range(n):
        out[t if t < sinks else sinks + (t - sinks) % window] = k[t]
    return out


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    x = x.double()
    d = x - x.mean(-1, keepdim=True)
    y = d / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    return y + bias.double() if bias is not None else y
