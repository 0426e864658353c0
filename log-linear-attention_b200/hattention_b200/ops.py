"""The kernels as `torch.library` operators (namespace `llattn`), for callers that want dispatcher-visible
ops: fake-tensor shape propagation (`torch.compile` tracing, `torch.export`), `torch.library.opcheck`.
Each operator calls the same C-ABI entry point as the Python drivers of this package; the drivers remain
the interface that mirrors the reference (`hattention/chunkwise.py`, `hattention/chunkwise_hgdn.py`,
`hattention/kernel.py:20-29`).

    llattn::mamba2_fwd(q, k, v, g, l)                        -> (o, g_cum, workspace)
    llattn::mamba2_bwd(q, k, v, g_cum, l, do, workspace)     -> (dq, dk, dv, dg, dl)
    llattn::gdn_fwd(q, k, v, beta, g, l)                     -> (g_cum, o, Aw, Au)
    llattn::gdn_bwd(q, k, v, beta, g_cum, l, Aw, Au, do)     -> (dq, dk, dv, dbeta, dg, dl)
    llattn::l2norm_scale_fwd(x, scale)                       -> y
    llattn::l2norm_scale_bwd(x, dy, scale)                   -> dx
    llattn::recurrence_fwd(x, g, h0)                         -> (o, h_last, states)
    llattn::recurrence_bwd(x, g, states, do, dh_last)        -> (dx, dg, dh0)
    llattn::window_fwd(q, k, v, window, sinks, scale)        -> (o, stats)
    llattn::window_bwd(q, k, v, o, stats, do, window, sinks, scale) -> (dq, dk, dv)
    llattn::layer_norm_fwd(x, weight, bias, eps)             -> (y, stats)
    llattn::layer_norm_bwd(x, weight, stats, dy)             -> (dx, dweight, dbias)

`workspace` of mamba2_fwd is the call's scratch (uint8); handing it to mamba2_bwd lets the backward read the
segment-level states instead of recomputing them (pass an empty tensor to recompute).  `states` and `stats` are what the forward
passes of the hybrid-stack operators keep for their backward passes.
"""
from typing import Optional, Tuple

import torch

from . import _lib
from .base import HType

_T = torch.Tensor


@torch.library.custom_op("llattn::mamba2_fwd", mutates_args=())
def mamba2_fwd(q: _T, k: _T, v: _T, g: _T, l: _T) -> Tuple[_T, _T, _T]:
    from .chunkwise import chunkwise_fwd
    kept = []
    o, g_cum, _ = chunkwise_fwd(q, k, v, g, l, False, 2, HType.WEAK, 64, False, keep_workspace=kept)
    return o, g_cum, kept[0]


@mamba2_fwd.register_fake
def _(q, k, v, g, l):
    B, T, G, K = k.shape
    H, V = v.shape[2], v.shape[3]
    n = _lib.lib().llattn_mamba2_fwd_workspace_bytes(B, T, H, G, K, V, l.shape[-1])
    return (torch.empty_like(v, dtype=torch.bfloat16), torch.empty_like(g, dtype=torch.float32),
            v.new_empty((max(int(n), 256),), dtype=torch.uint8))


@torch.library.custom_op("llattn::mamba2_bwd", mutates_args=())
def mamba2_bwd(q: _T, k: _T, v: _T, g_cum: _T, l: _T, do: _T, workspace: _T) -> Tuple[_T, _T, _T, _T, _T]:
    from .chunkwise import chunkwise_bwd
    return chunkwise_bwd(q, k, v, g_cum, l, do, False, 2, HType.WEAK, 64,
                         fwd_workspace=workspace if workspace.numel() > 0 else None)


@mamba2_bwd.register_fake
def _(q, k, v, g_cum, l, do, workspace):
    return (torch.empty_like(q, dtype=torch.bfloat16), torch.empty_like(k, dtype=torch.bfloat16),
            torch.empty_like(v, dtype=torch.bfloat16), torch.empty_like(g_cum, dtype=torch.float32),
            torch.empty_like(l, dtype=torch.float32))


@torch.library.custom_op("llattn::gdn_fwd", mutates_args=())
def gdn_fwd(q: _T, k: _T, v: _T, beta: _T, g: _T, l: _T) -> Tuple[_T, _T, _T, _T]:
    from .chunkwise_hgdn import chunkwise_fwd
    g_cum, o, Aw, Au, _ = chunkwise_fwd(q, k, v, beta, g, l, False, 2, HType.WEAK, 64, False)
    return g_cum, o, Aw, Au


@gdn_fwd.register_fake
def _(q, k, v, beta, g, l):
    B, T, H, _ = v.shape
    a = v.new_empty((B, T, H, 64), dtype=torch.bfloat16)
    return torch.empty_like(g, dtype=torch.float32), torch.empty_like(v, dtype=torch.bfloat16), a, torch.empty_like(a)


@torch.library.custom_op("llattn::gdn_bwd", mutates_args=())
def gdn_bwd(q: _T, k: _T, v: _T, beta: _T, g_cum: _T, l: _T, Aw: _T, Au: _T, do: _T) -> Tuple[_T, _T, _T, _T, _T, _T]:
    from .chunkwise_hgdn import chunkwise_bwd
    return chunkwise_bwd(q, k, v, beta, g_cum, l, Aw, Au, do, False, 2, HType.WEAK, 64)


@gdn_bwd.register_fake
def _(q, k, v, beta, g_cum, l, Aw, Au, do):
    f = torch.float32
    return (torch.empty_like(q, dtype=f), torch.empty_like(k, dtype=f), torch.empty_like(v, dtype=f),
            torch.empty_like(beta, dtype=f), torch.empty_like(g_cum, dtype=f), torch.empty_like(l, dtype=f))


@torch.library.custom_op("llattn::l2norm_scale_fwd", mutates_args=())
def l2norm_scale_fwd(x: _T, scale: float) -> _T:
    from .chunkwise_hgdn import l2norm_fwd
    return l2norm_fwd(x, scale)


@l2norm_scale_fwd.register_fake
def _(x, scale):
    return torch.empty_like(x, dtype=torch.bfloat16)


@torch.library.custom_op("llattn::l2norm_scale_bwd", mutates_args=())
def l2norm_scale_bwd(x: _T, dy: _T, scale: float) -> _T:
    from .chunkwise_hgdn import l2norm_bwd
    return l2norm_bwd(x, dy, scale)


@l2norm_scale_bwd.register_fake
def _(x, dy, scale):
    return torch.empty_like(x, dtype=torch.bfloat16)


def _taken(r, what: str):
    if r is None:
        raise ValueError(f"{what}: operands that the kernels do not take")
    return r


@torch.library.custom_op("llattn::recurrence_fwd", mutates_args=())
def recurrence_fwd(x: _T, g: _T, h0: Optional[_T]) -> Tuple[_T, _T, _T]:
    return _taken(_lib.host().recurrence_forward(x, g, h0), "recurrence_fwd")


@recurrence_fwd.register_fake
def _(x, g, h0):
    B, T, D = x.shape
    n = _lib.lib().llattn_recurrence_states_bytes(B, T, D) // 4
    f = torch.float32
    return x.new_empty(x.shape), x.new_empty((B, D), dtype=f), x.new_empty((int(n),), dtype=f)


@torch.library.custom_op("llattn::recurrence_bwd", mutates_args=())
def recurrence_bwd(x: _T, g: _T, states: _T, do: _T, dh_last: Optional[_T]) -> Tuple[_T, _T, _T]:
    return _taken(_lib.host().recurrence_backward(x, g, states, do, dh_last), "recurrence_bwd")


@recurrence_bwd.register_fake
def _(x, g, states, do, dh_last):
    return x.new_empty(x.shape), g.new_empty(g.shape), x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32)


@torch.library.custom_op("llattn::window_fwd", mutates_args=())
def window_fwd(q: _T, k: _T, v: _T, window: int, sinks: int, scale: float) -> Tuple[_T, _T]:
    return _taken(_lib.host().window_forward(q, k, v, window, sinks, scale, _lib.CHECK_STATUS), "window_fwd")


@window_fwd.register_fake
def _(q, k, v, window, sinks, scale):
    B, T, H, K = q.shape
    n = _lib.lib().llattn_window_stats_bytes(B, T, H, K, window, sinks)
    return q.new_empty(q.shape), q.new_empty((int(n),), dtype=torch.uint8)


@torch.library.custom_op("llattn::window_bwd", mutates_args=())
def window_bwd(q: _T, k: _T, v: _T, o: _T, stats: _T, do: _T, window: int, sinks: int, scale: float) -> Tuple[_T, _T, _T]:
    return _taken(_lib.host().window_backward(q, k, v, o, stats, do, window, sinks, scale, _lib.CHECK_STATUS), "window_bwd")


@window_bwd.register_fake
def _(q, k, v, o, stats, do, window, sinks, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


@torch.library.custom_op("llattn::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: _T, weight: _T, bias: Optional[_T], eps: float) -> Tuple[_T, _T]:
    return _taken(_lib.host().layer_norm_forward(x, weight, bias, eps), "layer_norm_fwd")


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps):
    rows = x.numel() // x.shape[-1]
    return x.new_empty(x.shape), x.new_empty((2, (rows + 3) // 4 * 4), dtype=torch.float32)


@torch.library.custom_op("llattn::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(x: _T, weight: _T, stats: _T, dy: _T) -> Tuple[_T, _T, _T]:
    return _taken(_lib.host().layer_norm_backward(x, weight, stats, dy), "layer_norm_bwd")


@layer_norm_bwd.register_fake
def _(x, weight, stats, dy):
    return x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty(weight.shape)
