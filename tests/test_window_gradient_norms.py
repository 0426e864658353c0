"""Gradients of the windowed attention in norm.

Elementwise bounds add up the worst case of every rounding, over all queries and heads that see a token; the gradient itself is a sum of random signs, and where it is long a lost share
of it stays below such a bound.  Errors of roundings are of random signs too: each of the two on the way to a gradient, of P or dS and of the result, is at most 2^-8 of what it rounds, and so
in norm; together sqrt(2) 2^-8, and with what is left (fp32 sums, exp2 to 2^-18, delta) less than 2 2^-8 of the norm of the gradient, and of any part of it that is long enough to have a
norm: the rows of sinks by themselves, which other CTAs sum."""
import math

import pytest
import torch

from oracle import hybrid_oracle as orc

BOUND = 2 * 2.0 ** -8
SHAPES = [(1, 1024, 4, 1, 256, 4), (1, 2000, 8, 1, 200, 16), (1, 1500, 16, 2, 1500, 0), (2, 1000, 6, 2, 1000, 0), (1, 1800, 5, 1, 130, 200), (1, 3000, 2, 1, 130, 300), (1, 700, 4, 4, 60, 5)]


def inputs(B, T, H, G, K, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda n: torch.randn(B, T, n, K, generator=gen).to(torch.bfloat16).to(device)
    return r(H), r(G), r(G), r(H)


def gradients(q, k, v, do, window, sinks, left_out=None):
    """(dq, dk, dv) in 64 bits from the formulas; `left_out` (T,T): pairs (t, s) whose part of dk is left out."""
    R, scale = q.shape[2] // k.shape[2], 1 / math.sqrt(q.shape[3])
    kd, vd = (x.double().repeat_interleave(R, 2) for x in (k, v))
    P = orc.window_probabilities(q, k, window, sinks)
    d, qd = do.double(), q.double()
    o = torch.einsum("bhts,bshk->bthk", P, vd)
    dS = P * (torch.einsum("bthk,bshk->bhts", d, vd) - (d * o).sum(-1).transpose(1, 2)[..., None])
    dq = scale * torch.einsum("bhts,bshk->bthk", dS, kd)
    if left_out is not None:
        dS = dS.masked_fill(left_out, 0)
    group = lambda x: x.unflatten(2, (-1, R)).sum(3)
    return dq, scale * group(torch.einsum("bhts,bthk->bshk", dS, qd)), group(torch.einsum("bhts,bthk->bshk", P, d))


def parts(sinks, dq, dk, dv):
    """What is held to the bound by itself, by name."""
    p = {"dq": dq, "dk": dk, "dv": dv}
    if sinks:
        p |= {"dk of sinks": dk[:, :sinks], "dv of sinks": dv[:, :sinks], "dk behind them": dk[:, sinks:], "dv behind them": dv[:, sinks:]}
    return p


def worst(got, ref, sinks):
    a, b = parts(sinks, *got), parts(sinks, *ref)
    off = {n: ((a[n].double() - b[n]).norm() / b[n].norm()).item() for n in b}
    name = max(off, key=off.get)
    return off[name], name


@pytest.mark.gpu
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", SHAPES)
def test_gradients(B, T, H, G, window, sinks, K):
    from hattention_b200 import sliding_window_attention
    q, k, v, do = inputs(B, T, H, G, K, "cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(sliding_window_attention(*leaves, window, sinks), leaves, do)
    off, name = worst(got, gradients(q.detach(), k.detach(), v.detach(), do, window, sinks), sinks)
    assert off <= BOUND, f"{name}: {off:.2e}"


@pytest.mark.parametrize("B,T,H,G,window,sinks,where", [
    (1, 1024, 4, 1, 256, 4, "far"),                 # the last 256 queries' part of the sinks' dk
    (1, 900, 8, 1, 200, 16, "far"),
    (1, 700, 4, 1, 700, 0, "head")])                # half of the keys' dk, of the later queries of one head
def test_the_bound_finds_a_share_of_dk_that_is_left_out(B, T, H, G, window, sinks, where):
    K = 64
    q, k, v, do = inputs(B, T, H, G, K, "cpu")
    ref = gradients(q, k, v, do, window, sinks)
    rounded = [x.to(torch.bfloat16) for x in ref]
    assert worst(rounded, ref, sinks)[0] <= BOUND
    t, s = torch.arange(T)[:, None], torch.arange(T)[None]
    out = ((t >= T - 256) & (s < sinks)).expand(H, T, T) if where == "far" else (t >= 2 * T // 3) & (s % 2 == 0) & (torch.arange(H) == 1)[:, None, None]
    off, name = worst([x.to(torch.bfloat16) for x in gradients(q, k, v, do, window, sinks, out)], ref, sinks)
    assert off > 2 * BOUND and name.startswith("dk"), f"{name}: {off:.2e}"
