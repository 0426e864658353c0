"""The hybrid-stack operators where autograd does more than one plain pass, and where values are not finite."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def bf(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(BF)


def _norm(x):
    from hattention_b200 import layer_norm
    return layer_norm(x, torch.ones(x.shape[-1], device="cuda"))


def _norm_weight(w):
    from hattention_b200 import layer_norm
    return layer_norm(bf(4, w.shape[-1]), w)


def _scan(x):
    from hattention_b200 import gated_recurrence
    return gated_recurrence(x, -bf(*x.shape, seed=1).abs())[0]


def _scan_state(h):
    from hattention_b200 import gated_recurrence
    return gated_recurrence(bf(2, 5, 64), -bf(2, 5, 64, seed=1).abs(), h.float())[0]


def _scan_step(x):
    from hattention_b200 import gated_recurrence_step
    return gated_recurrence_step(torch.ones(x.shape, device="cuda"), x, -bf(*x.shape, seed=1).abs())[0]


def _attention(q):
    from hattention_b200 import sliding_window_attention
    return sliding_window_attention(q, bf(1, 70, 1, 64, seed=1), bf(1, 70, 1, 64, seed=2), 20, 1)


def _prefill(q):
    from hattention_b200 import sliding_window_prefill
    return sliding_window_prefill(q, bf(1, 70, 1, 64, seed=1), bf(1, 70, 1, 64, seed=2), 20, 1)[0]


def _step(q):
    from hattention_b200 import WindowState, sliding_window_step
    return sliding_window_step(WindowState.empty(1, 1, 64, 8), q, bf(1, 1, 64, seed=1), bf(1, 1, 64, seed=2))[0]


CALLS = pytest.mark.parametrize("call,shape", [(_norm, (6, 64)), (_norm_weight, (64,)), (_scan, (2, 5, 64)), (_scan_state, (2, 64)), (_scan_step, (2, 64)),
                                               (_attention, (1, 70, 2, 64)), (_prefill, (1, 70, 2, 64)), (_step, (1, 2, 64))])


@CALLS
def test_forward_mode_is_refused(call, shape):
    x = bf(*shape)
    call(x)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        call(fwad.make_dual(x, torch.ones_like(x)))


@CALLS
def test_function_transforms_are_refused(call, shape):
    x = bf(*shape)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: call(t).float().sum())(x)
    with pytest.raises(Exception):
        torch.func.vmap(call, randomness="different")(torch.stack([x, x]))


def passes():
    """(name, a forward pass of its leaves, the leaves)"""
    from hattention_b200 import gated_recurrence, layer_norm, sliding_window_attention
    q, k, v = bf(2, 150, 4, 64, seed=1), bf(2, 150, 2, 64, seed=2), bf(2, 150, 2, 64, seed=3)
    x, w, b = bf(40, 96, seed=4), bf(96, seed=5), bf(96, seed=6)
    u, g, h = bf(2, 150, 34, seed=7), -bf(2, 150, 34, seed=8).abs(), bf(2, 34, seed=9).float()
    return [("window", lambda *t: sliding_window_attention(*t, 40, 2), [q, k, v]), ("norm", layer_norm, [x, w, b]), ("recurrence", lambda *t: gated_recurrence(*t)[0], [u, g, h])]


def _elsewhere(t):
    """The same values on the host, and back at an address between 16-byte boundaries."""
    kept = t.detach().cpu()

    def back():
        at = torch.empty(kept.numel() + 1, dtype=kept.dtype, device="cuda")[1:].view(kept.shape)
        return at.copy_(kept)
    return back


@pytest.mark.parametrize("which", range(3), ids=["window", "norm", "recurrence"])
def test_saved_tensors_that_hooks_moved(which):
    _, f, leaves = passes()[which]
    leaves = [t.requires_grad_(True) for t in leaves]
    y = f(*leaves)
    dy = bf(*y.shape, seed=11)
    want = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.saved_tensors_hooks(_elsewhere, lambda back: back()):
        y = f(*leaves)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(a, c)


@pytest.mark.parametrize("which", range(3), ids=["window", "norm", "recurrence"])
def test_checkpoints(which):
    from torch.utils.checkpoint import checkpoint
    _, f, leaves = passes()[which]
    leaves = [t.requires_grad_(True) for t in leaves]
    y = f(*leaves)
    dy = bf(*y.shape, seed=11)
    want = torch.autograd.grad(y, leaves, dy)
    y2 = checkpoint(f, *leaves, use_reentrant=False)
    assert torch.equal(y, y2)
    for a, c in zip(torch.autograd.grad(y2, leaves, dy), want):
        assert torch.equal(a, c)


def test_a_pass_that_changed_an_operand_is_noticed():
    for name, f, leaves in passes():
        leaves = [t.clone().requires_grad_(True) for t in leaves]
        y = f(*leaves)
        with torch.no_grad():
            leaves[0].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


# ------------------------------------------------------------------------------------------ the exponentials' polynomial
def test_polynomial_of_the_exponentials():
    """2^x from the polynomial of degree 4, which is off by 2.6e-6 of the value at most, and four additions' roundings; 2^-126 below -126, NaN for NaN."""
    from hattention_b200 import _lib
    f = _lib.lib().llattn_selftest_exp2_poly
    f.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]

    def poly(x):
        y = torch.empty_like(x)
        assert f(x.data_ptr(), y.data_ptr(), x.numel(), torch.cuda.current_stream().cuda_stream) == 0
        return y
    step = torch.arange(-126, 126, device="cuda").float()
    x = torch.cat([torch.linspace(-126, 126, 2 ** 21, device="cuda"), torch.linspace(-1, 1, 2 ** 20, device="cuda"), step, step + 0.5, torch.nextafter(step + 0.5, step), torch.nextafter(step + 0.5, step + 1)])
    ref = x.double().exp2()
    assert ((poly(x).double() - ref).abs() / ref).max() <= 2.65e-6 + 4 * 2.0 ** -24
    low = poly(torch.tensor([-126.0, -127.0, -1e30, -math.inf], device="cuda"))
    assert torch.allclose(low, torch.full_like(low, 2.0 ** -126), rtol=3e-6, atol=0)
    assert poly(torch.tensor([math.nan, 1.0], device="cuda"))[0].isnan()


# ------------------------------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("T,window", [(60, 20), (1500, 200)])
def test_window_gradients_of_a_key_that_is_not_finite(T, window, K):
    """It spoils the gradients of the queries that see it, and of the keys that those see; nothing of it reaches tiles of 128 that share no pair with a tile of those."""
    from hattention_b200 import sliding_window_attention
    q, k, v, do = bf(1, T, 2, K, seed=1), bf(1, T, 1, K, seed=2), bf(1, T, 1, K, seed=3), bf(1, T, 2, K, seed=4)
    s = T // 2

    def gradients(k):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(sliding_window_attention(*leaves, window), leaves, do)
    spoiled = k.clone()
    spoiled[0, s, 0, 3] = math.nan
    clean, got = gradients(k), gradients(spoiled)
    see = orc.seen(T, window, 0, "cuda")
    rows = see[:, s]
    keys = see[rows].any(0)
    assert got[0][0, rows].isnan().all() and got[1][0, keys].isnan().all() and got[2][0, keys].isnan().all()
    n = -(-T // 128)
    pad = torch.zeros(n * 128, n * 128, dtype=torch.bool, device="cuda")
    pad[:T, :T] = see
    tiles = pad.view(n, 128, n, 128).any(3).any(1)                # query tile i, key tile j
    hit = tiles[:, s // 128]
    far_rows = (~hit).repeat_interleave(128)[:T]
    far_keys = (~tiles[hit].any(0)).repeat_interleave(128)[:T]
    assert T < 128 or (far_rows.any() and far_keys.any())
    assert torch.equal(got[0][0, far_rows], clean[0][0, far_rows])
    for a, c in zip(got[1:], clean[1:]):
        assert torch.equal(a[0, far_keys], c[0, far_keys])


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("H,slots", [(4, 30), (24, 700)])
def test_steps_over_keys_that_are_not_finite(H, slots, K):
    """NaN in a key spoils the heads of its group; a key whose score is minus infinity has the weight 0; a query that is NaN spoils its own head."""
    from hattention_b200 import WindowState, sliding_window_step
    G = 2

    def step(change):
        kc, vc, q = bf(3, slots, G, K, seed=1), bf(3, slots, G, K, seed=2), bf(3, H, K, seed=3)
        q[..., 0] = 1.0
        change(kc, vc, q)
        n = torch.full((3, G), 5 * slots + 1, dtype=torch.int64, device="cuda")
        return sliding_window_step(WindowState(kc, vc, n, slots, 0), q, bf(3, G, K, seed=4), bf(3, G, K, seed=5))[0]
    clean = step(lambda kc, vc, q: None)
    R = H // G
    for at in (0, 15, 16, slots - 1):
        o = step(lambda kc, vc, q: kc[1, at, 1, 7].fill_(math.nan))
        assert o[1, R:].isnan().all() and torch.equal(o[1, :R], clean[1, :R]) and torch.equal(o[[0, 2]], clean[[0, 2]])
        o = step(lambda kc, vc, q: kc[1, at, 1, 0].fill_(-math.inf))
        far = step(lambda kc, vc, q: kc[1, at, 1, 0].fill_(-1e30))          # (its weight is 0 as well)
        assert o.isfinite().all() and torch.equal(o, far)
    o = step(lambda kc, vc, q: q[1, 1].fill_(math.nan))
    assert o[1, 1].isnan().all()
    o[1, 1] = clean[1, 1]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("D", [64, 30, 7])
@pytest.mark.parametrize("xt", [torch.float32, BF])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_recurrence_over_values_that_are_not_finite(bad, xt, D):
    """A value that is not finite spoils its channel from its token on, its gradient the tokens up to it, and no other channel."""
    from hattention_b200 import gated_recurrence
    x, g, do = bf(2, 700, D, seed=1).to(xt), -bf(2, 700, D, seed=2).abs().to(xt) / 64, bf(2, 700, D, seed=3).to(xt)

    def run(x, do):
        leaves = [x.clone().requires_grad_(True), g.clone().requires_grad_(True)]
        o, last = gated_recurrence(*leaves, output_final_state=True)
        return (o.detach(), last.detach()) + torch.autograd.grad(o, leaves, do)
    clean = run(x, do)
    for t in (0, 15, 16, 333, 699):
        x2, do2 = x.clone(), do.clone()
        x2[1, t, 3] = bad
        do2[0, t, 5] = bad
        o, last, dx, dg = run(x2, do2)
        assert not o[1, t:, 3].isfinite().any() and not last[1, 3].isfinite() and not dx[0, :t + 1, 5].isfinite().any()
        assert torch.equal(o[1, :t, 3], clean[0][1, :t, 3]) and torch.equal(dx[0, t + 1:, 5], clean[2][0, t + 1:, 5])
        for a, c in zip((o, last, dx, dg), clean):
            a, c = a.clone(), c.clone()
            for z in (a, c):
                z[1, ..., 3] = 0
                z[0, ..., 5] = 0
            assert torch.equal(a, c)


@pytest.mark.parametrize("rows,N", [(5, 31), (40, 256), (700, 96), (300, 2048), (4, 9000)])
@pytest.mark.parametrize("xt", [torch.float32, BF])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_norm_of_rows_that_are_not_finite(bad, xt, rows, N):
    """A row spoils itself, and the weight's gradient; a gradient of a row its row, and its column of the parameters'."""
    from hattention_b200 import layer_norm
    x, w, b, dy = bf(rows, N, seed=1).to(xt), bf(N, seed=2).to(xt), bf(N, seed=3).to(xt), bf(rows, N, seed=4).to(xt)

    def run(x, dy):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    clean = run(x, dy)
    for r in {0, rows // 2, rows - 1}:
        others = torch.arange(rows, device="cuda") != r
        x2 = x.clone()
        x2[r, N // 3] = bad
        y, dx, dw, db = run(x2, dy)
        assert y[r].isnan().all() and torch.equal(y[others], clean[0][others]) and dx[r].isnan().all() and torch.equal(dx[others], clean[1][others])
        assert dw.isnan().all() and torch.equal(db, clean[3])
        dy2 = dy.clone()
        dy2[r, N // 3] = bad
        y, dx, dw, db = run(x, dy2)
        cols = torch.arange(N, device="cuda") != N // 3
        assert torch.equal(y, clean[0]) and not dx[r].isfinite().any() and torch.equal(dx[others], clean[1][others])
        assert not dw[~cols].isfinite().any() and not db[~cols].isfinite().any() and torch.equal(dw[cols], clean[2][cols]) and torch.equal(db[cols], clean[3][cols])
