"""What rounding leaves of the hybrid-stack operators' outputs, in norm: elementwise bounds that add up worst cases over long sums cannot tell a rounding too many from none."""
import math

import pytest
import torch

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rel(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


# ------------------------------------------------------------------------------------------ steps of the windowed attention
def step_case(K, B, H, G, slots, seed=0):
    from hattention_b200 import WindowState
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(BF)
    state = WindowState(r(B, slots, G, K), r(B, slots, G, K), torch.full((B, G), slots - 1, dtype=torch.int64, device="cuda"), slots, 0)
    return state, r(B, H, K), r(B, G, K), r(B, G, K)


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("H,G,slots", [(8, 2, 1), (8, 2, 5), (12, 1, 20), (8, 8, 40), (34, 2, 33)])
def test_steps_lose_no_more_than_their_outputs_rounding(K, H, G, slots):
    """Outputs are sum P v (1 + e) rounded to bf16.  e: P in two bf16 terms, 2^-16; scores of 128 products that sum to at most 45 in magnitude, each addition within 2^-23 of that, times the
    scale: 128 * 45 * 2^-23 * 2^-3.5 < 2^-14, in P and once more in its sum.  In norm they are off by at most the rounding of the exact values and e of the magnitudes."""
    from hattention_b200 import sliding_window_step
    state, q, k, v = step_case(K, 64, H, G, slots)
    o, state = sliding_window_step(state, q, k, v)
    rep = lambda x: x.double().repeat_interleave(H // G, 2)
    P = (torch.einsum("bhk,bshk->bhs", q.double(), rep(state.k)) / math.sqrt(K)).softmax(-1)
    ref, mag = torch.einsum("bhs,bshk->bhk", P, rep(state.v)), torch.einsum("bhs,bshk->bhk", P, rep(state.v).abs())
    assert (o.double() - ref).norm() <= (ref.to(BF).double() - ref).norm() + (2.0 ** -16 + 2 * 2.0 ** -14) * mag.norm()


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("at", [0, 17, 39])
def test_values_of_infinity_stay_infinite_in_a_step(K, at):
    """Weights are positive: a row that sees an infinite value is infinite in that column, and as it was in the others."""
    from hattention_b200 import sliding_window_step
    (a, q, k, v), (b, *_) = step_case(K, 3, 8, 2, 40), step_case(K, 3, 8, 2, 40)
    b.v[:, at, :, 5], b.v[:, at, :, 6] = math.inf, -math.inf
    v2 = v.clone()
    if at == 39:
        v2[..., 5], v2[..., 6] = math.inf, -math.inf
    clean, _ = sliding_window_step(a, q, k, v)
    o, _ = sliding_window_step(b, q, k, v2)
    assert (o[..., 5] == math.inf).all() and (o[..., 6] == -math.inf).all()
    keep = [c for c in range(K) if c not in (5, 6)]
    assert torch.equal(o[..., keep], clean[..., keep])


# ------------------------------------------------------------------------------------------ the windowed attention
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("T,window", [(2, 2), (30, 12), (64, 64), (65, 40), (300, 64), (2100, 2048)])
def test_values_of_infinity_stay_infinite(T, window, K):
    """A row that sees an infinite value is infinite in that column (its weight there is at least 2^-25: scores within +-6 of each other, of at most 2048), and as it was in the others."""
    from hattention_b200 import sliding_window_attention
    gen = torch.Generator(device="cuda").manual_seed(T)
    q, k, v = (torch.randn(1, T, n, K, device="cuda", generator=gen).to(BF).clamp(-1, 1) for n in (2, 1, 1))
    clean = sliding_window_attention(q, k, v, window)
    for s in {0, T // 2, T - 1}:
        w = v.clone()
        w[0, s, 0, 5], w[0, s, 0, 6] = math.inf, -math.inf
        o = sliding_window_attention(q, k, w, window)
        rows = orc.seen(T, window, 0, "cuda")[:, s]
        assert (o[0, rows][..., 5] == math.inf).all() and (o[0, rows][..., 6] == -math.inf).all(), s
        keep = [c for c in range(K) if c not in (5, 6)]
        assert torch.equal(o[..., keep], clean[..., keep])


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("T,window,B", [(50, 20, 200), (100, 30, 80), (500, 500, 9)])
def test_gradients_of_a_sequence_are_those_of_any_batch(T, window, B, K):
    """Heads that share nothing, no sinks: every sum is one CTA's, so the same sequence has the same bits alone and among others."""
    from hattention_b200 import sliding_window_attention
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(B, T, 2, K, device="cuda", generator=gen).to(BF) for _ in range(4))

    def step(n):
        leaves = [t[:n].clone().requires_grad_(True) for t in (q, k, v)]
        o = sliding_window_attention(*leaves, window)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do[:n])
    for a, b in zip(step(1), step(B)):
        assert torch.equal(a, b[:1])


# ------------------------------------------------------------------------------------------ decays of the recurrence
@pytest.mark.parametrize("D", [100001, 100002, 100008])
@pytest.mark.parametrize("xt", [torch.float32, BF])
def test_decays(xt, D):
    """A state of ones after one token of zeros is exp(g): from a multiplication and ex2.approx, 2^-22 of the value, with one or two roundings more, 2^-24 each; expf is within two units, 2^-22 too.  bf16 callers have the rounding of
    the argument too, |g| 2^-24, and that of log2 e, |g| 2^-26.  Down to -87, where the value is about to leave fp32's normal range."""
    from hattention_b200 import gated_recurrence, gated_recurrence_step
    g = torch.linspace(-87, 0, D, device="cuda")[None]
    ref = g.double().exp()
    tol = 2.0 ** -22 + 2 * 2.0 ** -24 + (g.double().abs() * (2.0 ** -24 + 2.0 ** -26) if xt is BF else 0.0)
    x = torch.zeros_like(g, dtype=xt)
    _, h = gated_recurrence_step(torch.ones_like(g), x, g)
    assert ((h.double() - ref).abs() <= tol * ref).all()
    _, h = gated_recurrence(x[:, None], g[:, None], torch.ones_like(g), output_final_state=True)
    assert ((h.double() - ref).abs() <= tol * ref).all()


@pytest.mark.parametrize("D", [101, 128])
def test_fp32_states_are_as_exact_as_a_loop_in_fp32(D):
    """Long memories add up what decays are off on average: exponentials of a bias, however small, show here.  The same number of roundings a token in the kernel and in a loop of fp32 operations:
    errors of one size, a fourth for the order of sums."""
    from hattention_b200 import gated_recurrence
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, g = torch.randn(2, 1500, D, device="cuda", generator=gen), torch.nn.functional.logsigmoid(torch.randn(2, 1500, D, device="cuda", generator=gen) + 3)
    do = torch.randn(2, 1500, D, device="cuda", generator=gen)

    def gradients(f, dtype):
        leaves = [t.to(dtype).requires_grad_(True) for t in (x, g)]
        o = f(*leaves)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do.to(dtype))

    def loop(x, g):
        a, h, o = g.exp(), torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            h = a[:, t] * h + x[:, t]
            o.append(h)
        return torch.stack(o, 1)
    exact = gradients(loop, torch.float64)
    for ours, plain, ref in zip(gradients(lambda x, g: gated_recurrence(x, g)[0], torch.float32), gradients(loop, torch.float32), exact):
        assert rel(ours, ref) <= 1.25 * rel(plain, ref)


@pytest.mark.parametrize("xt", [torch.float32, BF])
def test_decays_that_are_not_finite(xt):
    from hattention_b200 import gated_recurrence, gated_recurrence_step
    g = torch.tensor([[-math.inf, math.nan, -100.0, -1e30, 0.0, -0.0]], device="cuda")
    want = torch.tensor([[0.0, math.nan, 0.0, 0.0, 1.0, 1.0]], device="cuda")
    x = torch.zeros_like(g, dtype=xt)
    _, h = gated_recurrence_step(torch.ones_like(g), x, g)
    assert torch.allclose(h, want, rtol=0, atol=1e-42, equal_nan=True)
    _, h = gated_recurrence(x[:, None], g[:, None], torch.ones_like(g), output_final_state=True)
    assert torch.allclose(h, want, rtol=0, atol=1e-42, equal_nan=True)


# ------------------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 5, 1), (2 ** 31, 1, 1), (1, 1, 2 ** 32 + 64)])
def test_recurrence_sizes_that_an_int_does_not_hold(shape):
    from hattention_b200 import gated_recurrence
    x = torch.zeros(1, 1, 1, dtype=BF, device="cuda").expand(shape)
    with pytest.raises(ValueError, match="2\\^31"):
        gated_recurrence(x, x)


def test_window_buffers_at_16_byte_boundaries():
    """Statistics that came back from elsewhere (a hook on saved tensors, a program of its own) start at any boundary of 16 bytes."""
    from hattention_b200 import ops  # noqa: F401
    q, k, v, do = (torch.randn(1, 200, 2, 64, device="cuda").to(BF) for _ in range(4))
    o, stats = torch.ops.llattn.window_fwd(q, k, v, 70, 2, 0.125)
    moved = torch.empty(stats.numel() + 16, dtype=torch.uint8, device="cuda")[16:].copy_(stats)
    assert moved.data_ptr() % 32 == 16
    for a, b in zip(torch.ops.llattn.window_bwd(q, k, v, o, moved, do, 70, 2, 0.125), torch.ops.llattn.window_bwd(q, k, v, o, stats, do, 70, 2, 0.125)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("xt,D", [(torch.float32, 40), (BF, 64), (BF, 33)])
def test_prompts_of_different_lengths(xt, D):
    """Padded with x = 0 and g = 0, a sequence has the state, outputs and gradients that it has alone.  (Other tiles and clusters, other orders of fp32 sums: states of at most 32, decays of a
    tenth a token at least, 2^-21 of what passes a token: 2^-21 * 32 * 10, twice.)"""
    from hattention_b200 import gated_recurrence
    gen = torch.Generator(device="cuda").manual_seed(5)
    lengths, T = [700, 1, 0, 333, 128], 700
    r = lambda: torch.randn(len(lengths), T, D, device="cuda", generator=gen)
    real = torch.arange(T, device="cuda")[None, :, None] < torch.tensor(lengths, device="cuda")[:, None, None]
    x, g, do = (r() * real).to(xt), (-(r().abs() + 0.1) * real), (r() * real).to(xt)
    h0, dlast = r()[:, 0].contiguous(), r()[:, 0].contiguous()
    leaves = [t.requires_grad_(True) for t in (x, g, h0)]
    o, last = gated_recurrence(*leaves, output_final_state=True)
    grads = torch.autograd.grad([o, last], leaves, [do, dlast])
    tol = 2 * 2.0 ** -21 * 32 * 10
    near = lambda a, b: ((a.float() - b.float()).abs() <= tol + 2.0 ** -7 * b.float().abs() * (a.dtype is BF)).all()
    for b, n in enumerate(lengths):
        if n == 0:
            assert torch.equal(last[b], h0[b]) and torch.equal(grads[2][b], dlast[b])
            continue
        part = [t.detach()[b:b + 1, :n].clone().requires_grad_(True) for t in (x, g)] + [h0.detach()[b:b + 1].clone().requires_grad_(True)]
        po, plast = gated_recurrence(*part, output_final_state=True)
        pg = torch.autograd.grad([po, plast], part, [do[b:b + 1, :n].contiguous(), dlast[b:b + 1]])
        assert near(o[b, :n], po[0]) and near(last[b], plast[0])
        assert near(grads[0][b, :n], pg[0][0]) and near(grads[1][b, :n], pg[1][0]) and near(grads[2][b], pg[2][0])
