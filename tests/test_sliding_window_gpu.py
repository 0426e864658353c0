"""Attention over a sliding window with sinks on the GPU against the 64-bit oracle.

Tolerances.  Products and softmax statistics are fp32; P and dS are rounded to bf16 for the matrix products, half a step h = 2^-8 relative each.  A score is off by at
most (K + 4) 2^-24 scale sum|q||k| <= 132 * 12 * 2^-24 (its accumulation) and 2^-19 (the scaled exponent, exp2), together d <= 2^-12 for inputs of unit variance; it
enters P as a factor 1 + d, and once more through the statistics.  So o is off by (h + 2 d) sum P|v| + h|o|;  dv by (h + 2 d) sum P|do| + h|dv|;  with delta from the
rounded o, off by (h + 2 d) sum|do|(sum P|v|), and dP by its accumulation 2^-16 sum|do||v|, dS is off by (h + 2 d)|dS| + P times those two, and dq, dk by the sums of that times
scale |k|, |q|, plus half a step of their own."""
import math

import pytest
import torch

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
HALF, D = 2.0 ** -8, 2.0 ** -12


def make(B, T, H, G, K, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n: torch.randn(B, T, n, K, device="cuda", generator=gen).to(torch.bfloat16)
    return r(H), r(G), r(G), r(H)


def within(got, ref, err, what):
    tol = err + HALF * ref.abs() * (1 + 2.0 ** -7) + 1e-30
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def reference(q, k, v, window, sinks, scale):
    R, K = q.shape[2] // k.shape[2], q.shape[3]
    s = scale if scale is not None else 1 / math.sqrt(K)
    P = orc.window_probabilities(q, k, window, sinks, s)
    heads = lambda x: x.double().repeat_interleave(R, 2)
    return R, s, P, heads(k), heads(v)


def check(q, k, v, window, sinks, o, scale=None, do=None, grads=None, half=HALF):
    q, k, v = q.detach(), k.detach(), v.detach()
    R, s, P, kd, vd = reference(q, k, v, window, sinks, scale)
    c = half + 2 * D
    ov = torch.einsum("bhts,bshk->bthk", P, vd)
    absv = torch.einsum("bhts,bshk->bthk", P, vd.abs())
    within(o, ov, c * absv, "o")
    if grads is None:
        return
    qd, d = q.double(), do.double()
    dP = torch.einsum("bthk,bshk->bhts", d, vd)
    dS = P * (dP - (d * ov).sum(-1).transpose(1, 2)[..., None])
    err = c * dS.abs() + P * (c * (d.abs() * absv).sum(-1).transpose(1, 2)[..., None] + 2.0 ** -16 * torch.einsum("bthk,bshk->bhts", d.abs(), vd.abs()))
    group = lambda x: x.unflatten(2, (-1, R)).sum(3)
    within(grads[0], s * torch.einsum("bhts,bshk->bthk", dS, kd), s * torch.einsum("bhts,bshk->bthk", err, kd.abs()), "dq")
    within(grads[1], s * group(torch.einsum("bhts,bthk->bshk", dS, qd)), s * group(torch.einsum("bhts,bthk->bshk", err, qd.abs())), "dk")
    within(grads[2], group(torch.einsum("bhts,bthk->bshk", P, d)), c * group(torch.einsum("bhts,bthk->bshk", P, d.abs())), "dv")


def run(B, T, H, G, K, window, sinks, scale=None, seed=0):
    from hattention_b200 import sliding_window_attention
    q, k, v, do = make(B, T, H, G, K, seed)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sliding_window_attention(q, k, v, window, sinks, scale)
    grads = torch.autograd.grad(o, leaves, do)
    check(q, k, v, window, sinks, o.detach(), scale, do, grads)
    with torch.no_grad():
        assert torch.equal(o, sliding_window_attention(q, k, v, window, sinks, scale))


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", [
    (1, 1, 1, 1, 1, 0), (1, 2, 2, 1, 2, 0), (2, 5, 4, 2, 3, 1), (1, 64, 2, 2, 64, 0), (1, 127, 2, 1, 1, 0), (1, 128, 2, 1, 128, 4), (2, 129, 3, 3, 50, 0),
    (1, 130, 5, 1, 1000, 0), (1, 255, 2, 2, 127, 1), (1, 256, 4, 4, 128, 16), (1, 257, 2, 1, 129, 100), (1, 300, 8, 2, 64, 128), (2, 385, 2, 2, 200, 130),
    (1, 512, 2, 1, 512, 0), (1, 513, 2, 1, 256, 257), (1, 700, 4, 1, 65, 3), (3, 640, 2, 1, 300, 600), (1, 1000, 2, 2, 100, 2000), (1, 1111, 2, 1, 385, 5)])
def test_forward_and_gradients(B, T, H, G, K, window, sinks):
    run(B, T, H, G, K, window, sinks)


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", [(1, 2, 1, 1, 2, 0), (2, 3, 2, 1, 2, 1), (1, 5, 4, 2, 3, 0), (3, 33, 2, 2, 7, 2), (1, 64, 8, 2, 64, 0), (40, 50, 2, 1, 20, 3)])
def test_short_sequences(B, T, H, G, K, window, sinks):
    """Up to 64 tokens the rounding of P and dS is made good by a second visit: what is left of it is the rounding of its rest, 2^-8 of 2^-8."""
    from hattention_b200 import sliding_window_attention
    q, k, v, do = make(B, T, H, G, K)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sliding_window_attention(*leaves, window, sinks)
    check(q, k, v, window, sinks, o.detach(), None, do, torch.autograd.grad(o, leaves, do), half=2.0 ** -16)


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", [(1, 500, 4, 2, 60, 3), (1, 1500, 5, 1, 130, 150), (2, 200, 8, 8, 200, 0), (1, 8192, 1, 1, 100, 0), (1, 8193, 1, 1, 100, 0), (1, 1025, 1, 1, 1025, 0)])
def test_few_rows(B, T, H, G, K, window, sinks):
    """Longer sequences whose backward visits each tile twice, and the first ones that do not."""
    run(B, T, H, G, K, window, sinks)


@pytest.mark.parametrize("B,T,H,G,window,sinks", [(1, 2048, 2, 1, 2048, 0), (2, 2305, 4, 2, 2048, 130), (1, 2500, 2, 2, 2100, 3), (1, 2177, 3, 1, 5000, 9), (1, 4200, 1, 1, 2050, 600)])
def test_long_windows(B, T, H, G, window, sinks):
    """Windows of thousands: two tiles of queries a CTA where heads are 128 wide."""
    run(B, T, H, G, 128, window, sinks)


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", [(1, 1024, 4, 1, 256, 4), (1, 2000, 8, 1, 200, 16), (1, 1500, 16, 2, 1500, 0), (2, 1000, 6, 2, 1000, 0), (1, 1800, 5, 1, 130, 200)])
def test_shared_out_sums(B, T, H, G, K, window, sinks):
    """Sums of dK and dV that several CTAs share: heads of a group, sinks, windows that reach back to the start."""
    run(B, T, H, G, K, window, sinks)


@pytest.mark.parametrize("scale", [0.01, 0.3])
def test_scale(scale):
    run(1, 200, 2, 1, 64, 90, 2, scale)


def test_long_sequence_of_one_head():
    run(1, 3000, 1, 1, 64, 700, 4)


def test_large_scores():
    """Scores of hundreds: the running maximum keeps every exponent in range, rows of one dominant token are that token."""
    from hattention_b200 import sliding_window_attention
    q, k, v, _ = make(1, 400, 2, 1, 64)
    o = sliding_window_attention(q * 40, k * 10, v, 150, 3)
    S = torch.einsum("bthk,bshk->bhts", (q * 40).double(), (k * 10).double().repeat_interleave(2, 2)) / 8
    P = S.masked_fill(~orc.seen(400, 150, 3, "cuda"), -math.inf).softmax(-1)
    ref = torch.einsum("bhts,bshk->bthk", P, v.double().repeat_interleave(2, 2))
    # products of magnitude 400 sum to scores of magnitude 2000 with an fp32 error of 2^-24 * 64 * 8 * 400 / 8: 2^-6 of a factor at most
    assert torch.isfinite(o).all()
    bound = (HALF + 2.0 ** -5) * torch.einsum("bhts,bshk->bthk", P, v.double().abs().repeat_interleave(2, 2)) + HALF * ref.abs()
    assert ((o.double() - ref).abs() <= bound).all()


def test_equal_scores():
    """q of zeros: every row is the mean of what it sees."""
    from hattention_b200 import sliding_window_attention
    _, k, v, _ = make(1, 500, 1, 1, 128)
    check(torch.zeros_like(k), k, v, 130, 7, sliding_window_attention(torch.zeros_like(k), k, v, 130, 7))


def test_keys_behind_a_query_do_not_reach_it():
    """Later tokens and tokens that left the window change nothing, not a bit, and get no gradient."""
    from hattention_b200 import sliding_window_attention
    q, k, v, do = make(1, 600, 2, 1, 64)
    o = sliding_window_attention(q, k, v, 100, 2)
    k2, v2 = k.clone(), v.clone()
    k2[:, 301:], v2[:, 301:] = 5.0, -7.0
    k2[:, 2:201], v2[:, 2:201] = 3.0, 9.0
    leaves = [t.requires_grad_(True) for t in (q, k2, v2)]
    o2 = sliding_window_attention(*leaves, 100, 2)
    assert torch.equal(o[:, 300], o2[:, 300].detach())
    d = torch.zeros_like(do)
    d[:, 300] = do[:, 300]
    dq, dk, dv = torch.autograd.grad(o2, leaves, d)
    for g in (dk, dv):
        assert (g[:, 301:] == 0).all() and (g[:, 2:201] == 0).all() and (g[:, :2] != 0).any() and (g[:, 201:301] != 0).any()
    assert (dq[:, :300] == 0).all() and (dq[:, 301:] == 0).all()


def test_strided_and_misaligned_operands():
    from hattention_b200 import sliding_window_attention
    B, T, H, G, K = 2, 150, 4, 2, 64
    fused = torch.randn(B, T, H + 2 * G, K, device="cuda").to(torch.bfloat16)
    q, k, v = fused[:, :, :H], fused[:, :, H:H + G], fused[:, :, H + G:]
    want = sliding_window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 40, 1)
    assert torch.equal(sliding_window_attention(q, k, v, 40, 1), want)
    off = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(B, T, H, K)
    assert off.data_ptr() % 16 != 0 and torch.equal(sliding_window_attention(off, k, v, 40, 1), want)
    first = q.transpose(1, 2).contiguous().transpose(1, 2)                    # stored head first
    assert torch.equal(sliding_window_attention(first, k, v, 40, 1), want)
    leaf = fused.clone().requires_grad_(True)
    o = sliding_window_attention(leaf[:, :, :H], leaf[:, :, H:H + G], leaf[:, :, H + G:], 40, 1)
    o.sum().backward()                                                        # a gradient of stride zero, into one leaf
    assert torch.isfinite(leaf.grad).all()


# ------------------------------------------------------------------------------------------ serving
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 2), (64, 4), (100, 0), (33, 150), (500, 3)])
def test_prefill_and_steps(window, sinks, K):
    """Prompts of different lengths, padded; then steps: outputs as those of the whole sequences, slots as filled a token at a time."""
    from hattention_b200 import sliding_window_prefill, sliding_window_step
    B, T, H, G, n = 4, 140, 6, 2, 5
    lengths = torch.tensor([140, 0, 1, 73], device="cuda")
    q, k, v, _ = make(B, T + n, H, G, K)
    o, state = sliding_window_prefill(q[:, :T], k[:, :T], v[:, :T], window, sinks, lengths=lengths)
    assert state.k.shape == (B, sinks + window, G, K) and torch.equal(state.lengths, lengths[:, None].expand(B, G))
    check(q[:, :T], k[:, :T], v[:, :T], window, sinks, o)
    for b, m in enumerate(lengths.tolist()):
        assert torch.equal(state.k[b], orc.window_slots(k[b], m, window, sinks)) and torch.equal(state.v[b], orc.window_slots(v[b], m, window, sinks))
    # the sequences as they really are: lengths[b] prompt tokens, then the n new ones
    seqs = [[torch.cat([x[b, :m], x[b, T:]])[None] for x in (q, k, v)] for b, m in enumerate(lengths.tolist())]
    for i in range(n):
        o, state = sliding_window_step(state, q[:, T + i], k[:, T + i], v[:, T + i])
        for b, m in enumerate(lengths.tolist()):
            qs, ks, vs = (x[:, :m + i + 1] for x in seqs[b])
            P = orc.window_probabilities(qs, ks, window, sinks)[:, :, -1]
            rep = vs.double().repeat_interleave(H // G, 2)
            ref, mag = torch.einsum("bhs,bshk->bhk", P, rep), torch.einsum("bhs,bshk->bhk", P, rep.abs())
            within(o[b:b + 1], ref, (HALF + 2 * D) * mag, f"step {i} of sequence {b}")
            assert torch.equal(state.k[b], orc.window_slots(ks[0], m + i + 1, window, sinks))
            assert torch.equal(state.v[b], orc.window_slots(vs[0], m + i + 1, window, sinks))
    assert torch.equal(state.lengths, (lengths + n)[:, None].expand(B, G))


@pytest.mark.parametrize("B,H,G,K,window,sinks,seen", [(1, 1, 1, 64, 5000, 0, 4999), (1, 32, 8, 128, 4096, 4, 9000), (3, 40, 1, 64, 700, 9, 800), (2, 5, 5, 128, 1000, 0, 50),
                                                       (17, 16, 2, 128, 300, 1, 10 ** 10), (2, 34, 2, 64, 2000, 100, 10 ** 12 + 7)])
def test_single_steps(B, H, G, K, window, sinks, seen):
    """Long caches, many and few heads a group, counts beyond 32 bits; slots that hold no token are NaN and must not be read."""
    from hattention_b200 import WindowState, sliding_window_step
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)
    slots = window + sinks
    kc, vc, q, k, v = r(B, slots, G, K), r(B, slots, G, K), r(B, H, K), r(B, G, K), r(B, G, K)
    n = torch.full((B, G), seen, dtype=torch.int64, device="cuda")
    if seen < slots:
        n[-1] = seen // 2
        for b in range(B):
            kc[b, int(n[b, 0]):], vc[b, int(n[b, 0]):] = math.nan, math.nan
    before = kc.clone()
    o, state = sliding_window_step(WindowState(kc, vc, n.clone(), window, sinks), q, k, v)
    assert torch.equal(state.lengths, n + 1)
    for b in range(B):
        m = int(n[b, 0])
        slot = m if m < sinks else sinks + (m - sinks) % window
        before[b, slot] = k[b]
        held = min(m + 1, slots)
        assert torch.equal(state.k[b, :held], before[b, :held]) and torch.equal(state.v[b, slot], v[b])
        rep = lambda x: x[b, :held].double().repeat_interleave(H // G, 1)
        P = (torch.einsum("hk,shk->hs", q[b].double(), rep(state.k)) / math.sqrt(K)).softmax(-1)
        vd = rep(state.v)
        within(o[b], torch.einsum("hs,shk->hk", P, vd), (HALF + 2 * D) * torch.einsum("hs,shk->hk", P, vd.abs()), f"sequence {b}")


def test_steps_from_nothing():
    from hattention_b200 import WindowState, sliding_window_step
    q, k, v, _ = make(2, 12, 4, 2, 64)
    state = WindowState.empty(2, 2, 64, window=4, sinks=2)
    outs = []
    for t in range(12):
        o, state = sliding_window_step(state, q[:, t], k[:, t], v[:, t])
        outs.append(o)
    check(q, k, v, 4, 2, torch.stack(outs, 1))
    assert torch.equal(outs[0], v[:, 0].repeat_interleave(2, 1))              # the first token sees itself alone


def test_captured_step_and_call():
    """A captured step advances the state at every replay; a captured call follows its inputs; both beside eager work on another stream."""
    from hattention_b200 import WindowState, sliding_window_attention, sliding_window_step
    q, k, v, _ = make(1, 300, 4, 2, 64)
    state = WindowState.empty(1, 2, 64, window=8, sinks=1)
    qs, ks, vs = q[:, 0].clone(), k[:, 0].clone(), v[:, 0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    from hattention_b200 import _lib
    _lib.CHECK_STATUS = False                        # reading the status word synchronises, which a capture refuses
    with torch.cuda.stream(side):
        sliding_window_step(WindowState.empty(1, 2, 64, 8, 1), qs, ks, vs)
        sliding_window_attention(q, k, v, 20, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = sliding_window_step(state, qs, ks, vs)
        whole = sliding_window_attention(q, k, v, 20, 1)
    outs = []
    for t in range(20):
        for dst, src in ((qs, q), (ks, k), (vs, v)):
            dst.copy_(src[:, t])
        graph.replay()
        with torch.cuda.stream(side):
            other = sliding_window_attention(q, k, v, 20, 1)
        outs.append(o.clone())
    check(q[:, :20], k[:, :20], v[:, :20], 8, 1, torch.stack(outs, 1))
    torch.cuda.synchronize()
    assert torch.equal(whole, other)
    check(q, k, v, 20, 1, whole)


def test_library_operators():
    from hattention_b200 import ops, sliding_window_attention  # noqa: F401
    q, k, v, do = make(1, 200, 4, 2, 64)
    o, lse = torch.ops.llattn.window_fwd(q, k, v, 70, 2, 0.125)
    assert torch.equal(o, sliding_window_attention(q, k, v, 70, 2, 0.125))
    check(q, k, v, 70, 2, o, 0.125, do, torch.ops.llattn.window_bwd(q, k, v, o, lse, do, 70, 2, 0.125))
    torch.library.opcheck(torch.ops.llattn.window_bwd.default, (q, k, v, o, lse, do, 70, 2, 0.125), test_utils=("test_schema", "test_faketensor"))
    with pytest.raises(ValueError):
        torch.ops.llattn.window_bwd(q, k, v, o, lse[1:], do, 70, 2, 0.125)


def test_refusals_on_the_gpu():
    from hattention_b200 import WindowState, sliding_window_prefill, sliding_window_step
    q, k, v, _ = make(2, 6, 4, 2, 64)
    with pytest.raises(TypeError):
        sliding_window_prefill(q, k, v, 4, lengths=torch.tensor([1, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        sliding_window_prefill(q, k, v, 4, lengths=torch.tensor([1, 2]))
    s = WindowState.empty(2, 2, 64, 4)
    with pytest.raises(ValueError):
        sliding_window_step(s._replace(window=5), q[:, 0], k[:, 0], v[:, 0])
    with pytest.raises(ValueError):
        sliding_window_step(s._replace(lengths=s.lengths.int()), q[:, 0], k[:, 0], v[:, 0])
    with pytest.raises(ValueError):
        sliding_window_step(s._replace(k=s.k.transpose(0, 1).contiguous().transpose(0, 1)), q[:, 0], k[:, 0], v[:, 0])


def test_calls_and_errors_of_a_thread():
    """A fresh thread makes the same calls, and gets an exception for one that the C entry refuses."""
    import threading
    from hattention_b200 import sliding_window_attention
    q, k, v, _ = make(1, 150, 2, 1, 64)
    many = torch.zeros(65536, 1, 1, 64, device="cuda", dtype=torch.bfloat16)
    got = []

    def call():
        got.append(sliding_window_attention(q, k, v, 50, 1))
        for _ in range(2):
            with pytest.raises(ValueError):
                sliding_window_attention(many, many, many, 1)
        got.append("refused")
    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert len(got) == 2 and torch.equal(got[0], sliding_window_attention(q, k, v, 50, 1))
    with pytest.raises(ValueError):
        sliding_window_attention(many, many, many, 1)


def test_empty_operands():
    from hattention_b200 import sliding_window_attention, sliding_window_prefill
    q = torch.zeros(2, 0, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    k = q.detach()[:, :, :2].requires_grad_(True)
    o = sliding_window_attention(q, k, k, 4)
    assert o.shape == q.shape and torch.autograd.grad(o.sum(), [q, k])[1].shape == k.shape
    _, state = sliding_window_prefill(q, k, k, 4, 1)
    assert state.k.shape == (2, 5, 2, 64) and (state.lengths == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("K,T,window", [(64, 500, 200), (128, 500, 200), (128, 2200, 2048)])
def test_non_finite_keys(K, T, window, bad):
    """A key that is not finite spoils the rows that see it, whatever its place in a tile, and none of the others."""
    from hattention_b200 import sliding_window_attention
    q, k, v = make(1, T, 2, 1, K)[:3]
    q[..., 0] = 1.0                                    # (a product with inf is +-inf, never NaN: of one sign in every row)
    clean = sliding_window_attention(q, k, v, window)
    for s in list(range(128, 144)) + [0, 255, 256, T - 1]:
        spoiled = k.clone()
        spoiled[0, s, 0, 0] = bad
        o = sliding_window_attention(q, spoiled, v, window)
        rows = orc.seen(T, window, 0, "cuda")[:, s]
        assert torch.equal(o[0, ~rows], clean[0, ~rows]), s
        if bad != -math.inf:
            assert o[0, rows].isnan().all(), s
            continue
        # weight 0: the row without that key; nothing is left of a row that sees it alone
        alone = rows & (torch.arange(T, device="cuda") == 0)
        assert o[0, alone].isnan().all()
        left = orc.seen(T, window, 0, "cuda")
        left[:, s] = False
        P = torch.einsum("thk,sk->ths", q[0].double(), k[0, :, 0].double()).mul(K ** -0.5).masked_fill(~left[:, None], -math.inf).softmax(-1)
        mean = lambda x: torch.einsum("ths,sk->thk", P, x[0, :, 0].double())[rows & ~alone]
        within(o[0, rows & ~alone], mean(v), (HALF + 2 * D) * mean(v.abs()), f"without {s}")
