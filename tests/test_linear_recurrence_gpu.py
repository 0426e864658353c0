"""Gated linear recurrence on the GPU against the 64-bit oracle.

Tolerances.  The kernels hold states in fp32.  A token's step multiplies by a decay that is off by at most 2^-22 (expf within 2 ulp) and
rounds at most four times (its own product and sum, once more where it is part of a run's summary): e = 2^-22 + 4 * 2^-24 = 2^-21 relative
to the magnitudes that pass it.  With S the recurrence of |x| from |h0|, the errors are at most e W, W_t = a_t W_{t-1} + S_t.  Outputs of a narrower type are
off by half a step more."""
import pytest
import torch

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
E = 2.0 ** -21
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


def half_step(t):
    return torch.finfo(t).eps / 2


def make(B, T, D, xt, gt, seed=0, state=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen)
    x, g = r(B, T, D).to(xt), torch.nn.functional.logsigmoid(r(B, T, D) * 2 + 2).to(gt)
    return x, g, r(B, D) * 3 if state else None, r(B, T, D).to(xt), r(B, D)


def within(got, ref, err, what):
    tol = err + half_step(got.dtype) * ref.abs() * (1 + 2.0 ** -7) + 1e-30
    worst = ((got.double() - ref).abs() / tol).max().item() if ref.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def magnitudes(a, x, start):
    """(S, W) of the docstring for inputs of magnitude x."""
    s, w, S, W = start, start, [], []
    for t in range(x.shape[1]):
        s = a[:, t] * s + x[:, t]
        w = a[:, t] * w + s
        S.append(s)
        W.append(w)
    return torch.stack(S, 1), torch.stack(W, 1)


def reference(x, g, h0, do, dlast):
    leaves = [t.detach().double().requires_grad_(True) for t in (x, g)] + ([h0.detach().double().requires_grad_(True)] if h0 is not None else [])
    o, last = orc.gated_recurrence(*leaves)
    loss = (o * do.double()).sum() + ((last * dlast.double()).sum() if dlast is not None else 0.0)
    grads = torch.autograd.grad(loss, leaves)
    return o.detach(), last.detach(), [t.detach() for t in grads]


def check(got_o, got_last, grads, x, g, h0, do, dlast):
    if grads is None:
        o, last = orc.gated_recurrence(x, g, h0)
    else:
        o, last, ref = reference(x, g, h0, do, dlast)
    a = g.double().exp()
    zero = torch.zeros_like(a[:, 0])
    S, W = magnitudes(a, x.double().abs(), h0.double().abs() if h0 is not None else zero)
    within(got_o, o, E * W, "o")
    if got_last is not None:
        within(got_last, last, E * W[:, -1], "last state")
    if grads is None:
        return
    # the walk from the other end: dh_t = do_t + a_{t+1} dh_{t+1}
    b = torch.cat([a[:, 1:], zero[:, None] + 1], 1).flip(1)
    U, V = magnitudes(b, do.double().abs().flip(1), dlast.double().abs() if dlast is not None else zero)
    U, V = U.flip(1), V.flip(1)
    before = torch.cat([(h0.double().abs() if h0 is not None else zero)[:, None], S[:, :-1]], 1)
    before_err = torch.cat([zero[:, None], W[:, :-1]], 1)
    within(grads[0], ref[0], E * V, "dx")
    within(grads[1], ref[1], 2 * E * a * (V * before + U * before_err + U * before), "dg")
    if h0 is not None:
        within(grads[2], ref[2], 2 * E * a[:, 0] * V[:, 0], "dh0")


@pytest.mark.parametrize("xt,gt", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 1, 64), (1, 2, 3), (3, 15, 2), (2, 16, 65), (1, 17, 130), (2, 127, 31), (1, 128, 64), (2, 129, 66), (1, 300, 33),
                                   (5, 257, 10), (1, 1025, 7), (1, 2500, 64), (2, 1300, 200)])
def test_forward_and_gradients(B, T, D, xt, gt):
    from hattention_b200 import gated_recurrence
    x, g, h0, do, dlast = make(B, T, D, xt, gt)
    leaves = [t.requires_grad_(True) for t in (x, g, h0)]
    o, last = gated_recurrence(x, g, h0, output_final_state=True)
    assert o.dtype == xt and last.dtype == torch.float32
    grads = torch.autograd.grad([o, last], leaves, [do, dlast])
    check(o.detach(), last.detach(), grads, x.detach(), g.detach(), h0.detach(), do, dlast)


@pytest.mark.parametrize("xt,gt", TYPES)
def test_without_states(xt, gt):
    from hattention_b200 import gated_recurrence
    x, g, _, do, _ = make(2, 200, 70, xt, gt)
    o, last = gated_recurrence(x, g)
    assert last is None
    check(o, None, None, x, g, None, do, None)
    x.requires_grad_(True), g.requires_grad_(True)
    o2, _ = gated_recurrence(x, g)
    assert torch.equal(o, o2.detach())
    check(o, None, torch.autograd.grad(o2, [x, g], do), x.detach(), g.detach(), None, do, None)


def test_gradient_of_the_last_state_alone():
    from hattention_b200 import gated_recurrence
    x, g, h0, do, dlast = make(2, 150, 12, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, g, h0)]
    _, last = gated_recurrence(x, g, h0, output_final_state=True)
    grads = torch.autograd.grad(last, leaves, dlast)
    o, _ = gated_recurrence(x, g, h0)
    check(o.detach(), None, grads, x.detach(), g.detach(), h0.detach(), torch.zeros_like(do), dlast)


def test_decays_of_minus_infinity_start_anew():
    """-inf at the first token of every sequence packs sequences into one; the states before do not reach across, whatever they are."""
    from hattention_b200 import gated_recurrence
    x, g, h0, do, _ = make(1, 400, 40, torch.float32, torch.float32)
    starts = [0, 1, 130, 256, 399]
    packed = g.clone()
    packed[:, starts] = -torch.inf
    leaves = [t.requires_grad_(True) for t in (x, packed)]
    o, _ = gated_recurrence(x, packed, h0)
    dx, dg = torch.autograd.grad(o, leaves, do)
    assert torch.isfinite(dg).all() and (dg[:, starts] == 0).all()
    for s, e in zip(starts, starts[1:] + [400]):
        part = [t[:, s:e].detach().clone().requires_grad_(True) for t in (x, g)]
        po, _ = gated_recurrence(*part)
        pdx, pdg = torch.autograd.grad(po, part, do[:, s:e].contiguous())
        S, W = magnitudes(part[1].detach().double().exp(), part[0].detach().double().abs(), torch.zeros(1, 40, device="cuda", dtype=torch.float64))
        assert ((o[:, s:e] - po).abs() <= 2 * E * W + 1e-30).all()
        assert torch.allclose(dx[:, s:e], pdx, rtol=1e-4, atol=1e-4)


def test_zero_and_vanishing_decays():
    """g = 0 sums, g far below sums nothing: no products that leave the range."""
    from hattention_b200 import gated_recurrence
    x = torch.ones(1, 1000, 4, device="cuda")
    g = torch.zeros_like(x)
    assert torch.equal(gated_recurrence(x, g)[0][0, :, 0], torch.arange(1, 1001, device="cuda", dtype=torch.float32))
    g.fill_(-200.0)
    assert torch.equal(gated_recurrence(x, g)[0], x)


def test_strided_and_misaligned_operands():
    from hattention_b200 import gated_recurrence
    big, gbig, _, do, _ = make(2, 100, 131, torch.bfloat16, torch.float32)
    x, g = big[:, :, 1:65], gbig.transpose(0, 1).contiguous().transpose(0, 1)[:, :, 3:67]
    check(gated_recurrence(x, g)[0], None, None, x, g, None, do, None)
    flat = torch.randn(1 + 100 * 64, device="cuda").to(torch.bfloat16)[1:].view(1, 100, 64)          # starts between 16-byte boundaries
    check(gated_recurrence(flat, g[:1])[0], None, None, flat, g[:1], None, do, None)
    x = x.detach().requires_grad_(True)
    o, _ = gated_recurrence(x, g)
    d = do[:, :, :64]
    expanded = d[:, :1].expand_as(o)                                                                 # a gradient of stride zero
    dx, = torch.autograd.grad(o, x, expanded)
    x2 = x.detach().clone().requires_grad_(True)
    dx2, = torch.autograd.grad(gated_recurrence(x2, g)[0], x2, expanded.contiguous())
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("B,D", [(1, 1), (3, 7), (64, 2048), (5, 1001)])
@pytest.mark.parametrize("xt,gt", TYPES)
def test_steps_follow_a_prompt(B, D, xt, gt):
    from hattention_b200 import gated_recurrence, gated_recurrence_step
    T, n = 37, 4
    x, g, h0, _, _ = make(B, T + n, D, xt, gt)
    o, state = gated_recurrence(x[:, :T], g[:, :T], h0, output_final_state=True)
    outs = [o]
    for t in range(T, T + n):
        o, same = gated_recurrence_step(state, x[:, t], g[:, t])
        assert same is state
        outs.append(o[:, None])
    check(torch.cat(outs, 1), state, None, x, g, h0, x, None)


def test_empty_operands():
    from hattention_b200 import gated_recurrence
    x = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    h0 = torch.ones(2, 8, device="cuda")
    o, last = gated_recurrence(x, x, h0, output_final_state=True)
    assert o.shape == (2, 0, 8) and torch.equal(last, h0)


def test_captured_and_replayed_on_another_stream():
    from hattention_b200 import gated_recurrence, gated_recurrence_step
    x, g, h0, _, _ = make(2, 300, 64, torch.bfloat16, torch.float32)
    state = h0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_recurrence(x, g, h0)
        gated_recurrence_step(state, x[:, 0], g[:, 0])
    torch.cuda.current_stream().wait_stream(side)
    state.copy_(h0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = gated_recurrence(x, g, h0)
        s, _ = gated_recurrence_step(state, x[:, 0], g[:, 0])
    x.neg_()
    graph.replay()
    graph.replay()
    want, _ = gated_recurrence(x, g, h0)
    assert torch.equal(o, want)
    again = h0.clone()
    for _ in range(2):
        w, _ = gated_recurrence_step(again, x[:, 0], g[:, 0])
    assert torch.equal(s, w) and torch.equal(state, again)


def test_library_operators():
    from hattention_b200 import gated_recurrence, ops  # noqa: F401
    x, g, h0, do, dlast = make(2, 200, 34, torch.bfloat16, torch.float32)
    o, last, states = torch.ops.llattn.recurrence_fwd(x, g, h0)
    want, wlast = gated_recurrence(x, g, h0, output_final_state=True)
    assert torch.equal(o, want) and torch.equal(last, wlast)
    grads = torch.ops.llattn.recurrence_bwd(x, g, states, do, dlast)
    check(o, last, grads, x, g, h0, do, dlast)
    torch.library.opcheck(torch.ops.llattn.recurrence_fwd.default, (x, g, h0), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.llattn.recurrence_bwd.default, (x, g, states, do, None), test_utils=("test_schema", "test_faketensor"))
    with pytest.raises(ValueError):
        torch.ops.llattn.recurrence_bwd(x, g, states[1:], do, None)


def test_same_call_same_bits():
    from hattention_b200 import gated_recurrence
    x, g, h0, do, _ = make(2, 3000, 96, torch.float32, torch.float32)
    x.requires_grad_(True), g.requires_grad_(True)
    runs = []
    for _ in range(3):
        o, _ = gated_recurrence(x, g, h0)
        runs.append((o.detach(),) + torch.autograd.grad(o, [x, g], do))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
