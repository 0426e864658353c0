"""The hybrid-stack operators in the ways that a program uses them beside plain calls: sizes whose offsets pass 32 bits, two streams at once, captured training steps, gradients
of gradients."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def test_recurrence_beyond_32_bits():
    """2^31 values and more: the last channels of the last sequence are those of the same channels by themselves."""
    from hattention_b200 import gated_recurrence
    B, T, D, W = 2, 2 ** 19 + 3, 2048, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(B, T, D, dtype=BF, device="cuda").normal_(generator=gen)
    g = torch.empty_like(x).normal_(generator=gen).abs_().neg_()
    do = torch.empty_like(x).normal_(generator=gen)
    part = [t[1:, :, -W:].contiguous() for t in (x, g, do)]
    x.requires_grad_(True), g.requires_grad_(True)
    o, last = gated_recurrence(x, g, output_final_state=True)
    dx, dg = torch.autograd.grad(o, (x, g), do)
    px, pg = part[0].requires_grad_(True), part[1].requires_grad_(True)
    po, plast = gated_recurrence(px, pg, output_final_state=True)
    pdx, pdg = torch.autograd.grad(po, (px, pg), part[2])
    # (strips of other widths: other orders of the fp32 sums; a value next to a border may round to the other side of it)
    for got, want in ((o, po), (dx, pdx), (dg, pdg)):
        got, want = got[1:, :, -W:].detach().float(), want.detach().float()
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-4).all()
    assert (last[1:, -W:] - plast).abs().max() < 1e-4


def test_window_beyond_32_bits():
    """The last tokens of 2^31 values of q see what they see by themselves, bit by bit (the cut falls between tiles)."""
    from hattention_b200 import sliding_window_attention
    T, H, G, K, window, tail = 2 ** 19 + 77, 32, 1, 128, 200, 1024 + 77
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda n: torch.empty(1, T, n, K, dtype=BF, device="cuda").normal_(generator=gen)
    leaves, do = [r(H), r(G), r(G)], r(H)
    part = [t[:, T - tail:].clone() for t in leaves]
    o = sliding_window_attention(*[t.requires_grad_(True) for t in leaves], window)
    d = torch.autograd.grad(o, leaves, do)
    po = sliding_window_attention(*[t.requires_grad_(True) for t in part], window)
    pd = torch.autograd.grad(po, part, do[:, T - tail:])
    for got, want in zip((o,) + d, (po,) + pd):
        got, want = got[:, T - 577:].detach(), want[:, -577:].detach()
        if got.shape[2] == H:
            assert torch.equal(got, want)
        else:                                # (dk, dv: shared out over CTAs in the short call, not in the long one)
            assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-3).all()


def test_window_step_beyond_32_bits():
    """A cache of more than 2^31 values: the new token goes to its last slot, and is what a query along its key sees."""
    from hattention_b200 import WindowState, sliding_window_step
    G, K, window = 8, 128, 2 ** 21 + 5
    state = WindowState.empty(1, G, K, window)
    state.lengths.fill_(window - 1)
    q = torch.full((1, 2 * G, K), 3.0, dtype=BF, device="cuda")
    k, v = q[:, :G].clone(), torch.randn(1, G, K, device="cuda").to(BF)
    o, state = sliding_window_step(state, q, k, v)       # (a score of 102 against zeros)
    assert torch.equal(state.k[0, -1], k[0]) and torch.equal(state.v[0, -1], v[0]) and (state.lengths == window).all()
    assert (o - v.repeat_interleave(2, 1)).abs().max() <= 2.0 ** -7 * v.abs().max()


def test_layer_norm_beyond_32_bits():
    from hattention_b200 import layer_norm
    rows, N, tail = 2 ** 20 + 9, 2048, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, N, dtype=BF, device="cuda").normal_(generator=gen)
    dy = torch.empty_like(x).normal_(generator=gen)
    w, b = torch.randn(N, device="cuda"), torch.randn(N, device="cuda")
    px = x[-tail:].clone().requires_grad_(True)
    x.requires_grad_(True)
    y, py = layer_norm(x, w, b), layer_norm(px, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    pdx, = torch.autograd.grad(py, px, dy[-tail:])
    assert torch.equal(y[-tail:], py) and torch.equal(dx[-tail:], pdx)


@pytest.mark.parametrize("B,T,D", [(150, 300, 64), (40, 2000, 128), (300, 65, 48), (10, 900, 2048)])
def test_recurrence_of_many_strips(B, T, D):
    """Enough strips to fill the chip without clusters, or with small ones."""
    from hattention_b200 import gated_recurrence
    from oracle import hybrid_oracle as orc
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B, T, D, device="cuda", generator=gen).requires_grad_(True)
    g = (-torch.randn(B, T, D, device="cuda", generator=gen).abs()).requires_grad_(True)
    do = torch.randn(B, T, D, device="cuda", generator=gen)
    o, _ = gated_recurrence(x, g)
    dx, dg = torch.autograd.grad(o, (x, g), do)
    pick = slice(0, None, max(1, B // 4))
    xd, gd = x.detach()[pick].double().requires_grad_(True), g.detach()[pick].double().requires_grad_(True)
    ref, _ = orc.gated_recurrence(xd, gd)
    rdx, rdg = torch.autograd.grad(ref, (xd, gd), do[pick].double())
    # states are sums of values of about 1 with weights that add up to at most a few tens: 2^-24 of that a step, a few hundred steps that count
    for got, want in ((o, ref), (dx, rdx), (dg, rdg)):
        assert (got.detach()[pick].double() - want.detach()).abs().max() < 2.0 ** -24 * 64 * 256


def stack(x, w, b, q, k, v, g):
    from hattention_b200 import gated_recurrence, layer_norm, sliding_window_attention
    h, _ = gated_recurrence(layer_norm(x, w, b), g)
    return sliding_window_attention(q + h.unflatten(-1, (4, 64)), k, v, 50, 2)


def leaves(seed, T=300):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(BF)
    return [r(2, T, 256), r(256), r(256), r(2, T, 4, 64), r(2, T, 2, 64), r(2, T, 2, 64), -r(2, T, 256).abs()], r(2, T, 4, 64)


def step(ts, do):
    o = stack(*ts)
    return (o.detach(),) + torch.autograd.grad(o, ts, do)


def test_captured_training_step():
    """Forward and backward of all three in one graph, twice, replayed in turn with other inputs."""
    from hattention_b200 import _lib
    ts, do = leaves(0)
    ts = [t.requires_grad_(True) for t in ts]
    status, _lib.CHECK_STATUS = _lib.CHECK_STATUS, False
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(ts, do)
        torch.cuda.current_stream().wait_stream(side)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(ts, do)
        with torch.cuda.graph(other):
            got2 = step(ts, do)
        for seed in (1, 2):
            new, ndo = leaves(seed)
            with torch.no_grad():
                for a, b in zip(ts, new):
                    a.copy_(b)
                do.copy_(ndo)
            graph.replay()
            other.replay()
            want = step(ts, do)
            for a, b, c in zip(got, got2, want):
                assert torch.equal(a, c) and torch.equal(b, c)
    finally:
        _lib.CHECK_STATUS = status


def test_two_streams_at_once():
    """Two training steps side by side, many times, give the bits of one alone."""
    from hattention_b200 import _lib
    sets = [leaves(s, 700) for s in (3, 4)]
    sets = [([t.requires_grad_(True) for t in ts], do) for ts, do in sets]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    status, _lib.CHECK_STATUS = _lib.CHECK_STATUS, False
    try:
        for _ in range(20):
            got = []
            for s, st in zip(sets, streams):
                with torch.cuda.stream(st):
                    got.append(step(*s))
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert all(torch.equal(a, b) for a, b in zip(g, w))
    finally:
        _lib.CHECK_STATUS = status


def test_one_tensor_in_several_places():
    """q, k and v from one leaf, a leaf broadcast over a batch: gradients add up."""
    from hattention_b200 import sliding_window_attention
    x = torch.randn(1, 200, 2, 64, device="cuda").to(BF).requires_grad_(True)
    do = torch.randn(3, 200, 2, 64, device="cuda").to(BF)
    a = [x.detach().expand(3, -1, -1, -1).contiguous().requires_grad_(True) for _ in range(3)]
    want = sum(torch.autograd.grad(sliding_window_attention(*a, 30), a, do)).float().sum(0, keepdim=True)
    e = x.expand(3, -1, -1, -1)
    o = sliding_window_attention(e, e, e, 30)
    got, = torch.autograd.grad(o, x, do)
    # (sums of nine bf16 gradients, in bf16 and in two orders)
    assert ((got.float() - want).abs() <= 2.0 ** -5 * want.abs() + 2.0 ** -5).all()


def test_gradients_of_gradients_raise():
    from hattention_b200 import gated_recurrence, layer_norm, sliding_window_attention
    x = torch.randn(2, 40, 2, 64, device="cuda").to(BF).requires_grad_(True)
    for f in (lambda x: layer_norm(x), lambda x: gated_recurrence(x.flatten(2), -x.flatten(2).abs())[0], lambda x: sliding_window_attention(x, x, x, 8)):
        plain, = torch.autograd.grad(f(x).float().square().sum(), x)
        first, = torch.autograd.grad(f(x).float().square().sum(), x, create_graph=True)
        assert torch.equal(first, plain) and first.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            first.float().square().sum().backward()


def test_cache_of_one_tensor_is_refused():
    from hattention_b200 import WindowState, sliding_window_step
    s = WindowState.empty(1, 2, 64, 8)
    q = torch.zeros(1, 2, 64, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="one tensor"):
        sliding_window_step(s._replace(v=s.k), q, q, q)


def test_steps_and_graphs():
    """A step has no graph, whatever its operands; a graph that kept a state notices that a step has advanced it; inference tensors are advanced too."""
    from hattention_b200 import WindowState, gated_recurrence, gated_recurrence_step, sliding_window_step
    x = torch.randn(2, 30, 64, device="cuda", requires_grad=True)
    _, h = gated_recurrence(x, -x.detach().abs(), output_final_state=True)
    loss = h.square().sum()                              # (keeps h)
    want = (-x[:, 0].detach().abs()).exp() * h.detach() + x[:, 0].detach()
    o, h2 = gated_recurrence_step(h, x[:, 0], -x[:, 0].abs())
    assert h2 is h and not o.requires_grad and torch.allclose(h.detach(), want, rtol=1e-5, atol=1e-6)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    q = torch.randn(1, 2, 64, device="cuda").to(BF).requires_grad_(True)
    s = WindowState.empty(1, 2, 64, 8)
    kept = s.k.float().requires_grad_(False)
    o, s = sliding_window_step(s, q, q, q)
    assert not o.requires_grad and torch.equal(o, q) and (kept == 0).all() and s.k._version == 1 and s.lengths._version == 1
    with torch.inference_mode():
        s = WindowState.empty(1, 2, 64, 8)
        h = torch.zeros(2, 64, device="cuda")
        for _ in range(2):
            o, s = sliding_window_step(s, q, q, q)
            gated_recurrence_step(h, x[:, 0], -x[:, 0].abs())
        assert (s.lengths == 2).all()
