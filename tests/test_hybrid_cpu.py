"""CPU side of the hybrid-stack operators (gated recurrence, windowed attention, layer norm): refusals of the Python entry points and of the C
ABI before a device is touched, empty operands, fake-tensor shapes, and the 64-bit oracle against differences."""
import ctypes
import math

import pytest
import torch

from oracle import hybrid_oracle as orc


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as ge
    ge.build()
    import hattention_b200
    return hattention_b200


def test_refusals(pkg):
    bf, f = torch.bfloat16, torch.float32
    x = torch.zeros(2, 5, 8, dtype=bf)
    with pytest.raises(RuntimeError):                                   # no CPU path
        pkg.gated_recurrence(x, x)
    with pytest.raises(ValueError):
        pkg.gated_recurrence(x, x[:, :4])
    with pytest.raises(ValueError):
        pkg.gated_recurrence(x[0], x[0])
    with pytest.raises(TypeError):
        pkg.gated_recurrence(x.half(), x)
    with pytest.raises(TypeError):
        pkg.gated_recurrence(x.float(), x)                              # g narrower than x
    with pytest.raises(TypeError):
        pkg.gated_recurrence(x, x, initial_state=torch.zeros(2, 8, dtype=bf))
    with pytest.raises(ValueError):
        pkg.gated_recurrence(x, x, initial_state=torch.zeros(2, 7))
    with pytest.raises(RuntimeError):
        pkg.gated_recurrence_step(torch.zeros(2, 8), x[:, 0], x[:, 0])
    with pytest.raises(ValueError):
        pkg.gated_recurrence_step(torch.zeros(3, 8), x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError):
        pkg.layer_norm(x)
    with pytest.raises(TypeError):
        pkg.layer_norm(x.half())
    with pytest.raises(TypeError):
        pkg.layer_norm(x, torch.ones(8), torch.ones(8, dtype=bf))
    with pytest.raises(ValueError):
        pkg.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        pkg.layer_norm(torch.zeros(3, 0))
    q, k = torch.zeros(1, 5, 4, 64, dtype=bf), torch.zeros(1, 5, 2, 64, dtype=bf)
    with pytest.raises(RuntimeError):
        pkg.sliding_window_attention(q, k, k, 4)
    for window, sinks in ((0, 0), (-1, 0), (4, -1), (2 ** 30, 0)):
        with pytest.raises(ValueError):
            pkg.sliding_window_attention(q, k, k, window, sinks)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            pkg.sliding_window_attention(q, k, k, 4, scale=scale)
    with pytest.raises(ValueError):
        pkg.sliding_window_attention(q[:, :, :3], k, k, 4)              # 3 heads over 2
    with pytest.raises(ValueError):
        pkg.sliding_window_attention(q, k[:, :4], k[:, :4], 4)
    with pytest.raises(NotImplementedError):
        pkg.sliding_window_attention(q.float(), k.float(), k.float(), 4)
    with pytest.raises(NotImplementedError):
        pkg.sliding_window_attention(q[..., :32], k[..., :32], k[..., :32], 4)
    with pytest.raises(RuntimeError):
        pkg.sliding_window_prefill(q, k, k, 4)
    state = pkg.WindowState.empty(1, 2, 64, 4, 1, device="cpu")
    assert state.k.shape == (1, 5, 2, 64) and state.lengths.shape == (1, 2)
    with pytest.raises(RuntimeError):
        pkg.sliding_window_step(state, q[:, 0], k[:, 0], k[:, 0])
    with pytest.raises(ValueError):
        pkg.sliding_window_step(state._replace(window=0), q[:, 0], k[:, 0], k[:, 0])


def test_c_entries_reject_bad_arguments(pkg):
    from hattention_b200 import _lib
    lib = _lib.lib()
    P, null = ctypes.c_void_p, ctypes.c_void_p(0)
    ok, odd = P(4096), P(4098)
    fwd = lambda x=ok, xf=0, gf=1, B=1, T=8, D=8: lib.llattn_recurrence_fwd(x, xf, ok, gf, null, ok, null, null, B, T, D, null)
    assert fwd(B=0) == -1 and fwd(T=0) == -1 and fwd(D=0) == -1 and fwd(xf=1, gf=0) == -1
    assert fwd(x=null) == -6 and fwd(x=odd) == -9
    bwd = lambda states=ok, dx=ok: lib.llattn_recurrence_bwd(ok, 0, ok, 1, states, ok, null, dx, ok, null, 1, 8, 8, null)
    assert bwd(states=null) == -6 and bwd(dx=odd) == -9
    assert lib.llattn_recurrence_step(null, ok, 0, ok, 0, ok, 1, 8, null) == -6
    assert lib.llattn_recurrence_step(ok, ok, 0, odd, 0, ok, 1, 8, null) == -9
    assert lib.llattn_recurrence_states_bytes(2, 1, 5) == 2 * 5 * 4 and lib.llattn_recurrence_states_bytes(1, 0, 5) == 0

    win = dict(B=1, T=8, H=4, G=2, K=64, window=4, sinks=0, scale=1.0)

    def wfwd(q=ok, ws=ok, n=256, **kw):
        a = {**win, **kw}
        return lib.llattn_window_fwd(q, ok, ok, ok, null, ws, n, a["B"], a["T"], a["H"], a["G"], a["K"], a["window"], a["sinks"], a["scale"], null)
    for bad in ({"B": 0}, {"T": 0}, {"H": 0}, {"G": 0}, {"K": 96}, {"window": 0}, {"sinks": -1}, {"scale": 0.0}, {"scale": math.nan}, {"T": 2 ** 24 + 1}):
        assert wfwd(**bad) == -1, bad
    assert wfwd(H=3) == -4 and wfwd(q=null) == -6 and wfwd(q=odd) == -9
    assert wfwd(ws=null) == -5 and wfwd(n=255) == -5 and wfwd(ws=P(4096 + 16)) == -5
    need = lib.llattn_window_workspace_bytes(1, 8, 4, 2, 64, 4, 0)
    assert need >= 256 + 4 * 8 * 4 and lib.llattn_window_stats_bytes(1, 8, 4, 64, 4, 0) >= 4 * 8 * 4
    wbwd = lambda stats, n: lib.llattn_window_bwd(*[ok] * 4, stats, *[ok] * 5, n, 1, 8, 4, 2, 64, 4, 0, 1.0, null)
    assert wbwd(null, need) == -6 and wbwd(odd, need) == -9 and wbwd(ok, need - 1) == -5
    assert lib.llattn_window_fill(null, ok, null, ok, ok, ok, 1, 8, 2, 64, 4, 0, null) == -6
    assert lib.llattn_window_fill(ok, ok, null, ok, odd, ok, 1, 8, 2, 64, 4, 0, null) == -9
    assert lib.llattn_window_step(*[ok] * 6, null, 1, 4, 2, 64, 4, 0, 1.0, null) == -6
    assert lib.llattn_window_step(*[ok] * 7, 1, 4, 2, 64, 0, 0, 1.0, null) == -1

    nf = lambda x=ok, mean=null, rstd=null, rows=4, N=8, xf=0, wf=1: lib.llattn_layer_norm_fwd(x, xf, null, null, wf, ok, mean, rstd, 1e-5, rows, N, null)
    assert nf(rows=0) == -1 and nf(N=0) == -1 and nf(xf=1, wf=0) == -1 and nf(x=null) == -6 and nf(mean=ok) == -6 and nf(x=odd) == -9
    nb = lambda dw, ws, n: lib.llattn_layer_norm_bwd(ok, 0, null, 1, ok, ok, ok, ok, dw, null, ws, n, 4, 8, null)
    need = lib.llattn_layer_norm_bwd_workspace_bytes(4, 8)
    assert need > 0 and nb(ok, null, need) == -5 and nb(ok, ok, need - 1) == -5 and nb(odd, ok, need) == -9


def test_operators_trace_with_fake_tensors(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    import hattention_b200.ops  # noqa: F401
    op = torch.ops.llattn
    with FakeTensorMode():
        x = torch.empty(2, 300, 6, dtype=torch.bfloat16)
        o, last, states = op.recurrence_fwd(x, x.float(), None)
        assert o.shape == x.shape and last.shape == (2, 6) and states.dtype == torch.float32
        dx, dg, dh = op.recurrence_bwd(x, x.float(), states, o, None)
        assert dx.dtype == torch.bfloat16 and dg.dtype == torch.float32 and dh.shape == (2, 6)
        q, k = torch.empty(1, 5, 4, 64, dtype=torch.bfloat16), torch.empty(1, 5, 2, 64, dtype=torch.bfloat16)
        o, stats = op.window_fwd(q, k, k, 3, 1, 0.125)
        assert [t.shape for t in op.window_bwd(q, k, k, o, stats, o, 3, 1, 0.125)] == [q.shape, k.shape, k.shape]
        w = torch.empty(6)
        y, stats = op.layer_norm_fwd(x, w, None, 1e-5)
        assert [t.shape for t in op.layer_norm_bwd(x, w, stats, y)] == [x.shape, w.shape, w.shape]


def test_oracle_gradients_against_differences():
    torch.manual_seed(0)
    d = dict(dtype=torch.float64, requires_grad=True)
    x, g, h = torch.randn(2, 7, 3, **d), (-torch.rand(2, 7, 3, dtype=torch.float64)).requires_grad_(True), torch.randn(2, 3, **d)
    assert torch.autograd.gradcheck(orc.gated_recurrence, (x, g, h))
    q, k, v = torch.randn(1, 9, 4, 3, **d), torch.randn(1, 9, 2, 3, **d), torch.randn(1, 9, 2, 3, **d)
    assert torch.autograd.gradcheck(lambda *a: orc.sliding_window_attention(*a, 3, 2), (q, k, v))
    w, b = torch.randn(3, **d), torch.randn(3, **d)
    assert torch.autograd.gradcheck(lambda *a: orc.layer_norm(*a), (x, w, b))


@pytest.mark.parametrize("T,window,sinks", [(9, 4, 2), (9, 20, 0), (5, 1, 9), (12, 3, 3)])
def test_window_and_sinks_of_the_oracle(T, window, sinks):
    """What a query sees, counted one by one; and the slots of a decoding state hold exactly what the next query sees."""
    see = orc.seen(T, window, sinks, "cpu")
    for t in range(T):
        assert see[t].nonzero().flatten().tolist() == [s for s in range(t + 1) if t - s < window or s < sinks]
    tokens = torch.arange(1, T + 1, dtype=torch.float64)[:, None]
    for n in range(1, T + 1):
        held = [int(i) - 1 for i in orc.window_slots(tokens, n, window, sinks).flatten() if i > 0]
        assert sorted(held) == see[n - 1].nonzero().flatten().tolist()
