"""The C entries of the hybrid-stack operators write what the header says and nothing beside it: every buffer lies between guard bytes, workspaces and kept statistics have
exactly the size that the library asks for."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
GUARD, FILL = 4096, 0xA5


class Buffers:
    """Tensors of exact size, 256-byte aligned, with guard bytes in front of and behind each."""

    def __init__(self):
        self.all = []

    def raw(self, nbytes):
        space = torch.full((GUARD + nbytes + GUARD + 256,), FILL, dtype=torch.uint8, device="cuda")
        at = GUARD + (-(space.data_ptr() + GUARD)) % 256
        self.all.append((space, at, nbytes))
        return space[at:at + nbytes]

    def empty(self, *shape, dtype=torch.bfloat16):
        n = 1
        for s in shape:
            n *= s
        return self.raw(n * torch.empty(0, dtype=dtype).element_size()).view(dtype).view(shape)

    def of(self, t):
        return self.empty(*t.shape, dtype=t.dtype).copy_(t)

    def check(self):
        torch.cuda.synchronize()
        for space, at, n in self.all:
            assert (space[:at] == FILL).all() and (space[at + n:] == FILL).all(), f"written beside a buffer of {n} bytes"


def lib():
    from hattention_b200 import _lib
    return _lib.lib()


def p(t):
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("xt,wt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,N", [(1, 1), (1, 7), (3, 33), (5, 128), (10, 1001), (11, 1000), (9, 2050), (150, 2048), (700, 96), (2, 8192), (3, 5001), (4, 9000)])
def test_layer_norm(rows, N, xt, wt):
    b = Buffers()
    x, dy, w, bias = b.of(torch.randn(rows, N, device="cuda").to(xt)), b.of(torch.randn(rows, N, device="cuda").to(xt)), b.of(torch.randn(N, device="cuda").to(wt)), \
        b.of(torch.randn(N, device="cuda").to(wt))
    y, dx, dw, db = b.empty(rows, N, dtype=xt), b.empty(rows, N, dtype=xt), b.empty(N, dtype=wt), b.empty(N, dtype=wt)
    mean, rstd = b.empty(rows, dtype=torch.float32), b.empty(rows, dtype=torch.float32)
    xf, wf = int(xt == torch.float32), int(wt == torch.float32)
    assert lib().llattn_layer_norm_fwd(p(x), xf, p(w), p(bias), wf, p(y), p(mean), p(rstd), 1e-5, rows, N, stream()) == 0
    n = lib().llattn_layer_norm_bwd_workspace_bytes(rows, N)
    ws = b.raw(n)
    assert lib().llattn_layer_norm_bwd(p(x), xf, p(w), wf, p(mean), p(rstd), p(dy), p(dx), p(dw), p(db), p(ws), n, rows, N, stream()) == 0
    b.check()


@pytest.mark.parametrize("xt,gt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 5, 3), (1, 64, 16), (3, 65, 30), (1, 600, 17), (2, 700, 100), (1, 1500, 72), (2, 3000, 33)])
def test_recurrence(B, T, D, xt, gt):
    b = Buffers()
    r = lambda *s: torch.randn(*s, device="cuda")
    x, g, do = b.of(r(B, T, D).to(xt)), b.of((-r(B, T, D).abs()).to(gt)), b.of(r(B, T, D).to(xt))
    h0, dl = b.of(r(B, D)), b.of(r(B, D))
    o, dx, dg = b.empty(B, T, D, dtype=xt), b.empty(B, T, D, dtype=xt), b.empty(B, T, D, dtype=gt)
    last, dh0 = b.empty(B, D, dtype=torch.float32), b.empty(B, D, dtype=torch.float32)
    states = b.raw(lib().llattn_recurrence_states_bytes(B, T, D))
    xf, gf = int(xt == torch.float32), int(gt == torch.float32)
    assert lib().llattn_recurrence_fwd(p(x), xf, p(g), gf, p(h0), p(o), p(last), p(states), B, T, D, stream()) == 0
    assert lib().llattn_recurrence_bwd(p(x), xf, p(g), gf, p(states), p(do), p(dl), p(dx), p(dg), p(dh0), B, T, D, stream()) == 0
    assert lib().llattn_recurrence_step(p(last), p(x), xf, p(g), gf, p(o), 1, D, stream()) == 0
    b.check()


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("B,T,H,G,window,sinks", [(1, 1, 1, 1, 1, 0), (2, 3, 2, 1, 2, 1), (1, 129, 4, 2, 40, 0), (2, 300, 2, 2, 20, 3), (1, 700, 8, 1, 100, 5), (1, 900, 2, 1, 130, 300),
                                                  (1, 1024, 4, 1, 256, 4), (1, 2000, 8, 1, 200, 16), (1, 2048, 16, 2, 2048, 0), (2, 1000, 16, 4, 1000, 0)])
def test_window(B, T, H, G, window, sinks, K):
    b = Buffers()
    r = lambda n: b.of(torch.randn(B, T, n, K, device="cuda").to(torch.bfloat16))
    q, k, v, do = r(H), r(G), r(G), r(H)
    o, dq, dk, dv = b.empty(B, T, H, K), b.empty(B, T, H, K), b.empty(B, T, G, K), b.empty(B, T, G, K)
    stats = b.raw(lib().llattn_window_stats_bytes(B, T, H, K, window, sinks))
    n = lib().llattn_window_workspace_bytes(B, T, H, G, K, window, sinks)
    small, ws = b.raw(256), b.raw(n)
    assert lib().llattn_window_fwd(p(q), p(k), p(v), p(o), p(stats), p(small), 256, B, T, H, G, K, window, sinks, 0.125, stream()) == 0
    assert lib().llattn_window_bwd(p(q), p(k), p(v), p(o), p(stats), p(do), p(dq), p(dk), p(dv), p(ws), n, B, T, H, G, K, window, sinks, 0.125, stream()) == 0
    kc, vc, counts = b.empty(B, sinks + window, G, K), b.empty(B, sinks + window, G, K), b.empty(B, G, dtype=torch.int64)
    lengths = b.of(torch.arange(B, device="cuda") * T // 2)
    assert lib().llattn_window_fill(p(k), p(v), p(lengths), p(kc), p(vc), p(counts), B, T, G, K, window, sinks, stream()) == 0
    q1, k1, v1, o1 = b.of(q[:, 0]), b.of(k[:, 0]), b.of(v[:, 0]), b.empty(B, H, K)
    for _ in range(3):
        assert lib().llattn_window_step(p(q1), p(k1), p(v1), p(kc), p(vc), p(counts), p(o1), B, H, G, K, window, sinks, 0.125, stream()) == 0
    b.check()
    assert torch.equal(counts, (lengths + 3)[:, None].expand(B, G))
    out = ctypes.c_int(-1)
    for w in (small, ws):
        assert lib().llattn_workspace_status(p(w), ctypes.byref(out), stream()) == 0 and out.value == 0


def test_negative_counts_start_at_the_first_slot():
    b = Buffers()
    q, k, v = (b.of(torch.randn(1, n, 64, device="cuda").to(torch.bfloat16)) for n in (2, 1, 1))
    kc, vc, o = b.empty(1, 5, 1, 64), b.empty(1, 5, 1, 64), b.empty(1, 2, 64)
    counts = b.of(torch.tensor([[-7]], device="cuda"))
    assert lib().llattn_window_step(p(q), p(k), p(v), p(kc), p(vc), p(counts), p(o), 1, 2, 1, 64, 4, 1, 0.125, stream()) == 0
    b.check()
    assert torch.equal(kc[0, 0], k[0]) and torch.equal(o[0], v[0].expand(2, 64)) and int(counts) == 1
