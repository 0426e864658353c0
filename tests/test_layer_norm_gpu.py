"""Layer norm on the GPU against the 64-bit oracle.

Tolerances.  A sum over a row adds at most 64 values in a thread and then at most 10 times across threads or warps, so it is off by at most e = 96 * 2^-24 times
the sum of magnitudes (further rounds of the terms themselves included).  The mean is off by e mean|x|, rstd by 2 e relative (a sum of squares, and a shift of the
mean that enters squared), so xhat by X = e rstd mean|x| + 2 e |xhat|.  Sums over rows: at most rows additions.  Outputs are off by half a step of their type more."""
import pytest
import torch

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
E = 96 * U
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


def make(rows, N, xt, wt, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen)
    return (r(rows, N) * 2 + 0.5).to(xt), (r(N) * 0.3 + 1).to(wt), r(N).to(wt), r(rows, N).to(xt)


def within(got, ref, err, what):
    half = torch.finfo(got.dtype).eps / 2
    tol = err + half * ref.abs() * (1 + 2.0 ** -7) + 1e-30
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def check(x, w, b, dy, y, grads, eps=1e-5):
    x, dy = x.detach().double(), dy.double()
    wd = w.detach().double() if w is not None else torch.ones_like(x[0])
    bd = b.detach().double() if b is not None else torch.zeros_like(x[0])
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xhat = (x - mean) * rstd
    X = E * rstd * x.abs().mean(-1, keepdim=True) + 2 * E * xhat.abs()
    within(y, orc.layer_norm(x, wd, bd, eps), X * wd.abs() + 2 * U * ((xhat * wd).abs() + bd.abs()), "y")
    if grads is None:
        return
    leaves = [x.requires_grad_(True), wd.requires_grad_(True), bd.requires_grad_(True)]
    ref = torch.autograd.grad(orc.layer_norm(*leaves, eps), leaves, dy)
    x, wd = x.detach(), wd.detach()
    z = (dy * wd).abs()
    m1, m2 = z.mean(-1, keepdim=True), (z * xhat.abs()).mean(-1, keepdim=True)
    err = rstd * (E * m1 + xhat.abs() * (E * m2 + (z * X).mean(-1, keepdim=True)) + X * m2 + 6 * E * (z + m1 + xhat.abs() * m2))
    within(grads[0], ref[0], err, "dx")
    n = (x.shape[0] + 8) * U
    if w is not None:
        within(grads[1], ref[1], (dy.abs() * X).sum(0) + n * (dy * xhat).abs().sum(0), "dw")
    if b is not None:
        within(grads[-1], ref[2], n * dy.abs().sum(0), "db")


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("rows,N", [(1, 1), (3, 2), (5, 31), (1, 64), (7, 100), (33, 256), (2, 1000), (65, 1001), (4, 1024), (300, 2048), (9, 2049), (3, 4096), (5, 5000),
                                    (4, 8192), (2, 10001)])
def test_forward_and_gradients(rows, N, xt, wt):
    from hattention_b200 import layer_norm
    x, w, b, dy = make(rows, N, xt, wt)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(x, w, b)
    assert y.dtype == xt
    grads = torch.autograd.grad(y, leaves, dy)
    assert [t.dtype for t in grads] == [xt, wt, wt]
    check(x, w, b, dy, y.detach(), grads)


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_absent_parameters(xt, has_w, has_b):
    from hattention_b200 import layer_norm
    x, w, b, dy = make(40, 333, xt, torch.float32)
    w, b = w if has_w else None, b if has_b else None
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = layer_norm(x, w, b, eps=1e-3)
    check(x, w, b, dy, y.detach(), torch.autograd.grad(y, leaves, dy), eps=1e-3)


def test_gradients_that_nobody_asks_for():
    from hattention_b200 import layer_norm
    x, w, b, dy = make(40, 256, torch.bfloat16, torch.float32)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(layer_norm(x, w, b), w, dy)
    x2, w2 = x.clone().requires_grad_(True), w.detach()
    dx, = torch.autograd.grad(layer_norm(x2, w2, b), x2, dy)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    all_ = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    assert torch.equal(dx, all_[0]) and torch.equal(dw, all_[1])


def test_many_rows():
    from hattention_b200 import layer_norm
    x, w, b, dy = make(20011, 96, torch.bfloat16, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(x, w, b)
    first = torch.autograd.grad(y, leaves, dy)
    check(x, w, b, dy, y.detach(), first)
    again = torch.autograd.grad(layer_norm(x, w, b), leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_shapes_strides_and_alignment():
    from hattention_b200 import layer_norm
    x, w, b, dy = make(24, 300, torch.bfloat16, torch.bfloat16)
    assert torch.equal(layer_norm(x.view(2, 3, 4, 300), w, b).view(24, 300), layer_norm(x, w, b))
    view = torch.cat([x, x], 1)[:, 300:]
    assert torch.equal(layer_norm(view, w, b), layer_norm(x, w, b))
    off = torch.cat([x.flatten()[:1], x.flatten()])[1:].view(24, 300)
    assert off.data_ptr() % 16 != 0 and torch.equal(layer_norm(off, w, b), layer_norm(x, w, b))
    assert torch.equal(layer_norm(x[0], w, b), layer_norm(x, w, b)[0])
    wide = torch.stack([w, w], 1)[:, 0]
    assert torch.equal(layer_norm(x, wide, b), layer_norm(x, w, b))


def test_constant_rows_and_far_means():
    """The variance comes from the differences to the mean: rows far from zero keep their digits, constant rows give zeros."""
    from hattention_b200 import layer_norm
    assert torch.equal(layer_norm(torch.full((3, 512), 7.0, device="cuda")), torch.zeros(3, 512, device="cuda"))
    x = torch.randn(3, 512, device="cuda") + 1000.0
    check(x, None, None, x, layer_norm(x), None)


def test_empty_operands():
    from hattention_b200 import layer_norm
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = layer_norm(torch.zeros(0, 8, device="cuda"), w)
    assert y.shape == (0, 8) and torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.zeros(8, device="cuda"))


def test_captured_and_library_operators():
    from hattention_b200 import layer_norm, ops  # noqa: F401
    x, w, b, dy = make(100, 640, torch.bfloat16, torch.float32)
    y, stats = torch.ops.llattn.layer_norm_fwd(x, w, b, 1e-5)
    grads = torch.ops.llattn.layer_norm_bwd(x, w, stats, dy)
    check(x, w, b, dy, y, grads)
    torch.library.opcheck(torch.ops.llattn.layer_norm_fwd.default, (x, w, b, 1e-5), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.llattn.layer_norm_bwd.default, (x, w, stats, dy), test_utils=("test_schema", "test_faketensor"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(x, w, b)
    x.mul_(3)
    graph.replay()
    assert torch.equal(y, layer_norm(x, w, b))
