"""The hybrid-stack operators together, as a model runs them: norm -> gated recurrence -> residual, norm -> windowed attention -> residual; a training step,
and a prompt with generation behind it against the same stack over the whole sequence."""
import pytest
import torch

from oracle import hybrid_oracle as orc

pytestmark = pytest.mark.gpu
H, G, K, WINDOW, SINKS = 4, 2, 64, 50, 3
WIDTH = H * K


def parameters(seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale=1.0, shift=0.0: torch.randn(s, device="cuda", generator=gen) * scale + shift
    return {"n1": r(WIDTH, scale=0.1, shift=1), "b1": r(WIDTH, scale=0.1), "n2": r(WIDTH, scale=0.1, shift=1), "gate": r(WIDTH, WIDTH, scale=WIDTH ** -0.5),
            "qkv": r(WIDTH, (H + 2 * G) * K, scale=WIDTH ** -0.5), "out": r(WIDTH, WIDTH, scale=WIDTH ** -0.5)}


class Kernels:
    def __init__(self):
        import hattention_b200 as p
        self.norm, self.attention = p.layer_norm, p.sliding_window_attention
        self.scan = lambda x, g: p.gated_recurrence(x, g)[0]


class Plain:
    norm = staticmethod(orc.layer_norm)
    attention = staticmethod(orc.sliding_window_attention)
    scan = staticmethod(lambda x, g: orc.gated_recurrence(x, g)[0])


def forward(x, p, ops):
    B, T, _ = x.shape
    t = lambda w: w.to(x.dtype)
    y = ops.norm(x, p["n1"], p["b1"])
    x = x + ops.scan(y, torch.nn.functional.logsigmoid(y @ t(p["gate"]) + 3))
    qkv = (ops.norm(x, p["n2"]) @ t(p["qkv"])).view(B, T, H + 2 * G, K)
    return x + ops.attention(qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:], WINDOW, SINKS).reshape(B, T, WIDTH) @ t(p["out"])


def test_training_step():
    """Outputs and gradients of all parameters against 64 bits.  A value passes about a dozen roundings to bf16 (half a step 2^-8 each, of independent signs) on its way
    through the stack and back: 4 * 2^-8 of the norm of a result, with a factor of two for the amplification by the norms."""
    p = {n: w.requires_grad_(True) for n, w in parameters().items()}
    x = torch.randn(2, 333, WIDTH, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    dy = torch.randn(2, 333, WIDTH, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.bfloat16)
    y = forward(x, p, Kernels())
    grads = torch.autograd.grad(y, list(p.values()), dy)
    pd = {n: w.detach().double().requires_grad_(True) for n, w in p.items()}
    ref = forward(x.double(), pd, Plain)
    rgrads = torch.autograd.grad(ref, list(pd.values()), dy.double())
    for name, a, b in zip(["y"] + list(p), (y,) + grads, (ref,) + rgrads):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= 8 * 2.0 ** -8, f"{name}: {rel:.4f}"


def test_prompt_and_generation():
    """A prompt, then token by token, gives what the stack gives over the whole sequence: every operator's serving form continues its state.  Differences are
    those of rounding an intermediate to bf16 at another neighbour, 2^-7 of the outputs' scale and a few of them along the way."""
    import hattention_b200 as hb
    p = parameters()
    T, n = 100, 30
    x = torch.randn(3, T + n, WIDTH, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    t = lambda w: w.to(x.dtype)
    with torch.no_grad():
        whole = forward(x, p, Kernels())
        y = hb.layer_norm(x[:, :T], p["n1"], p["b1"])
        o, h = hb.gated_recurrence(y, torch.nn.functional.logsigmoid(y @ t(p["gate"]) + 3), output_final_state=True)
        z = x[:, :T] + o
        qkv = (hb.layer_norm(z, p["n2"]) @ t(p["qkv"])).view(3, T, H + 2 * G, K)
        o, state = hb.sliding_window_prefill(qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:], WINDOW, SINKS)
        outs = [z + o.reshape(3, T, WIDTH) @ t(p["out"])]
        for i in range(T, T + n):
            y = hb.layer_norm(x[:, i], p["n1"], p["b1"])
            o, h = hb.gated_recurrence_step(h, y, torch.nn.functional.logsigmoid(y @ t(p["gate"]) + 3))
            z = x[:, i] + o
            qkv = (hb.layer_norm(z, p["n2"]) @ t(p["qkv"])).view(3, H + 2 * G, K)
            o, state = hb.sliding_window_step(state, qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:])
            outs.append((z + o.reshape(3, WIDTH) @ t(p["out"]))[:, None])
    got = torch.cat(outs, 1).double()
    assert ((got - whole.double()).norm() / whole.double().norm()).item() <= 4 * 2.0 ** -8
    assert (got - whole.double()).abs().max().item() <= 8 * 2.0 ** -7 * whole.double().abs().max().item()
