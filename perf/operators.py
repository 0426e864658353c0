"""Performance cases of the operators of hybrid stacks: the gated linear recurrence, attention over a sliding window with
sinks, and layer norm.  Each case is a dict of plain values; `prepare` makes what a program has in hand before the
call, `run` is one pass through an operator: its plain form in elementary torch operations, or, with `own`, the
package's calls.

    gated_recurrence          h_t = exp(g_t) h_{t-1} + x_t, a channel at a time
    sliding_window_attention  softmax over s <= t with t - s < window or s < sinks; H query heads share G heads of k and v
    layer_norm                (x - mean) / sqrt(var + eps) * weight + bias

Sizes: 32 heads of 64 = 2048 channels, 24 heads of 64 = 1536, sequences of 16384 and 8192 tokens and head widths of 64 and
128 as in the configurations of the benchmark and the test-suite; windows, odd lengths and odd widths are generic."""
import math
import os
import sys

import torch

own = False

BLOCK = 128        # query rows that the plain form of the windowed attention takes together


def listed():
    return [
        # one layer's training step at the headline length: log decays in fp32, as everywhere in the package
        {"name": "recurrence train T16384", "kind": "recurrence_train", "B": 2, "T": 16384, "D": 2048, "x": "bfloat16", "g": "float32", "state": False},
        # fp32 training of an odd batch of odd sequences, continued from a state that gets its gradient
        {"name": "recurrence train odd", "kind": "recurrence_train", "B": 3, "T": 1999, "D": 1001, "x": "float32", "g": "float32", "state": True},
        # a prompt of one sequence before generation: outputs and the state to go on from
        {"name": "recurrence prompt T1000", "kind": "recurrence_prompt", "B": 1, "T": 1000, "D": 2048, "x": "bfloat16", "g": "bfloat16"},
        # generation, a token of every sequence: the smallest calls, where launches and host work count
        {"name": "recurrence step B64", "kind": "recurrence_step", "B": 64, "D": 2048, "x": "bfloat16", "g": "bfloat16"},
        # one layer's training step over a long sequence, query heads in groups of four
        {"name": "window train T16384", "kind": "window_train", "B": 1, "T": 16384, "H": 32, "G": 8, "K": 128, "window": 2048, "sinks": 4},
        # narrow heads that share nothing, an odd length that ends inside a tile
        {"name": "window train odd K64", "kind": "window_train", "B": 2, "T": 1999, "H": 16, "G": 16, "K": 64, "window": 512, "sinks": 0},
        # prompts of different lengths, padded to the longest, and the caches to go on from
        {"name": "window prompt T1000", "kind": "window_prompt", "B": 4, "T": 1000, "H": 16, "G": 4, "K": 128, "window": 512, "sinks": 4},
        # generation of one sequence
        {"name": "window step B1", "kind": "window_step", "B": 1, "H": 32, "G": 8, "K": 128, "window": 4096, "sinks": 4, "position": 6000},
        # generation for a batch: the caches go through memory once a token, some are not full yet
        {"name": "window step B64", "kind": "window_step", "B": 64, "H": 32, "G": 8, "K": 128, "window": 2048, "sinks": 4, "position": 3000},
        # the norm before a layer of the headline training step, fp32 master parameters
        {"name": "norm train N2048", "kind": "norm_train", "rows": 32768, "N": 2048, "x": "bfloat16", "w": "float32", "bias": True},
        # fp32 rows of an odd width, no bias
        {"name": "norm train odd", "kind": "norm_train", "rows": 5997, "N": 1001, "x": "float32", "w": "float32", "bias": False},
        # the norm of a generation step
        {"name": "norm step B64", "kind": "norm_forward", "rows": 64, "N": 2048, "x": "bfloat16", "w": "bfloat16", "bias": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _types(rng):
    x = rng.choice(["bfloat16", "bfloat16", "float32"])
    return x, rng.choice([x, "float32"])


def draw(rng):
    kind = rng.choice(["recurrence_train", "recurrence_prompt", "recurrence_step", "window_train", "window_train", "window_prompt", "window_step",
                       "norm_train", "norm_forward"])
    c = {"kind": kind}
    if kind.startswith("recurrence"):
        c["x"], c["g"] = _types(rng)
        c["D"] = rng.choice([_log_int(rng, 60, 4096), 64 * _log_int(rng, 1, 64)])
        if kind == "recurrence_step":
            c["B"] = _log_int(rng, 1, 256)
            return c
        c["B"] = rng.choice([1, 1, 2, 3, 8])
        most = 2 * 16384 * 2048 // (2 if c["x"] == "float32" else 1)
        c["T"] = min(_log_int(rng, 1, 32768), max(1, most // (c["B"] * c["D"])))
        if kind == "recurrence_train":
            c["state"] = rng.random() < 0.3
        return c
    if kind.startswith("norm"):
        c["x"], c["w"] = _types(rng)
        c["N"] = rng.choice([_log_int(rng, 16, 8192), 64 * _log_int(rng, 1, 128)])
        c["rows"] = min(_log_int(rng, 1, 65536), max(1, 32768 * 2048 // (c["N"] * (2 if c["x"] == "float32" else 1))))
        c["bias"] = rng.random() < 0.7
        return c
    c["K"] = rng.choice([64, 128])
    c["G"] = rng.choice([1, 2, 4, 8, 16])
    c["H"] = c["G"] * rng.choice([1, 1, 2, 4, 5, 8])
    c["sinks"] = rng.choice([0, 1, 4, 16, 100])
    c["window"] = rng.choice([_log_int(rng, 1, 4096), 64 * _log_int(rng, 1, 64)])
    if kind == "window_step":
        c["B"] = _log_int(rng, 1, 64)
        c["window"] = min(c["window"], 64 * 2048 * 8 // (c["B"] * c["G"]))
        c["position"] = _log_int(rng, 1, 8000)
        return c
    c["B"] = rng.choice([1, 1, 2, 4])
    T = _log_int(rng, 2, 16384) if kind == "window_train" else _log_int(rng, 1, 8000)
    if kind == "window_train":
        c["window"] = max(c["window"], 2)       # tokens that see themselves alone have no gradients of q and k
    # pairs of the listed training step bound those of a drawn one
    while c["B"] * c["H"] * T * (min(c["window"], T) + c["sinks"] + BLOCK) > 32 * 16384 * 2048:
        T = T * 2 // 3
    c["T"] = T
    return c


# ------------------------------------------------------------------------------------------ inputs
class _Draws:
    """Tensors from one seed, made on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)

    def randn(self, *shape, dtype=torch.bfloat16, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=self.gen, device=self.dev) * scale + shift).to(dtype)

    def decay(self, *shape, dtype):
        """Log decays as a gate's logsigmoid gives them."""
        return torch.nn.functional.logsigmoid(self.randn(*shape, dtype=torch.float32, shift=3.0)).to(dtype)

    def lengths(self, B, lo, hi):
        n = torch.randint(lo, hi + 1, (B,), generator=self.gen, device=self.dev, dtype=torch.int64)
        n[0] = hi
        return n


def prepare(case, seed):
    r, c = _Draws(seed), case
    s = {"case": dict(case)}
    if c["kind"].startswith("recurrence"):
        xt, gt = getattr(torch, c["x"]), getattr(torch, c["g"])
        shape = (c["B"], c["D"]) if c["kind"] == "recurrence_step" else (c["B"], c["T"], c["D"])
        s["x"], s["g"] = r.randn(*shape, dtype=xt), r.decay(*shape, dtype=gt)
        if c["kind"] == "recurrence_step" or c.get("state"):
            s["h"] = r.randn(c["B"], c["D"], dtype=torch.float32, scale=3.0)
        if c["kind"] == "recurrence_train":
            s["do"] = r.randn(*shape, dtype=xt)
    elif c["kind"].startswith("norm"):
        xt, wt = getattr(torch, c["x"]), getattr(torch, c["w"])
        s["x"] = r.randn(c["rows"], c["N"], dtype=xt, scale=2.0, shift=0.5)
        s["w"] = r.randn(c["N"], dtype=wt, scale=0.2, shift=1.0)
        s["b"] = r.randn(c["N"], dtype=wt, scale=0.2) if c["bias"] else None
        if c["kind"] == "norm_train":
            s["do"] = r.randn(c["rows"], c["N"], dtype=xt)
    elif c["kind"] == "window_step":
        B, G, K, slots = c["B"], c["G"], c["K"], c["sinks"] + c["window"]
        s["q"], s["k"], s["v"] = r.randn(B, c["H"], K), r.randn(B, G, K), r.randn(B, G, K)
        n = r.lengths(B, c["position"] // 4, c["position"])
        held = (torch.arange(slots, device=r.dev) < n[:, None])[:, :, None, None]
        s["k_cache"], s["v_cache"] = r.randn(B, slots, G, K) * held, r.randn(B, slots, G, K) * held
        s["lengths"] = n[:, None].repeat(1, G)
    else:
        B, T, K = c["B"], c["T"], c["K"]
        s["q"], s["k"], s["v"] = r.randn(B, T, c["H"], K), r.randn(B, T, c["G"], K), r.randn(B, T, c["G"], K)
        if c["kind"] == "window_train":
            s["do"] = r.randn(B, T, c["H"], K)
        else:
            s["lengths"] = r.lengths(B, T // 4, T)
    if c["kind"].endswith("_train"):
        for name in ("x", "g", "h", "w", "b", "q", "k", "v"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    with torch.no_grad():
        return _PLAIN[kind](state)


def _package():
    at = os.path.join(os.getcwd(), "log-linear-attention_b200")     # the package's folder in the repository that is the working folder
    if at not in sys.path:
        sys.path.insert(0, at)
    import hattention_b200
    return hattention_b200


def _own_recurrence_train(s):
    leaves = [s["x"], s["g"]] + ([s["h"]] if "h" in s else [])
    o, _ = _package().gated_recurrence(s["x"], s["g"], initial_state=s.get("h"))
    d = torch.autograd.grad(o, leaves, s["do"])
    return dict(zip(("o", "dx", "dg", "dh"), (o.detach(),) + d))


def _own_recurrence_prompt(s):
    o, h = _package().gated_recurrence(s["x"], s["g"], output_final_state=True)
    return {"o": o, "h": h}


def _own_recurrence_step(s):
    o, h = _package().gated_recurrence_step(s["h"], s["x"], s["g"])
    return {"o": o, "h": h}


def _own_window_train(s):
    c = s["case"]
    o = _package().sliding_window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"])
    dq, dk, dv = torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_window_prompt(s):
    c = s["case"]
    o, w = _package().sliding_window_prefill(s["q"], s["k"], s["v"], c["window"], c["sinks"], lengths=s["lengths"])
    return {"o": o, "k": w.k, "v": w.v, "lengths": w.lengths}


def _own_window_step(s):
    c, p = s["case"], _package()
    w = p.WindowState(s["k_cache"], s["v_cache"], s["lengths"], c["window"], c["sinks"])
    o, w = p.sliding_window_step(w, s["q"], s["k"], s["v"])
    return {"o": o, "k": w.k, "v": w.v, "lengths": w.lengths}


def _own_norm_train(s):
    leaves = [s["x"], s["w"]] + ([s["b"]] if s["b"] is not None else [])
    y = _package().layer_norm(s["x"], s["w"], s["b"])
    d = torch.autograd.grad(y, leaves, s["do"])
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(),) + d))


def _own_norm_forward(s):
    return {"y": _package().layer_norm(s["x"], s["w"], s["b"])}


_OWN = {"recurrence_train": _own_recurrence_train, "recurrence_prompt": _own_recurrence_prompt, "recurrence_step": _own_recurrence_step,
        "window_train": _own_window_train, "window_prompt": _own_window_prompt, "window_step": _own_window_step,
        "norm_train": _own_norm_train, "norm_forward": _own_norm_forward}


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dimension 1, by doubling the span that an element has taken in."""
    T, d = x.shape[1], 1
    while d < T:
        x = torch.cat([x[:, :d], x[:, d:] + a[:, d:] * x[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return x


def _plain_recurrence(s):
    a, x = s["g"].float().exp(), s["x"].float()
    if s.get("h") is not None:
        x = torch.cat([x[:, :1] + a[:, :1] * s["h"][:, None], x[:, 1:]], 1)
    return a, _scan(a, x)


def _plain_recurrence_train(s):
    a, h = _plain_recurrence(s)
    h0 = s["h"] if s.get("h") is not None else torch.zeros_like(h[:, 0])
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)        # what h_t is multiplied by on its way to h_{t+1}
    dh = _scan(after.flip(1), s["do"].float().flip(1)).flip(1)
    out = {"o": h.to(s["x"].dtype), "dx": dh.to(s["x"].dtype), "dg": (dh * a * before).to(s["g"].dtype)}
    if s.get("h") is not None:
        out["dh"] = a[:, 0] * dh[:, 0]
    return out


def _plain_recurrence_prompt(s):
    _, h = _plain_recurrence(s)
    return {"o": h.to(s["x"].dtype), "h": h[:, -1].clone()}


def _plain_recurrence_step(s):
    s["h"].mul_(s["g"].float().exp()).add_(s["x"].float())
    return {"o": s["h"].to(s["x"].dtype), "h": s["h"]}


def _band(T, window, sinks, dev):
    """For blocks of query rows: the tokens whose keys a block looks at (blocks, columns), and which of them each row sees (blocks, rows, columns)."""
    reach, blocks = min(window, T), -(-T // BLOCK)
    first = torch.arange(blocks, device=dev)[:, None] * BLOCK
    t = (first + torch.arange(BLOCK, device=dev))[:, :, None]
    band = first - (reach - 1) + torch.arange(reach - 1 + BLOCK, device=dev)
    sink = torch.arange(min(sinks, T), device=dev).expand(blocks, -1)
    near = (band[:, None] >= 0) & (band[:, None] <= t) & (t - band[:, None] < window)
    far = t - sink[:, None] >= window
    seen = torch.cat([far, near], 2) & (t < T)
    return torch.cat([sink, band], 1).clamp(0, T - 1), seen


def _plain_window(s):
    c, q = s["case"], s["q"]
    B, T, H, K = q.shape
    G = s["k"].shape[2]
    cols, seen = _band(T, c["window"], c["sinks"], q.device)
    n = cols.shape[0]

    def blocks(x):
        x = torch.cat([x.float(), x.new_zeros(B, n * BLOCK - T, H, K, dtype=torch.float32)], 1)
        return x.view(B, n, BLOCK, G, H // G, K).permute(0, 1, 3, 4, 2, 5)

    def gathered(x):
        return x.float()[:, cols].permute(0, 1, 3, 4, 2)[:, :, :, None]         # (B, n, G, 1, K, columns)

    scale = K ** -0.5
    S = torch.matmul(blocks(q) * scale, gathered(s["k"]))
    S.masked_fill_(~seen[:, None, None], -math.inf)
    P = torch.exp(S - S.amax(-1, keepdim=True).clamp(min=-1e30))
    P /= P.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(P, gathered(s["v"]).transpose(-1, -2))

    def rows(x):
        return x.permute(0, 1, 4, 2, 3, 5).reshape(B, n * BLOCK, H, K)[:, :T]

    return cols, blocks, gathered, rows, scale, P, o


def _plain_window_train(s):
    cols, blocks, gathered, rows, scale, P, o = _plain_window(s)
    k, do = s["k"], blocks(s["do"])
    dS = P * (torch.matmul(do, gathered(s["v"])) - (do * o).sum(-1, keepdim=True))
    dq = torch.matmul(dS, gathered(k).transpose(-1, -2)) * scale

    def scattered(x, y):
        """Products summed over the rows of a block and the heads that share k and v, then over the blocks that look at a token."""
        z = torch.matmul(x.transpose(-1, -2), y).sum(3).permute(0, 1, 3, 2, 4).flatten(1, 2)
        return torch.zeros(k.shape, device=k.device).index_add_(1, cols.flatten(), z).to(k.dtype)

    return {"o": rows(o).to(s["q"].dtype), "dq": rows(dq).to(s["q"].dtype), "dk": scattered(dS, blocks(s["q"]) * scale), "dv": scattered(P, do)}


def _plain_window_prompt(s):
    c, k, v, n = s["case"], s["k"], s["v"], s["lengths"][:, None]
    _, _, _, rows, _, _, o = _plain_window(s)
    W, sinks = c["window"], c["sinks"]
    slot = torch.arange(sinks + W, device=k.device)[None]
    # the last of the sequence's tokens that goes to the slot: token `slot` among the sinks, then every W-th from there on
    token = torch.where(slot < sinks, slot, slot + torch.div(n - 1 - slot, W, rounding_mode="floor") * W)
    held = (slot < n)[:, :, None, None]
    at = token.clamp(0, k.shape[1] - 1)[:, :, None, None].expand(-1, -1, k.shape[2], k.shape[3])
    return {"o": rows(o).to(s["q"].dtype), "k": torch.gather(k, 1, at) * held, "v": torch.gather(v, 1, at) * held,
            "lengths": n.repeat(1, k.shape[2])}


def _plain_window_step(s):
    c, q, kc, vc, n = s["case"], s["q"], s["k_cache"], s["v_cache"], s["lengths"]
    B, H, K = q.shape
    G, slots = kc.shape[2], kc.shape[1]
    at = n[:, 0]
    slot = torch.where(at < c["sinks"], at, c["sinks"] + (at - c["sinks"]) % c["window"])
    which = torch.arange(B, device=q.device)
    kc[which, slot] = s["k"]
    vc[which, slot] = s["v"]
    n += 1
    held = torch.arange(slots, device=q.device) < n[:, :1]
    S = torch.matmul(q.float().view(B, G, H // G, K) * K ** -0.5, kc.float().permute(0, 2, 3, 1))
    S = S.masked_fill(~held[:, None, None], -math.inf)
    P = torch.exp(S - S.amax(-1, keepdim=True))
    o = torch.matmul(P / P.sum(-1, keepdim=True), vc.float().transpose(1, 2))
    return {"o": o.reshape(B, H, K).to(q.dtype), "k": kc, "v": vc, "lengths": n}


def _plain_norm(s):
    x = s["x"].float()
    m = x.mean(-1, keepdim=True)
    r = ((x - m).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xhat, w = (x - m) * r, s["w"].float()
    return xhat, r, w, (xhat * w + s["b"].float() if s["b"] is not None else xhat * w).to(s["x"].dtype)


def _plain_norm_train(s):
    xhat, r, w, y = _plain_norm(s)
    dy = s["do"].float()
    t = dy * w
    dx = r * (t - t.mean(-1, keepdim=True) - xhat * (t * xhat).mean(-1, keepdim=True))
    out = {"y": y, "dx": dx.to(y.dtype), "dw": (dy * xhat).sum(0).to(s["w"].dtype)}
    if s["b"] is not None:
        out["db"] = dy.sum(0).to(s["b"].dtype)
    return out


def _plain_norm_forward(s):
    return {"y": _plain_norm(s)[3]}


_PLAIN = {"recurrence_train": _plain_recurrence_train, "recurrence_prompt": _plain_recurrence_prompt, "recurrence_step": _plain_recurrence_step,
          "window_train": _plain_window_train, "window_prompt": _plain_window_prompt, "window_step": _plain_window_step,
          "norm_train": _plain_norm_train, "norm_forward": _plain_norm_forward}


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(T, window, sinks):
    """(t, s) with s <= t and t - s < window or s < sinks."""
    w = min(window, T)
    n = w * (w + 1) // 2 + (T - w) * w
    far = T - w                     # rows t >= window: of those, row window + i sees min(sinks, i + 1) tokens behind its window
    m = min(sinks, far)
    return n + m * (m + 1) // 2 + (far - m) * m


def work(case):
    c, kind = case, case["kind"]
    size = {"bfloat16": 2, "float32": 4}
    if kind.startswith("recurrence"):
        n, x, g = c["B"] * c.get("T", 1) * c["D"], size[c["x"]], size[c["g"]]
        state = 4 * c["B"] * c["D"]
        if kind == "recurrence_step":
            return {"bytes": n * (2 * x + g) + 2 * state, "flops": 3 * n}
        if kind == "recurrence_prompt":
            return {"bytes": n * (2 * x + g) + state, "flops": 3 * n}
        return {"bytes": n * (4 * x + 2 * g) + (2 * state if c["state"] else 0), "flops": 10 * n}
    if kind.startswith("norm"):
        n, x, p = c["rows"] * c["N"], size[c["x"]], size[c["w"]] * c["N"] * (2 if c["bias"] else 1)
        if kind == "norm_forward":
            return {"bytes": 2 * n * x + p, "flops": 8 * n}
        return {"bytes": 4 * n * x + 2 * p, "flops": 22 * n}
    B, H, G, K = c["B"], c["H"], c["G"], c["K"]
    if kind == "window_step":
        # the mean of the lengths, which are spread between a quarter of the position and all of it
        held = min(c["position"] * 5 // 8 + 1, c["sinks"] + c["window"])
        return {"bytes": 4 * B * G * K * (held + 1) + 4 * B * H * K + 16 * B * G, "flops": 4 * B * H * K * held}
    T = c["T"]
    pairs = B * H * _pairs(T, c["window"], c["sinks"])
    if kind == "window_prompt":
        slots = c["sinks"] + c["window"]
        return {"bytes": 4 * B * T * (H + G) * K + 4 * B * min(slots, T) * G * K, "flops": 4 * K * pairs}
    return {"bytes": 8 * B * T * (H + G) * K, "flops": 14 * K * pairs}


# ------------------------------------------------------------------------------------------ the operators in 64 bits, from their definitions
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    kind = case["kind"]
    if kind.startswith("recurrence"):
        return _exact_recurrence(s, kind)
    if kind.startswith("norm"):
        return _exact_norm(s, kind)
    return _exact_window_step(s) if kind == "window_step" else _exact_window(s, kind)


def _exact_recurrence(s, kind):
    """A loop over the tokens in spans: inside a span h_t = sum_s exp(g_{s+1} + .. + g_t) x_s, before it the state at its start."""
    x, g = s["x"].double(), s["g"].double()
    if kind == "recurrence_step":
        h = g.exp() * s["h"].double() + x
        return {"o": h, "h": h}
    B, T, D = x.shape
    span = 32
    h0 = s["h"].double() if "h" in s else x.new_zeros(B, D)
    before = torch.empty_like(x)

    def walk(decay, inputs, state, starts):
        out = torch.empty_like(inputs)
        for t0 in range(0, T, span):
            G = decay[:, t0:t0 + span].cumsum(1)
            n = G.shape[1]
            later = torch.ones(n, n, dtype=torch.bool, device=G.device).tril()[None, :, :, None]
            E = torch.where(later, (G[:, :, None] - G[:, None]).clamp(max=0), -math.inf).exp()
            if starts is not None:
                starts[:, t0] = state
            out[:, t0:t0 + n] = torch.einsum("btsd,bsd->btd", E, inputs[:, t0:t0 + n]) + G.exp() * state[:, None]
            state = out[:, t0 + n - 1]
        return out

    o = walk(g, x, h0, None)
    if kind == "recurrence_prompt":
        return {"o": o, "h": o[:, -1].clone()}
    before[:, 0], before[:, 1:] = h0, o[:, :-1]
    # the reverse walk: the decay from t + 1 to t
    turned = torch.cat([g.new_zeros(B, 1, D), g.flip(1)[:, :-1]], 1)
    dh = walk(turned, s["do"].double().flip(1), x.new_zeros(B, D), None).flip(1)
    out = {"o": o, "dx": dh, "dg": dh * before * g.exp()}
    if "h" in s:
        out["dh"] = dh[:, 0] * g[:, 0].exp()
    return out


def _exact_norm(s, kind):
    x, w = s["x"].double(), s["w"].double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = (var + 1e-5).sqrt()
    z = (x - mean) / sd
    y = z * w + (s["b"].double() if s["b"] is not None else 0.0)
    if kind == "norm_forward":
        return {"y": y}
    dy = s["do"].double()
    dz = dy * w
    N = x.shape[1]
    dx = (N * dz - dz.sum(-1, keepdim=True) - z * (dz * z).sum(-1, keepdim=True)) / (N * sd)
    out = {"y": y, "dx": dx, "dw": torch.einsum("rn,rn->n", dy, z)}
    if s["b"] is not None:
        out["db"] = torch.einsum("rn->n", dy)
    return out


def _exact_window_step(s):
    c = s["case"]
    B, H, K = s["q"].shape
    R = H // c["G"]
    o = torch.zeros(B, H, K, dtype=torch.float64, device=s["q"].device)
    for b in range(B):
        n = int(s["lengths"][b, 0])
        slot = n if n < c["sinks"] else c["sinks"] + (n - c["sinks"]) % c["window"]
        k, v = s["k_cache"][b].double(), s["v_cache"][b].double()
        k[slot], v[slot] = s["k"][b].double(), s["v"][b].double()
        k, v = k[:n + 1].repeat_interleave(R, 1), v[:n + 1].repeat_interleave(R, 1)
        p = torch.softmax(torch.einsum("hk,shk->hs", s["q"][b].double(), k) / math.sqrt(K), -1)
        o[b] = torch.einsum("hs,shk->hk", p, v)
    return {"o": o, "k": None, "v": None, "lengths": None}


def _exact_window(s, kind):
    """A head at a time, over spans of query rows and the keys that any of them sees."""
    c = s["case"]
    B, T, H, K = s["q"].shape
    R, W, sinks, scale = H // c["G"], c["window"], c["sinks"], 1.0 / math.sqrt(K)
    span = max(256, min(1024, W))
    dev = s["q"].device
    train = kind == "window_train"
    o = torch.empty(B, T, H, K, dtype=torch.float64, device=dev)
    dq = torch.empty_like(o) if train else None
    dk = torch.zeros(B, T, c["G"], K, dtype=torch.float64, device=dev) if train else None
    dv = torch.zeros_like(dk) if train else None
    for t0 in range(0, T, span):
        t1 = min(T, t0 + span)
        lo = max(0, t0 - W + 1)
        cols = torch.cat([torch.arange(min(sinks, lo), device=dev), torch.arange(lo, t1, device=dev)])
        t = torch.arange(t0, t1, device=dev)[:, None]
        hidden = (cols > t) | ((t - cols >= W) & (cols >= sinks))
        for h in range(H):
            g = h // R
            q, k, v = s["q"][:, t0:t1, h].double(), s["k"][:, cols, g].double(), s["v"][:, cols, g].double()
            p = torch.softmax((q @ k.mT * scale).masked_fill(hidden, -math.inf), -1)
            o[:, t0:t1, h] = p @ v
            if train:
                do = s["do"][:, t0:t1, h].double()
                dp = do @ v.mT
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[:, t0:t1, h] = ds @ k
                dk[:, cols, g] += ds.mT @ q
                dv[:, cols, g] += p.mT @ do
    if train:
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    return {"o": o, "k": None, "v": None, "lengths": None}
