"""Short causal convolution, selective state space scan and the norms around a block: the cases that are timed,
their inputs, plain forms and values in 64 bits.

Causal convolution.  Channel d of token t sees itself and the W - 1 tokens before it (zeros, or a given state):
  p_t = bias + sum_{w<W} weight_w x_{t-W+1+w},   y_t = silu(p_t).
The state is the last W - 1 inputs, oldest first.

Selective scan.  A channel keeps N states.  With s = softplus(dt + dt_bias) per token and channel, and B and C per
token and state,
  h_t = e^(s_t A) h_{t-1} + s_t x_t B_t,   y_t = (sum_n C_t h_t + skip x_t) silu(z_t).

Norms.  With rms(v) = v / sqrt(mean(v^2) + eps) over a row:
  gated:     y = rms(x) weight silu(gate)
  residual:  u = x, or rms(x) post_weight;  u = u silu(gate) where there is a gate;  s = residual + scale u
             y = rms(s) weight;  y and s are given.

`fwd` takes sequences (or rows) and gives the outputs and the states behind them, `train` the outputs and the
gradients, `step` one token a row, with its state updated in place.  Rows may be shorter than L: behind their end
the outputs are zero and the state is kept.

A case is a dict: "op" ("conv", "ssm" or "norm"), "way" ("fwd", "train" or "step"), its sizes and "dtype".
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
CHUNK = 128  # tokens between the states that the plain form of the scan carries one after another
DEVICE = "cuda"


def _conv(name, way, b, l, d, w, dtype, ragged=False, initial=False, sliced=False):
    return {"name": name, "op": "conv", "way": way, "b": b, "l": l, "d": d, "w": w, "dtype": dtype, "ragged": ragged,
            "initial": initial, "sliced": sliced}


def _ssm(name, way, b, l, d, n, dtype, gate=True, ragged=False, initial=False):
    return {"name": name, "op": "ssm", "way": way, "b": b, "l": l, "d": d, "n": n, "dtype": dtype, "gate": gate,
            "ragged": ragged, "initial": initial}


def _norm(name, way, kind, rows, d, dtype, gate=False, post=False, scale=False, wdtype="f32"):
    return {"name": name, "op": "norm", "way": way, "kind": kind, "rows": rows, "d": d, "dtype": dtype, "gate": gate,
            "post": post, "scale": scale, "wdtype": wdtype}


def listed():
    return [
        # one streaming frame of four videos: latency alone
        _conv("conv step frame", "step", 4, 1, 1024, 4, "bf16"),
        # four long videos before the streaming starts; x is one half of a projection's output
        _conv("conv fwd long", "fwd", 4, 16384, 1024, 4, "bf16", sliced=True),
        # the training step over eight videos of 8192 frames, 768 channels
        _conv("conv train long", "train", 8, 8192, 768, 4, "bf16"),
        # a short ragged batch with an odd width and three taps, half precision
        _conv("conv train ragged odd", "train", 3, 1001, 333, 3, "f16", ragged=True),
        # one frame of 64 videos with 2048 channels: the state's traffic
        _ssm("ssm step batch", "step", 64, 1, 2048, 16, "bf16"),
        # four long videos before the streaming starts, 1024 channels
        _ssm("ssm fwd long", "fwd", 4, 16384, 1024, 16, "bf16"),
        # a short ragged batch that carries on from a state, wide states, no gate
        _ssm("ssm fwd ragged", "fwd", 3, 1111, 768, 32, "f16", gate=False, ragged=True, initial=True),
        # the training step over eight videos of 8192 frames, 768 channels
        _ssm("ssm train long", "train", 8, 8192, 768, 16, "bf16"),
        # a short ragged batch in single precision, odd widths
        _ssm("ssm train ragged f32", "train", 2, 333, 250, 12, "f32", ragged=True),
        # the heads of a recurrence behind four videos of 4096 frames: 8 heads of 128, each normed by itself
        _norm("gated norm heads", "fwd", "gated", 4 * 4096 * 8, 128, "bf16", gate=True),
        # between two blocks of the training step over eight videos of 8192 frames
        _norm("residual norm train", "train", "residual", 8 * 8192, 768, "bf16", scale=True),
        # norms before and after a block, its gate and its scale: odd rows and an odd width
        _norm("residual norm all odd", "train", "residual", 1111, 999, "f16", gate=True, post=True, scale=True, wdtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "ssm", "ssm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        d = _log_int(rng, 24, 4096)
        rows = min(_log_int(rng, 1, 131072), (48 << 20) // d)
        kind = rng.choice(["gated", "residual", "residual"])
        c = _norm("", rng.choice(["fwd", "train"]), kind, rows, d, dtype, kind == "gated" or rng.random() < 0.4,
                  kind == "residual" and rng.random() < 0.4, kind == "residual" and rng.random() < 0.6,
                  rng.choice(["f32", dtype]))
    else:
        way = rng.choice(["fwd", "train", "train", "step"])
        d = _log_int(rng, 16, 4096)
        if way == "step":
            b, l = _log_int(rng, 1, 96), 1
        else:
            l = min(_log_int(rng, 1, 16384), (48 << 20) // d)
            b = max(1, min(_log_int(rng, 1, 8), (48 << 20) // (l * d)))
        ragged, initial = rng.random() < 0.4 and l > 1, rng.random() < 0.5 and way == "fwd"
        if op == "conv":
            c = _conv("", way, b, l, d, rng.choice([2, 3, 4, 4]), dtype, ragged, initial, rng.random() < 0.3 and way != "step")
        else:
            n = rng.choice([4, 8, 12, 16, 16, 16, 32, 64])
            while b * l * d * n > 800_000_000:
                b, l = max(1, b // 2), l if b > 1 else max(1, l // 2)
            c = _ssm("", way, b, l, d, n, dtype, rng.random() < 0.7, ragged and l > 1, initial)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    op, way = case["op"], case["way"]
    if op == "norm":
        rows, d, wdt = case["rows"], case["d"], DTYPES[case["wdtype"]]
        s = {"x": (normal(rows, d) * 1.5).to(dt), "weight": (1 + 0.2 * normal(d)).to(wdt),
             "gate": normal(rows, d).to(dt) if case["gate"] else None, "residual": None, "scale": None, "post_weight": None}
        if case["kind"] == "residual":
            s["residual"] = normal(rows, d).to(dt)
            if case["post"]:
                s["post_weight"] = (1 + 0.2 * normal(d)).to(wdt)
            if case["scale"]:
                s["scale"] = (0.3 + 0.1 * normal(d)).to(wdt)  # a block's share, one a channel
        leaves = [n for n in ("x", "gate", "residual", "weight", "scale", "post_weight") if s[n] is not None]
        if way == "train":
            s["dy"] = normal(rows, d).to(dt)
            s["ds"] = normal(rows, d).to(dt) if case["kind"] == "residual" else None
    else:
        B, L, D = (case[n] for n in ("b", "l", "d"))
        s = {"lengths": None, "initial": None}
        if case["ragged"]:
            s["lengths"] = (uniform(B) * L * 0.7 + 0.3 * L).round().int()
            s["lengths"][0] = L
            if B > 2:
                s["lengths"][1] = 0  # a video without a frame
        if op == "conv":
            W = case["w"]
            x = normal(B, L, D * (2 if case["sliced"] else 1)).to(dt)
            s["x"] = x[..., :D]
            s["weight"], s["bias"] = (normal(D, W) * W ** -0.5).to(dt), (0.1 * normal(D)).to(dt)
            if case["initial"] or way == "step":
                s["initial"] = normal(B, W - 1, D).to(dt)
            leaves = ["x", "weight", "bias"]
        else:
            N = case["n"]
            s["x"], s["B"], s["C"] = normal(B, L, D).to(dt), normal(B, L, N).to(dt), normal(B, L, N).to(dt)
            # steps of 0.001 to 0.1 at rest, made shorter or longer by each token; rates of 1 to N
            rest = torch.exp(math.log(1e-3) + uniform(D) * math.log(100.0))
            s["dt"], s["dt_bias"] = normal(B, L, D).to(dt), rest + torch.log(-torch.expm1(-rest))
            s["A"] = -(1 + torch.arange(N, device=DEVICE)).float() * torch.exp(0.1 * normal(D, N))
            s["skip"] = 1 + 0.1 * normal(D)
            s["z"] = normal(B, L, D).to(dt) if case["gate"] else None
            if case["initial"] or way == "step":
                s["initial"] = 0.3 * normal(B, D, N)
            leaves = ["x", "dt", "A", "B", "C", "skip", "dt_bias"] + (["z"] if case["gate"] else [])
        if way == "step":
            for n in ("x", "B", "C", "dt", "z"):
                if s.get(n) is not None:
                    s[n] = s[n][:, 0].contiguous()
        if way == "train":
            s["dy"] = normal(B, L, D).to(dt)
    if way == "train":
        for n in leaves:
            s[n] = s[n].detach().requires_grad_(True)
    s["leaves"], s["case"] = leaves, case
    return s


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _silu(v):
    return v * torch.sigmoid(v)


def _live(lengths, L):
    """(B, L, 1): the tokens before their row's end, as ones."""
    return (torch.arange(L, device=lengths.device) < lengths[:, None]).float()[..., None]


def _plain_conv(x, weight, bias, lengths, initial):
    B, L, D = x.shape
    W = weight.shape[1]
    before = torch.zeros(B, W - 1, D, device=x.device) if initial is None else initial.float()
    row = torch.cat([before, x.float()], 1)
    p = bias.float()
    for w in range(W):
        p = p + row[:, w:w + L] * weight[:, w].float()
    y = _silu(p)
    if lengths is None:
        return y.to(x.dtype), row[:, L:].to(x.dtype)
    at = lengths.long()[:, None] + torch.arange(W - 1, device=x.device)
    return (y * _live(lengths, L)).to(x.dtype), row.gather(1, at[..., None].expand(B, W - 1, D)).to(x.dtype)


def _plain_conv_step(x, weight, bias, state):
    row = torch.cat([state, x[:, None]], 1)
    y = _silu((row.float() * weight.float().t()).sum(1) + bias.float())
    state.copy_(row[:, 1:])
    return y.to(x.dtype)


def _states(a, b, h0):
    """All states of h_t = a_t h_{t-1} + b_t for a, b (B, L, D, N): chunks side by side from zero, then the states
    in front of the chunks, one after another."""
    B, L, D, N = a.shape
    n = -(-L // CHUNK)
    pad = n * CHUNK - L
    a, b = (torch.cat([t, t.new_zeros(B, pad, D, N)], 1) if pad else t for t in (a, b))
    a, b = (t.reshape(B, n, CHUNK, D, N) for t in (a, b))
    decay, local = torch.empty_like(a), torch.empty_like(b)
    decay[:, :, 0], local[:, :, 0] = a[:, :, 0], b[:, :, 0]
    for t in range(1, CHUNK):
        torch.mul(decay[:, :, t - 1], a[:, :, t], out=decay[:, :, t])
        torch.addcmul(b[:, :, t], local[:, :, t - 1], a[:, :, t], out=local[:, :, t])
    H = [h0]
    for c in range(n - 1):
        H.append(decay[:, c, -1] * H[-1] + local[:, c, -1])
    local.addcmul_(decay, torch.stack(H, 1)[:, :, None])
    return local.reshape(B, n * CHUNK, D, N)[:, :L]


def _ssm_terms(x, dt, dt_bias, lengths):
    raw = dt.float() + dt_bias
    s = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    x = x.float()
    if lengths is not None:
        live = _live(lengths, x.shape[1])
        s, x = s * live, x * live
    return raw, s, x


def _plain_ssm(x, dt, A, B, C, skip, z, dt_bias, lengths, initial, states=False):
    dtype, L = x.dtype, x.shape[1]
    _, s, x = _ssm_terms(x, dt, dt_bias, lengths)
    h0 = torch.zeros(x.shape[0], *A.shape, device=x.device) if initial is None else initial
    h = _states(torch.exp(s[..., None] * A), (s * x)[..., None] * B.float()[:, :, None], h0)
    o = (h * C.float()[:, :, None]).sum(-1) + skip * x
    y = o if z is None else o * _silu(z.float())
    if lengths is not None:
        y = y * _live(lengths, L)
    return (y.to(dtype), h, o) if states else (y.to(dtype), h[:, -1].contiguous())


def _plain_ssm_train(s):
    """Outputs and gradients.  With g_t the gradient of h_t, g_t = C_t do_t + e^(s_{t+1} A) g_{t+1}: the same scan
    backwards."""
    x, dt, A, Bs, Cs, skip, z, dt_bias = (None if s[n] is None else s[n].detach() for n in
                                          ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias"))
    dtype, lengths = x.dtype, s["lengths"]
    y, h, o = _plain_ssm(x, dt, A, Bs, Cs, skip, z, dt_bias, lengths, None, states=True)
    raw, step, xf = _ssm_terms(x, dt, dt_bias, lengths)
    Bf, Cf, do = Bs.float()[:, :, None], Cs.float()[:, :, None], s["dy"].float()
    if lengths is not None:
        do = do * _live(lengths, x.shape[1])
    out = {"y": y}
    if z is not None:
        sig = torch.sigmoid(z.float())
        out["dz"] = (do * o * sig * (1 + z.float() * (1 - sig))).to(dtype)
        do = do * z.float() * sig
    a = torch.exp(step[..., None] * A)
    ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    g = _states(ahead, (do[..., None] * Cf).flip(1), torch.zeros_like(a[:, 0])).flip(1)
    del ahead
    out["dC"] = (h * do[..., None]).sum(2).to(dtype)
    out["dB"] = (g * (step * xf)[..., None]).sum(2).to(dtype)
    du = (g * Bf).sum(-1)  # the gradient of s x
    w = a.mul_(g)
    w[:, 0] = 0  # nothing in front of the first token
    w[:, 1:] *= h[:, :-1]
    out["dA"] = (w * step[..., None]).sum((0, 1))
    dstep = (w * A).sum(-1) + du * xf
    draw = dstep * torch.sigmoid(raw)
    if lengths is not None:
        draw = draw * _live(lengths, x.shape[1])
    out["dx"], out["ddt"] = (du * step + do * skip).to(dtype), draw.to(dtype)
    out["dskip"], out["ddt_bias"] = (do * xf).sum((0, 1)), draw.sum((0, 1))
    return {n: out[n] for n in ["y"] + ["d" + n for n in s["leaves"]]}


def _plain_ssm_step(x, dt, A, B, C, skip, z, dt_bias, state):
    _, s, xf = _ssm_terms(x, dt, dt_bias, None)
    state.mul_(torch.exp(s[..., None] * A)).add_((s * xf)[..., None] * B.float()[:, None])
    y = (state * C.float()[:, None]).sum(-1) + skip * xf
    return (y if z is None else y * _silu(z.float())).to(x.dtype)


def _rms(v):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)


def _plain_norm(x, gate, residual, weight, scale, post_weight):
    u = x.float()
    if residual is None:
        return (_rms(u) * weight.float() * _silu(gate.float())).to(x.dtype)
    if post_weight is not None:
        u = _rms(u) * post_weight.float()
    if gate is not None:
        u = u * _silu(gate.float())
    s = residual.float() + (u if scale is None else u * scale.float())
    return (_rms(s) * weight.float()).to(x.dtype), s.to(x.dtype)


def _operators():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "longvideo-main_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from eacs_b200.ops import block_norm, causal_conv, selective_ssm
    return causal_conv, selective_ssm, block_norm


def _run_conv(s, way):
    args = s["x"], s["weight"], s["bias"]
    if way == "step":
        if own:
            y = _operators()[0].causal_conv_step(*args, s["initial"])
        else:
            y = _plain_conv_step(*args, s["initial"])
        return y, s["initial"]
    if not own:
        return _plain_conv(*args, s["lengths"], s["initial"])
    f = _operators()[0].causal_conv
    if way == "train":
        return f(*args, lengths=s["lengths"]), None
    return f(*args, initial_state=s["initial"], output_final_state=True, lengths=s["lengths"])


def _run_ssm(s, way):
    args = [s[n] for n in ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias")]
    if way == "step":
        if own:
            y = _operators()[1].selective_ssm_step(*args[:5], s["initial"], *args[5:])
        else:
            y = _plain_ssm_step(*args, s["initial"])
        return y, s["initial"]
    if not own:
        return _plain_ssm(*args, s["lengths"], s["initial"])
    f = _operators()[1].selective_ssm
    if way == "train":
        return f(*args, lengths=s["lengths"]), None
    return f(*args, initial_state=s["initial"], output_final_state=True, lengths=s["lengths"])


def _run_norm(s):
    if not own:
        return _plain_norm(*(s[n] for n in ("x", "gate", "residual", "weight", "scale", "post_weight")))
    ops = _operators()[2]
    if s["residual"] is None:
        return ops.gated_norm(s["x"], s["gate"], s["weight"], EPS)
    return ops.residual_norm(s["x"], s["residual"], s["weight"], scale=s["scale"], gate=s["gate"],
                             post_weight=s["post_weight"], eps=EPS)


def run(state):
    case = state["case"]
    op, way = case["op"], case["way"]
    if op == "ssm" and way == "train" and not own:
        return _plain_ssm_train(state)
    if op == "norm":
        y = _run_norm(state)
        outs = {"y": y} if state["residual"] is None else {"y": y[0], "s": y[1]}
    else:
        y, last = (_run_conv if op == "conv" else _run_ssm)(state, way)
        outs = {"y": y} if way == "train" else {"y": y, "state": last}
    if way != "train":
        return outs
    up = [state["dy"]] + ([state["ds"]] if "s" in outs else [])
    grads = torch.autograd.grad(list(outs.values()), [state[n] for n in state["leaves"]], up)
    return {**{n: t.detach() for n, t in outs.items()}, **{"d" + n: t for n, t in zip(state["leaves"], grads)}}


def work(case):
    e, train = SIZE[case["dtype"]], case["way"] == "train"
    if case["op"] == "norm":
        n, d, we = case["rows"] * case["d"], case["d"], SIZE[case["wdtype"]]
        ins = 1 + case["gate"] + (case["kind"] == "residual")
        outs = 2 if case["kind"] == "residual" else 1
        params = 1 + case["post"] + case["scale"]
        flops = 6 + 5 * case["gate"] + 5 * case["post"] + 2 * case["scale"]
        if not train:
            return {"bytes": n * e * (ins + outs) + params * d * we, "flops": flops * n}
        # inputs and upstream gradients in, outputs and gradients out
        return {"bytes": n * e * (2 * ins + 2 * outs) + 2 * params * d * we, "flops": 3 * flops * n}
    B, L, D = (case[n] for n in ("b", "l", "d"))
    n = B * L * D
    if case["op"] == "conv":
        W = case["w"]
        state = B * (W - 1) * D * e
        params = D * (W + 1) * e
        if train:  # x and dy in, y and dx out; weight and bias in, their gradients out
            return {"bytes": 4 * n * e + 2 * params, "flops": n * (6 * W + 16)}
        states = 2 if case["way"] == "step" or case["initial"] else 1
        return {"bytes": 2 * n * e + params + states * state, "flops": n * (2 * W + 5)}
    N = case["n"]
    rows, bc, params = 3 + case["gate"], 2 * B * L * N * e, (D * N + 2 * D) * 4
    if train:  # x, dt, z, dy, B and C in; y and the gradients out
        return {"bytes": (2 * rows) * n * e + 2 * bc + 2 * params, "flops": 23 * n * N}
    states = 2 if case["way"] == "step" or case["initial"] else 1
    return {"bytes": rows * n * e + bc + params + states * B * D * N * 4, "flops": 7 * n * N}


# ---------------------------------------------------------------------------------------------------------
# the definitions in 64 bits: sums written out, token by token, gradients by the chain rule
# ---------------------------------------------------------------------------------------------------------
def _sig(v):
    return 1 / (1 + (-v).exp())


def _dsilu(v):
    g = _sig(v)
    return g + v * g * (1 - g)


def _end(s, L):
    """Each row's number of tokens, as 64-bit whole numbers."""
    B = s["x"].shape[0]
    return torch.full((B,), L, device=s["x"].device) if s["lengths"] is None else s["lengths"].long()


def _exact_conv(s, way):
    x, weight, bias = (s[n].detach().double() for n in ("x", "weight", "bias"))
    if way == "step":
        x = x[:, None]
    B, L, D = x.shape
    W = weight.shape[1]
    pos = torch.arange(L, device=x.device)
    end = _end(s, L)
    live = (pos < end[:, None])[..., None]
    x = torch.where(live, x, torch.zeros_like(x))
    front = torch.zeros(B, W - 1, D, device=x.device, dtype=torch.float64)
    if s["initial"] is not None:
        front = s["initial"].double()

    def seen(back):  # the input `back` tokens before each token
        out = torch.zeros_like(x)
        out[:, back:] = x[:, :L - back] if back < L else x[:, :0]
        m = min(back, L)
        out[:, :m] = front[:, W - 1 - back:W - 1 - back + m]
        return out

    p = bias + sum(weight[:, W - 1 - back] * seen(back) for back in range(W))
    y = torch.where(live, p * _sig(p), torch.zeros_like(p))
    last = torch.empty_like(front)
    for j in range(W - 1):  # input number end - (W - 1) + j of each row
        at = end - (W - 1) + j
        inside = x[torch.arange(B, device=x.device), at.clamp(0, L - 1)]
        outside = front[torch.arange(B, device=x.device), (at + W - 1).clamp(0, max(W - 2, 0))]
        last[:, j] = torch.where((at >= 0)[:, None], inside, outside)
    if way == "step":
        return {"y": y[:, 0], "state": last}
    if way == "fwd":
        return {"y": y, "state": last}
    dp = torch.where(live, s["dy"].double() * _dsilu(p), torch.zeros_like(p))
    dx = torch.zeros_like(x)
    dweight = torch.empty_like(weight)
    for back in range(W):
        if back < L:
            dx[:, :L - back] += weight[:, W - 1 - back] * dp[:, back:]
        dweight[:, W - 1 - back] = (dp * seen(back)).sum((0, 1))
    return {"y": y, "dx": torch.where(live, dx, torch.zeros_like(dx)), "dweight": dweight, "dbias": dp.sum((0, 1))}


def _exact_ssm(s, way):
    x, dt, A, Bs, Cs, skip, dt_bias = (s[n].detach().double() for n in ("x", "dt", "A", "B", "C", "skip", "dt_bias"))
    z = None if s["z"] is None else s["z"].detach().double()
    if way == "step":
        x, dt, Bs, Cs = (t[:, None] for t in (x, dt, Bs, Cs))
        z = None if z is None else z[:, None]
    B, L, D = x.shape
    live = (torch.arange(L, device=x.device) < _end(s, L)[:, None])[..., None]
    nil = torch.zeros_like(x)
    raw = dt + dt_bias
    # log(1 + e^raw) without overflow, and without losing a small e^raw next to 1
    step = torch.where(live, torch.where(raw > 0, raw + (-raw).exp().log1p(), raw.clamp(max=0).exp().log1p()), nil)
    x = torch.where(live, x, nil)
    h = torch.zeros(B, D, A.shape[1], device=x.device, dtype=torch.float64)
    if s["initial"] is not None:
        h = h + s["initial"].double()

    def token(h, t):
        old = torch.exp(step[:, t, :, None] * A) * h
        return old, old + torch.einsum("bd,bn->bdn", step[:, t] * x[:, t], Bs[:, t])

    span = max(1, math.isqrt(L))
    kept, o = {}, torch.empty_like(x)
    for t in range(L):
        if way == "train" and t % span == 0:
            kept[t] = h
        h = token(h, t)[1]
        o[:, t] = torch.einsum("bdn,bn->bd", h, Cs[:, t])
    o = o + skip * x
    gain = torch.ones_like(x) if z is None else z * _sig(z)
    y = torch.where(live, o * gain, nil)
    if way != "train":
        return {"y": y[:, 0] if way == "step" else y, "state": h}
    dy = torch.where(live, s["dy"].double(), nil)
    out = {"y": y}
    if z is not None:
        out["dz"] = dy * o * _dsilu(z)
    do = dy * gain
    du, dstep = torch.empty_like(x), torch.empty_like(x)
    dA, dB, dC, g = torch.zeros_like(A), torch.empty_like(Bs), torch.empty_like(Cs), torch.zeros_like(h)
    for t0 in sorted(kept, reverse=True):
        h, seen = kept[t0], []
        for t in range(t0, min(L, t0 + span)):
            old, h = token(h, t)
            seen.append((old, h))
        for t in range(min(L, t0 + span) - 1, t0 - 1, -1):
            old, h = seen[t - t0]
            g = g + torch.einsum("bd,bn->bdn", do[:, t], Cs[:, t])
            dC[:, t] = torch.einsum("bdn,bd->bn", h, do[:, t])
            dB[:, t] = torch.einsum("bdn,bd->bn", g, step[:, t] * x[:, t])
            du[:, t] = torch.einsum("bdn,bn->bd", g, Bs[:, t])
            go = g * old
            dstep[:, t] = (go * A).sum(-1)
            dA += (go * step[:, t, :, None]).sum(0)
            g = g * torch.exp(step[:, t, :, None] * A)
    ddt = torch.where(live, (dstep + du * x) * _sig(raw), nil)
    out.update(dx=du * step + do * skip, ddt=ddt, dA=dA, dB=dB, dC=dC, dskip=(do * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))
    return out


def _exact_norm(s, way):
    x, gate, res, weight, scale, post = (None if s[n] is None else s[n].detach().double()
                                         for n in ("x", "gate", "residual", "weight", "scale", "post_weight"))
    D = x.shape[1]

    def norm(v):
        r = 1 / ((v ** 2).sum(1, keepdim=True) / D + EPS).sqrt()
        return v * r, r

    def back(dh, h, r):  # the gradient of v from that of h = v r
        return r * (dh - h * (dh * h).sum(1, keepdim=True) / D)

    out = {}
    first = weight if res is None else post
    h1, r1 = norm(x)
    u1 = x if first is None else h1 * first
    gain = 1 if gate is None else gate * _sig(gate)
    u2 = u1 * gain
    if res is None:
        out["y"] = u2
    else:
        sv = res + (u2 if scale is None else u2 * scale)
        h2, r2 = norm(sv)
        out["y"], out["s"] = h2 * weight, sv
    if way != "train":
        return out
    dy = s["dy"].double()
    if res is None:
        du2 = dy
    else:
        dsv = s["ds"].double() + back(dy * weight, h2, r2)
        out["dresidual"], out["dweight"] = dsv, (dy * h2).sum(0)
        du2 = dsv if scale is None else dsv * scale
        if scale is not None:
            out["dscale"] = (dsv * u2).sum(0)
    du1 = du2 * gain
    if gate is not None:
        out["dgate"] = du2 * u1 * _dsilu(gate)
    if first is None:
        out["dx"] = du1
    else:
        out["dx"] = back(du1 * first, h1, r1)
        out["dweight" if res is None else "dpost_weight"] = (du1 * h1).sum(0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        out = {"conv": _exact_conv, "ssm": _exact_ssm, "norm": _exact_norm}[case["op"]](s, case["way"])
    if case["way"] != "train":
        return out
    return {n: out[n] for n in ["y", "s"] + ["d" + n for n in s["leaves"]] if n in out}
