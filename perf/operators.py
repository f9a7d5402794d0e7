"""Layer norm and the gated delta rule: the cases that are timed, their inputs, plain forms and values in 64 bits.

Layer norm.  For a row s = x (+ residual) of D values, with mean m and variance w (over the row, biased):
  y = (s - m) / sqrt(w + eps) * weight + bias.

Gated delta rule.  A head keeps a state S (K x V).  With a decay e^g_t (g <= 0), a rate beta_t, a key k_t, a
value v_t and a query q_t, one token does
  S' = e^g_t S,  u_t = beta_t (v_t - S'^T k_t),  S = S' + k_t u_t^T,  o_t = scale S^T q_t.
`fwd` takes a sequence from an initial state and gives the outputs and the state behind it, `train` gives the
outputs and the gradients, and `step` takes one token and updates a state in place.  Several value heads may
share a key head.  Rows may be shorter than L: behind their end the outputs are zero and the state is kept.

A case is a dict: "op" ("norm" or "delta"), "way" (norm: "fwd", "train"; delta: "fwd", "train", "step"), its
sizes and "dtype".
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
CHUNK = 64  # tokens that the plain form of the delta rule takes at once
DEVICE = "cuda"


def _norm(name, way, rows, d, dtype, residual=False, wdtype="f32"):
    return {"name": name, "op": "norm", "way": way, "rows": rows, "d": d, "dtype": dtype, "residual": residual,
            "wdtype": wdtype}


def _delta(name, way, b, l, hk, hv, k, v, dtype, ragged=False, initial=False):
    return {"name": name, "op": "delta", "way": way, "b": b, "l": l, "hk": hk, "hv": hv, "k": k, "v": v,
            "dtype": dtype, "ragged": ragged, "initial": initial}


def listed():
    return [
        # one streaming frame of four videos through a layer's norm: latency alone
        _norm("norm fwd frame", "fwd", 4, 1024, "f32"),
        # the pre-norm of a three-branch layer over four long videos
        _norm("norm fwd long", "fwd", 4 * 16384, 1024, "bf16"),
        # the training step's norm over eight videos of 8192 frames, 768 channels
        _norm("norm train", "train", 8 * 8192, 768, "bf16"),
        # the epilogue norm of x + fused in training, odd rows and an odd width
        _norm("norm train residual odd", "train", 1111, 999, "f16", residual=True, wdtype="f16"),
        # one frame of one video: a state per head, latency alone
        _delta("delta step one", "step", 1, 1, 6, 6, 128, 128, "bf16"),
        # one frame of 64 videos with 2048 channels: the state's traffic
        _delta("delta step batch", "step", 64, 1, 16, 16, 128, 128, "bf16"),
        # four long videos before the streaming starts, 1024 channels in 8 heads
        _delta("delta fwd long", "fwd", 4, 16384, 8, 8, 128, 128, "bf16"),
        # a short ragged batch that carries on from a state; keys shared by two value heads
        _delta("delta fwd ragged", "fwd", 3, 1001, 4, 8, 64, 96, "f16", ragged=True, initial=True),
        # the training step over eight videos of 8192 frames, 768 channels in 6 heads
        _delta("delta train long", "train", 8, 8192, 6, 6, 128, 128, "bf16"),
        # two videos of 4096 frames, half precision, narrow heads
        _delta("delta train f16", "train", 2, 4096, 12, 12, 64, 64, "f16"),
        # a short ragged batch in single precision; keys shared by two value heads, odd widths
        _delta("delta train ragged f32", "train", 2, 333, 2, 4, 48, 40, "f32", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        d = _log_int(rng, 33, 4096)
        c = _norm("", rng.choice(["fwd", "train"]), min(_log_int(rng, 1, 65536), (50 << 20) // d), d,
                  rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.4, rng.choice(["f32", "same"]))
        c["wdtype"] = c["dtype"] if c["wdtype"] == "same" else c["wdtype"]
    else:
        way = rng.choice(["fwd", "train", "train", "step"])
        k, v = rng.choice([32, 48, 64, 72, 96, 128, 128]), rng.choice([24, 32, 64, 80, 96, 128, 128, 192])
        hk = _log_int(rng, 1, 12)
        hv = hk * rng.choice([1, 1, 2])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if way == "step":
            b, l = _log_int(rng, 1, 48), 1
        else:
            l = min(_log_int(rng, 1, 12000), 30_000_000 // (hv * v))
            b = max(1, min(_log_int(rng, 1, 8), 30_000_000 // (l * hv * v)))
        c = _delta("", way, b, l, hk, hv, k, v, dtype, rng.random() < 0.4 and l > 1, rng.random() < 0.5 and way == "fwd")
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

    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        s = {"case": case, "x": (normal(rows, d) * 1.5 + 0.3).to(dt), "residual": None,
             "weight": (1 + 0.2 * normal(d)).to(DTYPES[case["wdtype"]]), "bias": (0.2 * normal(d)).to(DTYPES[case["wdtype"]])}
        if case["residual"]:
            s["residual"] = normal(rows, d).to(dt)
        if case["way"] == "train":
            s["dy"] = normal(rows, d).to(dt)
        leaves = ["x", "weight", "bias"] + (["residual"] if case["residual"] else [])
    else:
        B, L, Hk, Hv, K, V = (case[n] for n in ("b", "l", "hk", "hv", "k", "v"))
        # neighbouring frames look alike: a share of every key is its head's, the rest is its own; unit length
        k = normal(B, L, Hk, K) + 0.7 * normal(B, 1, Hk, K)
        q = normal(B, L, Hk, K) + 0.3 * k
        s = {"case": case, "q": (q / q.norm(dim=-1, keepdim=True)).to(dt), "k": (k / k.norm(dim=-1, keepdim=True)).to(dt),
             "v": normal(B, L, Hv, V).to(dt), "beta": torch.sigmoid(normal(B, L, Hv)).to(dt), "scale": K ** -0.5,
             "lengths": None, "initial": None}
        # decays: a memory of 8 to 2048 frames for a head, made shorter or longer by each frame
        memory = torch.exp(math.log(8.0) + uniform(1, 1, Hv) * math.log(256.0))
        s["g"] = (-torch.nn.functional.softplus(normal(B, L, Hv)) / memory).to(dt)
        if case["ragged"]:
            s["lengths"] = (uniform(B) * L * 0.7 + 0.3 * L).round().int()
            s["lengths"][0] = L
            if B > 2:
                s["lengths"][1] = 0  # a video without a frame
        if case["initial"] or case["way"] == "step":
            s["initial"] = 0.3 * normal(B, Hv, K, V)
        if case["way"] == "step":
            for n in ("q", "k", "v", "g", "beta"):
                s[n] = s[n][:, 0].contiguous()
        if case["way"] == "train":
            s["dy"] = normal(B, L, Hv, V).to(dt)
        leaves = ["q", "k", "v", "g", "beta"]
    if case["way"] == "train":
        for n in leaves:
            s[n].requires_grad_(True)
    s["leaves"] = leaves
    return s


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _plain_norm(x, residual, weight, bias):
    s = x.float() if residual is None else x.float() + residual.float()
    c = s - s.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    return (c * rstd * weight.float() + bias.float()).to(x.dtype)


def _unit_lower_inverse(A):
    """(I + A)^-1 for strictly lower triangular A (..., C, C), C a power of two: by halves,
    [[P, 0], [R, Q]]^-1 = [[P^-1, 0], [-Q^-1 R P^-1, Q^-1]]."""
    C = A.shape[-1]
    T = A.new_ones(*A.shape[:-1], 1, 1)  # the blocks on the diagonal, each inverted
    size = 1
    while size < C:
        n = C // (2 * size)
        blocks = A.reshape(*A.shape[:-2], n, 2 * size, n, 2 * size).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        P, Q = T[..., 0::2, :, :], T[..., 1::2, :, :]
        R = -Q @ blocks[..., size:, :size] @ P
        T = torch.cat([torch.cat([P, torch.zeros_like(P)], -1), torch.cat([R, Q], -1)], -2)
        size *= 2
    return T[..., 0, :, :]


def _plain_delta(q, k, v, g, beta, scale, lengths, initial):
    """CHUNK tokens at once.  With G the running sum of g inside a chunk and S the state before it,
    u_i = beta_i (v_i - e^G_i S^T k_i) - sum_{j<i} A_ij u_j,  A_ij = beta_i e^(G_i - G_j) k_i.k_j."""
    dt = q.dtype
    B, L, Hk, K = q.shape
    Hv, V = v.shape[2:]
    q, k, v, g, beta = (t.float() for t in (q, k, v, g, beta))
    if lengths is not None:
        keep = (torch.arange(L, device=q.device) < lengths[:, None]).float()
        q, v, g, beta = q * keep[..., None, None], v * keep[..., None, None], g * keep[..., None], beta * keep[..., None]
    n = -(-L // CHUNK)

    def chunks(t):  # (B, L, H, ...) -> (B, H, n, CHUNK, ...), zeros behind the end
        t = torch.nn.functional.pad(t.transpose(1, 2), [0, 0] * (t.dim() - 3) + [0, n * CHUNK - L])
        return t.reshape(*t.shape[:2], n, CHUNK, *t.shape[3:])

    q, k = (chunks(t.repeat_interleave(Hv // Hk, 2)) for t in (q, k))
    v, g, beta = chunks(v), chunks(g), chunks(beta)
    G = g.cumsum(-1)
    ratio = torch.exp(torch.tril(G[..., :, None] - G[..., None, :])).tril()  # e^(G_i - G_j) for j <= i
    T = _unit_lower_inverse((beta[..., None] * ratio * (k @ k.transpose(-1, -2))).tril(-1))
    M = ratio * (q @ k.transpose(-1, -2))
    eG, last = torch.exp(G)[..., None], G[..., -1:]
    S = torch.zeros(B, Hv, K, V, device=q.device) if initial is None else initial.float()
    kr = k * torch.exp(last - G)[..., None]
    outs = []
    for c in range(n):
        u = T[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - eG[:, :, c] * (k[:, :, c] @ S)))
        outs.append((eG[:, :, c] * q[:, :, c]) @ S + M[:, :, c] @ u)
        S = torch.exp(last[:, :, c])[..., None] * S + kr[:, :, c].transpose(-1, -2) @ u
    o = torch.stack(outs, 2).reshape(B, Hv, n * CHUNK, V)[:, :, :L].transpose(1, 2) * scale
    return o.to(dt), S


def _plain_step(q, k, v, g, beta, scale, S):
    q, k, v, g, beta = (t.float() for t in (q, k, v, g, beta))
    r = v.shape[1] // k.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    S.mul_(torch.exp(g)[..., None, None])
    u = beta[..., None] * (v - (k[..., None] * S).sum(-2))
    S.add_(k[..., None] * u[..., None, :])
    return (q[..., None] * S).sum(-2) * scale


def _operators():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "longvideo-main_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from eacs_b200.ops import gated_delta, layer_norm
    return gated_delta, layer_norm


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        x, residual, weight, bias = (state[n] for n in ("x", "residual", "weight", "bias"))
        if own:
            y = _operators()[1].layer_norm(x, weight, bias, EPS, residual=residual)
        else:
            y = _plain_norm(x, residual, weight, bias)
    else:
        q, k, v, g, beta = (state[n] for n in ("q", "k", "v", "g", "beta"))
        if case["way"] == "step":
            if own:
                y = _operators()[0].gated_delta_step(q, k, v, g, beta, state["initial"], scale=state["scale"])
            else:
                y = _plain_step(q, k, v, g, beta, state["scale"], state["initial"]).to(q.dtype)
            return {"y": y, "state": state["initial"]}
        if own:
            y = _operators()[0].gated_delta_rule(q, k, v, g, beta, scale=state["scale"], initial_state=state["initial"],
                                                 output_final_state=case["way"] == "fwd", lengths=state["lengths"])
        else:
            y = _plain_delta(q, k, v, g, beta, state["scale"], state["lengths"], state["initial"])
            y = y if case["way"] == "fwd" else y[0]
        if case["way"] == "fwd":
            return {"y": y[0], "state": y[1]}
    if case["way"] == "fwd":
        return {"y": y}
    grads = torch.autograd.grad(y, [state[n] for n in state["leaves"]], state["dy"])
    return {"y": y.detach(), **{"d" + n: t for n, t in zip(state["leaves"], grads)}}


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, d, we = case["rows"] * case["d"], case["d"], SIZE[case["wdtype"]]
        sums = 2 if case["residual"] else 1
        if case["way"] == "fwd":
            return {"bytes": n * e * (sums + 1) + 2 * d * we, "flops": 8 * n}
        # x (and residual) and dy in, y and dx (and the residual's) out; weight and bias in, their gradients out
        return {"bytes": n * e * (2 * sums + 2) + 4 * d * we, "flops": 22 * n}
    B, L, Hk, Hv, K, V = (case[n] for n in ("b", "l", "hk", "hv", "k", "v"))
    qk, vo, gb = B * L * Hk * K * 2 * e, B * L * Hv * V * e, B * L * Hv * 2 * e
    step, S = 2 * B * L * Hv * K * V, B * Hv * K * V * 4
    if case["way"] == "train":  # q, k, v, g, beta, dy in; o and the five gradients out
        return {"bytes": 2 * qk + 4 * vo + 2 * gb, "flops": 10 * step}
    return {"bytes": qk + 2 * vo + gb + S * (2 if case["way"] == "step" or case["initial"] else 1), "flops": 3 * step}


# ---------------------------------------------------------------------------------------------------------
# the definitions in 64 bits: token by token, gradients by the chain rule of one token
# ---------------------------------------------------------------------------------------------------------
def _exact_norm(s, way):
    x, weight, bias = (s[n].detach().double() for n in ("x", "weight", "bias"))
    if s["residual"] is not None:
        x = x + s["residual"].detach().double()
    D = x.shape[1]
    m = x.sum(1, keepdim=True) / D
    rstd = 1 / ((((x - m) ** 2).sum(1, keepdim=True) / D) + EPS).sqrt()
    h = (x - m) * rstd
    out = {"y": h * weight + bias}
    if way == "train":
        dy = s["dy"].double()
        p = dy * weight
        out["dx"] = rstd * (p - p.sum(1, keepdim=True) / D - h * (p * h).sum(1, keepdim=True) / D)
        out["dweight"], out["dbias"] = (dy * h).sum(0), dy.sum(0)
        if s["residual"] is not None:
            out["dresidual"] = out["dx"]
    return out


def _exact_delta(s, way):
    q, k, v, g, beta = (s[n].detach().double() for n in ("q", "k", "v", "g", "beta"))
    if way == "step":
        q, k, v, g, beta = (t[:, None] for t in (q, k, v, g, beta))
    B, L, Hk, K = q.shape
    Hv, V = v.shape[2:]
    r = Hv // Hk
    live = torch.ones(B, L, device=q.device, dtype=torch.bool)
    if s["lengths"] is not None:
        live = torch.arange(L, device=q.device) < s["lengths"][:, None]
    q, k = (t[:, :, torch.arange(Hv, device=q.device) // r] for t in (q, k))
    a = torch.where(live[..., None], g.exp(), torch.ones_like(g))[..., None, None]
    beta = torch.where(live[..., None], beta, torch.zeros_like(beta))[..., None]
    q = torch.where(live[..., None, None], q, torch.zeros_like(q))

    def token(S, t):
        Sd = S * a[:, t]
        e = v[:, t] - torch.einsum("bhkv,bhk->bhv", Sd, k[:, t])
        return Sd, e, Sd + torch.einsum("bhk,bhv->bhkv", k[:, t], beta[:, t] * e)

    S = torch.zeros(B, Hv, K, V, device=q.device, dtype=torch.float64)
    if s["initial"] is not None:
        S = S + s["initial"].double()
    y = torch.empty(B, L, Hv, V, device=q.device, dtype=torch.float64)
    span = max(1, math.isqrt(L))
    kept = {}
    for t in range(L):
        if way == "train" and t % span == 0:
            kept[t] = S
        S = token(S, t)[2]
        y[:, t] = s["scale"] * torch.einsum("bhkv,bhk->bhv", S, q[:, t])
    if way == "step":
        return {"y": y[:, 0], "state": S}
    if way == "fwd":
        return {"y": y, "state": S}
    dy = s["dy"].double() * s["scale"]
    dy = torch.where(live[..., None, None], dy, torch.zeros_like(dy))
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, g, g))
    dS = torch.zeros_like(S)
    for t0 in sorted(kept, reverse=True):
        S, seen = kept[t0], []
        for t in range(t0, min(L, t0 + span)):
            Sd, e, S = token(S, t)
            seen.append((Sd, e, S))
        for t in range(min(L, t0 + span) - 1, t0 - 1, -1):
            Sd, e, S = seen[t - t0]
            dq[:, t] = torch.einsum("bhkv,bhv->bhk", S, dy[:, t])
            dS = dS + torch.einsum("bhk,bhv->bhkv", q[:, t], dy[:, t])
            du = torch.einsum("bhkv,bhk->bhv", dS, k[:, t])
            db[:, t] = (du * e).sum(-1)
            de = beta[:, t] * du
            dv[:, t] = de
            dk[:, t] = torch.einsum("bhkv,bhv->bhk", dS, beta[:, t] * e) - torch.einsum("bhkv,bhv->bhk", Sd, de)
            dS = dS - torch.einsum("bhk,bhv->bhkv", k[:, t], de)
            dg[:, t] = (dS * Sd).sum((-2, -1))
            dS = dS * a[:, t]
    m = live[..., None].double()
    return {"y": y, "dq": (dq * m[..., None]).unflatten(2, (Hk, r)).sum(3),
            "dk": (dk * m[..., None]).unflatten(2, (Hk, r)).sum(3), "dv": dv * m[..., None], "dg": dg * m, "dbeta": db * m}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s, case["way"]) if case["op"] == "norm" else _exact_delta(s, case["way"])
