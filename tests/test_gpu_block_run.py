"""A block of them together, as they would be used: norm, projection, causal convolution, selective scan (or gated delta
rule with a gated norm of its heads), projection, residual norm; trained, run over prompts and token by token.

The comparison is the same block in torch operations in 64 bits.  Tolerances: each operator is within 2^-16 of its terms
(their own tests), a block chains six of them with two matrix products of 64 terms between, whose conditions multiply
errors by a few: 2^-11 of the largest value in all for float32.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm
    from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step
    from eacs_b200.ops.gated_delta import gated_delta_rule, gated_delta_step
    from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step

d, D, N, W, EPS = 64, 96, 16, 4, 1e-5


def params(seed):
    g = torch.Generator(DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    p = dict(nw=1 + 0.1 * rnd(d), win=rnd(2 * D, d) * d ** -0.5, cw=rnd(D, W) * 0.5, cb=0.1 * rnd(D), wx=rnd(2 * N + D, D) * D ** -0.5,
             A=-(1 + torch.arange(N, device=DEV)).float().repeat(D, 1) * torch.exp(0.1 * rnd(D, N)), skip=rnd(D), bias=-3 + rnd(D),
             wout=rnd(d, D) * D ** -0.5, scale=0.5 + 0.1 * rnd(d), nw2=1 + 0.1 * rnd(d))
    return p, rnd


def block(p, x, res, lengths=None, states=None):
    """(y, s[, states]): norm of res + scale block(rms norm of x), and the sum itself."""
    h = gated_norm(x, None, p["nw"], EPS)
    xz = h @ p["win"].t()
    kw = {} if states is None else dict(output_final_state=True)
    u = causal_conv(xz[..., :D], p["cw"], p["cb"], lengths=lengths, initial_state=states and states[0], **kw)
    u, cs = u if states is not None else (u, None)
    bcd = u @ p["wx"].t()
    y = selective_ssm(u, bcd[..., 2 * N:], p["A"], bcd[..., :N], bcd[..., N:2 * N], p["skip"], xz[..., D:], p["bias"], lengths=lengths,
                      initial_state=states and states[1], **kw)
    y, hs = y if states is not None else (y, None)
    out = residual_norm(y @ p["wout"].t(), res, p["nw2"], scale=p["scale"], eps=EPS)
    return out if states is None else (*out, (cs, hs))


def plain(p, x, res, lengths):
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    silu = torch.nn.functional.silu
    b, L, _ = x.shape
    live = (torch.arange(L, device=x.device) < lengths[:, None])[..., None].double()
    xz = (rms(x) * p["nw"]) @ p["win"].t()
    row = torch.cat([xz.new_zeros(b, W - 1, D), xz[..., :D] * live], 1)
    u = silu(sum(row[:, k:k + L] * p["cw"][:, k] for k in range(W)) + p["cb"]) * live
    bcd = u @ p["wx"].t()
    s = torch.nn.functional.softplus(bcd[..., 2 * N:] + p["bias"]) * live
    h, ys = xz.new_zeros(b, D, N), []
    for t in range(L):
        h = torch.exp(s[:, t, :, None] * p["A"]) * h + (s[:, t] * u[:, t])[..., None] * bcd[:, t, None, :N]
        ys.append((h * bcd[:, t, None, N:2 * N]).sum(-1))
    y = (torch.stack(ys, 1) + p["skip"] * u) * silu(xz[..., D:]) * live
    sm = res + p["scale"] * (y @ p["wout"].t())
    return rms(sm) * p["nw2"], sm


def test_training_step_of_a_block():
    p, rnd = params(0)
    x, res, dy, ds = (rnd(3, 50, d) for _ in range(4))
    lengths = torch.tensor([50, 0, 33], device=DEV, dtype=torch.int32)
    leaves = {**p, "x": x, "res": res}
    leaves = {n: t.clone().requires_grad_(True) for n, t in leaves.items()}
    got = block(leaves, leaves["x"], leaves["res"], lengths)
    grads = torch.autograd.grad(got, list(leaves.values()), (dy, ds))
    wide = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    want = plain(wide, wide["x"], wide["res"], lengths.long())
    wgrads = torch.autograd.grad(want, list(wide.values()), (dy.double(), ds.double()))
    for n, a, b in [("y", got[0], want[0]), ("s", got[1], want[1])] + [(n, a, b) for n, a, b in zip(leaves, grads, wgrads)]:
        assert float((a.double() - b).abs().max()) <= 2.0 ** -11 * float(b.abs().max()), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """A prompt in two parts and then token by token gives what the whole sequence gives."""
    p, rnd = params(1)
    p = {n: t if n in ("A", "skip", "bias") else t.to(dtype) for n, t in p.items()}
    x, res = rnd(2, 30, d).to(dtype), rnd(2, 30, d).to(dtype)
    with torch.no_grad():
        zero = (torch.zeros(2, W - 1, D, device=DEV, dtype=dtype), torch.zeros(2, D, N, device=DEV))
        y, s, (cs, hs) = block(p, x, res, states=zero)
        parts = [block(p, x[:, :9], res[:, :9], states=zero)]
        parts.append(block(p, x[:, 9:20], res[:, 9:20], states=parts[0][2]))
        conv, state = (t.clone() for t in parts[1][2])
        tail = []
        for t in range(20, 30):
            xz = gated_norm(x[:, t], None, p["nw"], EPS) @ p["win"].t()
            u = causal_conv_step(xz[:, :D], p["cw"], p["cb"], conv)
            bcd = u @ p["wx"].t()
            o = selective_ssm_step(u, bcd[:, 2 * N:], p["A"], bcd[:, :N], bcd[:, N:2 * N], state, p["skip"], xz[:, D:], p["bias"])
            tail.append(residual_norm(o @ p["wout"].t(), res[:, t], p["nw2"], scale=p["scale"], eps=EPS))
    got = torch.cat([parts[0][0], parts[1][0], torch.stack([a for a, _ in tail], 1)], 1)
    sums = torch.cat([parts[0][1], parts[1][1], torch.stack([b for _, b in tail], 1)], 1)
    # matrix products of other shapes round otherwise; bfloat16 rounds each of them (2^-8 of a value, a few in a chain)
    tol = 2.0 ** -11 if dtype == torch.float32 else 2.0 ** -5
    for a, b in ((got, y), (sums, s), (conv, cs), (state, hs)):
        assert float((a.double() - b.double()).abs().max()) <= tol * float(b.double().abs().max())


def test_convolution_delta_rule_and_gated_norm():
    """Queries, keys and values through the convolution, heads normed and gated behind the recurrence."""
    g = torch.Generator(DEV).manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    H, K = 2, 32
    x = rnd(2, 40, 3 * H * K).requires_grad_(True)
    gate, w, cw = rnd(2, 40, H, K).requires_grad_(True), (1 + 0.1 * rnd(K)).requires_grad_(True), (0.5 * rnd(3 * H * K, W)).requires_grad_(True)
    decay, beta, dy = -torch.rand(2, 40, H, generator=g, device=DEV) * 0.2, torch.rand(2, 40, H, generator=g, device=DEV), rnd(2, 40, H, K)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)

    def run(x, gate, w, cw, conv, rule, norm):
        q, k, v = conv(x, cw).unflatten(-1, (3, H, K)).unbind(2)
        return norm(rule(unit(q), unit(k), v), gate, w)
    got = run(x, gate, w, cw, causal_conv, lambda q, k, v: gated_delta_rule(q, k, v, decay, beta), lambda o, g_, w_: gated_norm(o, g_, w_, EPS))
    grads = torch.autograd.grad(got, (x, gate, w, cw), dy)

    def conv64(x, cw):
        row = torch.cat([x.new_zeros(2, W - 1, x.shape[-1]), x], 1)
        return torch.nn.functional.silu(sum(row[:, k:k + 40] * cw[:, k] for k in range(W)))

    def rule64(q, k, v):
        S, outs = q.new_zeros(2, H, K, K), []
        for t in range(40):
            S = S * decay[:, t].double().exp()[..., None, None]
            u = beta[:, t].double()[..., None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t]))
            S = S + torch.einsum("bhk,bhv->bhkv", k[:, t], u)
            outs.append(K ** -0.5 * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
        return torch.stack(outs, 1)
    wide = [t.detach().double().requires_grad_(True) for t in (x, gate, w, cw)]
    want = run(*wide, conv64, rule64,
               lambda o, g_, w_: o * (o.square().mean(-1, keepdim=True) + EPS).rsqrt() * w_ * torch.nn.functional.silu(g_))
    for a, b in zip((got, *grads), (want, *torch.autograd.grad(want, wide, dy.double()))):
        assert float((a.double() - b).abs().max()) <= 2.0 ** -11 * float(b.abs().max())
    with torch.no_grad():  # and one more token
        conv_state, S = torch.zeros(2, W - 1, 3 * H * K, device=DEV), torch.zeros(2, H, K, K, device=DEV)
        for t in range(3):
            q, k, v = causal_conv_step(x[:, t], cw, None, conv_state).unflatten(-1, (3, H, K)).unbind(1)
            o = gated_norm(gated_delta_step(unit(q), unit(k), v, decay[:, t], beta[:, t], S), gate[:, t], w, EPS)
            assert float((o - got[:, t]).abs().max()) <= 2.0 ** -11 * float(got.abs().max())
