"""Saved-tensor hooks: what they give back holds the same values, but may be a copy with other strides, off its old alignment,
or back from the host.  Dense copies on their boundaries give the same bits as without hooks.  Off a boundary other kernels may
run, whose sums take the same terms in another order: each of at most n = 256 terms is off by n 2^-24 of the sum of their
sizes, twice; that sum is at most sqrt(n) = 16 times the largest of a tensor's sums of random terms: 2^-11 of it, and
half a step of the type for each of two roundings.
"""
import pytest
import torch

from inputs import cell_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm
    from eacs_b200.ops.causal_conv import causal_conv
    from eacs_b200.ops.continuous_query import cell_commits_train
    from eacs_b200.ops.continuous_ssm import ssm_forward
    from eacs_b200.ops.eacs_cell_train import GatedEACSCellFunction
    from eacs_b200.ops.gated_delta import gated_delta_rule
    from eacs_b200.ops.layer_norm import layer_norm
    from eacs_b200.ops.selective_ssm import selective_ssm

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def apart(t):
    """Elements two places apart."""
    return torch.empty(*t.shape, 2, dtype=t.dtype, device=t.device)[..., 0].copy_(t)


def shifted(t):
    """Dense, one element behind a boundary."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


def compare(run, seed=0, bits=True):
    """run(make) -> outputs, leaves; make(*shape, dtype) is the same random tensor in every run."""
    def once():
        g = torch.Generator(DEV).manual_seed(seed)
        return run(lambda *s, dtype=F32: torch.randn(*s, generator=g, device=DEV).to(dtype))
    g = torch.Generator(DEV).manual_seed(seed + 1)
    outs, leaves = once()
    ups = [torch.randn(o.shape, generator=g, device=DEV).to(o.dtype) for o in outs]
    want = torch.autograd.grad(outs, leaves, ups)
    assert all(bool(torch.isfinite(t).all()) for t in want)
    same = lambda t: t
    off = torch.autograd.graph.saved_tensors_hooks(shifted, same)
    for hooks in (torch.autograd.graph.saved_tensors_hooks(apart, same), torch.autograd.graph.save_on_cpu(), off):
        with hooks:
            outs, leaves = once()
        for t, u in zip(torch.autograd.grad(outs, leaves, ups), want):
            assert t.dtype == u.dtype and t.shape == u.shape
            if bits and hooks is not off:
                assert torch.equal(t, u)
            else:
                tol = 2.0 ** -11 * float(u.abs().max()) + (0 if u.dtype in (F32, torch.complex64) else torch.finfo(u.dtype).eps) * u.abs()
                assert bool(((t - u).abs() <= tol).all())


def leaf(t):
    return t.requires_grad_(True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("L,D,N", [(37, 48, 16), (70, 33, 12)])
def test_selective_scan(dtype, L, D, N):
    def run(rnd):
        x, dt, z = (leaf(rnd(2, L, D, dtype=dtype)) for _ in range(3))
        Bs, Cs, A = leaf(rnd(2, L, N, dtype=dtype)), leaf(rnd(2, L, N, dtype=dtype)), leaf(-rnd(D, N).abs())
        skip, bias, h0 = leaf(rnd(D)), leaf(rnd(D) - 3), leaf(rnd(2, D, N))
        n = torch.tensor([L, L - 9], device=DEV, dtype=torch.int32)
        outs = selective_ssm(x, dt, A, Bs, Cs, skip, z, bias, initial_state=h0, output_final_state=True, lengths=n)
        return outs, (x, dt, A, Bs, Cs, skip, z, bias, h0)
    compare(run)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [48, 50, 33])
def test_convolution(dtype, D):
    def run(rnd):
        x, w, b, h0 = leaf(rnd(2, 60, D, dtype=dtype)), leaf(rnd(D, 4)), leaf(rnd(D)), leaf(rnd(2, 3, D, dtype=dtype))
        n = torch.tensor([60, 41], device=DEV, dtype=torch.int32)
        return causal_conv(x, w, b, initial_state=h0, output_final_state=True, lengths=n), (x, w, b, h0)
    compare(run)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(40, 64), (3, 5, 99), (2, 768)])
def test_norms(dtype, shape):
    d = shape[-1]

    def gated(rnd):
        x, g, w = leaf(rnd(*shape, dtype=dtype)), leaf(rnd(*shape, dtype=dtype)), leaf(rnd(d))
        return (gated_norm(x, g, w),), (x, g, w)

    def residual(rnd):
        x, r, g = (leaf(rnd(*shape, dtype=dtype)) for _ in range(3))
        w, c, p = (leaf(rnd(d)) for _ in range(3))
        return residual_norm(x, r, w, c, g, p), (x, r, g, w, c, p)

    def layer(rnd):
        x, r, w, b = leaf(rnd(*shape, dtype=dtype)), leaf(rnd(*shape, dtype=dtype)), leaf(rnd(d)), leaf(rnd(d))
        return (layer_norm(x, w, b, residual=r),), (x, r, w, b)
    for f in (gated, residual, layer):
        compare(f)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gated_delta_rule(dtype):
    def run(rnd):
        q, k, v = (leaf(torch.nn.functional.normalize(rnd(2, 100, 2, 64), dim=-1).to(dtype)) for _ in range(3))
        g, beta, h0 = leaf(-rnd(2, 100, 2).abs()), leaf(torch.sigmoid(rnd(2, 100, 2))), leaf(rnd(2, 2, 64, 64))
        return gated_delta_rule(q, k, v, g, beta, initial_state=h0, output_final_state=True), (q, k, v, g, beta, h0)
    compare(run)


@pytest.mark.parametrize("which", ["ungated", "gated", "commits"])
def test_cells(which):
    d = cell_inputs(2, 50, 16, 8, seed=3)
    dev = lambda n: torch.from_numpy(d[n]).to(DEV)

    def run(rnd):
        lam, log_dt, u, Bc, Cc, t, D = (leaf(dev(n)) for n in ("lam", "log_dt", "u", "Bc", "Cc", "t", "D"))
        leaves = (lam, log_dt, u, Bc, Cc, t, D)
        if which == "ungated":
            return (ssm_forward(lam, log_dt, t, Bc, Cc, u, D),), leaves
        eps = leaf(torch.tensor(0.5, device=DEV))
        if which == "gated":
            outs = GatedEACSCellFunction.apply(u, Bc, Cc, t, lam, log_dt, D, eps, dev("mean"), dev("var"), 0.5, 1e-6, 1e-5, 1.0, "ste", True, 1e3)
            return outs[:1], (*leaves, eps)
        ys, _, _, c = cell_commits_train(lam, log_dt, u, Bc, Cc, t, D, dev("mean"), dev("var"), eps, 1e-6, 0.5, "ste")
        return (ys, c["h"].real), (*leaves, eps)
    compare(run, bits=False)
