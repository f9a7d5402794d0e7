"""The selective scan where a CTA of the backward takes several groups of channels (batches of wide rows: dB and dC are
summed over them), the single-token kernel that takes four rows a thread, and sums that carry nothing from token to token.

Oracle and bounds are those of test_gpu_selective.py.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

from test_gpu_selective import BF16, F16, F32, NAMES, call, check, close, inputs, oracle  # noqa: E402

if torch.cuda.is_available():
    from eacs_b200 import _lib
    from eacs_b200.ops.selective_ssm import selective_ssm_step


def groups(rows, L, D, N):
    """(groups of channels a CTA of the backward takes, whether they divide D), from the size of its partial rows."""
    p = _lib.SELECTIVE.pack(*[256] * 5, *[8] * 10, *[256] * 3, 0, 0, rows, L, D, N, 0, 1)
    up = lambda n: -(-n // 256) * 256
    padded = next(n for n in (8, 16, 32, 64) if n >= N)
    cw = 128 // padded
    both = _lib.lib().eacs_selective_bwd_workspace_size(p) - up(rows * D * padded * 4) - up(rows * 2 * D * 4)
    parts = both // 2 // (rows * L * padded * 4)
    fits = [g for g in range(1, 9) if -(-D // (g * cw)) == parts]
    return min(fits), any(D % (g * cw) == 0 for g in fits)


# rows, D, N and whether the groups divide D
SHAPES = [(16, 768, 8, True), (16, 1000, 8, False), (8, 600, 8, False), (8, 2560, 8, False), (8, 768, 16, True), (8, 600, 16, True),
          (4, 2048, 16, False), (8, 1000, 16, False), (16, 160, 16, False), (8, 1000, 12, False), (16, 96, 32, True),
          (8, 250, 32, False), (4, 1000, 32, False), (16, 64, 64, True), (8, 250, 64, False), (8, 249, 33, False)]


@pytest.mark.parametrize("rows,D,N,divide", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients_over_several_groups(rows, D, N, divide, dtype):
    L = 75  # more than a ring of eight warps holds at once, ending inside a slice
    g, whole = groups(rows, L, D, N)
    assert g > 1 and whole == divide
    for k, kw in enumerate([dict(), dict(gate=False, ragged=True, initial=True)]):
        i, rnd = inputs(rows, L, D, N, dtype, 20 + k, **kw)
        if k:
            i["lengths"][2:6] = torch.tensor([1, 8, 64, 74], device=DEV)[:rows - 2]
        check(i, L, rnd(rows, L, D).to(dtype), rnd(rows, D, N) if k else None, NAMES + ("initial",))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,D,N", [(8, 768, 16), (4, 2048, 16)])
def test_rows_off_their_boundaries_over_several_groups(rows, D, N, dtype):
    L = 19
    assert groups(rows, L, D, N)[0] > 1
    i, rnd = inputs(rows, L, D, N, dtype, 23)
    for n in ("x", "z"):
        i[n] = rnd(rows, L, D + 3).to(dtype)[..., 1:D + 1]
    for n in ("B", "C"):
        i[n] = rnd(rows, L, N + 1).to(dtype)[..., 1:]
    check(i, L, rnd(rows, L, D).to(dtype), None, NAMES)


def test_sums_without_a_carry():
    """dskip = sum dy silu(z) x takes nothing from token to token.  Each term is off by 2^-19 at most (silu 2^-20, two
    products); a lane adds a token in 64, then come 64 such sums a row and the rows: one rounding each."""
    rows, L, D, N = 2, 3000, 1200, 16
    i, rnd = inputs(rows, L, D, N, F32, 24)
    i["lengths"] = torch.tensor([3000, 1777], device=DEV, dtype=torch.int32)
    dy = rnd(rows, L, D)
    i["skip"] = i["skip"].requires_grad_(True)
    got = torch.autograd.grad(call(i), i["skip"], dy)[0]
    live = (torch.arange(L, device=DEV) < i["lengths"][:, None])[..., None]
    terms = dy.double() * torch.nn.functional.silu(i["z"].double()) * i["x"].double() * live
    tol = (2.0 ** -19 + (-(-L // 64) + 64 + rows) * 2.0 ** -24) * terms.abs().sum((0, 1))
    assert bool(((got.double() - terms.sum((0, 1))).abs() <= tol).all())


@pytest.mark.parametrize("b", [297, 298, 299, 300, 301])  # whole groups of four rows, and one to three rows over
@pytest.mark.parametrize("D,N,dtype", [(1024, 8, F32), (512, 16, BF16), (512, 12, F16), (256, 33, F32), (256, 64, BF16)])
def test_steps_of_many_rows(b, D, N, dtype):
    padded = next(n for n in (8, 16, 32, 64) if n >= N)
    assert D * padded // 4 // 256 * (-(-b // 4)) >= 148 * 4  # rows enough for the kernel that takes four at once
    for kw in (dict(), dict(gate=False, softplus=False), dict(skip=False, bias=False)):
        i, _ = inputs(b, 1, D, N, dtype, 25, initial=True, **kw)
        want, mag = oracle(i), oracle(i, magnitudes=True)
        state = i["initial"].clone()
        tok = lambda n: None if i[n] is None else i[n][:, 0]
        y = selective_ssm_step(tok("x"), tok("dt"), i["A"], tok("B"), tok("C"), state, i["skip"], tok("z"), i["dt_bias"],
                               softplus=i["softplus"])
        close("y", y[:, None], want["y"], mag["y"], 1, dtype)
        close("state", state, want["final"], mag["final"], 1, F32)
