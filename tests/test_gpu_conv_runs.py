"""The convolution on batches with runs of many stages: stages' places are used again, and whole stages take the kernels'
unrolled way.  Oracle and bounds are those of test_gpu_causal_conv.py; a channel's sum over a run of at most 608 tokens and
over 200 runs, a few in 32, is off by 640 2^-24 of its terms' sizes, with the terms' own 2^-18 less than the 2^-14 that they have."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

from test_gpu_causal_conv import BF16, F16, F32, check, inputs  # noqa: E402

if torch.cuda.is_available():
    from eacs_b200 import _lib

ROWS, L = 100, 603


def run_length(D, W):
    """Tokens that a run of the backward has at least, from its partial rows."""
    p = _lib.CONV.pack(256, 256, 256, 0, 0, L * D, D, ROWS, L, D, W, 0, 0, 1)
    parts = _lib.lib().eacs_conv_bwd_workspace_size(p) // (D * (W + 1) * 4)
    return L // -(-parts // ROWS)


def lengths():
    """Rows that end at every place of a stage, in the first, in inner and in the last run."""
    n = torch.arange(ROWS, device=DEV, dtype=torch.int32)
    out = torch.where(n < 20, L - n, torch.where(n < 40, 300 + n, torch.where(n < 60, n - 40, 97 + 7 * n)))
    return out.clamp(0, L).int()


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("D", [512, 510, 511])  # rows on 16 bytes (or 8), aligned to pairs of channels, odd
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_long_runs(D, W, dtype):
    assert run_length(D, W) > 5 * 8  # more stages than there is room for at once
    for k, kw in enumerate([dict(), dict(initial=True)]):
        i, rnd = inputs(ROWS, L, D, W, dtype, F32, 30 + k, **kw)
        if k:
            i["lengths"] = lengths()
        check(i)
        check(i, rnd(ROWS, L, D).to(dtype), rnd(ROWS, W - 1, D).to(dtype) if k else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_runs_of_a_slice(dtype):
    """x and dy as parts of wider tensors, on 16 bytes and aligned to pairs only."""
    i, rnd = inputs(ROWS, 300, 256, 4, dtype, dtype, 33)
    wide = rnd(ROWS, 300, 2 * 256 + 8).to(dtype)
    for at in (8, 258):
        check({**i, "x": wide[..., at:at + 248]} | {n: i[n][:248] for n in ("weight", "bias")}, wide.flip(1)[..., at:at + 248])
