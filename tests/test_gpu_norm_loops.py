"""The norms on more narrow rows than a grid holds at once (the heads of a recurrence), aligned and not: the kernels' loops
over rows, with the backward's next row on its way, and a last round that fills a warp in part.  Oracle and bounds are those of
test_gpu_block_norm.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

from test_gpu_block_norm import BF16, F16, F32, check, inputs  # noqa: E402


# at most 592 CTAs of a backward: 32 rows each up to 128 bytes, 16 to 256, 8 to 512; more resident CTAs forward
@pytest.mark.parametrize("rows,d", [(80003, 64), (80001, 40), (40003, 128), (20005, 256), (80003, 31), (20001, 100)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_narrow_rows(rows, d, dtype):
    for k, (kind, kw) in enumerate([("gated", dict(gate=True)), ("gated", {}), ("residual", dict(scale=True)), ("residual", {}),
                                    ("residual", dict(gate=True)), ("residual", dict(gate=True, scale=True, post=True))]):
        i, rnd = inputs((rows, d), dtype, F32, kind, 40 + k, **kw)
        check(i, rnd(rows, d).to(dtype), rnd(rows, d).to(dtype))


@pytest.mark.parametrize("rows,d", [(9001, 512), (4003, 768), (3001, 1024), (2003, 2048)])
def test_many_wide_rows(rows, d):
    for k, kw in enumerate([dict(scale=True), dict(gate=True, scale=True, post=True)]):
        i, rnd = inputs((rows, d), BF16, BF16, "residual", 50 + k, **kw)
        check(i, rnd(rows, d).bfloat16(), rnd(rows, d).bfloat16())
