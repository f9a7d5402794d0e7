"""Every gradient of the selective scan on more than 2^31 elements, near the end, against the same tokens as a small call.

The tokens in front of them are zeros with an empty state, and the part starts at a multiple of 8 tokens: both calls cut the
same slices, hand the same states from slice to slice, deal the slices to warps from the row's end, and add zeros for the
rest.  So every output, state and gradient is the same bits, float32 ones too.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
L, D, N, TAIL = (1 << 20) + 40, 2048, 16, 128

if torch.cuda.is_available():
    from eacs_b200.ops.selective_ssm import selective_ssm


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of device memory")
    yield
    torch.cuda.empty_cache()


def test_all_gradients():
    assert (L - TAIL) % 8 == 0
    g = torch.Generator(DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)

    def long(width):
        t = torch.zeros(1, L, width, device=DEV, dtype=torch.bfloat16)
        t[:, -TAIL:] = rnd(1, TAIL, width)
        return t
    A, skip, bias = -rnd(D, N).abs(), rnd(D), rnd(D) - 3
    seq = [long(D), long(D), long(N), long(N), long(D)]  # x, dt, B, C, z
    dy, dlast = long(D), rnd(1, D, N)

    def run(x, dt, Bs, Cs, z, dy):
        leaves = [t.requires_grad_(True) for t in (x, dt, A.clone(), Bs, Cs, skip.clone(), z, bias.clone())]
        y, last = selective_ssm(*leaves, output_final_state=True)
        return y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dy, dlast))
    tail = lambda t: t.detach()[:, -TAIL:].clone()
    want = run(*(tail(t) for t in seq), tail(dy))
    got = run(*seq, dy)
    names = ("y", "last", "dx", "ddt", "dA", "dB", "dC", "dskip", "dz", "dt_bias")
    for n, a, b in zip(names, got, want):
        assert bool(torch.isfinite(b).all()) and float(b.abs().max()) > 0, n
        a = a[:, -TAIL:] if a.dim() == 3 and n != "last" else a
        assert torch.equal(a, b), n
