"""The causal convolution, the selective scan and the block norms on tensors of more than 2^31 elements: what is computed
near their ends against the same places computed as small tensors (the convolution and the norms: the same bits; the scan,
whose slices then start elsewhere: within its own test's bounds, L 2^-21 for the tokens of the part)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
L, D, TAIL = (1 << 20) + 40, 2048, 64  # 2^31 elements and some more

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import residual_norm
    from eacs_b200.ops.causal_conv import causal_conv
    from eacs_b200.ops.selective_ssm import selective_ssm


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of device memory")
    yield
    torch.cuda.empty_cache()


def long(seed, scale=1.0):
    """(1, L, D) bfloat16, its last tokens random."""
    t = torch.zeros(1, L, D, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(DEV).manual_seed(seed)
    t[:, -2 * TAIL:] = torch.randn(1, 2 * TAIL, D, generator=g, device=DEV) * scale
    return t


def test_convolution():
    x, dy = long(0).requires_grad_(True), long(1)
    w = torch.randn(D, 4, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).requires_grad_(True)
    y, last = causal_conv(x, w, output_final_state=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    cut = x.detach()[:, -2 * TAIL:].clone().requires_grad_(True)
    y2, last2 = causal_conv(cut, w, output_final_state=True)
    dx2, dw2 = torch.autograd.grad(y2, (cut, w), dy[:, -2 * TAIL:])
    assert torch.equal(y[:, -2 * TAIL:], y2) and torch.equal(last, last2) and torch.equal(dx[:, -2 * TAIL:], dx2)
    # the same products in other runs: 128 of them at most 2^-24 of their size off each
    assert float((dw - dw2).abs().max()) <= 2.0 ** -16 * float(dw2.abs().max())
    assert float(y[:, :-2 * TAIL].abs().max()) == 0


def test_selective_scan():
    g = torch.Generator(DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    N = 4
    A = -torch.rand(D, N, generator=g, device=DEV) - 0.1
    Bs, Cs = rnd(1, L, N).bfloat16(), rnd(1, L, N).bfloat16()
    x, dt, dy = long(4).requires_grad_(True), long(5), long(6)
    y, last = selective_ssm(x, dt, A, Bs, Cs, output_final_state=True)
    dx = torch.autograd.grad(y, x, dy)[0]
    tail = lambda t: t.detach()[:, -2 * TAIL:].clone()
    cut = tail(x).requires_grad_(True)
    y2, last2 = selective_ssm(cut, tail(dt), A, tail(Bs), tail(Cs), output_final_state=True)  # nothing went in before them
    dx2 = torch.autograd.grad(y2, cut, tail(dy))[0]
    for a, b in ((y[:, -2 * TAIL:], y2), (last, last2), (dx[:, -2 * TAIL:], dx2)):
        scale = float(b.double().abs().max())
        assert float((a.double() - b.double()).abs().max()) <= (2 * TAIL * 2.0 ** -21 + 2.0 ** -8) * scale
    assert float(y[:, :-2 * TAIL].abs().max()) == 0


def test_norm():
    x, r, dy = long(7)[0].requires_grad_(True), long(8)[0], long(9)[0]
    y, s = residual_norm(x, r)
    dx = torch.autograd.grad((y, s), x, (dy, dy))[0]
    cut = x.detach()[-TAIL:].clone().requires_grad_(True)
    y2, s2 = residual_norm(cut, r[-TAIL:].clone())
    dx2 = torch.autograd.grad((y2, s2), cut, (dy[-TAIL:], dy[-TAIL:]))[0]
    assert torch.equal(y[-TAIL:], y2) and torch.equal(s[-TAIL:], s2) and torch.equal(dx[-TAIL:], dx2)


def test_rows_far_apart():
    """A batch whose second row starts past 2^31 elements."""
    big = torch.zeros((1 << 31) + 4096 * 64, device=DEV, dtype=torch.bfloat16)
    x = big.as_strided((2, 32, 64), (1 << 31, 64, 1))
    x.copy_(torch.randn(2, 32, 64, generator=torch.Generator(DEV).manual_seed(10), device=DEV))
    w = torch.ones(64, 3, device=DEV)
    assert torch.equal(causal_conv(x, w), causal_conv(x.contiguous(), w))
    A, B = -torch.ones(64, 8, device=DEV), torch.ones(2, 32, 8, device=DEV, dtype=torch.bfloat16)
    leaf = x.detach().requires_grad_(True)
    dense = x.contiguous().requires_grad_(True)
    y, y2 = selective_ssm(leaf, leaf, A, B, B, z=leaf), selective_ssm(dense, dense, A, B, B, z=dense)
    assert torch.equal(y, y2)
    assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0], torch.autograd.grad(y2.sum(), dense)[0])
