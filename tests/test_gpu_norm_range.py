"""GPU: layer norm at the ends of fp32's range: rows whose values, though finite, are so large that a square of the mean or
a product with 1 / sigma is not."""
import pytest
import torch

import graphsage_amd as gs

import norm_reference as ref

pytestmark = pytest.mark.gpu

# rows of two waves to sixteen that leave some of a workgroup's waves without elements, one that does not, and rows
# longer than a workgroup's registers (fp32 and 16 bits take other kernels at the same width)
LARGE = [(torch.float32, F) for F in (200, 900, 1500, 2000, 2500, 3400, 6000, 10_000, 16_384, 16_385, 40_000)] + \
        [(torch.bfloat16, F) for F in (1000, 1800, 3000, 4000, 5000, 7000, 9000, 20_000)]


@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("dtype,F", LARGE)
def test_means_whose_square_passes_the_range(dtype, F, joined):
    """Rows of 2^65, an element in 64 larger by 2^58: mean^2 = 2^130 is no fp32 number, the squares about the mean (2^116
    each, 2^126 in all) are."""
    gen = torch.Generator().manual_seed(F)
    x = torch.full((5, F), 2.0 ** 65)
    x[torch.rand(5, F, generator=gen) < 1 / 64] *= 1 + 2.0 ** -7
    x = x.to(dtype)
    residual = torch.zeros(5, F, dtype=dtype) if joined else None
    w, g = (1 + 0.2 * torch.randn(F, generator=gen)).to(dtype), torch.randn(5, F, generator=gen).to(dtype)
    want = ref.reference(x, residual, w, g=g)
    d = [t.cuda().requires_grad_() for t in (x, w)]
    y = gs.dropout_add_layer_norm(d[0], residual.cuda() if joined else None, d[1])
    ref.check(y, want["y"], f"{F} {dtype} y")
    for got, name in zip(torch.autograd.grad(y, d, g.cuda()), ("grad_x", "grad_weight")):
        ref.check(got, want[name], f"{F} {dtype} {name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("F", [2, 4, 8, 16, 32, 64, 256, 1024])
def test_constant_rows_whose_mean_over_sigma_passes_the_range(F, dtype):
    """Rows of one number c have h = 0 and sigma = sqrt(eps) whatever c is, so their gradients are those of c = 0, bit for
    bit; at c = 2^110 and eps = 1e-12, c / sigma is no fp32 number.  Widths whose 1 / F is exact: of another the kernel takes
    c - (c F) fl(1 / F), fused, which is c d, |d| <= 2^-24 the rounding of 1 / F; (c d)^2 = 2^172 is infinite, 1 / sigma 0,
    and so are the gradients, within what fp32 means allow (an error of L u c in the mean against sigma = 2^-20)."""
    c = 2.0 ** 110
    gen = torch.Generator().manual_seed(F)
    w, g = (1 + 0.2 * torch.randn(F, generator=gen)).to(dtype).cuda(), torch.randn(9, F, generator=gen).to(dtype).cuda()
    res = torch.zeros(9, F, dtype=dtype, device="cuda")
    outs = []
    for value in (0.0, c):
        x = torch.full((9, F), value, dtype=dtype, device="cuda").requires_grad_()
        wl = w.clone().requires_grad_()
        plain = torch.autograd.grad(gs.layer_norm(x, wl, eps=1e-12), [x, wl], g)
        joined = torch.autograd.grad(gs.dropout_add_layer_norm(x, res, wl, eps=1e-12), [x, wl], g)
        outs.append([*plain, *joined])
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(b).all())
    assert float(outs[0][0].abs().max()) > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,F", [(600, 6), (5000, 64), (600, 300), (600, 5000), (600, 12_000), (600, 20_000), (5, 40_000)])
def test_an_infinite_gradient_stays_infinite_in_its_column(M, F, dtype):
    """One gradient of +inf: its column's grad_bias is +inf and grad_weight the infinity of h's sign; the other columns are
    what they are without it, bit for bit."""
    gen = torch.Generator().manual_seed(F)
    x = torch.randn(M, F, generator=gen).to(dtype).cuda()
    w = torch.ones(F, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.zeros(F, dtype=dtype, device="cuda", requires_grad=True)
    g = torch.randn(M, F, generator=gen).to(dtype).cuda()
    y = gs.layer_norm(x, w, b)
    clean = torch.autograd.grad(y, [w, b], g, retain_graph=True)
    row, col, inf = M // 7, F // 2, float("inf")
    g[row, col] = inf
    gw, gb = torch.autograd.grad(y, [w, b], g)
    h = float(y.detach()[row, col])             # (weight one, bias zero)
    assert h != 0.0 and float(gb[col]) == inf and float(gw[col]) == (inf if h > 0 else -inf)
    rest = torch.arange(F, device="cuda") != col
    assert torch.equal(gw[rest], clean[0][rest]) and torch.equal(gb[rest], clean[1][rest])
