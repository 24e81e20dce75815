"""GPU: weight gradients of a layer whose input needs none, for gradients that start at odd addresses and for each kernel
that a caller may force: ReLU's derivative counts whichever kernel takes the call."""
import pytest
import torch

from graphsage_amd import _lib
from graphsage_amd.ops import project_bwd, project_fwd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epi", [_lib.EPI_RELU, _lib.EPI_RELU_DROPOUT])
@pytest.mark.parametrize("fi,fo", [(7, 64), (8, 64), (7, 128), (8, 128), (5, 192), (8, 256), (3, 100), (20, 128)])
@pytest.mark.parametrize("offset,force", [(0, 0), (1, 0), (2, 0), (0, 1), (0, 2), (3, 1)])
def test_weight_gradients_alone(fi, fo, offset, force, epi):
    n, p, seed = 333, 0.3, 77
    gen = torch.Generator().manual_seed(fi * 1000 + fo)
    agg, x, wl, bl, wr, g = (torch.randn(*s, generator=gen) for s in ((n, fi), (n, fi), (fo, fi), (fo,), (fo, fi), (n, fo)))
    rate = p if epi == _lib.EPI_RELU_DROPOUT else 0.0
    d = [t.cuda() for t in (agg, x, wl, bl, wr)]
    out, rnorm, sign = project_fwd(*d, epi, None, seed, rate, force_generic=force, want_relu_sign=True)
    grad = torch.empty(n * fo + 8, device="cuda")[offset:offset + n * fo].view(n, fo)
    grad.copy_(g)
    gwl, gb, gwr = project_bwd(grad, out, rnorm, d[0], d[1], d[2], d[4], None, epi, rate, False, force_generic=force,
                               relu_sign=sign)[2:]
    dpre = g.double() * (out.cpu() > 0) / (1.0 - rate)
    for got, want, size in ((gwl, dpre.t() @ agg.double(), dpre.abs().t() @ agg.double().abs()),
                            (gwr, dpre.t() @ x.double(), dpre.abs().t() @ x.double().abs()),
                            (gb, dpre.sum(0), dpre.abs().sum(0))):
        # 333 products and sums in fp32, or in two fp16 parts of 22 bits (4 u a product)
        assert bool(((got.cpu().double() - want).abs() <= (333 + 8) * 2.0 ** -24 * size + 1e-30).all())
