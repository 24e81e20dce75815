"""Layer norm, dropout and the two joined, from their formulas in float64 on the CPU, with the largest errors that
fp32 arithmetic and one rounding to the table's type can make.

Bounds, with u = 2^-24 (a rounding in fp32), t = finfo(type).eps / 2 (the one rounding of an output), A = the largest
|z| of the row, and L u the relative error of a sum (each partial sum is rounded at most L times: a lane's own
elements, then a tree over lanes and waves; L = 64 + F / 256 covers every width):

  z        : 3 u A                       1 / (1 - p), the product, the sum with the residual
  z - mean : E = (L + 4) u A             its operands' errors, the sum's, the subtraction's
  rstd     : R = rstd E + (L + 4) u      relative: half of var's, whose error is 2 sigma E + L u var; root, divide
  h        : H = rstd E + |h| (R + 2 u)
  y        : |w| H + 3 u (|h w| + |b|) + t |y|
  a = g w  : u |a|; mean(a): (L + 2) u mean|a|; mean(a h): mean(|a| H) + (L + 4) u mean|a h|
  dz       : rstd (u |a| + d mean(a) + |h| d mean(a h) + H |mean(a h)| + 3 u (|a| + |mean(a)| + |h mean(a h)|))
             + (R + 2 u) |dz|, and with the sum's gradient u (|dz| + |gsum|)
  dx       : 1 / (1 - p) times dz's, 2 u |dx|, t |dx|
  dw, db   : sum |g| H, and (Lr + 2) u sum |g h| (sum |g|) for sums over rows, Lr = 64 + M / 64
A type's smallest positive number is added to each: a result below the normal range is off by that at most.
"""
import torch

from graphsage_amd import rng

U = 2.0 ** -24


def keep(seed, shape, p, first=0):
    n = 1
    for s in shape:
        n *= s
    return torch.from_numpy(rng.dropout_keep_mask_range(seed, first, n, p)).view(shape).bool()


def drop(t, mask, p):
    return t if mask is None else torch.where(mask, t / (1.0 - p), torch.zeros((), dtype=torch.float64))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def reference(x, residual=None, weight=None, bias=None, p=0.0, eps=1e-5, seed=0, g=None, gsum=None, first=0):
    """All operands on the CPU, 2-D tables of one type, the rows of a larger table from element ``first`` on.  ->
     {name: (value, bound)} in float64."""
    dt = x.dtype
    wdt = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
    M, F = x.shape
    t, tiny = half_step(dt), _tiny(dt)
    mask = keep(seed, x.shape, p, first) if p > 0 else None
    z = drop(x.double(), mask, p)
    if residual is not None:
        z = z + residual.double()
    w = weight.double() if weight is not None else torch.ones(F, dtype=torch.float64)
    b = bias.double() if bias is not None else torch.zeros(F, dtype=torch.float64)
    L = 64 + F // 256
    # |z| here is the sum of the operands' sizes: what is rounded on the way to z
    size = drop(x.double(), mask, p).abs() + (residual.double().abs() if residual is not None else 0.0)
    A = size.max(1, keepdim=True).values
    mean = z.mean(1, keepdim=True)
    rstd = 1.0 / ((z - mean).square().mean(1, keepdim=True) + eps).sqrt()
    h = (z - mean) * rstd
    E = (L + 4) * U * A
    R = rstd * E + (L + 4) * U
    H = rstd * E + h.abs() * (R + 2 * U)
    y = h * w + b
    out = {"y": (y, w.abs() * H + 3 * U * ((h * w).abs() + b.abs()) + t * y.abs() + tiny),
           "sum": (z, 3 * U * size + t * z.abs() + tiny)}
    if g is None:
        return out
    g = g.double()
    a = g * w
    m1, m2 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    d1 = (L + 2) * U * a.abs().mean(1, keepdim=True)
    d2 = (a.abs() * H).mean(1, keepdim=True) + (L + 4) * U * (a * h).abs().mean(1, keepdim=True)
    dz = rstd * (a - m1 - h * m2)
    tz = rstd * (U * a.abs() + d1 + h.abs() * d2 + H * m2.abs() + 3 * U * (a.abs() + m1.abs() + (h * m2).abs())) \
        + (R + 2 * U) * dz.abs()
    if gsum is not None:
        tz = tz + U * (dz.abs() + gsum.double().abs())
        dz = dz + gsum.double()
    dx = drop(dz, mask, p)
    Lr = 64 + M // 64
    dw, db = (g * h).sum(0), g.sum(0)
    tw, wtiny = half_step(wdt), _tiny(wdt)
    out.update(grad_x=(dx, drop(tz, mask, p) + (2 * U + t) * dx.abs() + tiny),
               grad_residual=(dz, tz + t * dz.abs() + tiny),
               grad_weight=(dw, (g.abs() * H).sum(0) + (Lr + 2) * U * (g * h).abs().sum(0) + tw * dw.abs() + wtiny),
               grad_bias=(db, (Lr + 2) * U * g.abs().sum(0) + tw * db.abs() + wtiny))
    return out


def check(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, f"{what}: {tuple(got.shape)} for {tuple(value.shape)}"
    if not got.numel():
        return
    over = (got - value).abs() - bound * (1 + 1e-9)
    assert bool(torch.isfinite(got).all()) and float(over.max()) <= 0.0, (
        f"{what}: {int((~(over <= 0)).sum())} of {got.numel()} off by more than their bound, worst at "
        f"{int(over.argmax())}: {got.flatten()[over.argmax()].item()!r} for {value.flatten()[over.argmax()].item()!r}, "
        f"bound {bound.flatten()[over.argmax()].item():.3e}")
