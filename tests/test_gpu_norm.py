"""GPU: layer norm, dropout and the two joined with a residual sum against their formulas in float64
(norm_reference.py: every element within the bound that fp32 arithmetic and one rounding can reach)."""
import pytest
import torch

import graphsage_amd as gs
from graphsage_amd import _lib, rng

import norm_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# one column; rows shorter than a vector; each kernel's first and last width and the odd ones around them; rows longer
# than any register tile; no rows, one row, a few and enough to go round the grid
SHAPES = [(0, 64), (1, 1), (9, 1), (3, 3), (65, 7), (1, 8), (70, 9), (33, 31), (20_001, 33), (33, 64), (33, 65), (9, 127),
          (40_003, 128), (7, 200), (5, 255), (33, 256), (300, 257), (6, 511), (17, 513), (9, 1000), (1500, 1024), (3, 1029),
          (5, 2047), (2, 2049), (1, 4096), (700, 4097), (2, 5120), (3, 8191), (3, 8193), (2, 16_384), (3, 16_385),
          (2, 32_768), (2, 33_001), (1, 70_003)]


def _rand(gen, *size, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*size, generator=gen) * scale + shift).to(dtype)


def _case(M, F, dtype, seed, residual=True, wdtype=None, with_sum=False):
    gen = torch.Generator().manual_seed(seed)
    c = {"x": _rand(gen, M, F, dtype=dtype, scale=1.5, shift=0.25),
         "residual": _rand(gen, M, F, dtype=dtype) if residual else None,
         "weight": _rand(gen, F, dtype=wdtype or dtype, scale=0.2, shift=1.0), "bias": _rand(gen, F, dtype=wdtype or dtype)}
    return c, _rand(gen, M, F, dtype=dtype), _rand(gen, M, F, dtype=dtype) if with_sum else None


def _cuda(c, grad=True):
    return {k: v if v is None else v.cuda().requires_grad_(grad) for k, v in c.items()}


def _run(c, g, gsum, p, seed, what, eps=1e-5):
    """forward + backward through the public call, every output against its bound."""
    want = ref.reference(**c, p=p, eps=eps, seed=seed, g=g, gsum=gsum)
    d = _cuda(c)
    out = gs.dropout_add_layer_norm(**d, p=p, eps=eps, seed=seed, return_sum=gsum is not None)
    outs = list(out) if gsum is not None else [out]
    leaves = {k: v for k, v in d.items() if v is not None}
    grads = torch.autograd.grad(outs, list(leaves.values()), [t.cuda() for t in (g, gsum) if t is not None])
    ref.check(outs[0], want["y"], what + " y")
    if gsum is not None:
        ref.check(outs[1], want["sum"], what + " sum")
    for name, got in zip(leaves, grads):
        assert got.dtype == leaves[name].dtype
        ref.check(got, want["grad_" + name], f"{what} grad_{name}")
    # without autograd: the same numbers, bit for bit
    with torch.no_grad():
        again = gs.dropout_add_layer_norm(**d, p=p, eps=eps, seed=seed, return_sum=gsum is not None)
    for a, b in zip(outs, again if gsum is not None else [again]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,F", SHAPES)
def test_joined_forward_backward(M, F, dtype):
    c, g, gsum = _case(M, F, dtype, M + 7 * F, with_sum=F % 2 == 1)
    _run(c, g, gsum, 0.3, 0x1234567_89ABCDEF + F, f"{M}x{F} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,F", SHAPES)
def test_layer_norm_forward_backward(M, F, dtype):
    c, g, _ = _case(M, F, dtype, 3 * M + F, residual=False, wdtype=torch.float32 if F % 2 else None)
    _run(c, g, None, 0.0, 0, f"{M}x{F} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,F", [(900, 2571), (800, 5003), (700, 8201), (600, 12_347), (530, 16_384), (520, 16_500)])
def test_wide_rows_by_the_workgroup(M, F, dtype):
    """rows of nine to sixteen waves and longer, several of them a workgroup"""
    c, g, gsum = _case(M, F, dtype, M + F, wdtype=torch.float32 if F % 2 else None, with_sum=F % 4 == 0)
    _run(c, g, gsum, 0.3, F, f"{M}x{F} {dtype}")


@pytest.mark.parametrize("F", [5, 64, 300, 4096, 40_000])
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(F, weight, bias):
    c, g, _ = _case(37, F, torch.float32, F, residual=False)
    if not weight:
        c["weight"] = None
    if not bias:
        c["bias"] = None
    _run(c, g, None, 0.0, 0, f"37x{F} weight {weight} bias {bias}")


@pytest.mark.parametrize("F", [64, 65, 1024, 20_000])
def test_first_hidden_layer_has_no_residual(F):
    c, g, gsum = _case(41, F, torch.bfloat16, F, residual=False, wdtype=torch.float32, with_sum=True)
    _run(c, g, gsum, 0.5, 2 ** 63 + 5, f"41x{F} no residual")


@pytest.mark.parametrize("M,F", [(50, 8), (50, 64), (20, 1000)])
def test_rows_that_lose_every_element_and_constant_rows(M, F):
    """p = 0.97 empties whole rows of 8 and leaves one or two elements of 64; eps alone carries an empty row."""
    c, g, _ = _case(M, F, torch.float32, F, residual=False)
    c["x"][M // 2:] = 3.0
    _run(c, g, None, 0.97, 11, f"{M}x{F} emptied")
    c["x"][:] = -2.5
    _run(c, g, None, 0.0, 0, f"{M}x{F} constant")
    mask = ref.keep(11, (M, F), 0.97)
    if F == 8:
        assert bool((~mask).all(1).any())
        x = torch.full((M, F), 7.0, device="cuda")
        y = gs.dropout_add_layer_norm(x, bias=c["bias"].cuda(), p=0.97, seed=11).cpu()
        empty = (~mask).all(1)
        assert torch.equal(y[empty], c["bias"].expand(int(empty.sum()), F))


@pytest.mark.parametrize("F", [4, 64, 250, 1024, 9000])
def test_gradients_of_some_operands_only(F):
    c, g, gsum = _case(19, F, torch.float32, F, with_sum=True)
    want = ref.reference(**c, p=0.3, seed=5, g=g, gsum=gsum)
    for wanted in (["x"], ["residual"], ["weight"], ["bias"], ["x", "bias"], ["residual", "weight"]):
        d = {k: v.cuda().requires_grad_(k in wanted) for k, v in c.items()}
        out = gs.dropout_add_layer_norm(**d, p=0.3, seed=5, return_sum=True)
        for name, got in zip(wanted, torch.autograd.grad(out, [d[k] for k in wanted], [g.cuda(), gsum.cuda()])):
            ref.check(got, want["grad_" + name], f"only {wanted} grad_{name}")


def test_gradient_through_one_of_the_two_outputs():
    c, g, gsum = _case(23, 100, torch.float32, 1, with_sum=True)
    d = _cuda(c)
    y, z = gs.dropout_add_layer_norm(**d, p=0.3, seed=5, return_sum=True)
    only_y = torch.autograd.grad(y, [d["x"], d["residual"]], g.cuda(), retain_graph=True)
    want = ref.reference(**c, p=0.3, seed=5, g=g)
    ref.check(only_y[0], want["grad_x"], "through y alone")
    ref.check(only_y[1], want["grad_residual"], "through y alone")
    only_z = torch.autograd.grad(z, list(d.values()), gsum.cuda())
    want = ref.reference(**c, p=0.3, seed=5, g=torch.zeros_like(g), gsum=gsum)
    for name, got in zip(d, only_z):
        ref.check(got, want["grad_" + name], f"through the sum alone grad_{name}")


@pytest.mark.parametrize("M,F,dtype", [(9, 50, torch.float32), (4, 1500, torch.float32)])
def test_gradient_against_differences_of_the_kernel(M, F, dtype):
    """(loss(o + s v) - loss(o - s v)) / 2s from the kernel's forward against <gradient, v>.  What they may differ by:
    the formula's own truncation at this step (taken in float64), the forward's bounds over 2s, the gradients' bounds;
    s is a power of two and v small integers over 4, so the moved operands are rounded by at most a half step, which
    the float64 side sees as well (it is given the rounded operands)."""
    c, g, _ = _case(M, F, dtype, 3)
    p, seed, step = 0.3, 21, 2.0 ** -7
    gen = torch.Generator().manual_seed(8)
    v = {k: torch.randint(-4, 5, t.shape, generator=gen).to(t.dtype) / 4 for k, t in c.items()}
    want = ref.reference(**c, p=p, seed=seed, g=g)
    diff = diff64 = noise = 0.0
    for sign in (1.0, -1.0):
        moved = {k: t + sign * step * v[k] for k, t in c.items()}
        y = gs.dropout_add_layer_norm(**_cuda(moved, False), p=p, seed=seed).cpu().double()
        r = ref.reference(**moved, p=p, seed=seed)["y"]
        diff += sign * float((y * g.double()).sum()) / (2 * step)
        diff64 += sign * float((r[0] * g.double()).sum()) / (2 * step)
        noise += float((r[1] * g.double().abs()).sum()) / (2 * step)
    d = _cuda(c)
    y = gs.dropout_add_layer_norm(**d, p=p, seed=seed)
    grads = dict(zip(d, torch.autograd.grad(y, list(d.values()), g.cuda())))
    along = sum(float((grads[k].cpu().double() * v[k].double()).sum()) for k in d)
    along64 = sum(float((want["grad_" + k][0] * v[k].double()).sum()) for k in d)
    bound = sum(float((want["grad_" + k][1] * v[k].double().abs()).sum()) for k in d)
    assert abs(diff - along) <= abs(diff64 - along64) + noise + bound
    assert abs(diff64 - along64) <= 0.02 * abs(along64)        # (the step is small enough to say something)


# ------------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(0, 4), (1,), (7,), (64,), (1023,), (2049, 3), (5, 7, 129), (300_007,), (3_000_001,)])
def test_dropout_forward_backward(shape, dtype):
    gen = torch.Generator().manual_seed(len(shape))
    x, g = _rand(gen, *shape, dtype=dtype), _rand(gen, *shape, dtype=dtype)
    for p, seed in ((0.3, 2 ** 64 - 9), (0.9, 17)):
        mask = ref.keep(seed, shape, p)
        d = x.cuda().requires_grad_()
        y = gs.dropout(d, p, seed=seed)
        dx, = torch.autograd.grad(y, d, g.cuda())
        for got, t in ((y, x), (dx, g)):
            value = ref.drop(t.double(), mask, p)
            # 1 - p and its inverse, the product, the rounding to the type
            ref.check(got, (value, (4 * ref.U + ref.half_step(dtype)) * value.abs() + ref._tiny(dtype)), f"{shape} p {p}")
            assert bool((got.cpu() != 0)[~mask].sum() == 0)


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tables_that_start_anywhere(offset, dtype):
    """Views that begin off a 16-byte boundary; memory before and behind is left as it was."""
    c, g, _ = _case(13, 72, dtype, offset)
    n = 13 * 72

    def place(t, fill=1e4):
        buf = torch.full((t.numel() + 64,), fill, dtype=t.dtype, device="cuda")
        view = buf[16 + offset:16 + offset + t.numel()].view(t.shape)
        view.copy_(t)
        return buf, view
    ops = {k: place(t) for k, t in c.items()}
    want = ref.reference(**c, p=0.3, seed=4, g=g)
    lib = _lib.load()
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    v = {k: b[1] for k, b in ops.items()}
    bufs = {k: torch.full((n + 64,), 77.0, dtype=dtype, device="cuda") for k in ("y", "sum", "gx", "gres", "gw", "gb", "drop")}
    out = {k: b[16 + offset:16 + offset + (72 if k in ("gw", "gb") else n)] for k, b in bufs.items()}
    mean, rstd = torch.empty(13, device="cuda"), torch.empty(13, device="cuda")
    st = _lib.stream_handle()
    assert lib.gsage_layer_norm_fwd(v["x"].data_ptr(), v["residual"].data_ptr(), v["weight"].data_ptr(),
                                    v["bias"].data_ptr(), 13, 72, code, code, 1e-5, 0.3, 4, None, out["y"].data_ptr(),
                                    out["sum"].data_ptr(), mean.data_ptr(), rstd.data_ptr(), st) == 0
    gbuf, gv = place(g)
    size = lib.gsage_layer_norm_bwd_workspace_bytes(13, 72, code)
    ws = torch.full((size + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    assert lib.gsage_layer_norm_bwd(gv.data_ptr(), None, v["x"].data_ptr(), v["residual"].data_ptr(), v["weight"].data_ptr(),
                                    mean.data_ptr(), rstd.data_ptr(), 13, 72, code, code, 0.3, 4, None,
                                    out["gx"].data_ptr(), out["gres"].data_ptr(), out["gw"].data_ptr(),
                                    out["gb"].data_ptr(), ws.data_ptr(), size, st) == 0
    assert lib.gsage_dropout(v["x"].data_ptr(), n, code, 0.3, 4, None, out["drop"].data_ptr(), st) == 0
    for k, name in (("y", "y"), ("sum", "sum"), ("gx", "grad_x"), ("gres", "grad_residual"), ("gw", "grad_weight"),
                    ("gb", "grad_bias")):
        ref.check(out[k].view(want[name][0].shape), want[name], f"offset {offset} {name}")
    value = ref.drop(c["x"].double(), ref.keep(4, (13, 72), 0.3), 0.3)
    ref.check(out["drop"].view(13, 72), (value, (4 * ref.U + ref.half_step(dtype)) * value.abs() + ref._tiny(dtype)), "dropout")
    for k, b in bufs.items():
        used = out[k].numel()
        assert bool((b[:16 + offset] == 77.0).all()) and bool((b[16 + offset + used:] == 77.0).all()), k
    assert bool((ws[size:] == 0x5A).all())
    for k, (b, view) in ops.items():
        assert torch.equal(view.cpu(), c[k])


def test_strides_and_dimensions():
    gen = torch.Generator().manual_seed(0)
    base = _rand(gen, 40, 60).cuda()
    w = _rand(gen, 40).cuda()
    for x in (base.t(), base[:, 3:43], base[::2, :40], base[:1, :40].expand(7, 40)):
        F = x.size(1)
        y = gs.layer_norm(x, w[:F])
        assert torch.equal(y, gs.layer_norm(x.contiguous(), w[:F])) and y.shape == x.shape
        assert torch.equal(gs.dropout(x, 0.4, seed=3), gs.dropout(x.contiguous(), 0.4, seed=3))
    x3 = base.view(4, 10, 60)
    assert torch.equal(gs.layer_norm(x3), gs.layer_norm(base).view(4, 10, 60))
    assert torch.equal(gs.layer_norm(base[0]), gs.layer_norm(base)[0])
    # a gradient that is one number broadcast over the table
    x = base.clone().requires_grad_()
    wl = _rand(gen, 60).cuda().requires_grad_()
    gx, gw = torch.autograd.grad(gs.layer_norm(x, wl).sum(), [x, wl])
    want = ref.reference(base.cpu(), weight=wl.detach().cpu(), g=torch.ones(40, 60))
    ref.check(gx, want["grad_x"], "broadcast gradient")
    ref.check(gw, want["grad_weight"], "broadcast gradient")
    # the same tensor twice: both gradients count
    x = base.clone().requires_grad_()
    g = _rand(gen, 40, 60)
    got, = torch.autograd.grad(gs.dropout_add_layer_norm(x, x, p=0.3, seed=6), x, g.cuda())
    want = ref.reference(base.cpu(), base.cpu(), p=0.3, seed=6, g=g)
    both = want["grad_x"][0] + want["grad_residual"][0]
    ref.check(got, (both, want["grad_x"][1] + want["grad_residual"][1] + ref.U * both.abs()), "x is its own residual")


def test_masks_are_the_projections():
    from graphsage_amd.ops import project_fwd
    n, f, p, seed = 300, 64, 0.3, 987654321
    gen = torch.Generator().manual_seed(1)
    d = [_rand(gen, n, 7).cuda(), _rand(gen, n, 7).cuda(), _rand(gen, f, 7).cuda(), _rand(gen, f, shift=5.0).cuda(),
         _rand(gen, f, 7).cuda()]
    relu, _ = project_fwd(*d, _lib.EPI_RELU)
    both, _ = project_fwd(*d, _lib.EPI_RELU_DROPOUT, None, seed, p)
    assert torch.equal(gs.dropout(relu, p, seed=seed) != 0, both != 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_a_dropped_element_holds_does_not_matter(dtype):
    M, F, p, seed = 50, 96, 0.5, 31
    gen = torch.Generator().manual_seed(2)
    x, res, g = (_rand(gen, M, F, dtype=dtype) for _ in range(3))
    mask = ref.keep(seed, (M, F), p)
    bad = x.clone()
    fill = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], dtype=dtype)
    bad[~mask] = fill[torch.arange(int((~mask).sum())) % 4]
    clean = [gs.dropout(x.cuda(), p, seed=seed), *gs.dropout_add_layer_norm(x.cuda(), res.cuda(), p=p, seed=seed, return_sum=True)]
    xb = bad.cuda().requires_grad_()
    dirty = [gs.dropout(xb, p, seed=seed), *gs.dropout_add_layer_norm(xb, res.cuda(), p=p, seed=seed, return_sum=True)]
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    gx, = torch.autograd.grad(dirty[1], xb, g.cuda(), retain_graph=True)
    want = ref.reference(x, res, p=p, seed=seed, g=g)
    ref.check(gx, want["grad_x"], "dropped NaNs")
    gb = g.clone()
    gb[~mask] = float("nan")                   # ... nor what the gradient holds there
    gx, = torch.autograd.grad(dirty[0], xb, gb.cuda())
    assert bool((gx.cpu()[~mask] == 0).all()) and bool(torch.isfinite(gx).all())


@pytest.mark.parametrize("F", [6, 64, 200, 3000, 20_000])
def test_a_bad_row_stays_its_own(F):
    gen = torch.Generator().manual_seed(3)
    x, g = _rand(gen, 40, F), _rand(gen, 40, F)
    bad = x.clone()
    bad[3, 1], bad[11, F - 1], bad[39, 0] = float("nan"), float("inf"), -float("inf")
    rows = torch.tensor([r for r in range(40) if r not in (3, 11, 39)])
    outs = []
    for t in (x, bad):
        d = t.cuda().requires_grad_()
        y = gs.layer_norm(d)
        outs.append((y.detach(), torch.autograd.grad(y, d, g.cuda())[0]))
    for a, b in zip(*outs):
        assert torch.equal(a.cpu()[rows], b.cpu()[rows])
        assert bool(torch.isnan(b.cpu()[[3, 11, 39]]).all())


def test_refusals_on_the_device():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(8, device="cuda")
    bad = [lambda: gs.layer_norm(x.double()), lambda: gs.layer_norm(x.to(torch.int32)), lambda: gs.layer_norm(x, w[:7]),
           lambda: gs.layer_norm(x, w.view(1, 8)), lambda: gs.layer_norm(x, w.cpu()), lambda: gs.layer_norm(x, w.half()),
           lambda: gs.layer_norm(x.half(), w.half(), w), lambda: gs.layer_norm(x[:, :0]), lambda: gs.layer_norm(x[0, 0]),
           lambda: gs.dropout_add_layer_norm(x, x[:3]), lambda: gs.dropout_add_layer_norm(x, x.half()),
           lambda: gs.dropout_add_layer_norm(x, x.cpu()), lambda: gs.dropout(x.double()),
           lambda: gs.dropout(x, seed=torch.zeros(1, dtype=torch.int64)),
           lambda: gs.dropout(x, seed=torch.zeros(2, dtype=torch.int64, device="cuda")),
           lambda: gs.dropout(x, seed=torch.zeros(1, dtype=torch.int32, device="cuda"))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert gs.dropout(x, 0.5, training=False) is x and gs.dropout(x, 0.0) is x
    t = x.clone().requires_grad_()
    y = gs.layer_norm(t, w)
    dx, = torch.autograd.grad((y * y).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        dx.sum().backward()
    seed = torch.tensor([5], device="cuda")
    y = gs.dropout(t, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_seeds():
    x = torch.ones(500, 64, device="cuda")
    for seed in (0, 1, 2 ** 40 + 3, -1, 2 ** 63 - 1):
        t = torch.tensor([seed], device="cuda")
        a = gs.dropout(x, 0.3, seed=seed)
        assert torch.equal(a, gs.dropout(x, 0.3, seed=t)) and torch.equal(a, gs.dropout(x, 0.3, seed=t[0]))
        assert torch.equal(a.cpu() != 0, ref.keep(seed & (2 ** 64 - 1), (500, 64), 0.3))
        assert torch.equal(gs.dropout_add_layer_norm(x, p=0.3, seed=seed), gs.dropout_add_layer_norm(x, p=0.3, seed=t))
    torch.manual_seed(3)
    a, b = gs.dropout(x), gs.dropout(x)
    torch.manual_seed(3)
    assert torch.equal(a, gs.dropout(x)) and not torch.equal(a, b)


def test_results_repeat_and_do_not_depend_on_the_stream():
    c, g, gsum = _case(30_011, 96, torch.bfloat16, 4, with_sum=True)

    def once():
        d = _cuda(c)
        outs = gs.dropout_add_layer_norm(**d, p=0.2, seed=3, return_sum=True)
        return [*outs, *torch.autograd.grad(outs, list(d.values()), [g.cuda(), gsum.cuda()])]
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, d in zip(first, second, once()):
        assert torch.equal(a, b) and torch.equal(a, d)


@pytest.mark.parametrize("M,F,dtype", [(2000, 128, torch.float32), (3, 5000, torch.bfloat16)])
def test_captured_step_draws_new_masks_on_every_replay(M, F, dtype):
    """norm -> dropout -> joined, forward and backward, in one graph whose seeds live on the device."""
    c, g, _ = _case(M, F, dtype, 9)
    d = _cuda(c)
    g = g.cuda()
    seeds = torch.tensor([3, 4], device="cuda")

    def step():
        h = gs.layer_norm(d["x"], d["weight"], d["bias"])
        h = gs.dropout(h, 0.2, seed=seeds[0:1])
        y = gs.dropout_add_layer_norm(h, d["residual"], d["weight"], d["bias"], p=0.3, seed=seeds[1:2])
        return [y.detach(), *torch.autograd.grad(y, list(d.values()), g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        seeds.copy_(torch.tensor([100 + i, 200 + i]))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="needs a seed"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gs.dropout(c["x"].new_zeros(4, 4, device="cuda"), 0.5)


# ------------------------------------------------------------------------------------ past 32-bit indices
def test_dropout_past_2_to_the_32_elements():
    n, p, seed = (1 << 32) + 4099, 0.3, 2 ** 50 + 1
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = gs.dropout(x, p, seed=seed)
    for first in (0, (1 << 31) - 50, (1 << 32) - 2000, n - 2051):
        want = torch.from_numpy(rng.dropout_keep_mask_range(seed, first, 2051, p)).bool()
        assert torch.equal((y[first:first + 2051] != 0).cpu(), want), first


def test_joined_past_2_to_the_32_elements():
    M, F, p, seed, dt = (1 << 24) + 5, 256, 0.3, 8, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(M, F, dtype=dt, device="cuda").normal_(generator=gen)
    g = torch.empty(M, F, dtype=dt, device="cuda").normal_(generator=gen)
    w = torch.linspace(0.5, 1.5, F, device="cuda")
    x.requires_grad_()
    y = gs.dropout_add_layer_norm(x, None, w, p=p, seed=seed)
    dx, = torch.autograd.grad(y, x, g)
    for r0 in (0, (1 << 23) - 2, (1 << 24) - 3, M - 5):
        part = slice(r0, r0 + 5)
        want = ref.reference(x.detach()[part].cpu(), weight=w.cpu(), p=p, seed=seed, g=g[part].cpu(), first=r0 * F)
        ref.check(y[part], want["y"], f"rows from {r0}")
        ref.check(dx[part], want["grad_x"], f"rows from {r0}")


@pytest.mark.parametrize("M,F,dtype,joined", [
    (1_050_011, 64, torch.float32, False), (1_050_011, 64, torch.float32, True), (524_301, 128, torch.float32, False),
    (524_301, 128, torch.float32, True), (262_151, 256, torch.float32, False), (2_100_001, 64, torch.bfloat16, False),
    (2_100_001, 64, torch.float16, True), (1_050_011, 128, torch.bfloat16, False), (525_001, 256, torch.float16, False),
    (262_151, 512, torch.bfloat16, False), (350_003, 384, torch.bfloat16, True), (131_101, 1024, torch.bfloat16, True),
    (66_001, 2048, torch.float16, False), (33_001, 2048, torch.float32, True), (16_800, 8192, torch.bfloat16, False),
    (8_300, 8192, torch.float32, False), (4_300, 16_000, torch.float32, True), (8_500, 16_000, torch.bfloat16, True),
    (8_500, 16_000, torch.float16, False)])
def test_tables_beyond_the_caches(M, F, dtype, joined):
    """From 256 MB on whole-line tables take the streaming forms: sampled rows against the formulas, the column sums
    against sums over the whole table in float64 on the GPU."""
    p, seed = (0.3, 77) if joined else (0.0, 0)
    gen = torch.Generator(device="cuda").manual_seed(F)

    def rnd(*size):
        return torch.empty(*size, dtype=dtype, device="cuda").normal_(generator=gen)
    x, g = rnd(M, F).requires_grad_(), rnd(M, F)
    res = rnd(M, F).requires_grad_() if joined else None
    w = (1 + 0.1 * rnd(F).float()).requires_grad_()
    b = rnd(F).float().requires_grad_()
    y = gs.dropout_add_layer_norm(x, res, w, b, p=p, seed=seed)
    leaves = [t for t in (x, res, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, g)
    names = ["grad_x"] + (["grad_residual"] if joined else [])
    for r0 in (0, 17, M // 2 - 3, M - 13):
        part = slice(r0, r0 + 13)
        want = ref.reference(x.detach()[part].cpu(), res.detach()[part].cpu() if joined else None, w.detach().cpu(),
                             b.detach().cpu(), p=p, seed=seed, g=g[part].cpu(), first=r0 * F)
        ref.check(y[part], want["y"], f"rows from {r0}")
        for name, got in zip(names, grads):
            ref.check(got[part], want[name], f"rows from {r0} {name}")
    # h from y: (y - b) / w, off by y's bound over w >= 0.5 and y's rounding; g h summed over the rows
    dw = torch.zeros(F, dtype=torch.float64, device="cuda")
    size = torch.zeros(F, dtype=torch.float64, device="cuda")
    for r0 in range(0, M, 1 << 18):
        part = slice(r0, r0 + (1 << 18))
        gd = g[part].double()
        h = (y.detach()[part].double() - b.detach().double()) / w.detach().double()
        dw += (gd * h).sum(0)
        size += (gd.abs() * (h.abs() + 3)).sum(0)
    # every term: y's rounding (half a step of |w h + b| <= 2 (|h| + 3) over |w| >= 0.5: a factor 4), the bounds of h
    # (H <= 100 u (|h| + 3) for rows of unit spread) and the sum's (64 + M / 64 roundings at most)
    tol = (4 * ref.half_step(dtype) + 100 * ref.U + (66 + M / 64) * ref.U) * size
    assert bool(((grads[-2].double() - dw).abs() <= tol).all())
    db = g.sum(0, dtype=torch.float64)
    assert bool(((grads[-1].double() - db).abs() <= (66 + M / 64) * ref.U * g.abs().sum(0, dtype=torch.float64)).all())


def test_more_workgroups_than_one_launch_takes():
    """17 M rows of 64: the forward's workgroups are dealt to more than one launch."""
    M, F = (1 << 24) + 77, 64
    x = torch.empty(M, F, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    y = gs.layer_norm(x)
    for r0 in (0, (1 << 23) - 5, (1 << 24) - 5, M - 10):
        ref.check(y[r0:r0 + 10], ref.reference(x[r0:r0 + 10].cpu())["y"], f"rows from {r0}")
