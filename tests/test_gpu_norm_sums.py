"""GPU: the column sums of layer norm's backward (grad_weight, grad_bias), bit for bit: inputs whose every product and
partial sum is an fp32 number, so that a row lost, counted twice or added to the wrong column shows, however many rows."""
import pytest
import torch

import graphsage_amd as gs
from graphsage_amd import _lib

import norm_reference as ref

pytestmark = pytest.mark.gpu

U = ref.U


def _signs(gen, M, F):
    """[M, F] of +-1, a column and its neighbour of opposite signs: every pair of columns, hence every row, every wave's
    part of one and every vector of V columns, sums to exactly zero, its squares to the number of columns."""
    s = (torch.randint(0, 2, (M, F // 2, 1), device="cuda", generator=gen, dtype=torch.int8) * 2 - 1)
    return torch.cat([s, -s], 2).view(M, F)


def _exact(M, F, dtype, joined, wdtype):
    """x = +-1 (joined: the sum of two halves) has mean 0 and variance 1; eps = 3 makes sigma 2 and h = +-1/2.  Gradients
    are integers from -3 to 3: sums of at most 3 M < 2^24 halves, exact in any order."""
    assert 3 * M < 1 << 24 and F % 2 == 0
    gen = torch.Generator(device="cuda").manual_seed(M + F)
    signs = _signs(gen, M, F)
    g = torch.randint(-3, 4, (M, F), device="cuda", generator=gen, dtype=torch.int8)
    x = signs.to(dtype)
    w = torch.ones(F, dtype=wdtype, device="cuda", requires_grad=True)
    b = torch.zeros(F, dtype=wdtype, device="cuda", requires_grad=True)
    if joined:
        x = (x * 0.5).requires_grad_()
        y = gs.dropout_add_layer_norm(x, x.detach().clone(), w, b, eps=3.0)
    else:
        x.requires_grad_()
        y = gs.layer_norm(x, w, b, eps=3.0)
    assert torch.equal(y.detach(), signs.to(dtype) * 0.5)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], g.to(dtype))
    assert bool(torch.isfinite(gx).all())
    want_w, want_b = torch.zeros(F, dtype=torch.int64, device="cuda"), torch.zeros(F, dtype=torch.int64, device="cuda")
    for r0 in range(0, M, 1 << 18):
        part = g[r0:r0 + (1 << 18)].to(torch.int16)
        want_w += (part * signs[r0:r0 + (1 << 18)]).sum(0)
        want_b += part.sum(0)
    if M > 1000:
        assert int((want_w != 0).sum()) > F // 2 and int((want_b != 0).sum()) > F // 2
    assert torch.equal(gw, (want_w.double() * 0.5).to(wdtype)), f"{M}x{F} {dtype} grad_weight"
    assert torch.equal(gb, want_b.double().to(wdtype)), f"{M}x{F} {dtype} grad_bias"


# every width's kernel, whole vectors and moved ones, with rows from one to several flushes of a thread's registers
WIDTHS = [2, 6, 14, 20, 34, 64, 82, 96, 128, 130, 170, 192, 256, 300, 384, 512, 700, 1000, 1024, 1300, 2048, 2600, 4096, 5120,
          6002, 8000, 8192, 12_002, 16_000, 16_386, 20_002]


@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("F", WIDTHS)
def test_every_row_counts_once(F, dtype, joined):
    for M in (1, 17, 300, 5003, 70_001, 1_050_011, 5_000_011):
        if M * F <= 1 << 27:
            _exact(M, F, dtype, joined, torch.float32)


@pytest.mark.parametrize("F,M", [(64, 255), (1024, 40), (9000, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_in_the_tables_type(F, M, dtype):
    _exact(M, F, dtype, True, dtype)        # (sums of at most 3 M halves, rounded once)


@pytest.mark.parametrize("M,F,dtype,joined", [
    (1_050_011, 64, torch.float32, False), (1_050_011, 64, torch.float32, True), (524_301, 128, torch.float32, False),
    (700_001, 96, torch.float32, False), (5_300_003, 32, torch.float32, False), (524_301, 128, torch.float32, True),
    (262_151, 256, torch.float32, False), (262_151, 256, torch.float32, True), (2_100_001, 64, torch.bfloat16, False),
    (2_100_001, 64, torch.float16, True), (1_050_011, 128, torch.bfloat16, False), (525_001, 256, torch.float16, False),
    (350_003, 384, torch.bfloat16, True), (131_101, 1024, torch.bfloat16, True), (33_001, 2048, torch.float32, True),
    (16_800, 8192, torch.bfloat16, False), (8_300, 8192, torch.float32, False), (4_300, 16_000, torch.float32, True),
    (8_500, 16_000, torch.bfloat16, True)])
def test_tables_beyond_the_caches_count_every_row_once(M, F, dtype, joined):
    """The streaming forms (256 MB and whole lines), among them the slabs that are folded first (plain fp32, up to 128)."""
    _exact(M, F, dtype, joined, torch.float32)


@pytest.mark.parametrize("M,F,joined", [(1 << 25, 64, True), (1 << 25, 64, False), (1 << 25, 130, False), (1 << 22, 770, False)])
def test_thousands_of_rows_a_thread_lose_no_bits(M, F, joined):
    """Every gradient is v = 1 + 2^-18: sums of up to 32 are fp32 numbers, and the sum of 16 or 32 of them added to an fp32
    sum of 64 such or more is half a step past it and lost.  Left are a slab's rounding and the result's: 2 u (+ u^2)."""
    v = 1.0 + 2.0 ** -18
    x = torch.zeros(M, F, device="cuda")
    b = torch.zeros(F, device="cuda", requires_grad=True)
    y = gs.dropout_add_layer_norm(x, x if joined else None, None, b)
    gb, = torch.autograd.grad(y, b, torch.full((M, F), v, device="cuda"))
    assert float((gb.double() - M * v).abs().max()) <= 2.001 * U * M * v


@pytest.mark.parametrize("M,F,dtype", [(1_050_011, 64, torch.float32), (524_301, 128, torch.float32), (700_001, 96, torch.float32),
                                       (2_100_037, 32, torch.float32), (2_100_001, 64, torch.bfloat16), (33, 64, torch.float32),
                                       (1, 20_000, torch.float32), (300_007, 1, torch.float16), (9000, 5000, torch.float16)])
@pytest.mark.parametrize("joined", [False, True])
def test_workspaces_are_large_enough_and_no_larger_than_said(M, F, dtype, joined):
    """What a call is told to bring is enough (nothing behind it is written, less is refused), joined calls need no slab
    for every few rows, and sums are the same whatever the workspace held."""
    lib, code = _lib.load(), {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dtype]
    size = (lib.gsage_layer_norm_bwd_joined_workspace_bytes if joined else lib.gsage_layer_norm_bwd_workspace_bytes)(M, F, code)
    assert size <= lib.gsage_layer_norm_bwd_workspace_bytes(M, F, code)
    if joined:
        assert size <= max(1024 * 2 * F * 4, 256)
    gen = torch.Generator(device="cuda").manual_seed(F)
    x, g = (torch.empty(M, F, dtype=dtype, device="cuda").normal_(generator=gen) for _ in range(2))
    res = torch.zeros_like(x) if joined else None
    mean, rstd = x.float().mean(1), torch.ones(M, device="cuda")
    st, outs = _lib.stream_handle(), []
    for fill in (0x00, 0x7F):
        ws = torch.full((size + 4096,), fill, dtype=torch.uint8, device="cuda")
        gw, gb, gx = torch.empty(F, device="cuda"), torch.empty(F, device="cuda"), torch.empty_like(x)

        def call(nbytes):
            return lib.gsage_layer_norm_bwd(g.data_ptr(), None, x.data_ptr(), _lib.ptr(res), None, mean.data_ptr(),
                                            rstd.data_ptr(), M, F, code, _lib.F32, 0.0, 0, None, gx.data_ptr(), None,
                                            gw.data_ptr(), gb.data_ptr(), ws.data_ptr(), nbytes, st)
        assert call(size - 1) == -3
        assert call(size) == 0
        assert bool((ws[size:] == fill).all())
        outs.append((gw, gb))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    gbd, size_b = g.double().sum(0), g.double().abs().sum(0)
    assert bool(((outs[0][1].double() - gbd).abs() <= (66 + M / 64) * U * size_b).all())


@pytest.mark.parametrize("F,dtype,joined,rows", [
    (20, torch.float32, False, 64), (64, torch.float32, True, 64), (60, torch.bfloat16, False, 64), (62, torch.bfloat16, True, 64),
    (200, torch.float16, False, 32), (300, torch.float32, False, 16), (1000, torch.float32, False, 4), (1200, torch.float32, True, 4),
    (2000, torch.bfloat16, False, 4), (2600, torch.float32, False, 1), (5120, torch.bfloat16, False, 1),
    (5120, torch.float16, True, 1)])
def test_every_row_counts_once_around_each_flush(F, dtype, joined, rows):
    """As many rows as make a thread's number of them one less, as many and one more than the registers' sums are kept for:
    16 or 32, twice that, for 256 and 512 workgroups of `rows` rows at once."""
    for workgroups in (256, 512):
        for turns in (15, 16, 17, 23, 31, 32, 33, 63, 64, 65, 97):
            for M in (workgroups * rows * turns - 1, workgroups * rows * turns):
                if M * F <= 1 << 28 and 3 * M < 1 << 24:
                    _exact(M, F, dtype, joined, torch.float32)
