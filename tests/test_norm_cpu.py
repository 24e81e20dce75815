"""CPU: layer norm and dropout's checks of arguments, at the C ABI and in Python, and the tests' own reference: its
gradients against central differences, its mask against the projection's mirror."""
import pytest
import torch

import graphsage_amd as gs
from graphsage_amd import _lib, rng

import norm_reference as ref


def test_entry_points_validate_before_touching_the_device():
    lib = _lib.load()
    one = 16          # a pointer that is never followed: every call below is refused, or has nothing to do
    assert lib.gsage_dropout(None, 8, _lib.F32, 0.5, 1, None, None, None) == -1
    assert lib.gsage_dropout(one, -1, _lib.F32, 0.5, 1, None, one, None) == -1
    assert lib.gsage_dropout(one, 8, 3, 0.5, 1, None, one, None) == -1
    for p in (1.0, -0.1, float("nan")):
        assert lib.gsage_dropout(one, 8, _lib.F32, p, 1, None, one, None) == -1
    assert lib.gsage_dropout(one, 1 << 50, _lib.F32, 0.5, 1, None, one, None) == -2
    assert lib.gsage_dropout(None, 0, _lib.F32, 0.5, 1, None, None, None) == 0

    def fwd(x=one, M=4, F=8, dtype=_lib.F32, wdtype=_lib.F32, eps=1e-5, p=0.0, y=one, mean=None, rstd=None):
        return lib.gsage_layer_norm_fwd(x, None, None, None, M, F, dtype, wdtype, eps, p, 0, None, y, None, mean, rstd, None)
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(M=-1) == -1 and fwd(F=0) == -1
    assert fwd(dtype=7) == -1 and fwd(wdtype=_lib.F16) == -1 and fwd(dtype=_lib.BF16, wdtype=_lib.F16) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(p=1.0) == -1
    assert fwd(mean=one) == -1 and fwd(rstd=one) == -1
    assert fwd(F=(1 << 24) + 1) == -2 and fwd(M=1 << 40) == -2
    assert fwd(M=0) == 0

    def bwd(g=one, x=one, mean=one, M=4, F=8, gw=None, ws=None, ws_bytes=0, wdtype=_lib.F32):
        return lib.gsage_layer_norm_bwd(g, None, x, None, None, mean, one, M, F, _lib.F32, wdtype, 0.0, 0, None, None, None,
                                        gw, None, ws, ws_bytes, None)
    assert bwd(g=None) == -1 and bwd(x=None) == -1 and bwd(mean=None) == -1 and bwd(F=0) == -1
    assert bwd(wdtype=_lib.BF16) == -1
    assert bwd(gw=one) == -1 and bwd(gw=one, ws=one, ws_bytes=8) == -3
    assert bwd(M=0) == 0
    size = lib.gsage_layer_norm_bwd_workspace_bytes
    assert size(-1, 8, _lib.F32) == 0 and size(8, 0, _lib.F32) == 0 and size(8, 8, 9) == 0
    assert size(0, 8, _lib.F32) >= 2 * 8 * 4 and size(1, 1 << 20, _lib.F32) >= 2 * 4 << 20


def test_python_checks():
    x = torch.zeros(4, 8)
    for call in (lambda: gs.layer_norm(x), lambda: gs.dropout(x), lambda: gs.dropout_add_layer_norm(x)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for p in (1.0, -0.25, float("nan"), 2):
        with pytest.raises(ValueError, match="rate"):
            gs.dropout(x, p)
        with pytest.raises(ValueError, match="rate"):
            gs.dropout_add_layer_norm(x, p=p)
    with pytest.raises(ValueError, match="eps"):
        gs.layer_norm(x, eps=-1e-5)
    with pytest.raises(ValueError, match="last dimension"):
        gs.LayerNorm((4, 8))
    m = gs.LayerNorm(8)
    assert list(m.state_dict()) == ["weight", "bias"] and m.eps == 1e-5
    assert list(gs.LayerNorm(8, bias=False).state_dict()) == ["weight"]
    with pytest.raises(ValueError, match="columns"):
        m(torch.zeros(4, 7))
    with pytest.raises(ValueError, match="GPU"):
        m(x)


@pytest.mark.parametrize("p,with_residual,with_sum", [(0.0, False, False), (0.3, True, True), (0.5, True, False)])
def test_reference_gradients_against_differences(p, with_residual, with_sum):
    gen = torch.Generator().manual_seed(5)
    M, F = 6, 11

    def rnd(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)
    ops = {"x": rnd(M, F), "residual": rnd(M, F) if with_residual else None, "weight": rnd(F), "bias": rnd(F)}
    g, gsum = rnd(M, F), rnd(M, F) if with_sum else None

    def loss(o):
        r = ref.reference(**o, p=p, seed=77)
        return float((r["y"][0] * g).sum() + ((r["sum"][0] * gsum).sum() if with_sum else 0.0))
    grads = ref.reference(**ops, p=p, seed=77, g=g, gsum=gsum)
    for name, value in ops.items():
        if value is None:
            continue
        v, step = rnd(*value.shape), 1e-5
        diff = (loss({**ops, name: value + step * v}) - loss({**ops, name: value - step * v})) / (2 * step)
        # truncation ~ step^2 times a third derivative (rows of 11: up to ~1e3), rounding ~ 1e-16 |loss| / step
        assert abs(diff - float((grads["grad_" + name][0] * v).sum())) <= 1e-6


def test_mask_of_a_long_table_counts_in_64_bits():
    first = (1 << 32) - 3
    part = rng.dropout_keep_mask_range(99, first, 8, 0.5)
    assert (part[3:] != rng.dropout_keep_mask_range(99, 0, 5, 0.5)).any()      # not the first elements' again


def test_model_options():
    from graphsage_amd import GraphSAGE, create_model
    m = GraphSAGE(num_layers=3, norm="layer", residual=True)
    assert [k for k in m.state_dict() if k.startswith("norms")] == ["norms.0.weight", "norms.0.bias", "norms.1.weight",
                                                                   "norms.1.bias"]
    assert not any(k.startswith("norms") for k in GraphSAGE().state_dict())
    assert len(GraphSAGE(num_layers=1, norm="layer").norms) == 0
    for bad in (dict(norm="batch"), dict(residual=True), dict(input_dropout=1.0), dict(input_dropout=-0.1)):
        with pytest.raises(ValueError):
            GraphSAGE(**bad)
    cfg = {"model": {"num_layers": 3, "norm": "layer", "residual": True, "input_dropout": 0.25}}
    m = create_model(cfg)
    assert (m.norm, m.residual, m.input_dropout) == ("layer", True, 0.25)
    with torch.no_grad():
        m.norms[1].weight.zero_()
    m.reset_parameters()
    assert bool((m.norms[1].weight == 1).all())
    with pytest.raises(ValueError, match="GPU"):
        m.train()(torch.randn(5, 7), torch.zeros(2, 3, dtype=torch.int64))


def test_a_model_pickled_before_the_options_existed():
    from graphsage_amd import GraphSAGE
    m = GraphSAGE()
    for k in ("norm", "residual", "input_dropout"):
        del m.__dict__[k]
    m.reset_parameters()
    assert (m.norm, m.residual, m.input_dropout) == (None, False, 0.0)
    with pytest.raises(ValueError, match="GPU"):
        m.train()(torch.randn(5, 7), torch.zeros(2, 3, dtype=torch.int64))
