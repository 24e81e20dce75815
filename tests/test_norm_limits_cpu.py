"""CPU: layer norm and dropout's workspace sizes and the ends of the rate's range."""
import pytest

from graphsage_amd import _lib
from graphsage_amd.norm import _rate


def test_workspace_sizes():
    lib = _lib.load()
    plain, joined = lib.gsage_layer_norm_bwd_workspace_bytes, lib.gsage_layer_norm_bwd_joined_workspace_bytes
    # a slab of 2 F floats for every 64 rows of 64 columns, 128 of 32 or 96, 32 of 128, and 256 to fold them into
    for F, rows in ((32, 128), (64, 64), (96, 128), (128, 32)):
        M = 10_000_000
        assert plain(M, F, _lib.F32) == ((M + rows - 1) // rows + 256) * 2 * F * 4
        assert joined(M, F, _lib.F32) == 1024 * 2 * F * 4
    for M, F, dtype in ((10_000_000, 64, _lib.BF16), (1000, 64, _lib.F32), (10_000_000, 60, _lib.F32), (1 << 20, 4096, _lib.F16),
                        (0, 8, _lib.F32), (7, 1 << 20, _lib.F32)):
        assert 0 < joined(M, F, dtype) == plain(M, F, dtype) <= 1024 * 2 * F * 4 + 256
    assert joined(-1, 8, _lib.F32) == 0 and joined(8, 0, _lib.F32) == 0 and joined(8, 8, 9) == 0


def test_rates():
    assert _rate(0.0) == 0.0 and _rate(1e-60) == 0.0 and _rate(2.0 ** -149) == 2.0 ** -149 and _rate(0.5) == 0.5
    assert _rate(1.0 - 2.0 ** -24) == 1.0 - 2.0 ** -24
    for p in (-2.0 ** -149, 1.0 - 2.0 ** -25, 1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            _rate(p)
