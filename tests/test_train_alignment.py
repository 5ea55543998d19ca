"""Layer norm's statistics off float32's boundary are refused before any device work (the addresses are never read)."""
import pytest

from indecis_b200 import _capi, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


M = 1 << 20


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("which", [0, 1])
def test_statistics(lib, which, off):
    mean, rstd = 8 * M + off * (which == 0), 9 * M + off * (which == 1)
    assert lib.ig_layer_norm(M, 0, 64, 4, 64, None, None, 0, 1e-5, 2 * M, 0, 64, mean, rstd, None) == _capi.IG_ERR_BAD_ARG
    assert "aligned" in _capi.last_error()
    assert lib.ig_layer_norm_backward(M, 0, 64, 2 * M, 0, 64, 4, 64, None, 0, mean, rstd, 3 * M, 64, None, None, None, 0,
                                      None) == _capi.IG_ERR_BAD_ARG
    assert "aligned" in _capi.last_error()
