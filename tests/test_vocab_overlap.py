"""Outputs that share some of their input's memory are refused before any device work. The addresses are never read:
every call below is refused."""
import pytest

from indecis_b200 import _capi, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


P = 1 << 20


# (address of the output, its row stride) beside logits of 4 rows x 100 float32 at P, 120 apart.
@pytest.mark.parametrize("d,ldd", [(P + 4, 120), (P + 40, 120), (P - 4, 120), (P + 4 * 99, 120), (P + 4 * 21, 120),
                                   (P + 4 * (120 + 60), 120), (P - 4 * 3 * 120 - 4 * 90, 120), (P + 4 * (3 * 120 + 99), 120),
                                   (P + 4 * 100, 121), (P + 8, 200), (P - 4 * 300, 100), (P - 4 * 399, 100), (P, 121)])
def test_logits(lib, d, ldd):
    q = 1 << 30
    assert lib.ig_token_logprobs_backward(P, 0, 120, 4, 100, 1.0, q, 1, q, q, q, None, d, ldd, None) == _capi.IG_ERR_BAD_ARG
    assert "overlap" in _capi.last_error() or "in place" in _capi.last_error()
    assert lib.ig_distill_topk(P, 0, 120, 4, 100, 1.0, q, q, 3, 0, None, q, d, ldd, None) == _capi.IG_ERR_BAD_ARG
    assert "overlap" in _capi.last_error() or "in place" in _capi.last_error()


def test_head(lib):
    h, w, q = P, 2 * P, 1 << 30

    def call(dh, dw, ldh=64, lddh=64, lddw=64):
        return lib.ig_vocab_logprobs_backward(h, ldh, w, 64, 1, 8, 100, 64, 1.0, q, 1, q, q, q, q, None, dh, lddh, dw, lddw, q,
                                              1 << 40, None)
    for dh, dw in ((h, None), (h + 2, None), (h + 128, 3 * P), (w + 2, None), (None, h + 2), (None, w - 2), (None, w + 12798),
                   (3 * P, 3 * P), (3 * P + 2, 3 * P), (3 * P, 3 * P + 1022)):
        assert call(dh, dw) == _capi.IG_ERR_BAD_ARG, (dh, dw)
        assert "overlap" in _capi.last_error() or "replace" in _capi.last_error()
