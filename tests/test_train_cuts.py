"""How the gated block's calls are cut, as the library tells it (no GPU needed)."""
import ctypes

import pytest

from indecis_b200 import _capi, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def test_cuts(lib):
    c = (ctypes.c_int32 * 5)()
    for args, want in (((1, 768, 1152, 768, 0), [0, 0, 0, 0, 0]), ((1, 768, 1152, 768, 1), None), ((16384, 768, 1152, 768, 2), None)):
        assert lib.ig_check_gated_ff(*args, c) == _capi.IG_OK
        got = list(c)
        assert want is None or got == want
        if want is None:
            assert got[0] in (1, 2) and got[1] in (1, 2) and got[2] >= 1 and (got[3] >= 1) == (args[4] == 2)


@pytest.mark.parametrize("args", [(0, 8, 8, 8, 0), (-1, 8, 8, 8, 0), (4, 0, 8, 8, 0), (4, 8, 0, 8, 0), (4, 8, 8, 0, 0),
                                  (4, 8, 8, 8, 3), (4, 8, 8, 8, -1), (1 << 25, 8, 8, 8, 0), (4, 1 << 21, 8, 8, 0)])
def test_refusals(lib, args):
    assert lib.ig_check_gated_ff(*args, (ctypes.c_int32 * 5)()) == _capi.IG_ERR_BAD_ARG
    assert "ig_check_gated_ff" in _capi.last_error()


def test_no_place_for_the_answer(lib):
    assert lib.ig_check_gated_ff(4, 8, 8, 8, 0, None) == _capi.IG_ERR_BAD_ARG
