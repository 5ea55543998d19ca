"""Outputs and workspaces of the training operators that share memory with an operand or one another are refused before any
device work. The addresses are never read: every call with a device present is refused."""
import pytest
import torch

from indecis_b200 import _capi, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


M = 1 << 20  # apart by more than any of the arguments takes
ROWS, N = 6, 64


def refused(call, base, name, **kw):
    args = dict(base, **kw)
    assert call(**args) == _capi.IG_ERR_BAD_ARG, kw
    assert name in _capi.last_error() and "share memory" in _capi.last_error(), _capi.last_error()


def apart(call, base):
    """The base call itself is refused for nothing; it would run, so it is made without a device only."""
    if not torch.cuda.is_available():
        assert call(**base) not in (_capi.IG_OK, _capi.IG_ERR_BAD_ARG), _capi.last_error()


def near(at, size, other):
    """Addresses of `size` bytes that share their first or last four with the `other` bytes at `at`."""
    return at + other - 4, at - size + 4


# Bytes of float32 x, y, dx, dy; of weight and its kin; of mean and rstd.
MATRIX, VECTOR, STATS = 4 * ROWS * N, 4 * N, 4 * ROWS


def test_layer_norm(lib):
    def call(x, w, b, y, mean, rstd):
        return lib.ig_layer_norm(x, 0, N, ROWS, N, w, b, 0, 1e-5, y, 0, N, mean, rstd, None)
    base = dict(x=M, w=2 * M, b=3 * M, y=4 * M, mean=5 * M, rstd=6 * M)
    apart(call, base)
    size = dict(x=MATRIX, w=VECTOR, b=VECTOR, y=MATRIX, mean=STATS, rstd=STATS)
    for out in ("y", "mean", "rstd"):
        for other in base:
            if other == out or (out, other) == ("y", "x"):  # y and x: in place, or apart
                continue
            for at in (base[other], *near(base[other], size[out], size[other])):
                refused(call, base, "ig_layer_norm", **{out: at})


def test_layer_norm_between_rows(lib):
    """What lies between the rows of a strided result shares nothing with it; what reaches into a row does."""
    def call(w, y, mean):
        return lib.ig_layer_norm(M, 0, N, ROWS, N, w, None, 0, 1e-5, y, 0, 3 * N, mean, None, None)
    base = dict(w=4 * M + 4 * N, y=4 * M, mean=4 * M + 4 * 5 * N - STATS)
    apart(call, base)
    refused(call, base, "ig_layer_norm", w=4 * M + 4 * N - 4)
    refused(call, base, "ig_layer_norm", w=4 * M + 4 * 2 * N + 4)
    refused(call, base, "ig_layer_norm", mean=4 * M + 4 * 6 * N - STATS + 4)


def test_layer_norm_backward(lib):
    def call(dy, x, w, mean, rstd, dx, dw, db, ws):
        return lib.ig_layer_norm_backward(dy, 0, N, x, 0, N, ROWS, N, w, 0, mean, rstd, dx, N, dw, db, ws, M // 2, None)
    names = ("dy", "x", "w", "mean", "rstd", "dx", "dw", "db", "ws")
    base = {k: (i + 1) * M for i, k in enumerate(names)}
    apart(call, base)
    size = dict(dy=MATRIX, x=MATRIX, w=VECTOR, mean=STATS, rstd=STATS, dx=MATRIX, dw=VECTOR, db=VECTOR,
                ws=lib.ig_layer_norm_workspace(ROWS, N))
    assert size["ws"] == ROWS * 2 * 4 * N
    for out in ("dx", "dw", "db", "ws"):
        for other in names:
            if other == out or (out, other) in (("dx", "x"), ("dx", "dy")):  # in place, or apart
                continue
            spots = (base[other], *near(base[other], size[out], size[other]))
            for at in spots if out != "ws" else (base[other] // 16 * 16, (base[other] + size[other] - 4) // 16 * 16):
                refused(call, base, "ig_layer_norm_backward", **{out: at})


def test_layer_norm_backward_without_rows(lib):
    """No rows: the sums are set to 0 all the same, each in memory of its own."""
    def call(w, dw, db):
        return lib.ig_layer_norm_backward(None, 0, N, None, 0, N, 0, N, w, 0, None, None, None, N, dw, db, None, 0, None)
    base = dict(w=M, dw=2 * M, db=3 * M)
    apart(call, base)
    for kw in (dict(dw=M), dict(db=2 * M), dict(dw=3 * M - 4), dict(db=M + VECTOR - 4)):
        refused(call, base, "ig_layer_norm_backward", **kw)


H, I, O = 64, 32, 48


def test_gated_ff(lib):
    def call(x, wi, wo, y, saved, ws):
        return lib.ig_gated_ff(x, H, wi, H, wo, I, 1, ROWS, H, I, O, 0, y, O, saved, ws, M // 2, None)
    names = ("x", "wi", "wo", "y", "saved", "ws")
    base = {k: (i + 1) * M for i, k in enumerate(names)}
    apart(call, base)
    for saved in (base["saved"], None):  # 4 rows or fewer without it take another workspace
        size = dict(x=2 * ROWS * H, wi=4 * I * H, wo=2 * O * I, y=2 * ROWS * O, saved=lib.ig_gated_ff_saved(ROWS, I),
                    ws=lib.ig_gated_ff_workspace(ROWS, H, I, O, 0, int(saved is not None)))
        at = dict(base, saved=saved)
        for out in ("y", "saved", "ws"):
            for other in names:
                if other == out or at[other] is None or size[out] == 0 or size[other] == 0 or at[out] is None:
                    continue
                for spot in (at[other], (at[other] + size[other] - 2) // 256 * 256, at[other] - (size[out] - 1) // 256 * 256):
                    if spot + size[out] > at[other]:
                        refused(call, at, "ig_gated_ff", **{out: spot})


def test_gated_ff_backward(lib):
    names = ("dy", "x", "wi", "wo", "saved", "dx", "dwi", "dwo", "ws")

    def call(dy, x, wi, wo, saved, dx, dwi, dwo, ws):
        return lib.ig_gated_ff_backward(dy, O, x, H, wi, H, wo, I, 1, ROWS, H, I, O, 0, saved, dx, H, dwi, H, dwo, I, ws, M // 2, None)
    base = {k: (i + 1) * M for i, k in enumerate(names)}
    apart(call, base)
    size = dict(dy=2 * ROWS * O, x=2 * ROWS * H, wi=4 * I * H, wo=2 * O * I, saved=lib.ig_gated_ff_saved(ROWS, I), dx=2 * ROWS * H,
                dwi=4 * I * H, dwo=2 * O * I, ws=lib.ig_gated_ff_workspace(ROWS, H, I, O, 0, 2))
    for out in ("dx", "dwi", "dwo", "ws"):
        for other in names:
            if other != out:
                for spot in (base[other], (base[other] + size[other] - 2) // 256 * 256, base[other] - (size[out] - 1) // 256 * 256):
                    refused(call, base, "ig_gated_ff_backward", **{out: spot})
