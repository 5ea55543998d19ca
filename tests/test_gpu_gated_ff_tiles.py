"""The gated block at sizes that reach each of its cuts: h and [da | db] by the large tile, products by either tile, with
their sums over K in one part and in several. Every case says which cut it is there for, and that is looked at first."""
import ctypes

import pytest
import torch
import test_gpu_gated_ff as block

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
SMALL, LARGE = 1, 2


@pytest.fixture(autouse=True)
def activation_bound(monkeypatch):
    """The activation's own error relative to its value where |a| <= 6, as here: 4.4e-6 of R with its roundings, 3 half steps
    of the exponent a^2 / 2 times it (9e-8 a^2), and 2^-21 for the exponential, the reciprocal and the products."""
    monkeypatch.setattr(block, "ACT", 4.4e-6 + 9e-8 * 36 + 2.0 ** -21)


def cut(rows, H, I, O, backward):
    from indecis_b200 import _capi
    c = (ctypes.c_int32 * 5)()
    _capi.check(_capi.load().ig_check_gated_ff(rows, H, I, O, 2 if backward else 0, c))
    return list(c)


def reaches(sizes, h=None, z=None, y=None, grads=None):
    """y: (tile, split); grads: (tile, split of dw_in, dw_out, dx)."""
    f, b = cut(*sizes, False), cut(*sizes, True)
    assert h is None or f[0] == h
    assert z is None or b[0] == z
    assert y is None or (f[1], f[2] > 1) == y
    assert grads is None or (b[1], *[p > 1 for p in b[2:]]) == grads


# Rows whose last pair of tiles has a second CTA without any; inner sizes off multiples of 32 and 16, odd ones among them.
INNER = [(2817, 515, 1037, 517), (2900, 520, 1104, 504), (2944, 512, 1088, 512), (5930, 9, 213, 8)]


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("sizes", INNER[:2])
def test_large_inner_activations(igdev, sizes, kind):
    reaches(sizes, h=LARGE, z=LARGE)
    block.check(*sizes, BF16, kind, seed=1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes", INNER)
def test_large_inner(igdev, sizes, dtype):
    reaches(sizes, h=LARGE)
    block.check(*sizes, dtype, seed=2)


@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (0, 8), (3, 1)])
def test_large_inner_strides(igdev, pad, offset):
    reaches((2900, 520, 1104, 504), h=LARGE, z=LARGE)
    block.check(2900, 520, 1104, 504, BF16, pad=pad, offset=offset, seed=3)


@pytest.mark.parametrize("sizes,y,grads", [
    # y by the large tile: whole and odd columns.
    ((9001, 265, 401, 267), (LARGE, False), None),
    ((9000, 264, 400, 264), (LARGE, False), None),
    ((4354, 8, 9, 557), (LARGE, False), None),
    # its sums over K in parts, large and small tile.
    ((1661, 11, 3791, 711), (LARGE, True), None),
    ((1660, 16, 3792, 704), (SMALL, False), None),
    ((1700, 16, 3792, 712), (LARGE, True), None),
    ((1664, 16, 3792, 768), (LARGE, True), None),
    ((8, 64, 4096, 64), (SMALL, True), None),
    ((300, 63, 4001, 65), (SMALL, True), None),
    # The gradients by the large tile.
    ((2561, 700, 1000, 700), None, (LARGE, False, False, False)),
    ((2561, 701, 1003, 699), None, (LARGE, False, False, False)),
    ((2689, 704, 1024, 704), None, (LARGE, False, False, False)),
    # Their sums in parts: those of the weights over rows, those of the rows over columns.
    ((9687, 1020, 8, 57), None, (LARGE, True, True, False)),
    ((5, 164, 2614, 1184), None, (LARGE, False, False, True)),
    ((4000, 64, 64, 64), None, (SMALL, True, True, False)),
    ((1346, 12, 8, 11), None, (SMALL, True, True, False)),
    ((1805, 8, 159, 8), None, (SMALL, True, True, True)),
    ((20, 64, 8000, 100), (SMALL, True), (SMALL, False, False, True)),
])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_products(igdev, sizes, y, grads, dtype):
    reaches(sizes, y=y, grads=grads)
    block.check(*sizes, dtype, seed=4)


@pytest.mark.parametrize("rows", [2561, 2817])
def test_not_finite_rows_stay_alone(igdev, rows):
    from indecis_b200 import layers
    reaches((rows, 512, 1088, 512), h=LARGE)
    x, w_in, w_out = (block.matrix(r, c, BF16, i) for i, (r, c) in enumerate([(rows, 512), (2176, 512), (512, 1088)]))
    want = layers.gated_ff(x, w_in, w_out)
    for row in (5, 130, rows - 1):
        x[row, 7] = float("nan")
    y, saved = layers.gated_ff(x, w_in, w_out, save=True)
    bad = (~torch.isfinite(y)).any(1).nonzero().flatten().tolist()
    assert bad == [5, 130, rows - 1]
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(y[keep], want[keep])
    dx, _, _ = layers.gated_ff_backward(want, x, w_in, w_out, saved)
    assert (~torch.isfinite(dx)).any(1).nonzero().flatten().tolist() == bad


def test_two_streams_and_a_graph(igdev):
    """Large tiles and sums in parts, on two streams at once and recorded."""
    from indecis_b200 import layers
    for sizes in ((2817, 515, 1037, 517), (1661, 11, 3791, 711), (1805, 8, 159, 8)):
        x, w_in, w_out, dy, _, want = block.check(*sizes, BF16, seed=5)

        def run():
            y, saved = layers.gated_ff(x, w_in, w_out, save=True)
            return (y, *layers.gated_ff_backward(dy, x, w_in, w_out, saved))
        torch.cuda.synchronize()
        got = []
        for s in [torch.cuda.Stream() for _ in range(2)] * 2:
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for one in got for p, q in zip(one[1:], want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one = run()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(one[1:], want))
