"""Layer norm at sizes that reach its kernels for many rows (several to a warp), and the backward pass of its longest rows
off 16-byte boundaries."""
import pytest
import torch
from test_gpu_layer_norm import check_backward, check_forward, rows_of, vector

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture
def many(igdev):
    """Rows that are enough for four to a warp on every SM, and end inside a warp's."""
    return 16 * 4 * torch.cuda.get_device_properties(0).multi_processor_count + 5


@pytest.mark.parametrize("n", [1, 64, 250, 256, 257, 511, 512, 700, 768, 1000, 1023, 1024])
@pytest.mark.parametrize("tx,ty", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)])
def test_forward(many, n, tx, ty):
    check_forward(rows_of(many, n, tx, seed=n), vector(n, F32, 1), vector(n, F32, 2) if n % 2 else None, 1e-5, ty)


@pytest.mark.parametrize("n,pad,offset", [(256, 8, 0), (256, 0, 1), (500, 3, 0), (768, 1, 8), (1024, 8, 8)])
@pytest.mark.parametrize("tx", [F32, BF16])
def test_strides(many, n, pad, offset, tx):
    x, out = rows_of(many, n, tx, pad, offset), rows_of(many, n, BF16, pad + 8, offset)
    check_forward(x, vector(n, BF16, 1, 1), vector(n, BF16, 2, 1), 1e-5, BF16, out)
    check_forward(x, None, None, 1e-3)


@pytest.mark.parametrize("n", [200, 512, 768])
def test_not_finite_rows_and_in_place(many, n):
    from indecis_b200 import layers
    x = rows_of(many, n, BF16)
    want = layers.layer_norm(x).y
    rows = [0, 6, many - 1]
    for k, v in zip(rows, (float("nan"), float("inf"), float("nan"))):
        x[k, n - 1] = v
    y = layers.layer_norm(x).y
    bad = torch.isnan(y).any(1)
    assert bad.nonzero().flatten().tolist() == rows and torch.equal(y[~bad], want[~bad])
    got = layers.layer_norm(x, out=x).y
    assert got.data_ptr() == x.data_ptr() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("n,pad,offset", [(5121, 0, 0), (6001, 0, 0), (8191, 0, 0), (8192, 0, 1), (8192, 1, 0), (5600, 2, 3)])
@pytest.mark.parametrize("tx,ty", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])
def test_backward_long_rows(igdev, n, pad, offset, tx, ty):
    check_backward(rows_of(301, n, tx, pad, offset, 1), rows_of(301, n, ty, pad, offset, 2), vector(n, F32, 3))
