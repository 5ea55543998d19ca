"""AdamW on so many elements that a warp takes runs of several blocks from a tensor."""
import pytest
import torch
from test_gpu_adamw import check

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# Blocks of 256 elements: runs of two or three from 28,416 or 42,624 on with three CTAs an SM, of sixteen (the most) from
# 227,328. The tensors end inside a run, inside a block, or after a single one.
SOME = [(1 << 23) + 13, 5, 1 << 21, 255, 256 * 3]
MOST = [(60 << 20) + 300, 77, 256 * 17, 1, 256 * 15 + 1]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt,copies", [(F32, F32, False), (F32, BF16, True), (BF16, BF16, False), (F16, F32, False)])
def test_some(igdev, bits, pt, gt, copies):
    check(SOME, pt, gt, bits, copies=copies, steps=2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 4])
def test_off_boundaries(igdev, bits, offset):
    check(SOME, F32, BF16, bits, offset=offset, steps=1)


@pytest.mark.parametrize("bits", [32, 8])
def test_most(igdev, bits):
    check(MOST, F32, BF16, bits, copies=True, steps=2, scale=0.5)
