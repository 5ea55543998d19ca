"""AdamW on so many elements that a warp takes runs of several blocks from a tensor, and codes to the last bit."""
import pytest
import torch
from test_gpu_adamw import check, moments32, to8

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


def test_codes_of_the_root_are_those_of_its_definition(igdev):
    """Root and codes to the last bit, over three steps: a code that is another by a root half a step off would show in the
    next step's update. Blocks of very different sizes, elements without a gradient and blocks of zeros among them."""
    from indecis_b200 import optim
    n = 1 << 24
    g = torch.Generator(device="cuda").manual_seed(7)
    opt = optim.AdamW([torch.zeros(n, device="cuda")], lr=1e-3, betas=(0.9, 0.98), bits=8)
    size = torch.exp(3.0 * torch.randn(n // 256, 1, generator=g, device="cuda")) * 1e-3
    size[::50] = 0.0
    for step in range(1, 4):
        grad = (torch.randn(n // 256, 256, generator=g, device="cuda") * size).view(-1)
        grad[torch.rand(n, generator=g, device="cuda") < 0.05] = 0.0
        m0, r0 = opt.exp_avg[0].values(), opt.exp_avg_sq[0].values()
        opt.step([grad])
        m1, v1 = moments32(m0, r0 * r0, grad, 0.9, 0.98)
        for got, want, second in ((opt.exp_avg[0], m1, False), (opt.exp_avg_sq[0], v1.sqrt(), True)):
            codes, scales = to8(want, step, second)
            assert torch.equal(got.scales, scales)
            assert torch.equal(got.codes.view(torch.uint8), codes.view(torch.uint8)), int((got.codes.float() != codes.float()).sum())


@pytest.mark.parametrize("bits", [32, 8])
def test_roots_at_the_ends(igdev, bits):
    """v of 0, below the normal range, next to its ends, and past float32: the update is that of sqrt(v), to 2^-20."""
    from indecis_b200 import optim
    g = torch.tensor([0.0, 1e-22, 1e-21, 1e-20, 1e-19, 1.2e-19, 3e-19, 1e-15, 1e-5, 1.0, 1e10, 1e18, 1.8e19, 1e20, 1e30, -1e-20, -1e20],
                     device="cuda")
    for one in g:  # a tensor each: a scale of its own
        p = torch.zeros(1, device="cuda")
        opt = optim.AdamW([p], lr=1.0, betas=(0.0, 0.5), eps=1e-37, weight_decay=0.0, bits=bits)
        opt.step([one.reshape(1)])
        v = ((one * one) * torch.tensor(0.5, device="cuda")).double()  # float32 products
        want = -(one.double() / ((v / 0.5).sqrt() + 1e-37))
        if float(v) == 0.0 and float(one) != 0.0:
            want = -(one.double() / 1e-37)
        assert abs(float(p) - float(want)) <= 2.0 ** -20 * abs(float(want)), (float(one), float(p), float(want))
