"""Calls of the training operators beside torch's own autograd, with lists that have gaps, and with values at the ends of
their ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("of", ["y", "dx"])
def test_written_in_place_is_seen_by_autograd(igdev, of):
    """A graph that keeps a tensor refuses to go on once a call wrote over it, as with torch's own in-place operations."""
    from indecis_b200 import layers
    leaf = randn(5, 64, seed=1).requires_grad_()
    kept = leaf * 1.0
    z = (kept * kept).sum()
    r = layers.layer_norm(kept.detach().clone())
    if of == "y":
        layers.layer_norm(kept, out=kept)
    else:
        layers.layer_norm_backward(kept, randn(5, 64, seed=2), r.mean, r.rstd, out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_results_of_their_own_raise_no_version(igdev):
    from indecis_b200 import layers
    x, dy = randn(5, 64, seed=1), randn(5, 64, seed=2)
    r = layers.layer_norm(x)
    layers.layer_norm_backward(dy, x, r.mean, r.rstd)
    assert x._version == 0 and dy._version == 1 - 1
    with torch.inference_mode():  # tensors without a version
        y = torch.empty(5, 64, device="cuda")
        layers.layer_norm(x, out=y)
        layers.layer_norm_backward(dy, x, r.mean, r.rstd, out=y)
    with pytest.raises((RuntimeError, ValueError)):
        layers.layer_norm(x, eps=-1.0, out=dy)
    assert dy._version == 0  # refused: as it was


def test_refused_step_raises_no_version(igdev):
    """Only a step that was made changes parameters and copies for autograd."""
    from indecis_b200 import _capi, optim
    p = [randn(40, seed=i) for i in range(3)]
    copies = [t.bfloat16() for t in p]
    g = [randn(40, seed=10 + i) for i in range(3)]
    m, v = ([torch.zeros(40, device="cuda") for _ in p] for _ in range(2))
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = [t._version for t in p + copies]
    for grads, moments, kw in ((g, m, dict(lr=-1.0)), (g, m, dict(betas=(0.9, 1.0))), (g[:2] + [g[2][:39]], m, {}),
                               (g, m[:2] + [m[2].double()], {}), (g, m[:2] + [m[0]], {}), (g, m, dict(weight_decay=[0.0, 0.0, -1.0])),
                               (g, m, dict(skip=step))):
        with pytest.raises((ValueError, _capi.IgError)):
            optim.adamw_step(p, grads, moments, v, step, copies=copies, **kw)
        assert [t._version for t in p + copies] == before
    optim.adamw_step(p, g, m, v, step, copies=copies)
    assert [t._version for t in p + copies] == [k + 1 for k in before]
    optim.adamw_step(p, [g[0], None, g[2]], m, v, step, copies=copies)
    assert [t._version for t in p + copies] == [k + 1 + (i % 3 != 1) for i, k in enumerate(before)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gap", [0, 1, 2])
def test_moments_of_tensors_that_are_left_out(igdev, bits, gap):
    """A tensor without a gradient needs no moments, wherever it stands in the lists."""
    from indecis_b200 import optim
    p, q = ([randn(300, seed=i) for i in range(3)] for _ in range(2))
    g = [randn(300, seed=10 + i) for i in range(3)]
    moments = lambda: [None if i == gap else optim.new_moment(p[i], bits) for i in range(3)]  # noqa: E731
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    optim.adamw_step(p, [None if i == gap else g[i] for i in range(3)], moments(), moments(), step)
    rest = [i for i in range(3) if i != gap]
    full = [optim.new_moment(q[i], bits) for i in rest], [optim.new_moment(q[i], bits) for i in rest]
    optim.adamw_step([q[i] for i in rest], [g[i] for i in rest], *full, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert int(step) == 1 and all(torch.equal(a, b) for a, b in zip(p, q))
    assert all(not torch.equal(p[i], randn(300, seed=i)) for i in rest)


def test_moments_of_one_width(igdev):
    from indecis_b200 import optim
    p = [randn(300, seed=i) for i in range(2)]
    mixed = lambda first: [optim.new_moment(t, b) for t, b in zip(p, (first, 40 - first))]  # noqa: E731
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    for first in (8, 32):
        with pytest.raises(ValueError):
            optim.adamw_step(p, [torch.ones_like(t) for t in p], mixed(first), mixed(first), step)
    assert int(step) == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])  # whole blocks on boundaries of four, and single elements
@pytest.mark.parametrize("lr,decay", [(1e-5, 0.01), (1e-6, 0.01), (3e-6, 0.1)])
def test_small_decay(igdev, bits, offset, lr, decay):
    """The decay takes lr * decay of a parameter in the mean over many, however far that is below a step of float32, beside
    updates that differ from element to element: between runs with and without it the parameters differ by that. p in
    [0.5, 1) is stored to 2^-25 at most off, so is each run's result, evenly spread by the updates: both together leave
    a deviation of 2^-25 * sqrt(2 / 3) / sqrt(n) of the mean, of which six are allowed, and 2^-22 of it for the
    roundings of lr * decay and of the terms."""
    from indecis_b200 import optim
    n = (1 << 20) + offset
    g = torch.Generator(device="cuda").manual_seed(3)
    p = (torch.rand(n, generator=g, device="cuda") * 0.5 + 0.5)[offset:]
    grad, m = (torch.randn(n, generator=g, device="cuda")[offset:] for _ in range(2))
    v = (torch.rand(n, generator=g, device="cuda") + 0.1)[offset:]

    def moved(decay):
        q = torch.empty(n, device="cuda")[offset:].copy_(p)
        step = torch.full((1,), 10, dtype=torch.int32, device="cuda")
        if bits == 32:
            a, b = [torch.empty(n, device="cuda")[offset:].copy_(t) for t in (m, v)]
        else:
            a, b = optim.new_moment(q, 8), optim.new_moment(q, 8)
            for k, t in ((a, m), (b, v.sqrt())):
                k.scales.fill_(4.0 / 448)
                k.codes.copy_((t.clamp(-4, 4) * (448 / 4)).to(torch.float8_e4m3fn))
        optim.adamw_step([q], [grad], [a], [b], step, lr=lr, betas=(0.9, 0.99), weight_decay=decay)
        return q.double()
    want = lr * decay * float(p.double().mean())
    got = float((moved(0.0) - moved(decay)).mean())
    assert abs(got - want) <= 6 * 2.0 ** -25 * math.sqrt(2 / 3 / (1 << 20)) + 2.0 ** -22 * want, (got / want)


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation_of_the_largest_values(igdev, kind):
    """act(a) is a or 0 and act'(a) 1 or 0 for any finite a far from 0, those whose square is past float32 among them."""
    from indecis_b200 import layers
    top = 2.0 ** torch.arange(40, 128, device="cuda", dtype=torch.float64)
    a = torch.cat([top, -top, torch.tensor([torch.finfo(BF16).max, -torch.finfo(BF16).max], device="cuda", dtype=torch.float64)]).to(BF16)
    x = torch.stack([a, torch.ones_like(a)], 1)
    w_in, w_out = torch.eye(2, device="cuda", dtype=BF16), torch.ones(1, 1, device="cuda", dtype=BF16)
    y, saved = layers.gated_ff(x, w_in, w_out, kind, save=True)
    assert torch.equal(y[:, 0], a.clamp(min=0.0))
    dx, _, _ = layers.gated_ff_backward(torch.ones_like(y), x, w_in, w_out, saved, kind, need_in=False, need_out=False)
    assert torch.equal(dx[:, 0], (a > 0).to(BF16))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_through_a_file(igdev, tmp_path, bits):
    """torch.save and torch.load as they come (weights_only), into moments on the GPU again."""
    from indecis_b200 import optim
    a, b = [randn(700, seed=1)], [randn(700, seed=1)]
    one, two = optim.AdamW(a, bits=bits), optim.AdamW(b, bits=bits)
    one.step([randn(700, seed=2)])
    torch.save(one.state_dict(), tmp_path / "state.pt")
    b[0].copy_(a[0])
    two.load_state_dict(torch.load(tmp_path / "state.pt", map_location="cpu"))
    one.step([randn(700, seed=3)])
    two.step([randn(700, seed=3)])
    assert int(two.steps) == 2 and torch.equal(a[0], b[0])
