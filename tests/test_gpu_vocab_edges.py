"""Vocabulary operators where float32 or the inputs leave little room, against plain float64 forms.

Tolerances as in test_gpu_vocab.py (STAT_TOL, P_TOL) and test_gpu_vocab_head.py (LOGIT).
"""
import math

import pytest
import torch

from test_gpu_vocab import DTYPES, EPS, INF, P_TOL, STAT_TOL, TINY, close, make, ref_distill, ref_gradient

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def voc(igdev):
    from indecis_b200 import vocab
    return vocab


# ---- gradients of rows far from zero ---------------------------------------------------------------------------------


def gradient_close(d, x, ids, g, gh, temperature):
    """d against float64, with the tolerances of test_gpu_vocab.test_backward."""
    dtype = x.dtype
    want, p = ref_gradient(x, ids, g, gh, temperature)
    size = g.abs().sum(1, keepdim=True) + gh.abs()[:, None] * 40
    tol = P_TOL * p * size + 2e-6 * g.abs().sum(1, keepdim=True) / temperature * (want.abs() > p) + \
        EPS[dtype] / 2 * want.abs() * 1.01 + TINY[dtype]
    assert d.isfinite().all()
    assert ((d.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,pad,shift", [(12, 37, 0, 0), (12, 5003, 3, 1), (12, 262145, 0, 0), (2400, 2049, 0, 0)])
def test_gradient_of_masked_rows(voc, dtype, rows, V, pad, shift):
    """Rows wholly masked by a finite value are uniform, forward and backward, whatever the value; zero gradients stay
    zero there."""
    x = make(rows, V, dtype, 131 + V, pad, shift)
    values = [v for v in (-1e4, -1e9, -1e10, -1e30, torch.finfo(dtype).min) if abs(v) <= torch.finfo(dtype).max]
    for i, v in enumerate(values):
        x[2 * i] = v
    zero = 2 * len(values)  # the last masked row again, with gradients of zero
    x[zero] = values[-1]
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(-1, V, (rows, 5), generator=gen, device="cuda", dtype=torch.int32)
    ids[:, 4] = ids[:, 0]
    g = torch.randn((rows, 5), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    g[zero] = 0
    gh[zero] = 0
    for temperature in (0.5, 1.0, 5.5, 8.0):
        r = voc.token_logprobs(x, ids, temperature=temperature)
        d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, gh, temperature=temperature)
        gradient_close(d, x, ids, g, gh, temperature)
        assert (d[zero] == 0).all()
        y = x.contiguous().clone()
        voc.token_logprobs_backward(y, ids, r.lse, r.entropy, g, gh, temperature=temperature, out=y)
        gradient_close(y, x, ids, g, gh, temperature)


@pytest.mark.parametrize("rows,V", [(7, 4099), (3, 10007), (5, 27001), (3, 262145), (2400, 1025)])
@pytest.mark.parametrize("offset,temperature", [(-5000.0, 1.0), (20000.0, 1.0), (1e6, 3.0), (0.0, 0.005)])
def test_gradient_far_from_zero(voc, rows, V, offset, temperature):
    """float32 logits at a large offset, or scaled by a low temperature: the gradient does not lose the bits that the
    absolute logsumexp has lost. (x - m) / temperature is up to 64 where it counts, so the temperature's own rounding
    to float32 (2^-24 relative) is inside P_TOL."""
    x = make(rows, V, torch.float32, 141, scale=1.0 if temperature > 0.1 else 0.03) + offset
    if temperature < 0.1:
        x += 10.0
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(-1, V, (rows, 3), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 3), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    r = voc.token_logprobs(x, ids, temperature=temperature)
    d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, gh, temperature=temperature)
    gradient_close(d, x, ids, g, gh, temperature)
    # Rows that are no distribution, beside them.
    x[0] = -INF
    x[1, V // 2] = float("nan")
    x[2, V // 3] = INF
    ids[0, 1] = 5
    r = voc.token_logprobs(x, ids, temperature=temperature)
    y = x.clone()
    voc.token_logprobs_backward(y, ids, r.lse, r.entropy, g, gh, temperature=temperature, out=y)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2].isnan().all()
    if rows > 3:
        assert torch.equal(y[3:], d[3:])


def biased(rows, V, H, dtype, seed, bias):
    """hidden extended by a column of ones, weight by a column of the tokens' biases."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, H, generator=g, device="cuda")
    w = torch.randn(V, H, generator=g, device="cuda") * 0.1
    h[:, H - 1] = 1.0
    w[:, H - 1] = bias
    return h.to(dtype), w.to(dtype)


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, -1e4), (torch.bfloat16, -1e9), (torch.bfloat16, -1e10),
                                        (torch.bfloat16, -1e30), (torch.bfloat16, torch.finfo(torch.bfloat16).min),
                                        (torch.float16, -6e4), (torch.float16, torch.finfo(torch.float16).min)])
@pytest.mark.parametrize("rows", [5, 200])
def test_head_gradient_of_masked_rows(voc, dtype, bias, rows):
    """All tokens masked by a finite bias. Nothing is held of the states beside a bias of -1e9, but every probability is
    at most 1: the gradients are finite and bounded, and zero where the incoming ones are."""
    V, H = 999, 72
    h, w = biased(rows, V, H, dtype, 151, bias)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(0, V, (rows, 2), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 2), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    g[1] = 0
    gh[1] = 0
    for temperature in (0.5, 1.0, 5.5, 8.0):
        r = voc.vocab_logprobs(h, w, ids, temperature=temperature)
        dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh, temperature=temperature)
        dh, dw = dh[:, :H - 1], dw[:, :H - 1]  # the constant's own gradient is of the bias's size
        assert dh.isfinite().all() and dw.isfinite().all()
        assert (dh[1] == 0).all()
        size = (2 * g.abs().sum(1) + gh.abs() * (1 + math.log(V) + 1)) / temperature
        assert (dh.float().abs() <= 1.01 * size[:, None] * w[:, :H - 1].float().abs().sum(0)).all()
        assert (dw.float().abs() <= 1.01 * (size[:, None] * h[:, :H - 1].float().abs()).sum(0)).all()
        if r.lse.abs().max() < 1e5:
            # The distribution is still there: p is off by lse's rounding (|lse| 2^-24) and the logits' (LOGIT of |bias|).
            z = h.double() @ w.double().T / temperature
            logp = torch.log_softmax(z, 1)
            G = -g.double().sum(1, keepdim=True) * logp.exp()
            ent = -(logp.exp() * logp).sum(1, keepdim=True)
            G -= gh.double()[:, None] * logp.exp() * (logp + ent)
            G.scatter_add_(1, ids.long(), g.double())
            G /= temperature
            off = 2 * (float(r.lse.abs().max()) * 2.0**-24 + abs(bias) * 2.0**-20 / temperature)
            slack = (g.abs().sum(1) + gh.abs() * (1 + 2 * math.log(V)))[:, None].double() * logp.exp() / temperature
            err = slack * (P_TOL + math.expm1(off)) + torch.finfo(dtype).eps * G.abs() + 1e-7
            tol = err @ w[:, :H - 1].double().abs()
            want = G @ w[:, :H - 1].double()
            assert ((dh.double() - want).abs() <= tol + torch.finfo(dtype).eps * want.abs() + 1e-7).all()


# ---- entries that are not given --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("value", [1e6, 1e30, INF, -INF, math.nan])
def test_gradients_of_entries_not_given(voc, dtype, rows, value):
    """Whatever the gradient of an entry that is not given (padded, or past the vocabulary), it changes no bit, the
    scale of a float16 gradient included."""
    from indecis_b200 import ops
    V, H = 1003, 72
    gen = torch.Generator(device="cuda").manual_seed(17)
    h = torch.randn(rows, H, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(V, H, generator=gen, device="cuda") * 0.1).to(dtype)
    ids = torch.randint(0, V, (rows, 4), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 4), generator=gen, device="cuda") / rows
    ids[3, 1] = -1
    ids[7] = -5
    ids[11, 3] = V
    g[3] *= 100  # the row whose gradient sets the scale has an entry that is not given
    gone = (ids < 0) | (ids >= V)
    r = voc.vocab_logprobs(h, w, ids)
    x = (h.float() @ w.float().T).to(dtype)
    s = voc.token_logprobs(x, ids)
    want = got = None
    for v in (0.0, value):
        gv = torch.where(gone, torch.full_like(g, v), g)
        want, got = got, voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, gv) + (
            voc.token_logprobs_backward(x, ids, s.lse, s.entropy, gv),)
    assert ops.device_error() == 5
    for a, b in zip(got, want):
        assert b.isfinite().all() and (b != 0).any()
        assert torch.equal(a, b)


# ---- alternatives ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(2, 300), (3, 16384), (1, 70001), (9600, 257), (2400, 2049)])
def test_top_ties_of_signed_zeros(voc, dtype, rows, V):
    """-0 and +0 are the same value: the lowest column first."""
    gen = torch.Generator(device="cuda").manual_seed(23)
    none = torch.empty((rows, 0), dtype=torch.int32, device="cuda")
    x = torch.full((rows, V), -1.0, device="cuda", dtype=dtype)
    x[:, 0] = -0.0
    x[:, 100] = 0.0
    x[:, 200] = -0.0
    assert voc.token_logprobs(x, none, top_k=1).top_ids[:, 0].tolist() == [0] * rows
    assert voc.token_logprobs(x, none, top_k=3).top_ids.tolist() == [[0, 100, 200]] * rows
    pick = torch.randint(0, 40, (rows, V), generator=gen, device="cuda")
    x = torch.where(pick == 0, 0.0, torch.where(pick == 1, -0.0, -pick.float())).to(dtype)
    for k in (1, 5, 32):
        want = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(voc.token_logprobs(x, none, top_k=k).top_ids.long(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("left", [[], [5], [19], [0, 17, 18], [3, 40, 41, 42, 43, 44, 45, 999], list(range(16))])
def test_head_alternatives_of_masked_columns(voc, dtype, rows, left):
    """Tokens masked by a bias of -inf are no alternatives: past the unmasked ones, -1 and -inf."""
    V, H, K = 1000, 72, 8
    bias = torch.full((V,), -INF)
    bias[left] = 0.0
    h, w = biased(rows, V, H, dtype, 171, bias.cuda())
    h, w = h.contiguous(), w.contiguous()
    ids = torch.tensor([[5, 700]] * rows, dtype=torch.int32, device="cuda")
    for _ in range(2):
        junk = torch.full((1 << 16,), 7, dtype=torch.int32, device="cuda")  # what a forgotten output would show
        del junk
        r = voc.vocab_logprobs(h, w, ids, top_k=K)
        n = min(K, len(left))
        if not left:
            assert (r.lse == -INF).all() and (r.entropy == 0).all() and (r.logprobs == -INF).all()
        else:
            keep = torch.tensor(left, device="cuda")
            logp = torch.log_softmax(h.double()[:, :H - 1] @ w.double()[keep][:, :H - 1].T, 1)
            v, at = torch.sort(logp, dim=1, descending=True, stable=True)
            assert torch.equal(r.top_ids[:, :n].long(), keep[at[:, :n]])
            close(r.top_logprobs[:, :n], v[:, :n], STAT_TOL + 1e-4)
            assert (r.logprobs[:, 1] == -INF).all()
        assert (r.top_ids[:, n:] == -1).all() and (r.top_logprobs[:, n:] == -INF).all()


# ---- distillation ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,V", [(torch.float32, 1 << 20), (torch.float32, 300001), (torch.bfloat16, 1 << 20)])
def test_tail_loss_of_many_long_rows(voc, dtype, V):
    """The tail's loss without a gradient: rows enough that each would have one CTA, columns enough that their marks
    do not fit into one CTA's shared memory."""
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count
    gen = torch.Generator(device="cuda").manual_seed(29)
    x = torch.empty((rows, V), dtype=dtype, device="cuda")
    x.normal_(generator=gen)
    ids = torch.randint(0, V, (rows, 40), generator=gen, device="cuda", dtype=torch.int32)
    ids[3, 30:] = -1
    ids[4] = -1
    t = torch.log_softmax(torch.randn((rows, 41), generator=gen, device="cuda"), 1)[:, :40].contiguous()
    loss, none = voc.distill_topk(x, ids, t, tail=True, grad=False)
    assert none is None
    for n in (0, 3, 4, rows - 1):
        logp = torch.log_softmax(x[n].double(), 0)
        at, first = {}, {}
        for k, i in enumerate(ids[n].tolist()):
            if i >= 0:
                at.setdefault(i, []).append(float(t[n, k]))
        if not at:
            assert loss[n] == 0
            continue
        lp = logp[torch.tensor(list(at), device="cuda")].tolist()
        want = sum(math.exp(v) * (v - l) for l, vs in zip(lp, at.values()) for v in vs)
        rest = 1 - sum(math.exp(v) for vs in at.values() for v in vs)
        want += rest * (math.log(rest) - math.log1p(-sum(math.exp(l) for l in lp)))
        assert abs(float(loss[n]) - want) <= 4 * 7e-5 * (1 + abs(want))
    more, _ = voc.distill_topk(x, ids, t, tail=True, out=x)
    close(more, loss.double(), 4 * 7e-5)


# ---- where the gradient may go -----------------------------------------------------------------------------------------


def test_gradient_between_the_logits_rows(voc):
    """Rows of the output between those of the logits share nothing with them; an output that does is refused."""
    from indecis_b200 import _capi
    V = 1003
    buf = torch.empty((70, 2 * V + 5), device="cuda")
    x, out = buf[:, :V], buf[:, V + 2:2 * V + 2]
    x.copy_(make(70, V, torch.float32, 181))
    ids = torch.arange(70, dtype=torch.int32, device="cuda")[:, None].contiguous()
    r = voc.token_logprobs(x, ids)
    g = torch.ones_like(r.logprobs)
    want = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g)
    assert torch.equal(voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, out=out), want)
    t = torch.zeros((70, 1), device="cuda")
    want = voc.distill_topk(x, ids, t)[1]
    assert torch.equal(voc.distill_topk(x, ids, t, out=out)[1], want)
    for bad in (buf[:, 1:V + 1], buf[:, V - 1:2 * V - 1]):
        for call in (lambda: voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, out=bad),
                     lambda: voc.distill_topk(x, ids, t, out=bad)):
            with pytest.raises(_capi.IgError) as e:
                call()
            assert e.value.code == _capi.IG_ERR_BAD_ARG


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [7, 300])
def test_head_gradient_with_masked_columns(voc, dtype, rows):
    """Tokens masked by a bias of -inf, given ones among them: no probability, no gradient but a given token's own. (The
    bias column's own entry of dhidden is 0 times infinity.) Tolerances as in test_gpu_vocab_head.check_backward."""
    V, H = 1500, 72
    bias = torch.zeros(V)
    bias[::3] = -INF
    h, w = biased(rows, V, H, dtype, 191, bias.cuda())
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(0, V, (rows, 3), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 3), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    r = voc.vocab_logprobs(h, w, ids)
    assert ((r.logprobs == -INF) == (ids % 3 == 0)).all()
    dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh)
    hd, wd = h.double()[:, :H - 1], w.double()[:, :H - 1]
    z = hd @ wd.T + bias.cuda().double()
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    ent = torch.special.entr(p).sum(1, keepdim=True)
    G = -g.double().sum(1, keepdim=True) * p
    G -= gh.double()[:, None] * torch.where(p > 0, p * (logp + ent), torch.zeros_like(p))
    G.scatter_add_(1, ids.long(), g.double())
    slack = (g.double().abs().sum(1, keepdim=True) + gh.double().abs()[:, None] * 40) * p
    off = 2 * 2.0**-20 * float((hd.abs() @ wd.abs().T).max())
    u = torch.finfo(dtype).eps / 2
    floor = float((2 * g.abs().sum(1) + gh.abs() * 10).max()) * 2.0**-39 if dtype == torch.float16 else 0.0
    err = u * 1.01 * G.abs() + slack * (P_TOL + off) + floor
    tiny = 3e-8 if dtype == torch.float16 else 0.0
    want = G @ wd
    tol = err @ wd.abs() + 2.0**-20 * (G.abs() @ wd.abs()) + u * 1.01 * want.abs() + tiny
    assert ((dh[:, :H - 1].double() - want).abs() <= tol).all()
    want = G.T @ h.double()
    tol = err.T @ h.double().abs() + 2.0**-20 * (G.abs().T @ h.double().abs()) + u * 1.01 * want.abs() + tiny
    assert ((dw.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V", [(8, 37), (8, 70001), (2400, 2049)])
def test_distill_of_masked_rows(voc, dtype, tail, rows, V):
    """Rows wholly masked by a finite value are uniform."""
    x = make(rows, V, dtype, 201 + V)
    values = [v for v in (-1e4, -1e9, -1e30, torch.finfo(dtype).min) if abs(v) <= torch.finfo(dtype).max]
    for i, v in enumerate(values):
        x[2 * i] = v
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.rand((rows, V), generator=gen, device="cuda").topk(6, dim=1).indices.int().contiguous()
    t = torch.log_softmax(torch.randn((rows, 7), generator=gen, device="cuda"), 1)[:, :6].contiguous()
    for temperature in (0.5, 1.0, 8.0):
        loss, d = voc.distill_topk(x, ids, t, temperature=temperature, tail=tail)
        wl, wd, p, q = ref_distill(x, ids, t, temperature, tail, None)
        close(loss, wl, 4 * STAT_TOL, "loss")
        tol = (P_TOL * wd.abs() + 1e-6 * p + 4e-7) / min(temperature, 1.0) + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
        if tail:
            listed = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids.long(), True)
            mass = torch.where(listed, torch.zeros_like(p), p).sum(1).clamp(min=1e-300)
            tol = tol + (p * ((P_TOL * (1 - q.sum(1)).clamp(min=0) + 5e-7) / mass)[:, None]).clamp(max=1.0) / temperature
        assert ((d.double() - wd).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [0, 3])
def test_lse_says_whether_a_row_is_empty(voc, dtype, top):
    """-inf for a row with nothing left alone, also where the product with 1 / temperature leaves float32."""
    x = make(4, 3001, dtype, 211)
    x[0] = -INF
    x[1] = torch.finfo(dtype).min
    x[2] = -INF
    x[2, 7] = torch.finfo(dtype).min
    ids = torch.tensor([[7, 8]] * 4, dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, ids, temperature=0.5, top_k=top)
    assert r.lse[0] == -INF and r.lse[1:].isfinite().all()
    assert r.logprobs[0].tolist() == [-INF, -INF] and r.logprobs[2].tolist() == [0.0, -INF]
    g = torch.tensor([[1.0, 0.5]] * 4, device="cuda")
    d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, temperature=0.5)
    assert (d[0] == 0).all()
    want = torch.full((3001,), -3.0 / 3001, device="cuda", dtype=torch.float64)
    want[7] += 2.0
    want[8] += 1.0
    assert ((d[1].double() - want).abs() <= 4 * P_TOL / 3001 + EPS[dtype] * want.abs()).all()
    want = torch.zeros(3001, device="cuda", dtype=torch.float64)
    want[7], want[8] = -1.0, 1.0  # all of p in column 7: (1 - 1.5) / 0.5; the other given one has none
    assert ((d[2].double() - want).abs() <= 1e-6 + EPS[dtype] * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V,H,T", [(1, 2985, 1024, 1), (40, 2985, 1024, 4), (300, 2985, 1000, 8), (300, 70001, 768, 2),
                                        (129, 257, 520, 3)])
def test_head_log_probability_of_a_likely_token(voc, dtype, rows, V, H, T):
    """A token that takes nearly all of its row: its log probability is what the other columns leave, off by their own
    relative errors (LOGIT of sum |h w| in every logit, P_TOL) and by the roundings of a sum near 1 (2^-24 each, (terms
    per thread + 20) of them, at most 64), not by the difference of two ways to sum its logit."""
    gen = torch.Generator(device="cuda").manual_seed(221)
    w = (torch.randn(V, H, generator=gen, device="cuda") * 0.05).to(dtype)
    ids = torch.randint(0, V, (rows, T), generator=gen, device="cuda", dtype=torch.int32)
    h = torch.randn(rows, H, generator=gen, device="cuda")
    h = (h + 8.0 * w[ids[:, T - 1].long()].float()).to(dtype)
    z = (h.double() @ w.double().T) / 0.7
    off = float((h.double().abs() @ w.double().abs().T).max()) * 2.0**-20 / 0.7
    want = torch.log_softmax(z, 1).gather(1, ids.long())
    r = voc.vocab_logprobs(h, w, ids, temperature=0.7, top_k=3)
    likely = want[:, T - 1]
    assert likely.max() > -1e-2 and likely.min() > -8
    for got, lp in ((r.logprobs[:, T - 1], likely), (r.top_logprobs[:, 0], torch.log_softmax(z, 1).max(1).values)):
        assert ((got.double() - lp).abs() <= lp.abs() * (2 * off + P_TOL) + 2.0**-18).all()
    assert ((r.logprobs.double() - want).abs() <= (STAT_TOL + 2 * off) * (1 + want.abs())).all()
    # More tokens than are taken from the accumulators: the same up to the logits' error.
    many = torch.cat([ids, torch.randint(0, V, (rows, 9), generator=gen, device="cuda", dtype=torch.int32)], 1).contiguous()
    s = voc.vocab_logprobs(h, w, many, temperature=0.7, top_k=3)
    assert ((s.logprobs[:, :T] - r.logprobs).abs() <= 2 * off).all() and torch.equal(s.lse, r.lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,K", [(3, 40, 7), (6, 20011, 100), (2400, 2049, 33)])
def test_tail_of_a_list_that_holds_everything(voc, dtype, rows, V, K):
    """The teacher's list and the student's unmasked columns are the same: what float32 leaves of 1 does not count against
    columns masked by a finite value, however deep (the lowest value, -1e4)."""
    gen = torch.Generator(device="cuda").manual_seed(231)
    ids = torch.rand((rows, V), generator=gen, device="cuda").topk(K, dim=1).indices.int().contiguous()
    y = torch.randn((rows, K), generator=gen, device="cuda") * 2
    t = torch.log_softmax(torch.randn((rows, K), generator=gen, device="cuda").double() * 2, 1).float().contiguous()
    for mask in (-1e4, torch.finfo(dtype).min):
        x = torch.full((rows, V), mask, device="cuda").scatter_(1, ids.long(), y).to(dtype)
        for temperature in (0.3, 1.0):
            loss, d = voc.distill_topk(x, ids, t, temperature=temperature, tail=True)
            z = x.double() / temperature
            logp = torch.log_softmax(z, 1)
            q = t.double().exp()
            wl = (q * (t.double() - logp.gather(1, ids.long()))).sum(1)
            wd = (logp.exp() * q.sum(1, keepdim=True)).scatter_add_(1, ids.long(), -q) / temperature
            close(loss, wl, 4 * STAT_TOL, "loss")
            tol = (P_TOL * logp.exp() + P_TOL * wd.abs() + 1e-6) / temperature + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
            assert ((d.double() - wd).abs() <= tol).all()
