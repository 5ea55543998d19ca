"""Vocabulary operators on stored logits against plain float64 forms.

Tolerances, from the kernels' arithmetic. Statistics: (x - m) c log2 e takes two roundings of a value of magnitude
|y| <= 64 for terms that count (2^-64 adds nothing), so each term is off by at most 2 * 2^-24 * 64 * ln 2 = 5.3e-6
relative, ex2 by 2^-22, and a sum of up to 2^18 terms in threads, warps and parts by (terms per thread + 20) 2^-24
relative: under 7e-5 for the longest rows and 1.5e-5 for the rest, in practice far less because the roundings are
independent; logsumexp, log probabilities and entropies inherit that as absolute errors, plus one rounding of their own
size. Gradients: p carries the same relative error, then one rounding to the output type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = {dt: torch.finfo(dt).eps for dt in DTYPES}  # spacing at 1; a rounding is off by half of it
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 6e-8}  # half the smallest step, and more
STAT_TOL = 2e-5
P_TOL = 2e-5
INF = math.inf


@pytest.fixture(scope="module")
def voc(igdev):
    from indecis_b200 import vocab
    return vocab


def make(rows, V, dtype, seed, pad=0, shift=0, scale=3.0):
    """[rows, V] logits in a buffer with row stride V + pad, starting `shift` elements into it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((shift + rows * (V + pad) + 8,), float("nan"), dtype=dtype, device="cuda")
    x = buf[shift:shift + rows * (V + pad)].view(rows, V + pad)[:, :V]
    x.copy_((torch.randn(rows, V, generator=g, device="cuda") * scale).to(dtype))
    return x


def ref_forward(x, ids, temperature):
    z = x.double() / temperature
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    lp = torch.where(ids >= 0, logp.gather(1, ids.clamp(min=0).long()), torch.zeros((), dtype=torch.float64, device=x.device))
    return lp, lse, ent, logp


def close(got, want, tol, what=""):
    got, want = got.double(), want.float().double()  # a value past float32's range is its infinity
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol * (1 + want.abs()))
    assert not bad.any(), (what, got[bad][:5], want[bad][:5])


def ref_top(x, k):
    """Columns by (value descending, column ascending)."""
    v, i = torch.sort(x.float(), dim=1, descending=True, stable=True)
    return i[:, :k], v[:, :k]


SHAPES = [(1, 1, 0, 0), (3, 7, 0, 0), (2, 33, 3, 1), (5, 1000, 0, 0), (3, 4099, 0, 3), (2, 16384, 8, 0),
          (1, 50021, 0, 5), (64, 50021, 0, 0), (700, 2049, 1, 1), (1, 262144, 0, 0), (40, 262145, 7, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,pad,shift", SHAPES)
def test_forward(voc, dtype, rows, V, pad, shift):
    x = make(rows, V, dtype, 11 + V, pad, shift)
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(-1, V, (rows, 5), generator=g, device="cuda", dtype=torch.int32)
    for temperature, top in ((1.0, 0), (0.7, 1), (2.0, min(32, V))):
        r = voc.token_logprobs(x, ids, temperature=temperature, top_k=top)
        lp, lse, ent, logp = ref_forward(x, ids, temperature)
        close(r.lse, lse, STAT_TOL, "lse")
        close(r.logprobs, lp, STAT_TOL, "logprobs")
        close(r.entropy, ent, STAT_TOL, "entropy")
        assert (r.logprobs <= 0).all()
        if top:
            i, _ = ref_top(x, top)
            assert torch.equal(r.top_ids.long(), i)
            close(r.top_logprobs, logp.gather(1, i), STAT_TOL, "top")
        else:
            assert r.top_ids is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,pad", [(9600, 257, 0), (5000, 1023, 1), (2500, 2049, 0), (2400, 9001, 3)])
def test_many_short_rows(voc, dtype, rows, V, pad):
    """Enough rows for the CTAs of 32, 64 and 128 threads; more given tokens and teacher entries than threads."""
    x = make(rows, V, dtype, 45 + V, pad)
    g = torch.Generator(device="cuda").manual_seed(9)
    T = 70
    ids = torch.randint(-1, V, (rows, T), generator=g, device="cuda", dtype=torch.int32)
    x[5] = 2.0  # all columns equal
    r = voc.token_logprobs(x, ids, temperature=0.7, top_k=32)
    lp, lse, ent, logp = ref_forward(x, ids, 0.7)
    close(r.lse, lse, STAT_TOL, "lse")
    close(r.logprobs, lp, STAT_TOL, "logprobs")
    close(r.entropy, ent, STAT_TOL, "entropy")
    i, _ = ref_top(x, 32)
    assert torch.equal(r.top_ids.long(), i)
    close(r.top_logprobs, logp.gather(1, i), STAT_TOL, "top")
    del lp, logp
    gl = torch.randn((rows, T), generator=g, device="cuda") / T
    gh = torch.randn((rows,), generator=g, device="cuda")
    d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, gl, gh, temperature=0.7)
    want, p = ref_gradient(x, ids, gl, gh, 0.7)
    size = gl.abs().sum(1, keepdim=True) + gh.abs()[:, None] * 40
    tol = P_TOL * p * size + 2e-6 * gl.abs().sum(1, keepdim=True) / 0.7 * (want.abs() > p) + \
        EPS[dtype] / 2 * want.abs() * 1.01 + TINY[dtype]
    # Sums of up to T gradients in one column, in float32.
    tol = tol + T * 2.0**-24 * gl.abs().amax(1, keepdim=True) / 0.7
    assert ((d.double() - want).abs() <= tol).all()
    for tail in (False, True):
        tids, t = teacher(x, 100, tail, 7)
        tids[3, 5] = -1
        tids[4] = -1
        loss, d = voc.distill_topk(x, tids, t, temperature=0.7, tail=tail)
        wl, wd, p, q = ref_distill(x, tids, t, 0.7, tail, None)
        close(loss, wl, 4 * STAT_TOL, "loss")
        listed = torch.zeros_like(p, dtype=torch.bool).scatter_(1, tids.clamp(min=0).long(), tids >= 0)
        mass = torch.where(listed, torch.zeros_like(p), p).sum(1).clamp(min=1e-300)
        tol = (P_TOL * wd.abs() + 1e-6 * p / 0.7 + 4e-7) + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
        if tail:
            tol = tol + (p * ((P_TOL * (1 - q.sum(1)).clamp(min=0) + 5e-7) / mass)[:, None]).clamp(max=1.0) / 0.7
        assert ((d.double() - wd).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,rows", [(70, 2), (5000, 3), (70001, 1), (70001, 900)])
def test_top_ties(voc, dtype, V, rows):
    """Few distinct values, constant rows: ties go to the lowest column."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(0, 3, (rows, V), generator=g, device="cuda").to(dtype)
    x[0] = 1.5
    ids = torch.zeros((rows, 0), dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, ids, top_k=32)
    assert torch.equal(r.top_ids.long(), ref_top(x, 32)[0])
    # An increasing row makes every chunk the new best; a decreasing one only the first.
    up = (torch.arange(V, device="cuda").float() / V).to(dtype)
    for row in (up, up.flip(0)):
        r = voc.token_logprobs(row[None].contiguous(), ids[:1], top_k=32)
        assert torch.equal(r.top_ids.long(), ref_top(row[None], 32)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 3001, 60000])
def test_masks(voc, dtype, V):
    """Columns at -inf, rows with one or no column left, masks of the type's lowest value, NaN and +inf rows."""
    x = make(9, V, dtype, 21)
    low = torch.finfo(dtype).min
    x[1] = -INF
    x[2] = -INF
    x[2, V - 1] = 1.25
    x[3, : V - 2] = -INF
    x[4, 1:] = low
    x[5] = low
    x[6, V // 2] = float("nan")
    x[7, V // 3] = INF
    x[8, 0] = -INF
    ids = torch.tensor([[0, V - 1, -1]] * 9, dtype=torch.int32, device="cuda")
    top = 4
    for temperature in (1.0, 0.5):
        r = voc.token_logprobs(x, ids, temperature=temperature, top_k=top)
        ok = torch.tensor([0, 2, 3, 4, 8], device="cuda")
        lp, lse, ent, logp = ref_forward(x[ok], ids[ok], temperature)
        close(r.logprobs[ok], lp, STAT_TOL, "logprobs")
        close(r.lse[ok], lse, STAT_TOL, "lse")
        close(r.entropy[ok], ent, STAT_TOL, "entropy")
        i, v = ref_top(x[ok], top)
        i = torch.where(v == -INF, torch.full_like(i, -1), i)
        assert torch.equal(r.top_ids[ok].long(), i)
        # Nothing left.
        assert (r.lse[1] == -INF) and (r.entropy[1] == 0)
        assert r.logprobs[1].tolist() == [-INF, -INF, 0.0]
        assert r.top_ids[1].tolist() == [-1] * top and (r.top_logprobs[1] == -INF).all()
        assert r.top_ids[2].tolist() == [V - 1, -1, -1, -1]
        # All at the lowest value: uniform.
        close(r.logprobs[5, :2], torch.full((2,), -math.log(V), device="cuda"), STAT_TOL)
        close(r.entropy[5], torch.tensor(math.log(V), device="cuda"), STAT_TOL)
        # Not a distribution.
        for n in (6, 7):
            assert r.lse[n].isnan() and r.entropy[n].isnan() and r.logprobs[n, :2].isnan().all()
            assert r.logprobs[n, 2] == 0 and r.top_ids[n].tolist() == [-1] * top and r.top_logprobs[n].isnan().all()
        d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, torch.ones((9, 3), device="cuda"),
                                        torch.ones(9, device="cuda"), temperature=temperature)
        assert (d[1] == 0).all() and d[6].isnan().all() and d[7].isnan().all()
        assert d[ok].isfinite().all()
        assert (d[8, 1:] != 0).any() and (d[3, 1:V - 2] == 0).all()


def ref_gradient(x, ids, g, gh, temperature):
    z = (x.double() / temperature)
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    ent = -(p * logp).sum(1, keepdim=True)
    live = g.double() * (ids >= 0)
    d = -live.sum(1, keepdim=True) * p
    if gh is not None:
        d -= gh.double()[:, None] * p * (logp + ent)
    d.scatter_add_(1, ids.clamp(min=0).long(), live)
    return d / temperature, p / temperature


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,pad,shift", SHAPES)
def test_backward(voc, dtype, rows, V, pad, shift):
    x = make(rows, V, dtype, 31 + V, pad, shift)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(-1, V, (rows, 6), generator=gen, device="cuda", dtype=torch.int32)
    ids[:, 5] = ids[:, 0]  # a repeated token
    g = torch.randn((rows, 6), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    for temperature, h in ((1.0, None), (1.7, gh)):
        r = voc.token_logprobs(x, ids, temperature=temperature)
        d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, h, temperature=temperature)
        assert d.dtype == dtype
        want, p = ref_gradient(x, ids, g, h, temperature)
        # p's error against the sizes it is multiplied by (sum of gradients, |gH| (|log p| + H) <= |gH| 40), one rounding.
        size = g.abs().sum(1, keepdim=True) + (0 if h is None else h.abs()[:, None] * 40)
        tol = P_TOL * p * size + 2e-6 * g.abs().sum(1, keepdim=True) / temperature * (want.abs() > p) + \
            EPS[dtype] / 2 * want.abs() * 1.01 + TINY[dtype]
        assert ((d.double() - want).abs() <= tol).all()
        # Into a buffer with another alignment, and in place.
        buf = torch.empty(rows * (V + 3) + 1, dtype=dtype, device="cuda")
        out = buf[1:].view(rows, V + 3)[:, :V]
        voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, h, temperature=temperature, out=out)
        assert torch.equal(out, d)
        y = x.contiguous().clone()
        voc.token_logprobs_backward(y, ids, r.lse, r.entropy, g, h, temperature=temperature, out=y)
        assert torch.equal(y, d)


def test_backward_differences(voc):
    """Central differences of the forward in float32: h = 2^-5 leaves h^2/6 |f'''| <= 2^-10/6 and 2 * 1e-6 / (2 h) of
    the forward's rounding."""
    x = make(3, 61, torch.float32, 41, scale=1.0)
    ids = torch.tensor([[4, 60, 4], [0, -1, 7], [1, 2, 3]], dtype=torch.int32, device="cuda")
    g = torch.tensor([[0.5, -1.0, 0.25], [1.0, 9.0, -0.5], [0.3, 0.2, 0.1]], device="cuda")
    gh = torch.tensor([0.7, -0.4, 0.0], device="cuda")

    def loss(y):
        r = voc.token_logprobs(y, ids, temperature=1.3)
        return ((r.logprobs.double() * g * (ids >= 0)).sum(1) + r.entropy.double() * gh)

    r = voc.token_logprobs(x, ids, temperature=1.3)
    d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, g, gh, temperature=1.3)
    h = 2.0**-5
    for j in range(61):
        e = torch.zeros_like(x)
        e[:, j] = h
        num = (loss(x + e) - loss(x - e)) / (2 * h)
        assert ((num - d[:, j].double()).abs() <= 1e-3).all()


# ---- distillation ------------------------------------------------------------------------------------------------


def ref_distill(x, tids, t, temperature, tail, w):
    z = x.double() / temperature
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    there = tids >= 0
    at = tids.clamp(min=0).long()
    t = torch.where(there, t.double(), torch.full_like(t.double(), -INF))
    some = there.any(1)
    q = t.exp() if tail else torch.softmax(t / temperature, 1).nan_to_num(0.0)
    lq = torch.where(q > 0, q, torch.ones_like(q)).log()
    loss = torch.where(q > 0, q * (lq - logp.gather(1, at)), torch.zeros_like(q)).sum(1)
    listed = torch.zeros_like(p).scatter_add_(1, at, there.double()) > 0
    d = p * q.sum(1, keepdim=True) - torch.zeros_like(p).scatter_add_(1, at, q)
    if tail:
        rest = (1 - q.sum(1)).clamp(min=0)
        out = torch.where(listed, torch.zeros_like(p), p)
        mass = out.sum(1)
        has = (mass > 0) & (rest > 0)
        safe = torch.where(has, mass, torch.ones_like(mass))
        loss = loss + torch.where(has, rest * ((rest.clamp(min=1e-300)).log() - safe.log()), torch.zeros_like(rest))
        d = d + torch.where(has[:, None], p * rest[:, None] - out * (rest / safe)[:, None], torch.zeros_like(p))
    d = torch.where(some[:, None], d, torch.zeros_like(d))
    w = torch.ones_like(loss) if w is None else w.double()
    return torch.where(some, loss, torch.zeros_like(loss)) * w, d * (w[:, None] / temperature), p, q


def teacher(x, K, tail, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = x.float() + torch.randn(x.shape, generator=g, device="cuda")
    v, i = y.topk(min(K, x.shape[1]), dim=1)
    if tail:
        v = torch.log_softmax(y, 1).gather(1, i)
    return i.int().contiguous(), v.contiguous()


DSHAPES = [(1, 1, 1, 0, 0), (3, 9, 9, 0, 0), (4, 50, 7, 3, 1), (5, 1000, 64, 0, 0), (3, 4099, 200, 0, 3),
           (2, 16384, 8, 8, 0), (64, 50021, 32, 0, 0), (700, 2049, 5, 1, 1), (1, 262144, 256, 0, 0), (9, 262145, 64, 7, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V,K,pad,shift", DSHAPES)
def test_distill(voc, dtype, tail, rows, V, K, pad, shift):
    x = make(rows, V, dtype, 51 + V, pad, shift, scale=2.0)
    ids, t = teacher(x, K, tail, 7)
    if rows > 2 and K > 2:
        ids[1, 1] = -1
        ids[2] = -1
    w = torch.linspace(0.5, 2.0, rows, device="cuda")
    for temperature, weights in ((1.0, None), (2.0, w)):
        loss, d = voc.distill_topk(x, ids, t, temperature=temperature, tail=tail, weights=weights)
        wl, wd, p, q = ref_distill(x, ids, t, temperature, tail, weights)
        # The loss is a sum of terms of size q |log q - log p|, each off by STAT_TOL (1 + size).
        close(loss, wl, 4 * STAT_TOL, "loss")
        wmax = 1.0 if weights is None else 2.0
        # rest / mass multiplies p outside the list: its error is q_rest's (2e-7 absolute) and mass's (P_TOL relative).
        ratio = ((1 - q.sum(1)).clamp(min=0) / (wd.new_ones(()) * 1)).max() if tail else 0.0
        tol = (P_TOL * wd.abs() + 1e-6 * p + 4e-7) * wmax + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
        if tail:
            listed = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids.clamp(min=0).long(), ids >= 0)
            mass = torch.where(listed, torch.zeros_like(p), p).sum(1).clamp(min=1e-300)
            tol = tol + (p * ((P_TOL * (1 - q.sum(1)).clamp(min=0) + 5e-7) / mass)[:, None]).clamp(max=1.0) * wmax
        assert ((d.double() - wd).abs() <= tol).all()
        loss2, none = voc.distill_topk(x, ids, t, temperature=temperature, tail=tail, weights=weights, grad=False)
        assert none is None and torch.equal(loss2, loss)
        buf = torch.empty(rows * (V + 3) + 1, dtype=dtype, device="cuda")
        out = buf[1:].view(rows, V + 3)[:, :V]
        voc.distill_topk(x, ids, t, temperature=temperature, tail=tail, weights=weights, out=out)
        assert torch.equal(out, d)
        # In place; a copy has another alignment, so another order of summation than x.
        y = x.contiguous().clone()
        _, want = voc.distill_topk(y, ids, t, temperature=temperature, tail=tail, weights=weights)
        voc.distill_topk(y, ids, t, temperature=temperature, tail=tail, weights=weights, out=y)
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_edges(voc, dtype, tail):
    V = 3003
    x = make(8, V, dtype, 61)
    low = torch.finfo(dtype).min
    ids = torch.arange(6, dtype=torch.int32, device="cuda").repeat(8, 1).contiguous()
    t = torch.full((8, 6), math.log(0.125), device="cuda")
    x[1, 6:] = -INF       # nothing outside the list
    x[2, 3] = -INF        # a listed column is masked
    x[3] = -INF           # no distribution
    x[4, 100] = float("nan")
    x[5, 6:] = low        # masked by the lowest value
    ids[6, 4] = ids[6, 1]  # a repeated entry
    w = torch.ones(8, device="cuda")
    w[7] = 0
    x[7, 9] = INF
    loss, d = voc.distill_topk(x, ids, t, tail=tail, weights=w)
    ok = torch.tensor([0, 1, 6], device="cuda")
    wl, wd, p, q = ref_distill(x[ok], ids[ok], t[ok], 1.0, tail, None)
    close(loss[ok], wl, 4 * STAT_TOL)
    tol = 4 * P_TOL * (wd.abs() + p) + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
    assert ((d[ok].double() - wd).abs() <= tol).all()
    assert loss[2] == INF and d[2].isfinite().all()
    assert loss[3] == INF and (d[3] == 0).all()
    assert loss[4].isnan() and d[4].isnan().all()
    assert not loss[5].isnan() and d[5].isfinite().all()
    assert loss[7] == 0 and (d[7] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [50, 20000])
def test_distill_special(voc, dtype, tail, V):
    """NaN and +inf, in a listed column and outside; a teacher of -inf only; entries at and past the row's ends."""
    x = make(7, V, dtype, 63)
    ids = torch.tensor([[0, 3, V - 1, V - 2]] * 7, dtype=torch.int32, device="cuda")
    t = torch.tensor([[-1.0, -2.0, -3.0, -4.0]] * 7, device="cuda")
    x[1, 3] = INF
    x[2, 7] = INF
    x[3, 0] = float("nan")
    t[4] = -INF
    t[5, 2] = -INF
    ids[6] = -1
    loss, d = voc.distill_topk(x, ids, t, tail=tail)
    for n in (1, 2, 3):
        assert loss[n].isnan() and d[n].isnan().all()
    ok = torch.tensor([0, 5, 6], device="cuda")
    wl, wd, p, q = ref_distill(x[ok], ids[ok], t[ok], 1.0, tail, None)
    close(loss[ok], wl, 4 * STAT_TOL)
    tol = 4 * P_TOL * (wd.abs() + p) + EPS[dtype] / 2 * wd.abs() * 1.01 + TINY[dtype]
    assert ((d[ok].double() - wd).abs() <= tol).all()
    # No mass in the list: nothing without the tail, all of it outside with it.
    p4 = torch.softmax(x[4].double(), 0)
    inside = torch.zeros(V, dtype=torch.bool, device="cuda")
    inside[ids[4].long()] = True
    if tail:
        out = p4[~inside].sum()
        close(loss[4], -out.log(), 4 * STAT_TOL)
        want = p4 - torch.where(inside, torch.zeros_like(p4), p4 / out)
        assert ((d[4].double() - want).abs() <= 1e-4 * p4 + EPS[dtype] * want.abs() + TINY[dtype]).all()
    else:
        assert loss[4] == 0 and (d[4] == 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distill_long_rows(voc, tail):
    """Float32 rows of 2^20 columns: more than a cluster's shared memory holds, so the row is read twice."""
    x = make(2, 1 << 20, torch.float32, 65, pad=3, shift=1)
    ids, t = teacher(x, 40, tail, 7)
    loss, d = voc.distill_topk(x, ids, t, tail=tail)
    wl, wd, p, q = ref_distill(x, ids, t, 1.0, tail, None)
    close(loss, wl, 4 * 7e-5)
    assert ((d.double() - wd).abs() <= 1e-4 * (wd.abs() + p) + 1e-6 * p + 1e-9).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distill_differences(voc, tail):
    x = make(2, 40, torch.float32, 71, scale=1.0)
    ids, t = teacher(x, 5, tail, 8)
    w = torch.tensor([1.0, 0.5], device="cuda")
    _, d = voc.distill_topk(x, ids, t, temperature=1.5, tail=tail, weights=w)
    h = 2.0**-5
    for j in range(40):
        e = torch.zeros_like(x)
        e[:, j] = h
        up, _ = voc.distill_topk(x + e, ids, t, temperature=1.5, tail=tail, weights=w, grad=False)
        dn, _ = voc.distill_topk(x - e, ids, t, temperature=1.5, tail=tail, weights=w, grad=False)
        assert (((up.double() - dn.double()) / (2 * h) - d[:, j].double()).abs() <= 1e-3).all()


def test_tail_is_not_lost_to_cancellation(voc):
    """A student almost certain of the list: the tail's mass is 1e-9 of the whole."""
    x = torch.full((1, 2000), -21.0, device="cuda")
    x[0, 7] = 8.0
    ids = torch.tensor([[7]], dtype=torch.int32, device="cuda")
    t = torch.tensor([[math.log(0.9)]], device="cuda")
    loss, d = voc.distill_topk(x, ids, t, tail=True)
    wl, wd, _, _ = ref_distill(x, ids, t, 1.0, True, None)
    close(loss, wl, STAT_TOL)
    assert ((d.double() - wd).abs() <= 1e-5 * wd.abs() + 1e-9).all()


# ---- streams, offsets, refusals ------------------------------------------------------------------------------------


def test_other_stream_and_repeat(voc):
    x = make(300, 30011, torch.bfloat16, 81)
    ids = torch.randint(0, 30011, (300, 2), device="cuda", dtype=torch.int32)
    a = voc.token_logprobs(x, ids, top_k=8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = voc.token_logprobs(x, ids, top_k=8)
    st.synchronize()
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_offsets_past_32_bits(voc):
    """Rows that start beyond 2^32 bytes and 2^31 elements."""
    V, ld = 1000, (1 << 30) + 8
    buf = torch.empty(3 * ld, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (3, V), (ld, 1))
    x.copy_(make(3, V, torch.bfloat16, 91))
    ids = torch.tensor([[1], [2], [999]], dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, ids, top_k=3)
    s = voc.token_logprobs(x.contiguous(), ids, top_k=3)
    for u, v in zip(r, s):
        assert torch.equal(u, v)
    d = voc.token_logprobs_backward(x, ids, r.lse, r.entropy, torch.ones((3, 1), device="cuda"), out=x)
    e = voc.token_logprobs_backward(make(3, V, torch.bfloat16, 91), ids, r.lse, r.entropy, torch.ones((3, 1), device="cuda"))
    assert torch.equal(d, e)


def test_empty(voc):
    x = torch.empty((0, 100), device="cuda")
    ids = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, ids, top_k=2)
    assert r.logprobs.shape == (0, 2)
    assert voc.token_logprobs_backward(x, ids, r.lse, r.entropy, r.logprobs).shape == (0, 100)
    loss, d = voc.distill_topk(x, ids, r.logprobs)
    assert loss.shape == (0,) and d.shape == (0, 100)
    x = make(2, 100, torch.float32, 1)
    none = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, none)
    d = voc.token_logprobs_backward(x, none, r.lse, r.entropy, torch.empty((2, 0), device="cuda"), torch.ones(2, device="cuda"))
    want, _ = ref_gradient(x, torch.full((2, 1), -1, device="cuda"), torch.zeros((2, 1), device="cuda"),
                           torch.ones(2, device="cuda"), 1.0)
    assert ((d.double() - want).abs() <= 1e-5 * (want.abs() + 1e-3)).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distill_without_entries(voc, tail):
    """Lists of length zero: no loss and no gradient, whatever the rows hold."""
    x = make(3, 100, torch.bfloat16, 1)
    x[1] = float("nan")
    none = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    loss, d = voc.distill_topk(x, none, torch.empty((3, 0), device="cuda"), tail=tail)
    assert (loss == 0).all() and (d == 0).all()


def test_two_streams_at_once(voc):
    """Calls in flight on two streams do not touch one another."""
    xs = [make(600, 20011, torch.bfloat16, 83 + i) for i in range(2)]
    ids = torch.randint(0, 20011, (600, 2), device="cuda", dtype=torch.int32)
    want = [voc.token_logprobs(x, ids, top_k=8) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (st, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(st):
                got[i].append(voc.token_logprobs(x, ids, top_k=8))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_bad_ids(voc):
    from indecis_b200 import ops
    ops.device_error()
    x = make(2, 100, torch.float32, 1)
    ids = torch.tensor([[5, 100], [-7, 3]], dtype=torch.int32, device="cuda")
    r = voc.token_logprobs(x, ids)
    assert r.logprobs[0, 1].isnan() and r.logprobs[1, 0] == 0 and r.logprobs[0, 0].isfinite()
    assert ops.device_error() == 5
    voc.distill_topk(x, ids, torch.zeros((2, 2), device="cuda"))
    assert ops.device_error() == 5
    assert ops.device_error() == 0


def test_refusals(voc):
    from indecis_b200 import _capi
    x = make(2, 100, torch.float32, 1)
    ids = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    f = torch.zeros((2, 2), device="cuda")
    bad = [lambda: voc.token_logprobs(x.double(), ids), lambda: voc.token_logprobs(x.cpu(), ids),
           lambda: voc.token_logprobs(x.t(), ids), lambda: voc.token_logprobs(x, ids.long()),
           lambda: voc.token_logprobs(x, ids[:1]), lambda: voc.token_logprobs(x[0], ids),
           lambda: voc.token_logprobs(x.expand(2, 100)[:1].expand(2, 100), ids),
           lambda: voc.distill_topk(x, ids, f.half()), lambda: voc.distill_topk(x, ids, f, out=x[:1]),
           lambda: voc.token_logprobs_backward(x, ids, f[0], f[0], f[:, 0], out=x.bfloat16())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    codes = [lambda: voc.token_logprobs(x, ids, temperature=0.0), lambda: voc.token_logprobs(x, ids, temperature=-1.0),
             lambda: voc.token_logprobs(x, ids, temperature=math.nan), lambda: voc.token_logprobs(x, ids, temperature=INF),
             lambda: voc.token_logprobs(x, ids, top_k=33), lambda: voc.token_logprobs(x, ids, top_k=-1),
             lambda: voc.token_logprobs(x, torch.zeros((2, 257), dtype=torch.int32, device="cuda"))]
    for call in codes:
        with pytest.raises(_capi.IgError) as e:
            call()
        assert e.value.code == _capi.IG_ERR_BAD_ARG
    L = _capi.load()
    assert L.ig_token_logprobs(None, 0, 100, 2, 100, 1.0, None, 0, None, None, None, 0, None, None, None) == _capi.IG_ERR_BAD_ARG
    assert L.ig_token_logprobs(x.data_ptr(), 3, 100, 2, 100, 1.0, None, 0, None, None, None, 0, None, None, None) == _capi.IG_ERR_BAD_ARG
    assert L.ig_token_logprobs(x.data_ptr() + 2, 0, 100, 1, 50, 1.0, None, 0, None, None, None, 0, None, None, None) == _capi.IG_ERR_BAD_ARG
    assert L.ig_distill_topk(x.data_ptr(), 0, 99, 2, 100, 1.0, None, None, 0, 0, None, x.data_ptr(), None, 0, None) == _capi.IG_ERR_BAD_ARG
    assert L.ig_distill_topk(x.data_ptr(), 0, 1 << 21, 1, 1 << 21, 1.0, None, None, 0, 1, None, x.data_ptr(), None, 0, None) == _capi.IG_ERR_UNSUPPORTED
    assert "ig_distill_topk" in _capi.last_error()
