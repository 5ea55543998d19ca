"""Vocabulary operators from hidden states (tensor-core products) against plain float64 forms.

Tolerances. A logit is a float32 sum of exact products: off by at most LOGIT (2^-20) of sum |h w| (a truncation of 2^-23 per
step of 16, and the partial sums stay well under that sum). Statistics add what the stored-logits kernels' do (STAT_TOL).
Gradients: the logits' gradient G has relative error P_TOL plus the logit's error in p, then one rounding to 16 bits
(u = eps / 2 relative, or half the smallest step), so a product is off by at most that times sum |G| |operand|, plus its
float32 accumulation (LOGIT) and the rounding of the result.
"""
import math

import pytest
import torch

from test_gpu_vocab import STAT_TOL, P_TOL, close, ref_top

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
LOGIT = 2.0**-20


@pytest.fixture(scope="module")
def voc(igdev):
    from indecis_b200 import vocab
    return vocab


def make(rows, V, H, dtype, seed, wstd=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, H, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, H, generator=g, device="cuda") * wstd).to(dtype)
    return h, w


def check_forward(r, h, w, ids, temperature, top):
    hd, wd = h.double(), w.double()
    z = hd @ wd.T / temperature
    off = float((hd.abs() @ wd.abs().T).max()) * LOGIT / temperature
    tol = STAT_TOL + off
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    lp = torch.where(ids >= 0, logp.gather(1, ids.clamp(min=0).long()), torch.zeros_like(lse)[:, None])
    close(r.lse, lse, tol, "lse")
    close(r.logprobs, lp, tol, "logprobs")
    # d(entropy)/dx_j = -p_j (log p_j + entropy): at most (1/e + entropy) in all.
    close(r.entropy, ent, STAT_TOL + off * (1 + float(ent.max())), "entropy")
    if top:
        # The columns chosen have the k-th largest values, within the logits' error, in descending order.
        at = r.top_ids.long()
        assert (at >= 0).all() and (at.sort(1).values.diff(dim=1) > 0).all()
        want = logp.topk(top, dim=1).values
        close(logp.gather(1, at), want, tol, "top columns")
        close(r.top_logprobs, logp.gather(1, at), tol, "top values")
        assert (r.top_logprobs.diff(dim=1) <= 0).all()


SHAPES = [(1, 1, 1), (1, 257, 8), (3, 1000, 70), (33, 50021, 256), (128, 4096, 64), (129, 4096, 72), (300, 5000, 200),
          (513, 777, 40), (1, 262144, 768), (700, 33000, 768), (2000, 300, 1000), (4097, 2500, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,H", SHAPES)
def test_forward(voc, dtype, rows, V, H):
    h, w = make(rows, V, H, dtype, 3 + V)
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(-1, V, (rows, 5), generator=g, device="cuda", dtype=torch.int32)
    for temperature, top in ((1.0, 0), (0.7, 1), (2.0, min(32, V))):
        check_forward(voc.vocab_logprobs(h, w, ids, temperature=temperature, top_k=top), h, w, ids, temperature, top)
    from indecis_b200 import ops
    assert ops.device_error() == 0


@pytest.mark.parametrize("rows", [2, 200])
def test_forward_exact_ties(voc, rows):
    """Small integers: the logits are exact, many are equal, and ties go to the lowest column."""
    g = torch.Generator(device="cuda").manual_seed(7)
    h = torch.randint(-2, 3, (rows, 24), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randint(-1, 2, (30011, 24), generator=g, device="cuda").to(torch.bfloat16)
    h[1] = 0  # all columns equal
    ids = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
    r = voc.vocab_logprobs(h, w, ids, top_k=32)
    x = h.double() @ w.double().T
    assert torch.equal(r.top_ids.long(), ref_top(x, 32)[0])
    s = voc.token_logprobs(x.float(), ids, top_k=32)
    for a, b in zip(r, s):
        close(a.float(), b.float(), STAT_TOL)


def test_forward_special(voc):
    """NaN and infinite states reach their rows only; more alternatives than columns; a column at the lowest value."""
    h, w = make(140, 20, 64, torch.bfloat16, 9)
    h[3, 5] = float("nan")
    h[130, 0] = math.inf
    ids = torch.zeros((140, 1), dtype=torch.int32, device="cuda")
    r = voc.vocab_logprobs(h, w, ids, top_k=32)
    for n in (3, 130):
        assert r.lse[n].isnan() and r.entropy[n].isnan() and r.logprobs[n].isnan().all()
        assert (r.top_ids[n] == -1).all() and r.top_logprobs[n].isnan().all()
    ok = torch.ones(140, dtype=torch.bool, device="cuda")
    ok[[3, 130]] = False
    assert (r.top_ids[ok][:, 20:] == -1).all() and (r.top_logprobs[ok][:, 20:] == -math.inf).all()
    part = type(r)(*[t[ok] if t.shape[1:] != (32,) else t[ok][:, :20].contiguous() for t in r])
    check_forward(part, h[ok], w, ids[ok], 1.0, 20)


def check_backward(voc, h, w, ids, g, gh, temperature, step=1 << 20):
    rows, V, H = h.shape[0], w.shape[0], h.shape[1]
    dtype = h.dtype
    r = voc.vocab_logprobs(h, w, ids, temperature=temperature)
    dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh, temperature=temperature)
    assert dh.dtype == dw.dtype == dtype and dh.shape == h.shape and dw.shape == w.shape
    u = torch.finfo(dtype).eps / 2
    wd, wa = w.double(), w.double().abs()
    want_w, size_w = torch.zeros_like(wd), torch.zeros_like(wd)
    live = g.double() * (ids >= 0)
    # float16: dZ is scaled so that the largest bound is at least 2^14; half the smallest step is 2^-25.
    size_g = (2 * g.double().abs().sum(1) + (0 if gh is None else gh.double().abs() * (1 + r.entropy.double()))) / temperature
    floor = float(size_g.max()) * 2.0**-25 * 2.0**-14 if dtype == torch.float16 else 0.0
    for lo in range(0, rows, step):
        s = slice(lo, lo + step)
        hd = h[s].double()
        z = hd @ wd.T / temperature
        off = (hd.abs() @ wa.T) * (LOGIT / temperature)
        logp = torch.log_softmax(z, 1)
        p = logp.exp()
        ent = -(p * logp).sum(1, keepdim=True)
        G = -live[s].sum(1, keepdim=True) * p
        slack = live[s].abs().sum(1, keepdim=True) * p
        if gh is not None:
            G -= gh[s].double()[:, None] * p * (logp + ent)
            slack = slack + gh[s].double().abs()[:, None] * p * (logp.abs() + ent + 1)
        G.scatter_add_(1, ids[s].clamp(min=0).long(), live[s])
        G /= temperature
        err = u * 1.01 * G.abs() + slack / temperature * (P_TOL + 2 * off.amax(1, keepdim=True)) + floor
        want = G @ wd
        tol = err @ wa + LOGIT * (G.abs() @ wa) + u * 1.01 * want.abs() + (3e-8 if dtype == torch.float16 else 0)
        assert ((dh[s].double() - want).abs() <= tol).all(), "dhidden"
        want_w += G.T @ hd
        size_w += err.T @ hd.abs() + LOGIT * (G.abs().T @ hd.abs())
    tol = size_w + u * 1.01 * want_w.abs() + (3e-8 if dtype == torch.float16 else 0)
    assert ((dw.double() - want_w).abs() <= tol).all(), "dweight"
    return r, dh, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,H", SHAPES)
def test_backward(voc, dtype, rows, V, H):
    h, w = make(rows, V, H, dtype, 13 + V)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(-1, V, (rows, 4), generator=gen, device="cuda", dtype=torch.int32)
    ids[:, 3] = ids[:, 0]
    scale = 64.0 / rows
    g = torch.randn((rows, 4), generator=gen, device="cuda") * scale
    gh = torch.randn((rows,), generator=gen, device="cuda") * scale
    check_backward(voc, h, w, ids, g, None, 1.0)
    r, dh, dw = check_backward(voc, h, w, ids, g, gh, 1.7)
    a, none = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh, temperature=1.7, need_weight=False)
    assert none is None and torch.equal(a, dh)
    none, b = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh, temperature=1.7, need_hidden=False)
    assert none is None and torch.equal(b, dw)
    from indecis_b200 import ops
    assert ops.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,H,T", [(40, 300, 64, 200), (300, 5003, 72, 17), (300, 5003, 72, 16), (130, 50, 64, 16)])
def test_many_given_tokens(voc, dtype, rows, V, H, T):
    """Many given tokens in a row, most of the columns given."""
    h, w = make(rows, V, H, dtype, 15)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(-1, V, (rows, T), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, T), generator=gen, device="cuda")
    gh = torch.randn((rows,), generator=gen, device="cuda")
    check_backward(voc, h, w, ids, g, gh, 0.8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,H", [(1, 5000, 256), (7, 33001, 72), (128, 1000, 136)])
def test_few_rows_keep_more_bits(voc, dtype, rows, V, H):
    """At most 128 rows: dZ in two 16-bit parts, so the gradients are off by their own rounding and little else (the
    second part's rounding is 2^-8 of the first's: u (1 + 2^-6) bounds both, in the norm over a gradient)."""
    h, w = make(rows, V, H, dtype, 19)
    gen = torch.Generator(device="cuda").manual_seed(8)
    ids = torch.randint(0, V, (rows, 1), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.rand((rows, 1), generator=gen, device="cuda") + 0.5
    r = voc.vocab_logprobs(h, w, ids)
    dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g)
    G = -g.double() * torch.softmax(h.double() @ w.double().T, 1)
    G.scatter_add_(1, ids.long(), g.double())
    u = torch.finfo(dtype).eps / 2
    for got, want in ((dh, G @ w.double()), (dw, G.T @ h.double())):
        rounded = (want.to(dtype).double() - want).norm()
        assert (got.double() - want).norm() <= 1.1 * rounded + u * 2**-6 * want.norm()


def test_backward_column_chunks(voc):
    """A logits' gradient of more than its workspace's chunk: two chunks of columns."""
    rows, V, H = 8192, 70001, 64
    h, w = make(rows, V, H, torch.bfloat16, 17)
    gen = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(0, V, (rows, 2), generator=gen, device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 2), generator=gen, device="cuda") / 64
    check_backward(voc, h, w, ids, g, None, 1.0, step=1024)


def test_backward_differences(voc):
    """Central differences of the forward in the states: a step of 2^-5 in float16 is exact for these values; the
    second-order term is at most 2^-10 |w|^3 ~ 1e-5, the forward's rounding 2e-6 / 2^-4."""
    g0 = torch.Generator(device="cuda").manual_seed(23)
    h = (torch.randint(-32, 33, (3, 8), generator=g0, device="cuda").float() / 32).half()
    w = (torch.randn(50, 8, generator=g0, device="cuda") * 0.2).half()
    ids = torch.tensor([[4, 49], [7, -1], [2, 2]], dtype=torch.int32, device="cuda")
    g = torch.tensor([[0.5, -1.0], [1.0, 3.0], [0.25, 0.5]], device="cuda")
    gh = torch.tensor([0.5, 0.0, -1.0], device="cuda")

    def loss(hh, ww):
        r = voc.vocab_logprobs(hh, ww, ids)
        return (r.logprobs.double() * g * (ids >= 0)).sum(1) + r.entropy.double() * gh

    r = voc.vocab_logprobs(h, w, ids)
    dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g, gh)
    step = 2.0**-5
    for k in range(8):
        e = torch.zeros_like(h)
        e[:, k] = step
        num = (loss(h + e, w) - loss(h - e, w)) / (2 * step)
        assert ((num - dh[:, k].double()).abs() <= 2e-3).all()
    for v in (4, 2, 30):
        up, dn = w.clone(), w.clone()
        up[v, 3] += step
        dn[v, 3] -= step
        width = float(up[v, 3].double() - dn[v, 3].double())
        num = (loss(h, up) - loss(h, dn)).sum() / width
        assert abs(float(num - dw[v, 3].double())) <= 4e-3


def test_strides_streams_and_repeats(voc):
    h, w = make(300, 5003, 90, torch.bfloat16, 31)
    ids = torch.randint(0, 5003, (300, 3), device="cuda", dtype=torch.int32)
    g = torch.randn((300, 3), device="cuda")
    r = voc.vocab_logprobs(h, w, ids, top_k=4)
    d = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g)
    # Rows in wider buffers, aligned and not.
    for ld, shift in ((96, 0), (128, 8), (97, 1)):
        hb = torch.full((300 * ld + 8,), float("nan"), dtype=h.dtype, device="cuda")
        wb = torch.full((5003 * ld + 8,), float("nan"), dtype=h.dtype, device="cuda")
        h2 = hb[shift:shift + 300 * ld].view(300, ld)[:, :90]
        w2 = wb[shift:shift + 5003 * ld].view(5003, ld)[:, :90]
        h2.copy_(h)
        w2.copy_(w)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            r2 = voc.vocab_logprobs(h2, w2, ids, top_k=4)
            d2 = voc.vocab_logprobs_backward(h2, w2, ids, r2.logprobs, r2.lse, r2.entropy, g)
        st.synchronize()
        for a, b in zip(tuple(r) + tuple(d), tuple(r2) + tuple(d2)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [3, 300])
def test_no_given_tokens(voc, rows):
    """Entropy alone: no given tokens, forward and backward."""
    h, w = make(rows, 500, 64, torch.bfloat16, 41)
    none = torch.empty((rows, 0), dtype=torch.int32, device="cuda")
    gh = torch.linspace(-1, 1, rows, device="cuda")
    r = voc.vocab_logprobs(h, w, none, top_k=2)
    assert r.logprobs.shape == (rows, 0)
    dh, dw = voc.vocab_logprobs_backward(h, w, none, r.logprobs, r.lse, r.entropy, torch.empty((rows, 0), device="cuda"), gh)
    one = torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    zero = torch.zeros((rows, 1), device="cuda")
    s = voc.vocab_logprobs(h, w, one, top_k=2)
    for a, b in zip(r[1:], s[1:]):
        assert torch.equal(a, b)
    eh, ew = voc.vocab_logprobs_backward(h, w, one, zero, s.lse, s.entropy, zero, gh)
    assert torch.equal(dh, eh) and torch.equal(dw, ew) and (dw != 0).any()


def test_graph_capture(voc):
    """Every operator recorded in one CUDA graph and replayed on new inputs."""
    h, w = make(200, 3001, 72, torch.float16, 37)
    ids = torch.randint(0, 3001, (200, 2), device="cuda", dtype=torch.int32)
    g = torch.full((200, 2), -0.005, device="cuda")

    def all_of_them():
        r = voc.vocab_logprobs(h, w, ids, top_k=3)
        dh, dw = voc.vocab_logprobs_backward(h, w, ids, r.logprobs, r.lse, r.entropy, g)
        x = h @ w.T
        s = voc.token_logprobs(x, ids, top_k=3)
        d = voc.token_logprobs_backward(x, ids, s.lse, s.entropy, g)
        loss, e = voc.distill_topk(x, s.top_ids, s.top_logprobs, tail=True)
        return tuple(r) + (dh, dw) + tuple(s) + (d, loss, e)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        all_of_them()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = all_of_them()
    h.copy_(make(200, 3001, 72, torch.float16, 38)[0])
    graph.replay()
    for a, b in zip(out, all_of_them()):
        assert torch.equal(a, b)


def test_unaligned_gradients(voc):
    """The C entry point writes gradients at any stride and alignment."""
    from indecis_b200 import _capi
    rows, V, H = 200, 700, 100
    h, w = make(rows, V, 104, torch.bfloat16, 33)
    ids = torch.randint(0, V, (rows, 1), device="cuda", dtype=torch.int32)
    g = torch.randn((rows, 1), device="cuda")
    r = voc.vocab_logprobs(h[:, :H], w[:, :H], ids)
    dh, dw = voc.vocab_logprobs_backward(h[:, :H], w[:, :H], ids, r.logprobs, r.lse, r.entropy, g)
    L = _capi.load()
    n = L.ig_vocab_workspace(rows, V, H, 0, 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    bh = torch.full((rows, 103), 7.0, dtype=h.dtype, device="cuda")
    bw = torch.full((V, 101), 7.0, dtype=h.dtype, device="cuda")
    _capi.check(L.ig_vocab_logprobs_backward(h.data_ptr(), 104, w.data_ptr(), 104, 1, rows, V, H, 1.0, ids.data_ptr(), 1,
                                             r.logprobs.data_ptr(), r.lse.data_ptr(), r.entropy.data_ptr(), g.data_ptr(),
                                             None, bh.data_ptr() + 2, 103, bw.data_ptr() + 2, 101, ws.data_ptr(), n,
                                             torch.cuda.current_stream().cuda_stream))
    assert torch.equal(bh[:, 1:101], dh) and (bh[:, 101:] == 7).all() and (bh[:, 0] == 7).all()
    assert torch.equal(bw[:, 1:], dw) and (bw[:, 0] == 7).all()


def test_empty_and_refusals(voc):
    from indecis_b200 import _capi
    h, w = make(4, 100, 64, torch.bfloat16, 35)
    none = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    r = voc.vocab_logprobs(h[:0], w, none, top_k=3)
    assert r.logprobs.shape == (0, 2) and r.top_ids.shape == (0, 3)
    dh, dw = voc.vocab_logprobs_backward(h[:0], w, none, r.logprobs, r.lse, r.entropy, r.logprobs)
    assert dh.shape == (0, 64) and (dw == 0).all()
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for call in (lambda: voc.vocab_logprobs(h.float(), w.float(), ids), lambda: voc.vocab_logprobs(h, w.half(), ids),
                 lambda: voc.vocab_logprobs(h[:, :32], w, ids), lambda: voc.vocab_logprobs(h, w, ids[:2]),
                 lambda: voc.vocab_logprobs(h.cpu(), w, ids), lambda: voc.vocab_logprobs(h, w, ids.long())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: voc.vocab_logprobs(h, w, ids, temperature=0), lambda: voc.vocab_logprobs(h, w, ids, top_k=33)):
        with pytest.raises(_capi.IgError) as e:
            call()
        assert e.value.code == _capi.IG_ERR_BAD_ARG
    L = _capi.load()
    n = L.ig_vocab_workspace(4, 100, 64, 0, 0)
    assert n > 0 and L.ig_vocab_workspace(0, 100, 64, 0, 0) == 0 and L.ig_vocab_workspace(4, 100, 64, 33, 0) == 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    out = torch.empty((4, 2), device="cuda")

    def c(hp=h.data_ptr(), ldh=64, dt=1, wsp=ws.data_ptr(), wsn=n):
        return L.ig_vocab_logprobs(hp, ldh, w.data_ptr(), 64, dt, 4, 100, 64, 1.0, ids.data_ptr(), 2, out.data_ptr(), None,
                                   None, 0, None, None, wsp, wsn, None)

    for kw in (dict(ldh=63), dict(ldh=65), dict(hp=h.data_ptr() + 2), dict(hp=None), dict(dt=0), dict(dt=3), dict(wsp=None),
               dict(wsn=n - 1), dict(wsp=ws.data_ptr() + 1)):
        assert c(**kw) == _capi.IG_ERR_BAD_ARG, kw
    assert c() == 0
    torch.cuda.synchronize()
