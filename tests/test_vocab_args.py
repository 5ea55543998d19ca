"""Refusals of the vocabulary entry points that need no GPU: bad arguments fail before any device work."""
import math

import pytest
import torch

from indecis_b200 import _capi, build, vocab


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


P = 4096  # an address that is never read: every call below is refused, or has no rows


def logprobs(L, x=P, dt=0, ld=100, rows=2, V=100, t=1.0, ids=P, n=1, lp=P, top=0, ti=None, tl=None):
    return L.ig_token_logprobs(x, dt, ld, rows, V, t, ids, n, lp, None, None, top, ti, tl, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(dt=3), dict(dt=-1), dict(ld=99), dict(rows=-1), dict(V=0), dict(V=-5),
                                dict(t=0.0), dict(t=-1.0), dict(t=math.nan), dict(t=math.inf), dict(t=1e-60), dict(ids=None),
                                dict(n=-1), dict(n=257), dict(lp=None), dict(top=33), dict(top=-1), dict(top=3),
                                dict(x=P + 2), dict(rows=1 << 40), dict(V=(1 << 30) + 1, ld=1 << 31)])
def test_token_logprobs(lib, kw):
    assert logprobs(lib, **kw) == _capi.IG_ERR_BAD_ARG
    assert "ig_token_logprobs" in _capi.last_error()


def test_nothing_to_do(lib):
    assert logprobs(lib, x=None, rows=0, ids=None, lp=None) == _capi.IG_OK
    assert lib.ig_token_logprobs_backward(None, 1, 100, 0, 100, 1.0, None, 0, None, None, None, None, None, 100, None) == 0
    assert lib.ig_distill_topk(None, 1, 100, 0, 100, 1.0, None, None, 0, 1, None, None, None, 0, None) == 0
    assert lib.ig_vocab_logprobs(None, 64, P, 64, 1, 0, 100, 64, 1.0, None, 0, None, None, None, 0, None, None, None, 0,
                                 None) == 0


def test_token_logprobs_backward(lib):
    def call(lse=P, ent=P, g=P, gh=None, d=P, ldd=100, x=P, ld=100):
        return lib.ig_token_logprobs_backward(x, 0, ld, 2, 100, 1.0, P, 1, lse, ent, g, gh, d, ldd, None)
    for kw in (dict(lse=None), dict(g=None), dict(ent=None, gh=P), dict(d=None), dict(ldd=50), dict(d=P + 1),
               dict(ld=128, ldd=100)):
        assert call(**kw) == _capi.IG_ERR_BAD_ARG, kw


def test_distill_topk(lib):
    def call(x=P, dt=0, ld=100, V=100, ids=P, t=P, k=3, tail=0, loss=P, d=2 * P, ldd=100):
        return lib.ig_distill_topk(x, dt, ld, 2, V, 1.0, ids, t, k, tail, None, loss, d, ldd, None)
    for kw in (dict(x=None), dict(dt=7), dict(ld=10), dict(ids=None), dict(t=None), dict(k=257), dict(k=-1), dict(loss=None),
               dict(ldd=99), dict(d=P, ldd=101), dict(d=P + 2)):
        assert call(**kw) == _capi.IG_ERR_BAD_ARG, kw
    assert call(V=(1 << 20) + 1, ld=1 << 21, ldd=1 << 21, tail=1) == _capi.IG_ERR_UNSUPPORTED


def test_vocab(lib):
    def fwd(h=P, ldh=64, w=P, ldw=64, dt=1, rows=2, V=100, H=64, top=0, ws=P, n=1 << 30):
        return lib.ig_vocab_logprobs(h, ldh, w, ldw, dt, rows, V, H, 1.0, P, 1, P, None, None, top, None, None, ws, n, None)
    for kw in (dict(h=None), dict(w=None), dict(ldh=60), dict(ldh=68), dict(ldw=63), dict(h=P + 8), dict(dt=0), dict(dt=3),
               dict(H=0), dict(H=1 << 21, ldh=1 << 21, ldw=1 << 21), dict(rows=(1 << 24) + 1), dict(top=40), dict(top=2),
               dict(ws=None), dict(n=16), dict(ws=P + 16)):
        assert fwd(**kw) == _capi.IG_ERR_BAD_ARG, kw

    def bwd(lp=P, lse=P, ent=P, g=P, gh=None, dh=2 * P, dw=3 * P, ws=P, n=1 << 40, lddh=64):
        return lib.ig_vocab_logprobs_backward(P, 64, P, 64, 1, 2, 100, 64, 1.0, P, 1, lp, lse, ent, g, gh, dh, lddh, dw, 64, ws,
                                              n, None)
    for kw in (dict(lp=None), dict(lse=None), dict(g=None), dict(ent=None, gh=P), dict(dh=P), dict(dw=P), dict(lddh=63),
               dict(ws=None), dict(n=0)):
        assert bwd(**kw) == _capi.IG_ERR_BAD_ARG, kw
    assert bwd(dh=None, dw=None) == _capi.IG_OK


def test_workspace(lib):
    W = lib.ig_vocab_workspace
    for bad in ((0, 100, 64, 0, 0), (-1, 100, 64, 0, 0), (2, 0, 64, 0, 0), (2, 100, 0, 0, 1), (2, 100, 64, 33, 0),
                ((1 << 24) + 1, 100, 64, 0, 0)):
        assert W(*bad) == 0
    assert 0 < W(2, 100, 64, 0, 0) < W(2, 100, 64, 5, 0)
    # The gradient's workspace is bounded whatever the vocabulary and the rows.
    for rows, V, H in ((8192, 262144, 768), (65536, 50021, 256), (100, 262144, 768)):
        assert W(rows, V, H, 0, 1) < (1 << 30) + (1 << 24) + 65 * rows * (H + 3) * 4 + 64 * rows
    assert W(1 << 24, 1 << 30, 64, 0, 1) > 0


def test_wrapper_checks():
    x = torch.zeros(2, 100)
    ids = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: vocab.token_logprobs(x, ids), lambda: vocab.vocab_logprobs(x.bfloat16(), x.bfloat16(), ids),
                 lambda: vocab.distill_topk(x, ids, x[:, :1])):
        with pytest.raises(ValueError):
            call()
