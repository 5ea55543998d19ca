"""Vocabulary operators on torch CUDA tensors: log probabilities of tokens with
entropy and top alternatives (from stored logits, or straight from hidden
states and the vocabulary matrix), distillation from a teacher's top logits.

Thin wrappers over the C ABI: each checks shapes, types and strides, allocates
the outputs, enqueues the kernels on the current stream of the inputs' device
and raises on a non-zero status. Logits are [rows, vocab] float32, bfloat16 or
float16 with a unit column stride and any row stride.

No call records anything for torch's autograd, whatever its inputs require:
gradients come from the *_backward functions and from distill_topk.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi

IDS_MAX = 256  # given tokens, or teacher entries, per row
TOP_MAX = 32   # alternatives per row

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenLogProbs(NamedTuple):
    """Pieces of one allocation: clone() what is kept on its own."""
    logprobs: torch.Tensor                # float32 [rows, given]
    lse: torch.Tensor                     # float32 [rows]
    entropy: torch.Tensor                 # float32 [rows]
    top_ids: Optional[torch.Tensor]       # int32 [rows, top_k]
    top_logprobs: Optional[torch.Tensor]  # float32 [rows, top_k]


def _matrix(t, name):
    """Row stride of a CUDA matrix with a unit column stride."""
    shape = t.shape
    if len(shape) == 2 and t.is_cuda and t.dtype in _DT:
        ld, unit = t.stride()
        n = shape[1]
        if shape[0] <= 1:
            ld = n
        if (unit == 1 or n <= 1) and ld >= n:
            return ld
    raise ValueError(f"{name}: expected a CUDA float32, bfloat16 or float16 matrix with a unit column stride, rows apart "
                     "by at least their length")


def _dense(t, dtype, shape, like, name):
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on {like.device}")
    return t.data_ptr()


# The current stream's handle. torch.cuda.current_stream builds a Stream object
# on every call (3 us); torch's own generated code takes the raw handle.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(like, fn, *args):
    """fn on the current stream of like's device."""
    index = like.device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _capi.check(rc)


def _outputs(like, N, T, K):
    """The forward's outputs as pieces of one allocation of 32-bit words, and the addresses of logprobs,
    lse, entropy, top_ids and top_logprobs. (Taken from the allocation: the data_ptr of an empty piece is 0.)"""
    K = max(K, 0)  # a negative top_k is refused by the call
    buf = torch.empty(N * (T + 2 + 2 * K), dtype=torch.float32, device=like.device)
    base, n = buf.data_ptr(), N * T
    tl = ti = None
    if K > 0:
        tl = buf.as_strided((N, K), (K, 1), n + 2 * N)
        ti = buf.view(torch.int32).as_strided((N, K), (K, 1), n + 2 * N + N * K)
    r = TokenLogProbs(buf.as_strided((N, T), (T, 1)), buf.as_strided((N,), (1,), n), buf.as_strided((N,), (1,), n + N), ti,
                      tl)
    ptrs = (base, base + 4 * n, base + 4 * (n + N), base + 4 * (n + 2 * N + N * K) if K > 0 else None,
            base + 4 * (n + 2 * N) if K > 0 else None)
    return r, ptrs


def token_logprobs(logits, ids, temperature=1.0, top_k=0) -> TokenLogProbs:
    """log softmax(logits / temperature) at ids (int32 [rows, given], negative:
    none, reported as 0), with each row's logsumexp, entropy and top_k largest
    columns (ties: the lowest first)."""
    ld = _matrix(logits, "logits")
    N, V = logits.shape
    if ids.dim() != 2:
        raise ValueError("ids: expected a matrix")
    T = ids.shape[1]
    pid = _dense(ids, torch.int32, (N, T), logits, "ids")
    r, (lp, lse, ent, ti, tl) = _outputs(logits, N, T, top_k)
    _call(logits, _capi.load().ig_token_logprobs, logits.data_ptr(), _DT[logits.dtype], ld, N, V, temperature, pid, T, lp,
          lse, ent, top_k, ti, tl)
    return r


def token_logprobs_backward(logits, ids, lse, entropy, dlogprobs, dentropy=None, temperature=1.0, out=None):
    """Gradient with respect to the logits, in their type, from the gradients
    of token_logprobs' logprobs and entropy. out: where to write it (may be
    logits itself, but not overlap it otherwise)."""
    ld = _matrix(logits, "logits")
    N, V = logits.shape
    if ids.dim() != 2:
        raise ValueError("ids: expected a matrix")
    T = ids.shape[1]
    out, ldd = _out_like(logits, out)
    _call(logits, _capi.load().ig_token_logprobs_backward, logits.data_ptr(), _DT[logits.dtype], ld, N, V, temperature,
          _dense(ids, torch.int32, (N, T), logits, "ids"), T, _dense(lse, torch.float32, (N,), logits, "lse"),
          _dense(entropy, torch.float32, (N,), logits, "entropy"),
          _dense(dlogprobs, torch.float32, (N, T), logits, "dlogprobs"),
          _dense(dentropy, torch.float32, (N,), logits, "dentropy"), out.data_ptr(), ldd)
    return out


def _out_like(logits, out):
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    ldd = _matrix(out, "out")
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out: expected the logits' shape, type and device")
    return out, ldd


def distill_topk(logits, teacher_ids, teacher_logits, temperature=1.0, tail=False, weights=None, grad=True, out=None):
    """Divergence of softmax(logits / temperature) from a teacher's top entries
    (int32 ids [rows, k], negative where a list is shorter; float32 values).

    tail=False: the teacher's softmax over its list. tail=True: the values are
    log probabilities, and the mass they leave is one more outcome. Returns
    (loss float32 [rows], already weighted by `weights`; the gradient of its
    sum with respect to the logits, or None with grad=False). out: where to
    write the gradient (may be logits itself, but not overlap it otherwise)."""
    ld = _matrix(logits, "logits")
    N, V = logits.shape
    if teacher_ids.dim() != 2:
        raise ValueError("teacher_ids: expected a matrix")
    K = teacher_ids.shape[1]
    loss = torch.empty(N, dtype=torch.float32, device=logits.device)
    d, ldd = _out_like(logits, out) if grad else (None, 0)
    _call(logits, _capi.load().ig_distill_topk, logits.data_ptr(), _DT[logits.dtype], ld, N, V, temperature,
          _dense(teacher_ids, torch.int32, (N, K), logits, "teacher_ids"),
          _dense(teacher_logits, torch.float32, (N, K), logits, "teacher_logits"), K, 1 if tail else 0,
          _dense(weights, torch.float32, (N,), logits, "weights"), loss.data_ptr(),
          d.data_ptr() if d is not None else None, ldd)
    return loss, d


def aligned(t):
    """t itself if its rows start at multiples of 16 bytes, else a copy that does. Lay a weight out once: the calls
    below do it on every call for what is not."""
    ld = _matrix(t, "matrix")
    if t.data_ptr() % 16 == 0 and ld % 8 == 0:
        return t
    n, h = t.shape
    buf = torch.empty((n, (h + 7) // 8 * 8), dtype=t.dtype, device=t.device)
    return buf[:, :h].copy_(t)


def _operands(hidden, weight):
    ldh, ldw = _matrix(hidden, "hidden"), _matrix(weight, "weight")
    dtype = hidden.dtype
    if dtype is torch.float32 or weight.dtype is not dtype:
        raise ValueError("hidden and weight: expected both bfloat16 or both float16")
    H = hidden.shape[1]
    if weight.shape[1] != H or hidden.device != weight.device:
        raise ValueError("hidden and weight: expected one device and row length")
    if ldh % 8 or hidden.data_ptr() % 16:
        hidden, ldh = aligned(hidden), (H + 7) // 8 * 8
    if ldw % 8 or weight.data_ptr() % 16:
        weight, ldw = aligned(weight), (H + 7) // 8 * 8
    return hidden, ldh, weight, ldw


def _workspace(like, *sizes):
    L = _capi.load()
    if like.device.index == torch.cuda.current_device():
        n = L.ig_vocab_workspace(*sizes)
    else:
        with torch.cuda.device(like.device):
            n = L.ig_vocab_workspace(*sizes)
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=like.device)


def vocab_logprobs(hidden, weight, ids, temperature=1.0, top_k=0) -> TokenLogProbs:
    """token_logprobs of the logits hidden @ weight.T (hidden [rows, H], weight
    [vocab, H], both bfloat16 or both float16), which are never stored."""
    hidden, ldh, weight, ldw = _operands(hidden, weight)
    N, H = hidden.shape
    V = weight.shape[0]
    if ids.dim() != 2:
        raise ValueError("ids: expected a matrix")
    T = ids.shape[1]
    pid = _dense(ids, torch.int32, (N, T), hidden, "ids")
    r, (lp, lse, ent, ti, tl) = _outputs(hidden, N, T, top_k)
    ws = _workspace(hidden, N, V, H, max(top_k, 0), 0)
    _call(hidden, _capi.load().ig_vocab_logprobs, hidden.data_ptr(), ldh, weight.data_ptr(), ldw, _DT[hidden.dtype], N, V,
          H, temperature, pid, T, lp, lse, ent, top_k, ti, tl, ws.data_ptr(), ws.numel())
    return r


def vocab_logprobs_backward(hidden, weight, ids, logprobs, lse, entropy, dlogprobs, dentropy=None, temperature=1.0,
                            need_hidden=True, need_weight=True):
    """Gradients with respect to hidden and weight, in their type (None where
    not needed), from the gradients of vocab_logprobs' logprobs and entropy and
    its results. The logits' gradient in between is held in the operands' type
    for more than 128 rows, which adds an error of the gradients' own rounding's
    size."""
    hidden, ldh, weight, ldw = _operands(hidden, weight)
    N, H = hidden.shape
    V = weight.shape[0]
    if ids.dim() != 2:
        raise ValueError("ids: expected a matrix")
    T = ids.shape[1]
    dh = torch.empty((N, H), dtype=hidden.dtype, device=hidden.device) if need_hidden else None
    dw = torch.empty((V, H), dtype=weight.dtype, device=hidden.device) if need_weight else None
    ws = _workspace(hidden, N, V, H, 0, 1)
    _call(hidden, _capi.load().ig_vocab_logprobs_backward, hidden.data_ptr(), ldh, weight.data_ptr(), ldw,
          _DT[hidden.dtype], N, V, H, temperature, _dense(ids, torch.int32, (N, T), hidden, "ids"), T,
          _dense(logprobs, torch.float32, (N, T), hidden, "logprobs"), _dense(lse, torch.float32, (N,), hidden, "lse"),
          _dense(entropy, torch.float32, (N,), hidden, "entropy"),
          _dense(dlogprobs, torch.float32, (N, T), hidden, "dlogprobs"),
          _dense(dentropy, torch.float32, (N,), hidden, "dentropy"), dh.data_ptr() if dh is not None else None, H,
          dw.data_ptr() if dw is not None else None, H, ws.data_ptr(), ws.numel())
    return dh, dw
