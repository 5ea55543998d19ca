"""Cases for timing and checking the vocabulary operators (indecis_b200.vocab).

Three operators, each with its backward pass:

  logprobs / logprobs_grad  log probabilities of given tokens, entropy and top alternatives from stored logits
  distill                   divergence from a teacher's top logits: loss and gradient in one call
  vocab / vocab_grad        the same log probabilities from hidden states and the vocabulary matrix

With own = False the operators run in plain torch (32-bit arithmetic, rounded once at the end), with own = True
through the library. exact() computes the same outputs in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _logprobs(name, dtype, rows, vocab, given=1, top=0, temperature=1.0, masked=False, op="logprobs"):
    return dict(name=name, op=op, dtype=dtype, rows=rows, vocab=vocab, given=given, top=top, temperature=temperature,
                masked=masked)


def _distill(name, dtype, rows, vocab, k, tail=False, temperature=1.0):
    return dict(name=name, op="distill", dtype=dtype, rows=rows, vocab=vocab, k=k, tail=tail, temperature=temperature)


def _vocab(name, dtype, rows, vocab, hidden, given=1, top=0, temperature=1.0, op="vocab"):
    return dict(name=name, op=op, dtype=dtype, rows=rows, vocab=vocab, hidden=hidden, given=given, top=top,
                temperature=temperature)


def listed():
    """Vocabularies of 16384 and 262144 and hidden sizes of 256 and 768 are the framework's own model shapes; 50021 is
    an odd vocabulary, whose rows start off any vector boundary."""
    return [
        # One masked position answered: latency.
        _logprobs("logprobs_one", "f32", 1, 16384, given=4, top=5),
        # 32 texts x 128 tokens scored, with alternatives, over the small vocabulary.
        _logprobs("logprobs_4096x16384", "bf16", 4096, 16384, top=8),
        # A page of positions over the large vocabulary, special tokens masked out, sampled with a temperature.
        _logprobs("logprobs_1024x262144", "bf16", 1024, 262144, given=2, top=20, temperature=0.7, masked=True),
        # Training on given tokens with an entropy bonus, odd vocabulary.
        _logprobs("logprobs_grad_2047x50021", "bf16", 2047, 50021, op="logprobs_grad"),
        # A small distillation batch in float32.
        _distill("distill_32x16384", "f32", 32, 16384, 8, temperature=2.0),
        # Distillation of 4096 tokens, odd vocabulary.
        _distill("distill_4096x50021", "bf16", 4096, 50021, 32, temperature=2.0),
        # The large vocabulary, the teacher's remaining mass counted as one more outcome.
        _distill("distill_tail_1024x262144", "f16", 1024, 262144, 64, tail=True),
        # One masked position answered from its hidden state: the weights are read once.
        _vocab("vocab_one_262144x768", "bf16", 1, 262144, 768, given=4, top=5),
        # A batch of texts, one answer position each, odd sizes.
        _vocab("vocab_33x50021x256", "f16", 33, 50021, 256, given=5, top=3),
        # 4096 tokens scored over the large vocabulary.
        _vocab("vocab_4096x262144x768", "bf16", 4096, 262144, 768),
        # A small training batch of the small model.
        _vocab("vocab_grad_500x16384x256", "f16", 500, 16384, 256, given=2, op="vocab_grad"),
        # A training batch of 8192 tokens: gradients of the hidden states and of the vocabulary matrix.
        _vocab("vocab_grad_8192x50021x768", "bf16", 8192, 50021, 768, given=8, op="vocab_grad"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_grad", "distill", "vocab", "vocab_grad"])
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op in ("vocab", "vocab_grad"):
        hidden = 8 * _log_uniform(rng, 8, 128)
        vocab = _log_uniform(rng, 1000, 262144)
        most = 4096 * 262144 * 768 // (3 if op == "vocab_grad" else 1)
        rows = _log_uniform(rng, 1, max(1, min(8192, most // (vocab * hidden))))
        top = rng.choice([0, 1, 3]) if op == "vocab" and rows <= 32 else 0
        c = _vocab("", rng.choice(["bf16", "f16"]), rows, vocab, hidden, rng.randint(1, 8), top, temperature, op)
    else:
        vocab = _log_uniform(rng, 1000, 262144)
        rows = _log_uniform(rng, 1, max(1, min(8192, (1024 * 262144) // vocab // 2)))
        dtype = rng.choice(["bf16", "f16", "f32"])
        if op == "distill":
            c = _distill("", dtype, rows, vocab, rng.randint(1, 64), rng.random() < 0.5, temperature)
        else:
            top = rng.choice([0, 1, 5, 32]) if op == "logprobs" else 0
            c = _logprobs("", dtype, rows, vocab, rng.randint(1, 8), top, temperature, rng.random() < 0.5, op)
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    N, V, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    s = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def integers(hi, *shape):
        return torch.randint(0, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    if case["op"] in ("vocab", "vocab_grad"):
        H, T = case["hidden"], case["given"]
        s["weight"] = (normal(V, H) * 0.05).to(dt)
        s["hidden"] = normal(N, H).to(dt)
        s["ids"] = integers(V, N, T)
        # The states lean towards their first token, as a trained model's do.
        s["hidden"] = (s["hidden"].float() + 4.0 * s["weight"][s["ids"][:, 0].long()].float()).to(dt)
        if N > 4:
            s["ids"][N // 3, T - 1] = -1  # a padded entry
        if case["op"] == "vocab_grad":
            z = (s["hidden"].float() @ s["weight"].float().T) * (1.0 / case["temperature"])
            s["logprobs"], s["lse"], s["entropy"] = _stats(z, s["ids"])
            s["dlogprobs"] = -(0.5 + torch.rand((N, T), generator=g, device="cuda")) / N
            s["dentropy"] = normal(N) * (0.01 / N)
        return s
    s["logits"] = normal(N, V) * 2.0
    if case["op"] == "distill":
        K = case["k"]
        teacher = (s["logits"] + normal(N, V)).topk(K, dim=1)
        t = teacher.values
        if case["tail"]:
            t = t - math.log(V) - 2.0  # log probabilities whose sum leaves some mass over
            t = torch.where(t.exp().sum(1, keepdim=True) < 0.98, t, torch.log_softmax(t, 1) - 0.05)
        s["teacher_ids"], s["teacher_logits"] = teacher.indices.int(), t.contiguous()
        if N > 4 and K > 2:
            s["teacher_ids"][N // 3, K - 2:] = -1  # a shorter list
            s["teacher_ids"][N // 2] = -1  # a row with none
        # The mean over the rows, times the loss scale that float16 gradients are trained with.
        s["weights"] = torch.full((N,), (4096.0 if case["dtype"] == "f16" else 1.0) / N, device="cuda")
        s["logits"] = s["logits"].to(dt)
        return s
    s["ids"] = integers(V - 4, N, case["given"]) + 4
    s["logits"].scatter_add_(1, s["ids"][:, :1].long(), torch.full((N, 1), 8.0, device="cuda"))
    if case["masked"]:
        s["logits"][:, :4] = -math.inf  # special tokens are no answers
        if N > 4:
            s["logits"][N // 2] = -math.inf  # a row with nothing left
    s["logits"] = s["logits"].to(dt)
    if N > 4:
        s["ids"][N // 3, case["given"] - 1] = -1
    if case["op"] == "logprobs_grad":
        _, s["lse"], s["entropy"] = _stats(s["logits"].float() * (1.0 / case["temperature"]), s["ids"])
        scale = (4096.0 if case["dtype"] == "f16" else 1.0) / N  # float16 gradients come with a loss scale
        s["dlogprobs"] = -(0.5 + torch.rand((N, case["given"]), generator=g, device="cuda")) * scale
        s["dentropy"] = normal(N) * (0.01 * scale)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------


def _stats(z, ids):
    """Log probabilities of ids, logsumexp and entropy of the rows of z."""
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(z - m)
    s = e.sum(1)
    lse = m[:, 0] + torch.log(s)
    mean = torch.where(e > 0, e * (z - m), torch.zeros_like(e)).sum(1)
    empty = s == 0
    entropy = torch.where(empty, torch.zeros_like(s), torch.log(s) - mean / s)
    lp = torch.gather(z, 1, ids.clamp(min=0).long()) - lse[:, None]
    lp = torch.where(empty[:, None], torch.full_like(lp, -math.inf), lp)
    return torch.where(ids < 0, torch.zeros_like(lp), lp), lse, entropy


def _top(x, k):
    """The k largest of each row and their columns, ties to the lowest column; -1 where only -inf is left."""
    if k == 0:
        return None, None
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    column = torch.arange(x.shape[1], device=x.device)
    key = (order << 32) | (0x7FFFFFFF - column)
    key = torch.topk(key, k, dim=1).values
    at = 0x7FFFFFFF - (key & 0xFFFFFFFF)
    v = torch.gather(x, 1, at)
    return torch.where(v == -math.inf, torch.full_like(at, -1), at).int(), v


def _forward(x, s):
    c = 1.0 / s["temperature"]
    ids, v = _top(x, s["top"])
    lp, lse, entropy = _stats(x * c, s["ids"])
    out = dict(logprobs=lp, lse=lse, entropy=entropy)
    if ids is not None:
        out["top_ids"] = ids
        out["top_logprobs"] = torch.where(ids < 0, torch.full_like(v, -math.inf), v * c - lse[:, None])
    return out


def _gradient(x, s):
    """d(loss)/d(x) from the gradients of the log probabilities and of the entropy."""
    c = 1.0 / s["temperature"]
    logp = x * c - s["lse"][:, None]
    p = torch.exp(logp)
    live = (s["ids"] >= 0).to(x.dtype)
    g = s["dlogprobs"] * live
    h = torch.where(p > 0, p * (logp + s["entropy"][:, None]), torch.zeros_like(p))
    d = -g.sum(1, keepdim=True) * p - s["dentropy"][:, None] * h
    d.scatter_add_(1, s["ids"].clamp(min=0).long(), g)
    d = torch.where(s["lse"][:, None] == -math.inf, torch.zeros_like(d), d)
    return d * c


def _distill_terms(z, s):
    """Loss and gradient with respect to z of the divergence from the teacher's list, before the rows' weights."""
    ids, t = s["teacher_ids"], s["teacher_logits"].to(z.dtype)
    there = ids >= 0
    at = ids.clamp(min=0).long()
    none = torch.zeros((), dtype=z.dtype, device=z.device)
    if s["tail"]:
        q = torch.where(there, torch.exp(t), none)
    else:
        u = torch.where(there, t * (1.0 / s["temperature"]), torch.full_like(t, -math.inf))
        top = u.amax(1, keepdim=True)
        e = torch.where(there, torch.exp(u - torch.where(top == -math.inf, torch.zeros_like(top), top)), none)
        q = e / e.sum(1, keepdim=True).clamp(min=1e-30)
    z = z - z.amax(1, keepdim=True)
    lse = torch.log(torch.exp(z).sum(1, keepdim=True))
    logp = z - lse
    p = torch.exp(logp)
    term = torch.where(q > 0, q * (torch.log(q.clamp(min=1e-37)) - torch.gather(logp, 1, at)), none)
    loss = term.sum(1)
    q_sum = q.sum(1, keepdim=True)
    some = there.any(1, keepdim=True)
    listed_ = torch.zeros(z.shape, dtype=z.dtype, device=z.device).scatter_add_(1, at, there.to(z.dtype)) > 0
    spread = torch.zeros_like(z).scatter_add_(1, at, q)
    if s["tail"]:
        q_rest = torch.where(some, (1.0 - q_sum).clamp(min=0.0), none)
        p_rest = torch.where(listed_, none, p).sum(1, keepdim=True)
        loss = loss + torch.where(q_rest > 0, q_rest * (torch.log(q_rest.clamp(min=1e-37)) - torch.log(p_rest)), none)[:, 0]
        q_sum = q_sum + q_rest
        spread = torch.where(listed_, spread, p * (q_rest / p_rest))
    d = torch.where(some, p * q_sum - spread, none)
    return torch.where(some[:, 0], loss, none), d


def _distilled(x, s):
    loss, d = _distill_terms(x * (1.0 / s["temperature"]), s)
    w = s["weights"].to(x.dtype)
    return dict(loss=loss * w, dlogits=d * (w[:, None] * (1.0 / s["temperature"])))


def run(state):
    if own:
        return _run_own(state)
    s, op = state, state["op"]
    if op == "logprobs":
        return _forward(s["logits"].float(), s)
    if op == "logprobs_grad":
        return dict(dlogits=_gradient(s["logits"].float(), s).to(s["logits"].dtype))
    if op == "distill":
        out = _distilled(s["logits"].float(), s)
        return dict(loss=out["loss"], dlogits=out["dlogits"].to(s["logits"].dtype))
    h, w = s["hidden"].float(), s["weight"].float()
    x = h @ w.T
    if op == "vocab":
        return _forward(x, s)
    d = _gradient(x, s)
    return dict(dhidden=(d @ w).to(s["hidden"].dtype), dweight=(d.T @ h).to(s["weight"].dtype))


# ---- the library's calls ---------------------------------------------------------------------------------------


def _run_own(s):
    from indecis_b200 import vocab
    op, t = s["op"], s["temperature"]
    if op == "logprobs":
        r = vocab.token_logprobs(s["logits"], s["ids"], temperature=t, top_k=s["top"])
    elif op == "vocab":
        r = vocab.vocab_logprobs(s["hidden"], s["weight"], s["ids"], temperature=t, top_k=s["top"])
    elif op == "logprobs_grad":
        return dict(dlogits=vocab.token_logprobs_backward(s["logits"], s["ids"], s["lse"], s["entropy"], s["dlogprobs"],
                                                          s["dentropy"], temperature=t))
    elif op == "distill":
        loss, d = vocab.distill_topk(s["logits"], s["teacher_ids"], s["teacher_logits"], temperature=t, tail=s["tail"],
                                     weights=s["weights"])
        return dict(loss=loss, dlogits=d)
    else:
        dh, dw = vocab.vocab_logprobs_backward(s["hidden"], s["weight"], s["ids"], s["logprobs"], s["lse"], s["entropy"],
                                               s["dlogprobs"], s["dentropy"], temperature=t)
        return dict(dhidden=dh, dweight=dw)
    out = dict(logprobs=r.logprobs, lse=r.lse, entropy=r.entropy)
    if s["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    N, V, e = case["rows"], case["vocab"], SIZE[case["dtype"]]
    op = case["op"]
    if op == "logprobs":
        return {"bytes": N * V * e + N * (8 * case["given"] + 8 + 8 * case["top"]), "flops": 8 * N * V}
    if op == "logprobs_grad":
        return {"bytes": 2 * N * V * e + N * (8 * case["given"] + 12), "flops": 8 * N * V}
    if op == "distill":
        return {"bytes": 2 * N * V * e + N * (8 * case["k"] + 8), "flops": 10 * N * V}
    H = case["hidden"]
    if op == "vocab":
        return {"bytes": (N + V) * H * e + N * (8 * case["given"] + 8 + 8 * case["top"]), "flops": 2 * N * V * H}
    return {"bytes": 2 * (N + V) * H * e + N * (12 * case["given"] + 12), "flops": 6 * N * V * H}


# ---- in 64 bits ----------------------------------------------------------------------------------------------------


def exact(case, seed):
    """run()'s outputs in float64, computed over slices of rows, each output from its definition."""
    s = prepare(case, seed)
    N, V, op = case["rows"], case["vocab"], case["op"]
    c = 1.0 / case["temperature"]
    step = max(1, (1 << 27) // V)
    parts, dweight = [], None
    w = s["weight"].double() if "weight" in s else None
    for lo in range(0, N, step):
        r = slice(lo, lo + step)
        h = s["hidden"][r].double() if w is not None else None
        z = (h @ w.T if w is not None else s["logits"][r].double()) * c
        logp = torch.log_softmax(z, 1)
        p = torch.exp(logp)
        if op == "distill":
            parts.append(_exact_distill(z, logp, p, s, r, c))
            continue
        lse = torch.logsumexp(z, 1)
        empty = lse == -math.inf
        entropy = torch.special.entr(p).sum(1).masked_fill(empty, 0.0)
        ids = s["ids"][r].long()
        if op in ("logprobs", "vocab"):
            lp = logp.gather(1, ids.clamp(min=0)).masked_fill(empty[:, None], -math.inf).masked_fill(ids < 0, 0.0)
            out = dict(logprobs=lp, lse=lse, entropy=entropy)
            if case["top"]:
                out["top_logprobs"] = logp.topk(case["top"], dim=1).values.masked_fill(empty[:, None], -math.inf)
            parts.append(out)
            continue
        g = s["dlogprobs"][r].double().masked_fill(ids < 0, 0.0)
        gh = s["dentropy"][r].double()[:, None]
        surprise = torch.where(p > 0, logp + entropy[:, None], torch.zeros_like(p))
        d = -p * (g.sum(1, keepdim=True) + gh * surprise)
        d = d.scatter_add(1, ids.clamp(min=0), g).masked_fill(empty[:, None], 0.0) * c
        if op == "logprobs_grad":
            parts.append(dict(dlogits=d))
        else:
            parts.append(dict(dhidden=d @ w))
            dweight = d.T @ h if dweight is None else dweight.addmm_(d.T, h)
        del z, logp, p, surprise, d
    out = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if dweight is not None:
        out["dweight"] = dweight
    if case.get("top"):
        out["top_ids"] = None
    return out


def _exact_distill(z, logp, p, s, r, c):
    ids, w = s["teacher_ids"][r].long(), s["weights"][r].double()
    there = ids >= 0
    some = there.any(1)
    t = s["teacher_logits"][r].double().masked_fill(~there, -math.inf)
    q = torch.exp(t) if s["tail"] else torch.softmax(t * c, 1).nan_to_num(0.0)
    # One spare column takes the entries that are not there.
    at = torch.where(there, ids, torch.full_like(ids, z.shape[1]))
    full = torch.zeros((z.shape[0], z.shape[1] + 1), dtype=torch.float64, device=z.device)
    target = full.scatter_add(1, at, q)[:, :-1]
    inside = full.scatter_add(1, at, there.double())[:, :-1] > 0
    loss = (torch.special.xlogy(q, q) - q * logp.gather(1, ids.clamp(min=0))).masked_fill(~there, 0.0).sum(1)
    d = p * q.sum(1, keepdim=True) - target
    if s["tail"]:
        rest = (1.0 - q.sum(1)).clamp(min=0.0).masked_fill(~some, 0.0)
        outside = p.masked_fill(inside, 0.0)
        mass = outside.sum(1)
        loss = loss + torch.special.xlogy(rest, rest) - torch.special.xlogy(rest, mass)
        d = d + p * rest[:, None] - outside * (rest / mass)[:, None]
    d = d.masked_fill(~some[:, None], 0.0)
    return dict(loss=loss.masked_fill(~some, 0.0) * w, dlogits=d * (w * c)[:, None])
