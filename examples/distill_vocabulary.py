"""Teaches a vocabulary head on the int8 encoder from a teacher's recorded top logits, then answers with it.

The encoder (seeded random weights, as no checkpoint ships with the repository) turns texts into hidden states on the
GPU. A teacher's answers are known only as its top entries for every token, as a language model's interface returns
them. The student is a vocabulary matrix over the encoder's states:

  1. distillation: logits = states . weight^T, ig_distill_topk gives the loss and the logits' gradient in one call (the
     teacher's remaining mass counted as one more outcome);
  2. training on given tokens with ig_vocab_logprobs and its backward pass, which never store the logits;
  3. answers: the states' last tokens scored over the vocabulary with the entropy and the top alternatives.

    python examples/distill_vocabulary.py [--steps 60]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from indecis_b200 import synthetic, vocab  # noqa: E402
from indecis_b200.model import Config, Model  # noqa: E402


def states_of(cfg, nseq=48, seed=3):
    """Hidden states [tokens, hidden] (bfloat16) of seeded texts, their ids and the texts' last rows."""
    model = Model.from_arrays(Config.from_dict(cfg), synthetic.weights(cfg, seed=42), device=0)
    ids, offs = synthetic.ids_varlen(nseq, 8, 64, cfg["vocab"], seed=seed)
    h = torch.from_numpy(np.asarray(model.EncodeTokens((ids, offs)))).cuda()
    model.close()
    return h.bfloat16(), torch.from_numpy(ids).cuda(), torch.from_numpy(offs[1:] - 1).cuda()


def main(steps=60, top=16, rate=0.5, log=print):
    torch.manual_seed(0)
    cfg = synthetic.tiny(layers=3, hidden=256, heads=4, intermediate=384, vocab=4001)
    h, ids, last = states_of(cfg)
    rows, V = h.shape[0], cfg["vocab"]

    # The teacher: a sharper head of its own, recorded as its top entries' log probabilities.
    teacher = torch.randn(V, cfg["hidden"], device="cuda") * 0.15
    known = torch.log_softmax(h.float() @ teacher.T, 1).topk(top, dim=1)
    t_ids, t_logp = known.indices.int().contiguous(), known.values.contiguous()

    weight = torch.zeros(V, cfg["hidden"], device="cuda")  # the float32 master copy
    share = torch.full((rows,), 1.0 / rows, device="cuda")
    losses = []
    for step in range(steps):
        w = weight.bfloat16()
        logits = h @ w.T
        loss, grad = vocab.distill_topk(logits, t_ids, t_logp, tail=True, weights=share, out=logits)
        losses.append(float(loss.sum()))
        weight -= rate * rows ** 0.5 * (grad.T @ h).float()
        if step % 20 == 0 or step == steps - 1:
            log(f"distillation step {step}: {losses[-1]:.4f} nats")

    # The teacher's first choice as the given token.
    given = t_ids[:, :1].contiguous()
    nll = []
    for step in range(steps):
        w = weight.bfloat16()
        r = vocab.vocab_logprobs(h, w, given)
        nll.append(float(-r.logprobs.mean()))
        pull = torch.full_like(r.logprobs, -1.0 / rows)  # d(mean negative log probability)
        _, dw = vocab.vocab_logprobs_backward(h, w, given, r.logprobs, r.lse, r.entropy, pull, need_hidden=False)
        weight -= rate * rows ** 0.5 * dw.float()
    log(f"given tokens: {nll[0]:.4f} -> {nll[-1]:.4f} nats")

    w = weight.bfloat16()
    r = vocab.vocab_logprobs(h[last].contiguous(), w, given[last].contiguous(), top_k=5)
    agree = float((r.top_ids[:, 0] == t_ids[last][:, 0]).float().mean())
    log(f"answers at {len(last)} last tokens: {100 * agree:.0f}% the teacher's first choice, entropy "
        f"{float(r.entropy.mean()):.2f} nats")
    stored = vocab.token_logprobs(h[last] @ w.T, given[last].contiguous(), top_k=5)
    log(f"the same from stored logits: log probabilities within {float((stored.logprobs - r.logprobs).abs().max()):.1e}")
    return losses, nll, agree


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    main(**vars(ap.parse_args()))
