"""Oracle for top alternatives and for distillation from a teacher's (CPU torch, meant to be run in fp64).

Test infrastructure only; see ``oracle/__init__.py``.  Written from the definitions, entry by entry where the rules about
padding, ties and masked logits decide; gradients are autograd's through these expressions.  Nothing of the reference holds
values for them: parity unpinned, checked against hand-computed values in ``tests/test_oracle_topk.py``.
"""

from __future__ import annotations

import math

import torch


def order_of_alternatives(logits, k):
    """Columns of the ``k`` largest logits per row: largest first, the lowest column among equals, NaN below -inf."""
    last = torch.isnan(logits)
    first = torch.sort(torch.where(last, -math.inf, logits), dim=-1, descending=True, stable=True).indices
    # NaN after every number: a stable sort of the found columns by whether they hold one
    moved = torch.sort(last.gather(-1, first).to(torch.int8), dim=-1, stable=True).indices
    return first.gather(-1, moved)[..., :k]


def topk_logprobs(logits, labels, k, temperature=1.0):
    """``(logprobs, entropy, top, index)``: log-probability of ``labels`` (0 for one outside the vocabulary), entropy with
    ``0 log 0 = 0``, and the ``k`` largest."""
    z = logits / temperature
    log_q = torch.log_softmax(z, dim=-1)
    inside = (labels >= 0) & (labels < logits.shape[-1])
    lp = log_q.gather(-1, torch.where(inside, labels, 0)[..., None])[..., 0]
    lp = torch.where(inside, lp, 0.0)
    q = log_q.exp()
    entropy = -torch.where(q == 0, 0.0, q * torch.where(q == 0, 0.0, log_q)).sum(-1)
    index = order_of_alternatives(logits, k)
    return lp, entropy, log_q.gather(-1, index), index


def divergence(kind, t, log_q, beta):
    """Sum over the last dimension of the terms of a divergence between log-probabilities; ``exp(-inf) * x = 0``."""
    p, q = t.exp(), log_q.exp()
    weigh = lambda w, x: torch.where(w == 0, 0.0, w * torch.where(w == 0, 0.0, x))
    if kind == "forward_kl":
        return weigh(p, t - log_q).sum(-1)
    if kind == "reverse_kl":
        return weigh(q, log_q - t).sum(-1)
    log_m = torch.logaddexp(t + math.log(beta), log_q + math.log(1 - beta))
    return (weigh(beta * p, t - log_m) + weigh((1 - beta) * q, log_q - log_m)).sum(-1)


def topk_distillation(logits, teacher_logprobs, teacher_indices, kind="forward_kl", beta=0.5, temperature=1.0):
    """Per-token loss; entries outside the vocabulary or with log-probability -inf add nothing."""
    log_q = torch.log_softmax(logits / temperature, dim=-1)
    counts = (teacher_indices >= 0) & (teacher_indices < logits.shape[-1]) & (teacher_logprobs != -math.inf)
    losses = []
    for row, t, i, ok in zip(log_q.reshape(-1, log_q.shape[-1]), *(x.reshape(-1, x.shape[-1])
                                                                 for x in (teacher_logprobs, teacher_indices, counts))):
        losses.append(divergence(kind, t[ok], row[i[ok]], beta))
    return torch.stack(losses).reshape(logits.shape[:-1])
