"""The vocabulary losses in 64 bits, row by row from the definition, and their gradients
in the logits by the formula (checked against autograd in test_vocab_losses_host.py)."""

import math

import torch


def targets_as_known(targets, ignore_index=-100):
    """A target as a teacher's one token of probability 1 (-1: none)."""
    ids = torch.where(targets == ignore_index, -1, targets)[:, None]
    return ids, torch.zeros(ids.shape, dtype=torch.float32, device=ids.device)


def divergence(logits, ids, log_q, temperature=1.0, rest=True):
    """Losses [rows] and dloss / dlogits [rows, vocab] of finite or -inf logits and ids
    below the vocabulary; also q's mass and the probabilities, for tolerances."""
    z = logits.double() / temperature
    R, V = z.shape
    lp = z.log_softmax(-1)
    empty = (z == -math.inf).all(-1)
    lp = torch.where(empty[:, None], -math.inf, lp)
    p = lp.exp()
    given = ids >= 0
    at = torch.where(given, ids, V)
    q = torch.where(given, log_q.double().exp(), 0.0)
    log_q = torch.where(q > 0, log_q.double(), 0.0)
    wide = torch.cat((lp, torch.zeros_like(lp[:, :1])), 1)
    own = wide.gather(1, at)
    loss = torch.where(q > 0, q * (log_q - torch.where(q > 0, own, 0.0)), 0.0).sum(-1)
    Q = q.sum(-1)
    known = torch.zeros(R, V + 1, dtype=torch.float64, device=z.device).scatter_add_(1, at, q)[:, :V]
    among = torch.zeros(R, V + 1, dtype=torch.bool, device=z.device).scatter_(1, at, True)[:, :V]
    log_others = lp.masked_fill(among, -math.inf).logsumexp(-1)
    others = log_others > -math.inf
    q_rest = torch.zeros_like(Q)
    if rest:
        q_rest = torch.where(others & given.any(-1), (1.0 - Q).clamp(min=0), 0.0)
        safe = torch.where(q_rest > 0, q_rest, 1.0)
        loss = loss + torch.where(q_rest > 0, safe * (safe.log() - torch.where(others, log_others, 0.0)), 0.0)
    part = torch.where(others[:, None], (lp - torch.where(others, log_others, 0.0)[:, None]).exp(), 0.0)
    part = part.masked_fill(among, 0.0)
    grad = (p * (Q + q_rest)[:, None] - known - part * q_rest[:, None]) / temperature
    grad = torch.where(empty[:, None], 0.0, grad)
    return loss, grad, Q + q_rest, p


def reduced(loss, ids, reduction):
    if reduction == "none":
        return loss
    return loss.sum() / (max(int((ids >= 0).any(-1).sum()), 1) if reduction == "mean" else 1)


def upstream(ids, reduction, d_loss):
    """What each row's gradient is times."""
    if reduction == "none":
        return d_loss.double()
    n = max(int((ids >= 0).any(-1).sum()), 1) if reduction == "mean" else 1
    return (d_loss.double() / n).expand(ids.shape[0])


def tokens(R, V, K, gen, device, mass=(0.6, 0.99)):
    """Different tokens in no order with log probabilities, some rows with fewer tokens,
    some without any."""
    ids = torch.stack([torch.randperm(V, generator=gen, device=device)[:K] for _ in range(R)])
    share = mass[0] + (mass[1] - mass[0]) * torch.rand(R, 1, generator=gen, device=device)
    log_q = ((2.0 * torch.randn(R, K, generator=gen, device=device)).softmax(-1) * share).log()
    few = torch.rand(R, 1, generator=gen, device=device)
    gone = (few < 0.15) | ((few < 0.4) & (torch.rand(R, K, generator=gen, device=device) < 0.5))
    gone[0] = False
    return torch.where(gone, -1, ids), torch.where(gone, math.nan, log_q)
