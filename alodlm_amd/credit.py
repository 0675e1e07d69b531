"""Sequence credit primitives on the HIP kernels (drop-in for alodlm/credit.py).

``masked_sequence_ids(masked_indices, cum_seqlens)`` gives the sequence of
every masked row; ``sequence_score_function(credit, log_prob, sequence_ids,
sequence_count)`` is the score-function surrogate (1/M) sum_s R_s Q_s, R_s and
Q_s the per-sequence sums of the detached credit and of log q.  Arguments are
validated with the reference's ValueError messages (alodlm/credit.py:8-35);
the sums run in one workgroup with a fixed order (float32), so results are
deterministic.

``token_log_probs(logits, targets)`` gives the per-token log probabilities that the
score function takes, with the entropy and the top alternatives, from logits over
the vocabulary.
"""

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, call_on, ptr, query


def _require_gpu(t, what):
    if t.device.type != "cuda":
        raise ValueError(f"{what} runs on the HIP kernels; move the tensors to a CUDA (ROCm) device")


def _refuse_tangents(what, *tensors):
    """Forward-mode derivatives are refused: a tensor with a tangent need not require a
    gradient, and a result without one would count as constant."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _ignored_id(ignore_index):
    """As the library takes it: ctypes would drop what passes 64 bits."""
    i = int(ignore_index)
    if not -2 ** 63 <= i < 2 ** 63:
        raise ValueError('ignore_index must fit 64 bits')
    return i


def check_sequence_boundaries(masked_indices, cum_seqlens):
    """The argument checks of alodlm/credit.py:8-19."""
    if masked_indices.ndim != 1 or masked_indices.dtype != torch.bool:
        raise ValueError('masked_indices must be a one-dimensional boolean tensor')
    if cum_seqlens is None or cum_seqlens.ndim != 1 or cum_seqlens.numel() < 2:
        raise ValueError('Outcome credit requires packed sequence boundaries')
    if cum_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError('Sequence boundaries must use an integer dtype')
    if cum_seqlens.device != masked_indices.device:
        raise ValueError('Sequence boundaries and mask must share a device')
    bounds = cum_seqlens.tolist()
    if bounds[0] != 0 or bounds[-1] != masked_indices.numel():
        raise ValueError('Sequence boundaries must cover the actual packed stream')
    if any(b < a for a, b in zip(bounds, bounds[1:])):
        raise ValueError('Sequence boundaries must be nondecreasing')


def masked_sequence_ids(masked_indices, cum_seqlens):
    """Sequence index of every masked row, in row order (alodlm/credit.py:7-21:
    bucketize(arange(N), cum_seqlens[1:], right=True)[masked])."""
    check_sequence_boundaries(masked_indices, cum_seqlens)
    _require_gpu(masked_indices, "masked_sequence_ids")
    rows = masked_indices.numel()
    bounds = cum_seqlens.to(torch.int64).contiguous()
    out = torch.empty(rows, dtype=torch.int64, device=masked_indices.device)
    count = torch.empty(1, dtype=torch.int64, device=masked_indices.device)
    mask = masked_indices.contiguous().view(torch.uint8)
    call("alodlm_masked_sequence_ids", ptr(mask), ptr(bounds), bounds.numel() - 1, rows,
         ptr(out), ptr(count), _lib.stream_handle(masked_indices.device))
    return out[:int(count.item())]


class _SequenceScore(torch.autograd.Function):
    @staticmethod
    def forward(ctx, credit, log_prob, sequence_ids, sequence_count):
        n = credit.numel()
        dev = credit.device
        value = torch.empty(1, dtype=torch.float32, device=dev)
        dlogq = torch.empty(n, dtype=torch.float32, device=dev)
        ws = torch.empty(2 * sequence_count, dtype=torch.float32, device=dev)
        c32 = credit.detach().to(torch.float32).contiguous()
        q32 = log_prob.detach().to(torch.float32).contiguous()
        ids = sequence_ids.contiguous()
        call("alodlm_sequence_score", ptr(c32), ptr(q32), ptr(ids), n, sequence_count,
             ptr(value), ptr(dlogq), ptr(ws), _lib.stream_handle(dev))
        ctx.save_for_backward(dlogq)
        ctx.dtype = log_prob.dtype
        return value[0].to(log_prob.dtype)

    @staticmethod
    def backward(ctx, grad):
        (dlogq,) = ctx.saved_tensors
        return None, (dlogq * grad.to(torch.float32)).to(ctx.dtype), None, None


def sequence_score_function(credit, log_prob, sequence_ids, sequence_count):
    """dot(segment_sum(credit.detach()), segment_sum(log_prob)) / len(credit)
    (alodlm/credit.py:23-40); differentiable in ``log_prob``."""
    if credit.ndim != 1 or log_prob.shape != credit.shape or sequence_ids.shape != credit.shape:
        raise ValueError('Credit, log probabilities, and sequence IDs must be equal-length vectors')
    if sequence_ids.dtype != torch.int64 or sequence_count < 1:
        raise ValueError('Sequence IDs must be int64 and sequence_count must be positive')
    if not credit.device == log_prob.device == sequence_ids.device:
        raise ValueError('Credit, log probabilities, and IDs must share a device')
    if credit.dtype != log_prob.dtype:
        raise ValueError('Credit and log probabilities must share a dtype')
    if credit.numel() == 0:
        return log_prob.sum() * 0
    if bool(((sequence_ids < 0) | (sequence_ids >= sequence_count)).any()):
        raise ValueError('Sequence IDs must be within the declared sequence count')
    _require_gpu(credit, "sequence_score_function")
    return _SequenceScore.apply(credit, log_prob, sequence_ids, int(sequence_count))


class TokenLogProbs(NamedTuple):
    """What ``token_log_probs`` returns."""
    log_prob: torch.Tensor  # float32 [rows]
    entropy: torch.Tensor  # float32 [rows]
    top_log_prob: torch.Tensor  # float32 [rows, top]
    top_ids: torch.Tensor  # int64 [rows, top]


MAX_TOP = 64


def _vocabulary_rows(logits):
    """The logits with a vocabulary in a row, and the rows' stride."""
    R, V = logits.shape
    row, column = logits.stride()
    if V == 1 or column == 1:
        if R < 2:  # one row's stride says nothing
            return logits, V
        if row >= V:
            return logits, row
    return logits.contiguous(), V


def _log_probs(logits, targets, top, inv_temperature, ignore_index):
    """The four results and the buffer that starts with the backward's statistics."""
    R, V = logits.shape
    dev = logits.device
    x, ld = _vocabulary_rows(logits)
    log_prob = torch.empty(R, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(log_prob)
    top_log_prob = torch.empty(R, top, dtype=torch.float32, device=dev)
    top_ids = torch.empty(R, top, dtype=torch.int64, device=dev)
    # statistics [R, 2], then the workspace (8-byte aligned)
    buf = torch.empty(2 * R + query("alodlm_token_log_probs_workspace", R, V, top),
                      dtype=torch.float32, device=dev)
    stats = buf.data_ptr()
    call_on(dev, "alodlm_token_log_probs", x.data_ptr(), ld, targets.data_ptr(), R, V, top,
            inv_temperature, ignore_index, log_prob.data_ptr(), entropy.data_ptr(), stats,
            top_log_prob.data_ptr(), top_ids.data_ptr(), stats + 8 * R, _lib.dtype_code(x.dtype))
    return log_prob, entropy, top_log_prob, top_ids, buf


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, inv_temperature, ignore_index):
        *outs, buf = _log_probs(logits, targets, top, inv_temperature, ignore_index)
        ctx.save_for_backward(logits, targets, outs[3], outs[1], buf)
        ctx.args = top, inv_temperature, ignore_index
        ctx.mark_non_differentiable(outs[3])
        ctx.set_materialize_grads(False)
        return tuple(outs)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_log_prob, d_entropy, d_top, _d_ids):
        logits, targets, top_ids, entropy, buf = ctx.saved_tensors
        top, inv_temperature, ignore_index = ctx.args
        R, V = logits.shape
        x, ld = _vocabulary_rows(logits)
        out = torch.empty(R, V, dtype=logits.dtype, device=logits.device)
        grads = [g if g is None or (g.dtype == torch.float32 and g.is_contiguous())
                 else g.to(torch.float32).contiguous() for g in (d_log_prob, d_entropy, d_top)]
        call_on(x.device, "alodlm_token_log_probs_bwd", ptr(x), ld, ptr(targets), ptr(top_ids),
                ptr(buf), ptr(entropy), *map(ptr, grads), R, V, top, inv_temperature, ignore_index,
                ptr(out), _lib.dtype_code(x.dtype))
        return out, None, None, None, None


def token_log_probs(logits, targets, top=0, temperature=1.0, ignore_index=-100):
    """Log probabilities of the tokens ``targets`` (int64 [rows]) under logits [rows,
    vocab] over ``temperature``, with each row's entropy and its ``top`` most likely
    tokens (up to 64, in order, the lower id first among equal logits) and their log
    probabilities: a ``TokenLogProbs``, all float32 but the ids.  Differentiable in
    ``logits``, through the entropies and the alternatives' log probabilities too;
    forward-mode derivatives are refused.

    A target of ``ignore_index`` has log probability 0 and no gradient; any other
    target outside the vocabulary gives NaN, in the gradient too unless the log
    probability takes no part.  A logit of -inf is a token that cannot
    be; in a row of nothing else the log_prob of a target in the vocabulary is -inf, the
    entropy 0 and, unless that is NaN as above, the gradient 0.
    A NaN in a row makes its results NaN.

    A backward that is captured into a graph must not find an eager autograd graph of the
    same logits alive (its nodes are tied to the eager stream): drop its outputs first."""
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError('Logits must be [rows, vocabulary]')
    _lib.dtype_code(logits.dtype)
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:1]:
        raise ValueError('Targets must be int64, one per row of logits')
    if targets.device != logits.device:
        raise ValueError('Targets and logits must share a device')
    if not 0 <= top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f'top must be between 0 and {MAX_TOP} and at most the vocabulary')
    if not 0 < temperature < float("inf"):
        raise ValueError('temperature must be positive and finite')
    ignored = _ignored_id(ignore_index)
    _refuse_tangents("token_log_probs", logits)
    _require_gpu(logits, "token_log_probs")
    args = logits, targets.contiguous(), int(top), 1.0 / temperature, ignored
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogProbs(*_TokenLogProbs.apply(*args))
    return TokenLogProbs(*_log_probs(*args)[:4])
