"""The training objective's public functions on the HIP kernels (drop-in for
alodlm/loss.py).

``outcome_loss(ce, gate_logits, depths, batch, config)`` returns the NELBO
denoising term plus the sequence score-function actor and the reference's
seven metrics (alodlm/loss.py:35-90); ``autoregressive_loss(logits, labels,
packed_boundaries)`` the count-weighted next-token cross-entropy of each
segment's clean stream (alodlm/loss.py:12-32).  Both are differentiable:
outcome_loss in ``ce`` (through the detached truncated stick) and in the gate
logits (through log q), autoregressive_loss in ``logits``.

``linear_cross_entropy(hidden, weight, targets)`` is the cross entropy of hidden states
times the output projection without the logits being kept;
``distillation_loss(logits, teacher_ids, teacher_log_probs)`` and
``linear_distillation_loss(hidden, weight, ...)`` the divergence from a teacher of which
each row's most likely tokens are known (``credit.token_log_probs(..., top=k)`` of the
teacher's logits), from the student's logits or from its hidden states.

The objective kernel accumulates in float32 where the reference's bf16 run
keeps the stick and the denoising sum in bf16; sums run in one workgroup in a
fixed order.
"""

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, call_on, ptr, query
from .credit import _ignored_id, _refuse_tangents, _require_gpu, _vocabulary_rows, check_sequence_boundaries

METRIC_KEYS = ("denoising", "actor", "sampled_mean_depth", "prediction_cost",
               "regularization_cost", "profile_mean_depth", "first_pass_halt_probability")


class _OutcomeLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ce, gates, depths, masked, mask_probability, boundaries, config):
        K, N = gates.shape
        dev = gates.device
        rows = torch.nonzero(masked).flatten()
        ce_full = torch.zeros(K, N, dtype=torch.float32, device=dev)
        ce_full[:, rows] = ce.detach().to(torch.float32)
        g32 = gates.detach().to(torch.float32).contiguous()
        exits = depths.to(torch.int32).contiguous()
        mask = masked.contiguous().view(torch.uint8)
        prob = mask_probability.to(torch.float32).contiguous()
        bounds = boundaries.to(torch.int64).contiguous()
        S = bounds.numel() - 1
        out = torch.empty(10, dtype=torch.float32, device=dev)
        dgate = torch.empty(K, N, dtype=torch.float32, device=dev)
        dce = torch.empty(K, N, dtype=torch.float32, device=dev)
        ws = torch.empty(query("alodlm_objective_workspace", N, S, K), dtype=torch.float32,
                         device=dev)
        call("alodlm_outcome_loss", ptr(g32), ptr(exits), ptr(mask), ptr(prob), ptr(ce_full),
             ptr(bounds), S, N, K, float(config.depth_prior_c), float(config.kl_beta_mi),
             float(config.kl_beta_marg), ptr(out), ptr(dgate), ptr(dce), ptr(ws),
             _lib.stream_handle(dev))
        ctx.save_for_backward(dgate, dce[:, rows])
        ctx.dtypes = (ce.dtype, gates.dtype)
        metrics = out[1:8].clone()
        ctx.mark_non_differentiable(metrics)
        return out[1] + out[2], metrics

    @staticmethod
    def backward(ctx, grad, _grad_metrics):
        dgate, dce = ctx.saved_tensors
        g = grad.to(torch.float32)
        ce_dtype, gate_dtype = ctx.dtypes
        return (dce * g).to(ce_dtype), (dgate * g).to(gate_dtype), None, None, None, None, None


def outcome_loss(ce, gate_logits, depths, batch, config):
    """Denoising + actor loss and metrics (alodlm/loss.py:35-90).

    ce [K, M] masked-token cross-entropies, ``gate_logits`` K tensors [N],
    ``depths`` [N] sampled exits in 1..K, ``batch`` with ``masked``,
    ``mask_probability`` and ``boundaries``; ``config`` a ModelConfig."""
    selected = batch.masked
    count = int(selected.sum())
    if count == 0:
        zero = ce.sum() + sum(g.sum() * 0 for g in gate_logits)
        return zero, {key: zero.detach() for key in METRIC_KEYS}
    check_sequence_boundaries(selected, batch.boundaries)
    _require_gpu(ce, "outcome_loss")
    if ce.shape != (config.max_depth, count) or len(gate_logits) != config.max_depth:
        raise ValueError("ce must be [max_depth, masked rows] with one gate tensor per depth")
    loss, metrics = _OutcomeLoss.apply(ce, torch.stack(list(gate_logits)), depths, selected,
                                       batch.mask_probability, batch.boundaries, config)
    return loss, dict(zip(METRIC_KEYS, metrics.unbind()))


class _AutoregressiveLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, sel, target, n_rows, R):
        dev, (N, V) = logits.device, logits.shape
        buf = torch.empty(R, V, dtype=logits.dtype, device=dev)
        src = logits.detach().contiguous()
        coef = torch.full((R,), 1.0 / R, dtype=torch.float32, device=dev)
        ce = torch.empty(R, dtype=torch.float32, device=dev)
        # ce[r] = logsumexp - logit[target] in float32 for bf16 logits too: rounding
        # each term to bf16 first adds up to 2^-9 of it, which the mean of a few
        # hundred terms leaves at about 5e-5 of the loss; buf <- (softmax - onehot) / R
        call("alodlm_cross_entropy_rows", ptr(src), ptr(sel), ptr(buf), ptr(target), ptr(coef),
             ptr(n_rows), R, V, ptr(ce), None, _lib.dtype_code(logits.dtype),
             _lib.stream_handle(dev))
        ctx.save_for_backward(buf, sel[:R])
        ctx.shape = (N, V)
        return ce.sum() / R

    @staticmethod
    def backward(ctx, grad):
        buf, sel = ctx.saved_tensors
        N, V = ctx.shape
        out = torch.empty(N, V, dtype=buf.dtype, device=buf.device)
        scale = grad.to(torch.float32).reshape(1)
        call("alodlm_spread_rows", ptr(buf), ptr(sel), sel.numel(), ptr(scale), ptr(out), N, V,
             _lib.dtype_code(buf.dtype), _lib.stream_handle(buf.device))
        return out, None, None, None, None


def autoregressive_loss(logits, labels, packed_boundaries):
    """Average next-token loss without crossing segments (alodlm/loss.py:12-32):
    clean row start + i of each dual-stream segment [start, end) predicts
    labels[start // 2 + 1 + i] (i < L - 1, L = (end - start) // 2); ignored
    labels (-100) do not count.  Returns a float32 scalar (0 with
    requires_grad when no target counts)."""
    _require_gpu(logits, "autoregressive_loss")
    N = logits.shape[0]
    bounds = packed_boundaries.to(device=logits.device, dtype=torch.int64).contiguous()
    lab = labels.to(device=logits.device, dtype=torch.int64).contiguous()
    sel = torch.empty(2 * N + 1, dtype=torch.int32, device=logits.device)
    target, n_rows = sel[N:2 * N], sel[2 * N:]
    call("alodlm_ar_rows", ptr(lab), ptr(bounds), bounds.numel() - 1, N, ptr(sel), ptr(target),
         ptr(n_rows), _lib.stream_handle(logits.device))
    R = int(n_rows.item())
    if R == 0:
        return torch.tensor(0.0, device=logits.device, requires_grad=True)
    return _AutoregressiveLoss.apply(logits, sel, target, n_rows, R)


MAX_KNOWN = 256
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _aligned_rows(t):
    """A matrix whose rows the kernels can take (elements of a row next to each other, whole
    16 bytes, 16-byte aligned), and their stride; rows of other widths have zeros behind them."""
    rows, width = t.shape
    step = 16 // t.element_size()
    if width % step:
        out = torch.zeros(rows, -(-width // step) * step, dtype=t.dtype, device=t.device)
        out[:, :width] = t
        return out, out.shape[1]
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, width
        stride = width if rows < 2 else t.stride(0)
        if t.stride(1) == 1 and stride >= width and stride % step == 0:
            return t, stride
    t = t.contiguous()
    return (t if t.data_ptr() % 16 == 0 else t.clone()), width


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device)


def _upstream(d_loss):
    if d_loss.dtype == torch.float32 and d_loss.is_contiguous():
        return d_loss
    return d_loss.to(torch.float32).contiguous()


@functools.lru_cache(maxsize=256)
def _distill_sizes(R, V, known):
    return query("alodlm_vocab_loss_state", R, known), query("alodlm_distillation_workspace", R, V)


def _distill(logits, ids, log_q, inv_temperature, rest, reduction):
    R, V = logits.shape
    dev = logits.device
    x, ld = _vocabulary_rows(logits)
    state, ws = _distill_sizes(R, V, ids.shape[1])
    loss = _floats(() if reduction else R, dev)
    # the state, then the workspace (8-byte aligned: the state's floats are even)
    buf = _floats(state + ws, dev)
    at = buf.data_ptr()
    call_on(dev, "alodlm_distillation", x.data_ptr(), ld, ids.data_ptr(), log_q.data_ptr(), R, V,
            ids.shape[1], inv_temperature, rest, reduction, loss.data_ptr(), at, at + 4 * state,
            _lib.dtype_code(x.dtype))
    return loss, buf


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, log_q, inv_temperature, rest, reduction):
        loss, state = _distill(logits, ids, log_q, inv_temperature, rest, reduction)
        ctx.save_for_backward(logits, state)
        ctx.args = ids.shape[1], inv_temperature, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        logits, state = ctx.saved_tensors
        R, V = logits.shape
        x, ld = _vocabulary_rows(logits)
        out = torch.empty(R, V, dtype=logits.dtype, device=logits.device)
        up = _upstream(d_loss)
        call_on(x.device, "alodlm_distillation_bwd", x.data_ptr(), ld, state.data_ptr(), up.data_ptr(),
                R, V, *ctx.args, out.data_ptr(), _lib.dtype_code(x.dtype))
        return out, None, None, None, None, None


@functools.lru_cache(maxsize=256)
def _linear_sizes(R, V, H, known, code, keep, dh, dw):
    """Floats of a call's state, kept logits, forward and backward workspaces."""
    kept = query("alodlm_linear_loss_kept", R, V, H, code) if keep else 0
    return (query("alodlm_vocab_loss_state", R, known), kept,
            query("alodlm_linear_loss_workspace", R, V, H, kept > 0, code),
            query("alodlm_linear_loss_bwd_workspace", R, V, H, kept > 0, dh, dw, code))


def _linear(hidden, weight, targets, ids, log_q, inv_temperature, ignore_index, rest, reduction, keep=False):
    V, dev = weight.shape[0], hidden.device
    known = 1 if ids is None else ids.shape[1]
    h, ldh = _aligned_rows(hidden)
    w, ldw = _aligned_rows(weight)
    (R, H), code = h.shape, _lib.dtype_code(h.dtype)
    state, kept, ws, _ = _linear_sizes(R, V, H, known, code, keep, True, True)
    loss, ws = _floats(() if reduction else R, dev), _floats(ws, dev)
    saved = _floats(state + kept, dev)  # (the state's floats are whole 16 bytes)
    at = saved.data_ptr()
    call_on(dev, "alodlm_linear_loss", h.data_ptr(), ldh, w.data_ptr(), ldw, ptr(targets), ptr(ids),
            ptr(log_q), R, V, H, known, inv_temperature, ignore_index, rest, reduction, loss.data_ptr(),
            at, at + 4 * state if kept else None, ws.data_ptr(), code)
    return loss, saved


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, *args):
        loss, saved = _linear(hidden, weight, *args, keep=True)
        ctx.save_for_backward(hidden, weight, saved)
        ids = args[1]
        ctx.args = 1 if ids is None else ids.shape[1], args[3], args[6]
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        hidden, weight, saved = ctx.saved_tensors
        width, V, dev = hidden.shape[1], weight.shape[0], hidden.device
        h, ldh = _aligned_rows(hidden)
        w, ldw = _aligned_rows(weight)
        (R, H), code = h.shape, _lib.dtype_code(h.dtype)
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = torch.empty(R, H, dtype=h.dtype, device=dev) if need_h else None
        # room for whole 32 rows: the kernels' tiles
        dw = (torch.empty if R else torch.zeros)(-(-V // 32) * 32, H, dtype=h.dtype, device=dev) if need_w else None
        state, kept, _, ws = _linear_sizes(R, V, H, ctx.args[0], code, True, need_h, need_w)
        ws, up, at = _floats(ws, dev), _upstream(d_loss), saved.data_ptr()
        call_on(dev, "alodlm_linear_loss_bwd", h.data_ptr(), ldh, w.data_ptr(), ldw, at,
                at + 4 * state if kept else None, up.data_ptr(), R, V, H, *ctx.args, ptr(dh), ptr(dw), ws.data_ptr(), code)
        if dw is not None:
            dw = dw[:V]
        if H != width:
            dh, dw = (g if g is None else g[:, :width].contiguous() for g in (dh, dw))
        return (dh, dw) + (None,) * 7


def _check_options(temperature, reduction):
    if not 0 < temperature < float("inf"):
        raise ValueError('temperature must be positive and finite')
    if reduction not in _REDUCTIONS:
        raise ValueError('reduction must be "none", "sum" or "mean"')


def _check_factors(hidden, weight):
    if hidden.ndim != 2 or weight.ndim != 2 or min(weight.shape) < 1 or hidden.shape[1] != weight.shape[1]:
        raise ValueError('Hidden states must be [rows, width] and the weight [vocabulary, width]')
    _lib.dtype_code(hidden.dtype)
    if weight.dtype != hidden.dtype or weight.device != hidden.device:
        raise ValueError('Hidden states and weight must share a dtype and a device')


def _check_teacher(x, teacher_ids, teacher_log_probs):
    if (teacher_ids.dtype != torch.int64 or teacher_ids.ndim != 2
            or teacher_ids.shape[0] != x.shape[0] or not 1 <= teacher_ids.shape[1] <= MAX_KNOWN):
        raise ValueError(f'Teacher ids must be int64 [rows, 1 to {MAX_KNOWN}]')
    if teacher_log_probs.dtype != torch.float32 or teacher_log_probs.shape != teacher_ids.shape:
        raise ValueError('Teacher log probabilities must be float32, one per id')
    if not teacher_ids.device == teacher_log_probs.device == x.device:
        raise ValueError('The teacher\'s tensors and the student\'s must share a device')
    if teacher_log_probs.requires_grad and torch.is_grad_enabled():
        raise ValueError('Teacher log probabilities have no gradient here: detach them')


def linear_cross_entropy(hidden, weight, targets, temperature=1.0, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the tokens ``targets`` (int64 [rows]) under the logits
    ``hidden`` [rows, width] times ``weight`` [vocabulary, width] transposed, over
    ``temperature``: float32, the mean over the rows whose target is not ``ignore_index``
    (0 if there is none), their sum, or with ``reduction="none"`` the rows' own.  The logits
    are not rounded, and more than 2^25 of them are not kept: the backward computes them
    again, a piece of the vocabulary at a time, in a workspace of half a GiB for the piece
    and, with a gradient in ``hidden``, up to 1 GiB (or once its size in float32, if that is
    more) for its sums.
    Differentiable in ``hidden`` and ``weight`` (either may be without gradient, which saves
    its product); forward-mode derivatives are refused.

    A row of ``ignore_index`` has loss 0 and no gradient; any other target outside the
    vocabulary makes its loss NaN, and its gradients where the loss takes part.  A row that
    takes no part (ignored, or of upstream gradient 0) may hold NaN where the weight has no
    gradient; the weight's is a product that multiplies such a row by 0.

    A backward that is captured into a graph must not find an eager autograd graph of the
    same leaves alive (its nodes are tied to the eager stream): drop its outputs first."""
    _check_factors(hidden, weight)
    if targets.dtype != torch.int64 or targets.shape != hidden.shape[:1]:
        raise ValueError('Targets must be int64, one per row of hidden states')
    if targets.device != hidden.device:
        raise ValueError('Targets and hidden states must share a device')
    _check_options(temperature, reduction)
    ignored = _ignored_id(ignore_index)
    _refuse_tangents("linear_cross_entropy", hidden, weight)
    _require_gpu(hidden, "linear_cross_entropy")
    args = (hidden, weight, targets.contiguous(), None, None, 1.0 / temperature, ignored, False,
            _REDUCTIONS[reduction])
    if (hidden.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _Linear.apply(*args)
    return _linear(*args)[0]


def distillation_loss(logits, teacher_ids, teacher_log_probs, temperature=1.0, rest=True, reduction="mean"):
    """Divergence of the student p = softmax(``logits`` / ``temperature``) ([rows,
    vocabulary]) from a teacher whose most likely tokens a row are ``teacher_ids`` (int64
    [rows, up to 256]) with log probabilities ``teacher_log_probs`` (float32, taken at the
    same temperature):

        sum_k q_k (log q_k - log p[id_k])  and with ``rest``  + q_r (log q_r - log p_r),

    all other tokens taken as one, q_r = max(0, 1 - sum_k q_k); where no other token can be
    (all are known, or their logits -inf) it takes no part: of a vocabulary that teacher and
    student mask alike, q_r is what rounding leaves of 1.  float32, the mean over the rows
    that have a teacher's token (0 if none has), their sum, or each row's with
    ``reduction="none"``.  Differentiable in ``logits``; forward-mode derivatives are refused.

    An id below 0 is no token (rows of fewer, down to none: loss 0 and no gradient); one
    given twice counts twice; one outside the vocabulary makes the row's loss NaN, and its
    gradient where the loss takes part.  A logit of -inf is a token that cannot be: the
    loss is inf where the teacher gives it probability.

    A backward that is captured into a graph must not find an eager autograd graph of the
    same logits alive (its nodes are tied to the eager stream): drop its outputs first."""
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError('Logits must be [rows, vocabulary]')
    _lib.dtype_code(logits.dtype)
    _check_teacher(logits, teacher_ids, teacher_log_probs)
    _check_options(temperature, reduction)
    _refuse_tangents("distillation_loss", logits, teacher_log_probs)
    _require_gpu(logits, "distillation_loss")
    args = (logits, teacher_ids.contiguous(), teacher_log_probs.contiguous(), 1.0 / temperature, bool(rest),
            _REDUCTIONS[reduction])
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distillation.apply(*args)
    return _distill(*args)[0]


def linear_distillation_loss(hidden, weight, teacher_ids, teacher_log_probs, temperature=1.0, rest=True,
                             reduction="mean"):
    """``distillation_loss`` of the logits ``hidden`` [rows, width] times ``weight``
    [vocabulary, width] transposed, without keeping them, as ``linear_cross_entropy``:
    differentiable in ``hidden`` and ``weight``."""
    _check_factors(hidden, weight)
    _check_teacher(hidden, teacher_ids, teacher_log_probs)
    _check_options(temperature, reduction)
    _refuse_tangents("linear_distillation_loss", hidden, weight, teacher_log_probs)
    _require_gpu(hidden, "linear_distillation_loss")
    args = (hidden, weight, None, teacher_ids.contiguous(), teacher_log_probs.contiguous(), 1.0 / temperature,
            0, bool(rest), _REDUCTIONS[reduction])
    if (hidden.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _Linear.apply(*args)
    return _linear(*args)[0]
