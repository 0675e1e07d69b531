"""The vocabulary losses without a GPU: the oracle against autograd, what the entry points
refuse, and what the library's calls and size queries refuse."""

import math

import pytest
import torch

from alodlm_amd import _lib
from alodlm_amd.loss import MAX_KNOWN, distillation_loss, linear_cross_entropy, linear_distillation_loss
from tests.vocab_loss_oracle import divergence, targets_as_known, tokens

F32, BF16, I64 = torch.float32, torch.bfloat16, torch.int64


@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_oracle_against_autograd(temperature, rest):
    gen = torch.Generator().manual_seed(3)
    logits = (2 * torch.randn(9, 31, generator=gen, dtype=torch.float64)).requires_grad_()
    ids, log_q = tokens(9, 31, 6, gen, "cpu")
    ids[1] = torch.tensor([3, -1, 8, 1, 8, 30])  # one given twice
    log_q[1] = torch.tensor([-2.0, math.nan, -1.9, -3.0, -1.5, -2.5])
    loss, grad, _, _ = divergence(logits.detach(), ids, log_q, temperature, rest)
    total = 0.0
    for r in range(9):
        lp = (logits[r] / temperature).log_softmax(-1)
        known = [(int(i), math.exp(float(q))) for i, q in zip(ids[r], log_q[r]) if i >= 0]
        row = sum((q * (math.log(q) - lp[i]) for i, q in known), torch.zeros((), dtype=torch.float64))
        left = 1.0 - sum(q for _, q in known)
        if rest and known:
            others = [j for j in range(31) if j not in {i for i, _ in known}]
            row = row + left * (math.log(left) - lp[others].logsumexp(0))
        torch.testing.assert_close(row.detach(), loss[r], rtol=1e-12, atol=1e-12)
        total = total + row
    torch.testing.assert_close(torch.autograd.grad(total, logits)[0], grad, rtol=1e-10, atol=1e-12)


def test_oracle_cross_entropy():
    gen = torch.Generator().manual_seed(4)
    logits = torch.randn(7, 12, generator=gen, dtype=torch.float64)
    targets = torch.randint(0, 12, (7,), generator=gen)
    targets[3] = -100
    loss, _, _, _ = divergence(logits, *targets_as_known(targets), 1.0, False)
    torch.testing.assert_close(loss, torch.nn.functional.cross_entropy(logits, targets, reduction="none"))


def ids_and_q(R=4, K=3):
    return torch.zeros(R, K, dtype=I64), torch.full((R, K), -2.0)


@pytest.mark.parametrize("bad", [
    dict(logits=torch.zeros(4)), dict(logits=torch.zeros(4, 0)), dict(logits=torch.zeros(4, 9, dtype=torch.float16)),
    dict(ids=torch.zeros(4, 3, dtype=torch.int32)), dict(ids=torch.zeros(3, 3, dtype=I64)),
    dict(ids=torch.zeros(4, dtype=I64)), dict(ids=torch.zeros(4, 0, dtype=I64)),
    dict(ids=torch.zeros(4, MAX_KNOWN + 1, dtype=I64), q=torch.zeros(4, MAX_KNOWN + 1)),
    dict(q=torch.zeros(4, 2)), dict(q=torch.zeros(4, 3, dtype=BF16)), dict(q=torch.zeros(4, 3, requires_grad=True)),
    dict(ids=torch.zeros(4, 3, dtype=I64, device="meta")), dict(temperature=0.0), dict(temperature=-1.0),
    dict(temperature=math.inf), dict(temperature=math.nan), dict(reduction="batchmean"), dict()])
def test_distillation_refusals(bad):
    """(The last: tensors that are not on a GPU.)"""
    ids, q = ids_and_q()
    args = (bad.get("logits", torch.zeros(4, 9)), bad.get("ids", ids), bad.get("q", q))
    options = {k: v for k, v in bad.items() if k in ("temperature", "reduction")}
    with pytest.raises(ValueError):
        distillation_loss(*args, **options)
    if "logits" not in bad:
        with pytest.raises(ValueError):
            linear_distillation_loss(torch.zeros(4, 8), torch.zeros(9, 8), *args[1:], **options)


@pytest.mark.parametrize("bad", [
    dict(hidden=torch.zeros(4)), dict(weight=torch.zeros(9)), dict(weight=torch.zeros(9, 7)),
    dict(weight=torch.zeros(0, 8)), dict(hidden=torch.zeros(4, 0), weight=torch.zeros(9, 0)),
    dict(weight=torch.zeros(9, 8, dtype=BF16)), dict(hidden=torch.zeros(4, 8, dtype=torch.float64)),
    dict(weight=torch.zeros(9, 8, device="meta")), dict(targets=torch.zeros(4, dtype=torch.int32)),
    dict(targets=torch.zeros(3, dtype=I64)), dict(targets=torch.zeros(4, 1, dtype=I64)),
    dict(targets=torch.zeros(4, dtype=I64, device="meta")), dict(temperature=0.0), dict(reduction="max"), dict()])
def test_cross_entropy_refusals(bad):
    args = (bad.get("hidden", torch.zeros(4, 8)), bad.get("weight", torch.zeros(9, 8)),
            bad.get("targets", torch.zeros(4, dtype=I64)))
    with pytest.raises(ValueError):
        linear_cross_entropy(*args, **{k: v for k, v in bad.items() if k in ("temperature", "reduction")})


def library():
    if not _lib.LIBRARY.exists():
        pytest.skip("library not built (run python -m alodlm_amd.build)")


def distill(logits=16, ld=9, ids=16, q=16, rows=4, vocab=9, known=3, inv_t=1.0, reduction=0, loss=16, state=16, ws=16,
            dtype=0):
    return "alodlm_distillation", (logits, ld, ids, q, rows, vocab, known, inv_t, 1, reduction, loss, state, ws, dtype,
                                   None)


def distill_bwd(logits=16, ld=9, state=16, d_loss=16, rows=4, vocab=9, known=3, inv_t=1.0, reduction=0, out=16, dtype=0):
    return "alodlm_distillation_bwd", (logits, ld, state, d_loss, rows, vocab, known, inv_t, reduction, out, dtype, None)


def linear(hidden=16, ldh=8, weight=16, ldw=8, targets=16, ids=None, q=None, rows=4, vocab=9, width=8, known=1,
           inv_t=1.0, rest=0, reduction=0, loss=16, state=16, kept=None, ws=16, dtype=1):
    return "alodlm_linear_loss", (hidden, ldh, weight, ldw, targets, ids, q, rows, vocab, width, known, inv_t, -100, rest,
                                  reduction, loss, state, kept, ws, dtype, None)


def linear_bwd(hidden=16, ldh=8, weight=16, ldw=8, state=16, kept=None, d_loss=16, rows=4, vocab=9, width=8, known=1,
               inv_t=1.0, reduction=0, dh=16, dw=16, ws=16, dtype=1):
    return "alodlm_linear_loss_bwd", (hidden, ldh, weight, ldw, state, kept, d_loss, rows, vocab, width, known, inv_t,
                                      reduction, dh, dw, ws, dtype, None)


ALL = [distill, distill_bwd, linear, linear_bwd]


@pytest.mark.parametrize("make,bad", [(f, b) for f in ALL for b in (
    dict(rows=-1), dict(rows=1 << 24), dict(vocab=0), dict(vocab=1 << 30), dict(known=0), dict(known=257),
    dict(inv_t=0.0), dict(inv_t=-1.0), dict(inv_t=math.nan), dict(inv_t=math.inf), dict(inv_t=3e38), dict(reduction=3),
    dict(reduction=-1), dict(state=None))]
    + [(f, b) for f in ALL[:2] for b in (dict(ld=8), dict(logits=None), dict(rows=1 << 22, vocab=1 << 20, ld=1 << 20))]
    + [(distill, dict(ids=None)), (distill, dict(q=None)), (distill, dict(ws=None)), (distill, dict(loss=None)),
       (distill, dict(ws=20)), (distill_bwd, dict(d_loss=None)), (distill_bwd, dict(out=None))]
    + [(f, b) for f in ALL[2:] for b in (
        dict(dtype=2), dict(width=0), dict(width=1 << 20), dict(ldh=7), dict(ldw=7), dict(ldh=1 << 22), dict(hidden=None),
        dict(weight=None), dict(hidden=24), dict(weight=24), dict(ldh=12), dict(ldw=12), dict(ws=None), dict(ws=24),
        dict(rows=1 << 20, vocab=1000, kept=16), dict(rows=1 << 23, vocab=1 << 20))]
    + [(f, dict(dtype=0, **b)) for f in ALL[2:] for b in (dict(hidden=24), dict(weight=24), dict(ldh=10), dict(ldw=10))]
    + [(linear, dict(targets=None)), (linear, dict(known=2)), (linear, dict(rest=1)), (linear, dict(loss=None)),
       (linear_bwd, dict(d_loss=None)), (linear_bwd, dict(dh=24)), (linear_bwd, dict(dw=24))])
def test_library_refusals(make, bad):
    """Refused on the host: nothing is launched (and there may be no GPU)."""
    library()
    name, args = make(**bad)
    with pytest.raises(ValueError):
        _lib.call(name, *args)


def test_calls_without_rows_need_no_arrays():
    library()
    for make, none in ((distill, dict(logits=None, ids=None, q=None, loss=None, ws=None)), (distill_bwd, dict(logits=None, out=None)), (linear_bwd, dict(hidden=None, dh=None, dw=None)),
                       (linear, dict(hidden=None, weight=None, targets=None, loss=None))):
        name, args = make(rows=0, state=None, **none)
        _lib.call(name, *args)


def test_sizes():
    """Logits are kept up to 2^25 of them; a backward's workspace is bounded by pieces of
    the vocabulary, whatever that is."""
    library()
    q = _lib.query
    for dtype in (0, 1):
        assert q("alodlm_linear_loss_kept", 100, 151936, 2048, dtype) == 100 * 151936
        assert q("alodlm_linear_loss_kept", 3, 10007, 520, dtype) == 3 * 10008
        assert q("alodlm_linear_loss_kept", 4096, 151936, 2048, dtype) == 0
    small, large = (q("alodlm_linear_loss_bwd_workspace", 4096, V, 2048, 0, 1, 0, 1) for V in (1 << 18, 1 << 19))
    planes = 4 * 4096 * 2048  # of d_hidden: one or two a piece
    assert large - small <= 2 * 4 * planes
    assert small <= (512 << 20) // 4 + 9 * 2 * planes
    assert q("alodlm_linear_loss_workspace", 4096, 151936, 2048, 0, 1) == 2 * 4096 * 594
    assert q("alodlm_vocab_loss_state", 10, 20) == 4 + 10 * (8 + 80)


@pytest.mark.parametrize("make", [linear, linear_bwd])
@pytest.mark.parametrize("bad", [dict(width=12, ldh=16, ldw=16), dict(width=6, ldh=8, ldw=8, dtype=0)])
def test_library_takes_rows_of_whole_16_bytes(make, bad):
    library()
    name, args = make(**bad)
    with pytest.raises(ValueError, match="16 bytes"):
        _lib.call(name, *args)
