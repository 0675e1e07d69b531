"""The vocabulary losses at their edges: operands past 2 GiB, pieces of the vocabulary that
add to one plane, upstream gradients that are NaN or inf.  Against 64 bits, with the
tolerances of test_vocab_losses_gpu.py."""

import math

import pytest
import torch

from alodlm_amd.loss import distillation_loss, linear_cross_entropy, linear_distillation_loss
from tests.helpers import log
from tests.test_vocab_losses_gpu import B, BF16, DEV, EPS, F32, check_linear, factors, generator, sizes
from tests.vocab_loss_oracle import divergence, targets_as_known, tokens

pytestmark = pytest.mark.gpu


def check_repeated(R, V, H, dtype, n=1000, seed=0):
    """R rows of which only n differ: row i is row i % n.  What 64 bits say of n rows holds for all."""
    hidden, weight, targets = factors(n, V, H, dtype, seed)
    at = torch.arange(R, device=DEV) % n
    h, w = hidden[at].requires_grad_(), weight.clone().requires_grad_()
    loss = linear_cross_entropy(h, w, targets[at], reduction="sum")
    gh, gw = torch.autograd.grad(loss, (h, w))
    del h
    loss = float(loss.detach())
    ids, log_q = targets_as_known(targets)
    h64, w64 = hidden.double(), weight.double()
    logits = h64 @ w64.T
    want, D, mass, p = divergence(logits, ids, log_q, 1.0, False)
    count = torch.bincount(at, minlength=n).double()
    # as in check_linear: a log probability's error, D's rounding, the products' sums
    noise = (H / 32 + 8) * EPS * (h64.abs().amax(-1) * w64.abs().sum(-1).amax())
    tol = sizes(logits, V, 1.0, noise)
    assert abs(loss - float((want * count).sum())) <= float(((tol + 8 * EPS * want) * count).sum()) + EPS * loss
    own = torch.zeros(n, V + 1, dtype=torch.float64, device=DEV).scatter_(1, torch.where(ids >= 0, ids, V), 1.0)[:, :V]
    size = p * mass[:, None] + own + mass[:, None] * torch.where(own > 0, 0.0, p)
    step = B if dtype == BF16 else 0.0
    one = B if dtype == BF16 else EPS
    far = 8 * (tol[:, None] + 2 * EPS) * size + step * D.abs()
    each, wide = D @ w64, (far + V / 32 * EPS * D.abs()) @ w64.abs()
    assert bool((gh == gh[:n][at]).all())
    assert bool(((gh[:n].double() - each).abs() <= wide + 2 * one * each.abs()).all())
    D, far = D * count[:, None], (far + R / 32 * EPS * D.abs()) * count[:, None]
    ref, wide = D.T @ h64, far.T @ h64.abs()
    off = (gw.double() - ref).abs()
    assert bool((off <= wide + 2 * one * ref.abs()).all())
    if dtype == BF16:
        rms = ((D * D).T @ (h64 * h64)).sqrt()
        assert float(off.norm()) <= B * (float(ref.norm()) + float(rms.norm()))


def test_gradients_past_4_gib():
    """2^23 rows: the logits' gradient of 256 tokens takes 4 GiB, and both its products must
    not wrap their 32-bit offsets (the last 8 tokens and 40 rows fill no tile)."""
    log("linear cross entropy 2^23 + 40 rows")
    check_repeated(2 ** 23 + 40, 200, 64, BF16)


@pytest.mark.parametrize("stride", [2 ** 19, 2 ** 22 - 8])
def test_rows_far_apart(stride):
    """Weight rows, and hidden rows, of more than 2 GiB from the first to the last: several
    launches a product, or several a part of one."""
    for R, V, which in ((90, 3000, 1), (3000, 40, 0)):
        log(f"linear cross entropy, rows {stride} apart, {R} x {V}")
        data = list(factors(R, V, 64, BF16))
        rows = data[which].shape[0]
        buf = torch.empty(rows * stride, dtype=BF16, device=DEV)
        data[which] = buf.as_strided((rows, 64), (stride, 1)).copy_(data[which])
        check_linear(*data, reduction="mean")
        check_linear(*data, reduction="none")
        del data, buf


# bf16 tiles of 128 and of 256 rows, float32 with and without tokens left over (the latter adds
# to the gradient itself); the planes of all pieces would be 1 to 2.3 GiB
@pytest.mark.parametrize("R,V,H,dtype", [(2 ** 20 + 100, 1000, 64, BF16), (300000, 2001, 512, BF16),
                                         (300000, 901, 512, F32), (300040, 896, 512, F32)])
def test_pieces_add_to_one_plane(R, V, H, dtype):
    log(f"linear cross entropy {R} x {V} x {H} {dtype}, one plane")
    check_repeated(R, V, H, dtype)


def check_wild_upstream(call, leaves, ignored):
    """call(leaves, reduction) -> loss; row i of leaves[0] is ignored where ignored[i]."""
    R = ignored.numel()
    grads = lambda reduction, up: torch.autograd.grad(call(leaves, reduction), leaves, up)
    up = torch.randn(R, generator=generator(R), device=DEV)
    clean = grads("none", torch.where(ignored, 0.0, up))
    for value in (math.nan, math.inf, -math.inf):
        for a, b in zip(grads("none", torch.where(ignored, value, up)), clean):
            assert torch.equal(a, b)
        for reduction in ("mean", "sum"):
            g = grads(reduction, torch.tensor(value, device=DEV))[0]
            assert not bool(g[ignored].any())
            assert not bool(g[~ignored].isfinite().all(1).any())


@pytest.mark.parametrize("R,V,H,dtype", [(300, 1500, 64, BF16), (300, 120001, 64, BF16), (40, 1500, 64, BF16),
                                         (40, 40000, 72, BF16), (20, 20000, 64, F32), (70, 900, 64, F32)])
def test_upstream_of_rows_that_are_ignored(R, V, H, dtype):
    """An ignored row has no gradient whatever its upstream gradient is: one a row (0 / 0 of a
    row's weight, say), or a reduced loss's."""
    log(f"wild upstream {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    check_wild_upstream(lambda x, reduction: linear_cross_entropy(*x, targets, reduction=reduction), (h, w),
                        targets == -100)
    ids, log_q = tokens(R, V, 3, generator(R), DEV)
    ids[::5] = -1
    ignored = (ids < 0).all(1)
    for rest in (True, False):
        check_wild_upstream(lambda x, reduction: linear_distillation_loss(*x, ids, log_q, rest=rest, reduction=reduction),
                            (h, w), ignored)
        z = (h @ w.T).detach().requires_grad_()
        check_wild_upstream(lambda x, reduction: distillation_loss(*x, ids, log_q, rest=rest, reduction=reduction), (z,),
                            ignored)
