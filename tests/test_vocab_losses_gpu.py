"""linear_cross_entropy, distillation_loss and linear_distillation_loss against 64 bits:
losses, gradients (the formula and differences), few and many rows, odd sizes, pieces of
the vocabulary, tokens that are absent, given twice or outside, masked vocabularies, NaN,
strides, streams and graphs, and a run of them together.

Tolerances (EPS = 2^-24, half a float32 step).  A logit that the library computes is a sum
of `width` products in chains of 32 terms: off by at most (width / 32 + 8) EPS of the sum
of its terms' sizes, `noise`; logits in memory are exact.  Over the temperature it is
rounded twice more.  A sum over V exponentials in parts of at most V / 256 terms is off by
(V / 256 + 20) EPS of itself.  So a log probability is off by `tol` = 2 noise / T + (4 size +
V / 256 + 30) EPS, size the largest |logit| / T + 1; a loss by its mass times that, and by a
few EPS of its terms (q (|ln q| + |ln p|), their sum's EPS apiece).

A gradient in the logits is (mass p - q) and p is off by tol of itself.  bf16: one rounding,
half a step, 2^-8 of the value (B).  Products of a rounded D: each product's term carries its
own rounding, so with random signs an element is off by B times the root of its terms' sum
of squares; the test bounds the whole's 2-norm by that (a rounding's root mean square is
1 / sqrt 3 of its bound), and each element by the sum of its terms' bounds."""

import math

import pytest
import torch

from alodlm_amd.credit import token_log_probs
from alodlm_amd.loss import distillation_loss, linear_cross_entropy, linear_distillation_loss
from tests.helpers import log
from tests.vocab_loss_oracle import divergence, reduced, targets_as_known, tokens, upstream

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
EPS, B = 2.0 ** -24, 2.0 ** -8


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def sizes(logits, V, temperature, noise):
    finite = torch.where(logits.abs() < 1e30, logits.double(), 0.0)
    return 2 * noise / temperature + (4 * (finite.abs().amax(-1) / temperature + 1) + V / 256 + 30) * EPS


def check_losses(got, want, ids, log_q, tol, mass, reduction):
    q = torch.where(ids >= 0, log_q.double().exp(), 0.0)
    terms = torch.where(q > 0, q * log_q.double().abs(), 0.0).sum(-1) + want.abs() + mass + 1
    off = mass * tol + (ids.shape[1] + 8) * EPS * terms
    if reduction != "none":
        n = max(int((ids >= 0).any(-1).sum()), 1) if reduction == "mean" else 1
        want, off = reduced(want, ids, reduction), off.sum() / n
        off = off + 2 * EPS * want.abs()
    assert got.dtype == F32 and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= off).all()), float((got.double() - want).abs().max())


def check_distill(logits, ids, log_q, temperature=1.0, rest=True, reduction="none", grad=True, seed=0):
    R, V = logits.shape
    want, dz, mass, p = divergence(logits.detach(), ids, log_q, temperature, rest)
    x = logits.detach().requires_grad_(grad)
    got = distillation_loss(x, ids, log_q, temperature=temperature, rest=rest, reduction=reduction)
    tol = sizes(logits, V, temperature, 0.0)
    check_losses(got, want, ids, log_q, tol, mass, reduction)
    if not grad:
        return
    up = torch.randn(got.shape, generator=generator(seed), device=DEV)
    g, = torch.autograd.grad(got, x, up)
    assert g.dtype == logits.dtype and g.shape == logits.shape
    row = upstream(ids, reduction, up)[:, None]
    ref = dz * row
    # mass p, q and the rest's share each have their own error
    err = (8 * tol[:, None] * p * mass[:, None] + 8 * EPS * (dz * temperature).abs()) / temperature * row.abs()
    own = torch.zeros(R, V + 1, dtype=torch.float64, device=DEV)
    q = torch.where(ids >= 0, log_q.double().exp(), 0.0)
    own.scatter_add_(1, torch.where(ids >= 0, ids, V), q)
    among = own[:, :V] > 0
    left = torch.where(among, 0.0, p).sum(-1, keepdim=True)
    part = torch.where(among, 0.0, p) / left.clamp(min=1e-300)
    q_rest = (mass - q.sum(-1)).clamp(min=0)[:, None]
    err = err + (8 * EPS * own[:, :V] + 4 * (tol[:, None] + EPS) * part * q_rest) / temperature * row.abs()
    if logits.dtype == BF16:
        err = err + B * ref.abs()
    assert bool(((g.double() - ref).abs() <= err + 1e-30).all())


def make(R, V, K, dtype, seed=0, scale=2.5):
    gen = generator(seed + R + V)
    logits = scale * torch.randn(R, V, generator=gen, device=DEV)
    ids, log_q = tokens(R, V, K, gen, DEV)
    lift = torch.where(ids >= 0, 5.0 + log_q, 0.0)
    logits.scatter_add_(1, ids.clamp(min=0), lift)
    return logits.to(dtype), ids, log_q


SHAPES = [(1, 1, 1), (3, 2, 1), (5, 11, 4), (2, 300, 256), (7, 1003, 5), (17, 8192, 20), (33, 64, 64),
          (4, 151936, 64), (2, 151937, 3), (600, 4099, 20), (2, 300001, 7), (530, 262145, 2)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V,K", SHAPES)
def test_distill_against_64_bits(R, V, K, dtype):
    log(f"distill {R} x {V} known {K} {dtype}")
    data = make(R, V, K, dtype)
    for rest in (True, False):
        check_distill(*data, rest=rest)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("temperature", [0.2, 1.5])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_temperature_and_reductions(dtype, temperature, reduction):
    log(f"distill temperature {temperature} {reduction} {dtype}")
    check_distill(*make(50, 3001, 9, dtype, seed=2), temperature, True, reduction)
    check_distill(*make(50, 3001, 9, dtype, seed=2), temperature, False, reduction, grad=False)


@pytest.mark.parametrize("K", [2, 5, 64, 65, 130, 256])
def test_tokens_given_twice(K):
    """Pairs, whole rows of one token, absent ones between them: every occurrence counts."""
    log(f"distill twice {K}")
    logits, ids, log_q = make(40, 1200, K, F32, seed=3)
    gen = generator(K)
    other = torch.randint(0, K, (40, K), generator=gen, device=DEV)
    ids = torch.where(torch.rand(40, K, generator=gen, device=DEV) < 0.5, ids.gather(1, other), ids)
    ids[1] = 77
    ids[2, ::2] = -1
    log_q = torch.where(log_q.isnan(), -9.0, log_q) - 1.0
    for rest in (True, False):
        check_distill(logits, ids, log_q, rest=rest)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", [(6, 900), (3, 151936), (520, 2001)])
def test_masked_vocabularies(R, V, dtype):
    """Few tokens that can be: all of them known (the rest takes no part), or not; the
    type's lowest value elsewhere; rows of which no token can be."""
    log(f"distill masked {R} x {V} {dtype}")
    logits, _, _ = make(R, V, 1, dtype, seed=4)
    live = torch.tensor([3, V // 3, V - 2, V // 2], device=DEV)
    keep = torch.zeros(R, V, dtype=torch.bool, device=DEV)
    keep[:, live] = True
    for low in (-math.inf, torch.finfo(dtype).min):
        x = torch.where(keep, logits, low)
        for known in (live[:3], live):
            ids = known.flip(0).repeat(R, 1)
            log_q = torch.tensor([0.5, 0.2, 0.1, 0.05], device=DEV)[:known.numel()].log().repeat(R, 1)
            ids[0, 1] = -1
            if known.numel() == 4 and low != -math.inf:
                ids[:, 3] = -1  # the rest's logit is finite
            for rest in (True, False):
                check_distill(x, ids, log_q, rest=rest)
    x = torch.full((R, V), -math.inf, dtype=dtype, device=DEV).requires_grad_()
    out = distillation_loss(x, ids, log_q, reduction="none")
    assert bool((out == math.inf).all())
    g, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert not bool(g.any())
    x = torch.full((R, V), torch.finfo(dtype).min, dtype=dtype, device=DEV)  # all alike
    check_distill(x, ids, log_q)
    # a token that the teacher gives probability and the student cannot give any
    x = logits.clone()
    x[:, live[0]] = -math.inf
    out = distillation_loss(x, live[:1].repeat(R, 1), torch.full((R, 1), -0.5, device=DEV), reduction="none")
    assert bool((out == math.inf).all())
    # and one that neither can be
    out = distillation_loss(x, live[:2].repeat(R, 1), torch.tensor([[-math.inf, -0.5]], device=DEV).repeat(R, 1),
                            reduction="none")
    want = divergence(x, live[1:2].repeat(R, 1), torch.full((R, 1), -0.5, device=DEV))[0]
    assert bool(((out.double() - want).abs() <= 4 * sizes(x, V, 1.0, 0.0)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_inf_and_tokens_outside(dtype):
    log(f"distill nan {dtype}")
    logits, ids, log_q = make(9, 5000, 3, dtype, seed=5)
    ids[:], log_q[:] = torch.tensor([17, 400, 4999], device=DEV), torch.tensor([-1.0, -2.0, -3.0], device=DEV)
    clean = distillation_loss(logits, ids, log_q, reduction="none")
    logits[1, 4000] = math.nan
    logits[2, 9] = math.inf
    logits[3, 400] = math.nan
    logits[4, 17] = math.inf
    ids[5, 1], ids[6, 0], log_q[7, 2] = 5000, 2 ** 40, math.nan
    x = logits.clone().requires_grad_()
    out = distillation_loss(x, ids, log_q, reduction="none")
    bad = torch.tensor([False] + [True] * 7 + [False], device=DEV)
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad].detach(), clean[~bad])
    g, = torch.autograd.grad(out, x, torch.ones(9, device=DEV), retain_graph=True)
    assert torch.equal(g.isnan().any(1), bad) and bool(g[5].isnan().all()) and bool(g[6].isnan().all())
    # a loss that takes no part: ids outside the vocabulary leave no trace
    g, = torch.autograd.grad(torch.where(bad, 0.0, out).sum(), x)
    assert not bool(g[5:7].any()) and bool(g[[0, 8]].isfinite().all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_without_tokens(reduction):
    log(f"rows without tokens {reduction}")
    logits, ids, log_q = make(5, 700, 3, F32, seed=6)
    ids[:] = -1
    x = logits.requires_grad_()
    out = distillation_loss(x, ids, log_q, reduction=reduction)
    assert not bool(out.any())
    assert not bool(torch.autograd.grad(out, x, torch.ones_like(out))[0].any())
    hidden, weight = torch.randn(70, 64, device=DEV).to(BF16), torch.randn(300, 64, device=DEV).to(BF16)
    for h, w in ((hidden, weight), (hidden.float(), weight.float())):
        h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
        out = linear_cross_entropy(h, w, torch.full((70,), 5, device=DEV), ignore_index=5, reduction=reduction)
        assert not bool(out.any())
        assert not any(bool(g.any()) for g in torch.autograd.grad(out, (h, w), torch.ones_like(out)))
        # no rows at all
        out = linear_cross_entropy(h[:0], w, torch.zeros(0, dtype=torch.int64, device=DEV), reduction=reduction)
        assert out.shape == ((0,) if reduction == "none" else ()) and not bool(out.any())
        gh, gw = torch.autograd.grad(out, (h, w), torch.ones_like(out))
        assert not bool(gh.any()) and gw.shape == w.shape and not bool(gw.any())
    out = distillation_loss(torch.zeros(0, 9, device=DEV).requires_grad_(), ids[:0], log_q[:0], reduction=reduction)
    assert out.shape == ((0,) if reduction == "none" else ()) and not bool(out.any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_strides(dtype):
    """Slices of wider buffers, row starts off every alignment, transposes, expanded rows."""
    log(f"distill strides {dtype}")
    wide, _, _ = make(6, 3001, 1, dtype, seed=7)
    gen = generator(8)
    for view in (wide[:, 1:2050], wide[:, :2048], wide[::2], wide[:, 7:], wide[:, :1000].t().contiguous().t(),
                 wide[:1].expand(6, 3001), wide[::2][:, ::3], wide.as_strided((1, 3001), (0, 1)), wide[:, 5:6],
                 wide[2:3, 1:4], wide.flip(0)[::2, 3:]):
        R, V = view.shape
        ids, log_q = tokens(R, V, min(4, V), gen, DEV)
        check_distill(view, ids, log_q)
        check_distill(view, ids.t().contiguous().t(), log_q.t().contiguous().t(), reduction="mean")
        both = torch.stack((ids, ids), -1)[..., 0]
        check_distill(view, both, log_q, grad=False)


def test_distill_against_differences():
    """Central differences along directions of largest size 1, step h.  The third derivative
    of a log probability along one is a third central moment of values in [-1, 1], at most 2;
    a row's loss has mass at most 2 of them.  Rounding adds the losses' errors over h."""
    log("distill differences")
    logits, ids, log_q = make(6, 23, 4, F32, seed=9)
    h = 2.0 ** -6
    for rest in (True, False):
        x = logits.clone().requires_grad_()
        out = distillation_loss(x, ids, log_q, rest=rest, reduction="none")
        g, = torch.autograd.grad(out, x, torch.ones(6, device=DEV))
        for s in range(4):
            d = 2 * torch.rand(6, 23, generator=generator(s), device=DEV) - 1
            lo, hi = (distillation_loss(logits + t * h * d, ids, log_q, rest=rest, reduction="none") for t in (-1, 1))
            off = ((g * d).sum(-1) - (hi - lo) / (2 * h)).abs()
            assert bool((off <= h * h / 6 * 2 * 2 + 200 * EPS * (1 + out.detach()) / h).all())


# ----------------------------------------------------------------------------
# From hidden states
# ----------------------------------------------------------------------------

def factors(R, V, H, dtype, seed=0):
    gen = generator(seed + R + V + H)
    hidden = torch.randn(R, H, generator=gen, device=DEV)
    weight = (2.5 * H ** -0.5 * torch.randn(V, H, generator=gen, device=DEV)).to(dtype)
    targets = torch.randint(0, V, (R,), generator=gen, device=DEV)
    hidden += torch.rand(R, 1, generator=gen, device=DEV) * weight[targets].float()
    targets[::6] = -100
    targets[0] = V - 1
    return hidden.to(dtype), weight, targets


def check_linear(hidden, weight, targets=None, ids=None, log_q=None, temperature=1.0, rest=True, reduction="mean",
                 grads=(True, True), seed=0):
    (R, H), V = hidden.shape, weight.shape[0]
    h, w = (x.detach().requires_grad_(g) for x, g in zip((hidden, weight), grads))
    if targets is not None:
        got = linear_cross_entropy(h, w, targets, temperature=temperature, reduction=reduction)
        ids, log_q = targets_as_known(targets)
        rest = False
    else:
        got = linear_distillation_loss(h, w, ids, log_q, temperature=temperature, rest=rest, reduction=reduction)
    up = torch.randn(got.shape, generator=generator(seed), device=DEV)
    leaves = [x for x in (h, w) if x.requires_grad]
    found = torch.autograd.grad(got, leaves, up) if leaves else []
    row = upstream(ids, reduction, up)
    h64, w64 = hidden.detach().double(), weight.detach().double()
    losses, masses, tols = [], [], []
    dh, dh_far, dh_rms = (torch.zeros(R, H, dtype=torch.float64, device=DEV) for _ in range(3))
    dw, dw_far, dw_rms = (torch.zeros(V, H, dtype=torch.float64, device=DEV) for _ in range(3))
    for r in range(0, R, 512):
        part = slice(r, r + 512)
        logits = h64[part] @ w64.T
        noise = (H / 32 + 8) * EPS * (h64[part].abs().amax(-1) * w64.abs().sum(-1).amax())
        loss, dz, mass, p = divergence(logits, ids[part], log_q[part], temperature, rest)
        tol = sizes(logits, V, temperature, noise)
        losses.append(loss), masses.append(mass), tols.append(tol)
        if not leaves:
            continue
        D = dz * row[part, None]
        q = torch.zeros(dz.shape[0], V + 1, dtype=torch.float64, device=DEV)
        q.scatter_add_(1, torch.where(ids[part] >= 0, ids[part], V), torch.where(ids[part] >= 0, log_q[part].double().exp(), 0.0))
        size = (p * mass[:, None] + q[:, :V] + mass[:, None] * torch.where(q[:, :V] > 0, 0.0, p)
                / torch.where(q[:, :V] > 0, 0.0, p).sum(-1, keepdim=True).clamp(min=1e-300)) / temperature * row[part, None].abs()
        # errors of D in every term, all of one sign; its rounding
        # (of up to 64 rows in two parts: the second's rounding)
        step = 0.0 if hidden.dtype != BF16 else B if R > 64 else B * B
        far = 8 * (tol[:, None] + 2 * EPS) * size + step * D.abs()
        far = far + (R + V) / 32 * EPS * D.abs()  # the products' sums
        dh[part] = D @ w64
        dh_far[part] = far @ w64.abs()
        dh_rms[part] = ((D * D) @ (w64 * w64)).sqrt()
        dw += D.T @ h64[part]
        dw_far += far.T @ h64[part].abs()
        dw_rms += (D * D).T @ (h64[part] ** 2)
    check_losses(got, torch.cat(losses), ids, log_q, torch.cat(tols), torch.cat(masses), reduction)
    wanted = [(dh, dh_far, dh_rms)] * grads[0] + [(dw, dw_far, dw_rms.sqrt())] * grads[1]
    for g, (ref, far, rms) in zip(found, wanted):
        assert g.dtype == hidden.dtype and g.shape == ref.shape
        one = B if hidden.dtype == BF16 else EPS
        off = (g.double() - ref).abs()
        assert bool((off <= far + 2 * one * ref.abs() + 1e-30).all())
        if hidden.dtype == BF16 and ref.numel() > 4000:
            assert float(off.norm()) <= B * (float(ref.norm()) + float(rms.norm()))
    return got, found


SMALL = [(1, 1, 8), (1, 31, 40), (3, 5, 64), (5, 33, 40), (7, 1000, 72), (64, 1003, 64), (65, 700, 64), (33, 300, 8),
         (300, 264, 128), (3, 9001, 132), (8, 20000, 64), (16, 1100, 1028), (24, 2051, 640), (32, 1200, 2052), (257, 2049, 192), (1000, 40, 256), (5, 40000, 64), (40, 33000, 136), (64, 151936, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V,H", SMALL)
def test_linear_cross_entropy(R, V, H, dtype):
    log(f"linear cross entropy {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    check_linear(hidden, weight, targets)
    check_linear(hidden, weight, targets, grads=(False, False), reduction="none")


@pytest.mark.parametrize("R,V,H,dtype", [
    (257, 131101, 64, BF16), (300, 151936, 128, BF16), (1000, 33601, 72, BF16), (4100, 70001, 64, BF16),
    (64, 600001, 64, BF16), (65, 524321, 8, BF16), (4100, 40001, 32, F32), (3, 12000001, 4, F32), (31, 1200001, 12, F32)])
def test_logits_that_are_not_kept(R, V, H, dtype):
    """More than 2^25 logits: computed twice, some in several pieces of the vocabulary."""
    log(f"linear not kept {R} x {V} x {H} {dtype}")
    assert R * V > 1 << 25
    hidden, weight, targets = factors(R, V, H, dtype)
    check_linear(hidden, weight, targets, reduction="mean")
    check_linear(hidden, weight, targets, reduction="none", temperature=0.7, grads=(True, False))


@pytest.mark.parametrize("R,V,H,dtype", [(300, 1500, 64, BF16), (300, 120001, 64, BF16), (40, 1500, 64, BF16),
                                         (300, 1501, 60, F32), (20, 30000, 64, F32)])
def test_rows_that_take_no_part_may_hold_nan(R, V, H, dtype):
    """Rows of NaN or infinite hidden states that are ignored, or whose loss has no upstream
    gradient, leave the others as they are and have no gradient themselves."""
    log(f"linear no part {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    up = torch.rand(R, device=DEV) + 0.5
    bad = torch.tensor([0, 3, 7, R - 1], device=DEV)
    targets[bad[:2]] = -100
    targets[bad[2:]] = 5
    up[bad[2:]] = 0.0
    wild = hidden.clone()
    wild[bad[0]], wild[bad[1], 3] = math.nan, math.inf
    wild[bad[2], 1], wild[bad[3]] = math.nan, -math.inf
    got = []
    for x in (hidden, wild):
        h = x.clone().requires_grad_()
        loss = linear_cross_entropy(h, weight, targets, reduction="none")
        g, = torch.autograd.grad(loss, h, up)
        got.append((loss.detach(), g))
    assert bool((got[1][0][bad[:2]] == 0).all())
    keep = torch.ones(R, dtype=torch.bool, device=DEV)
    keep[bad[2:]] = False
    assert torch.equal(got[0][0][keep], got[1][0][keep])
    assert torch.equal(got[0][1], got[1][1]) and bool((got[1][1][bad] == 0).all())
    # a teacher without tokens, the mean
    h = wild.clone()
    h[bad[2:]] = hidden[bad[2:]]
    h.requires_grad_()
    ids = torch.randint(0, V, (R, 3), device=DEV)
    ids[bad[:2]] = -1
    log_q = torch.full((R, 3), -2.0, device=DEV)
    out = linear_distillation_loss(h, weight, ids, log_q)
    g, = torch.autograd.grad(out, h)
    assert bool(out.isfinite()) and bool(g.isfinite().all()) and bool((g[bad[:2]] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V,H", [(3, 40, 1), (70, 900, 3), (20, 30000, 37), (90, 1003, 513), (300, 120001, 34)])
def test_rows_of_any_width(R, V, H, dtype):
    """Rows of any width, dense, in wider buffers and transposed; either gradient alone."""
    log(f"linear odd widths {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    _, (gh, gw) = check_linear(hidden, weight, targets)
    assert gh.is_contiguous() and gw.is_contiguous()
    wide = torch.full((V, H + 11), math.nan, dtype=dtype, device=DEV)
    wide[:, 5:5 + H] = weight
    for h, w, grads in ((hidden.t().contiguous().t(), wide[:, 5:5 + H], (True, False)), (hidden, weight, (False, True))):
        _, (g,) = check_linear(h, w, targets, grads=grads)
        assert torch.equal(g, gh if grads[0] else gw)


@pytest.mark.parametrize("R,V,H,dtype", [(3, 10000001, 64, BF16), (2, 9000003, 40, BF16), (2, 8500001, 4, F32)])
def test_kept_logits_of_several_pieces(R, V, H, dtype):
    """Few rows against a vocabulary whose gradient is taken in pieces and whose logits are
    kept whole, or computed in other pieces."""
    log(f"linear kept, pieces {R} x {V} x {H} {dtype}")
    assert R * V <= 1 << 25
    hidden, weight, targets = factors(R, V, H, dtype)
    check_linear(hidden, weight, targets, reduction="none", grads=(True, False))
    h, w = hidden.clone().requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets)
    assert torch.equal(loss, linear_cross_entropy(hidden, weight.detach(), targets))
    gw, = torch.autograd.grad(loss, w)
    rows = torch.cat([torch.arange(0, V, V // 7, device=DEV), targets[targets >= 0], torch.arange(V - 40, V, device=DEV)])
    lp = (hidden.double() @ weight.detach().double().T).log_softmax(-1)
    n = int((targets >= 0).sum())
    D = lp.exp()[:, rows] - (targets[:, None] == rows[None]).double()
    ref = (D * (targets >= 0)[:, None] / n).T @ hidden.double()
    one = B if dtype == BF16 else 64 * EPS
    size = (D.abs() * (targets >= 0)[:, None] / n).T @ hidden.double().abs()
    assert bool(((gw[rows].double() - ref).abs() <= 2 * one * size + 1e-30).all())


@pytest.mark.parametrize("temperature", [0.004, 0.05, 40.0])
@pytest.mark.parametrize("R,V", [(300, 120001), (90, 3000)])
def test_linear_temperatures(R, V, temperature):
    """Exponents of up to some thousands, and nearly flat ones.  (Logits of few values: the
    sums' own error over the temperature stays small.)"""
    log(f"linear temperature {temperature} {R} x {V}")
    gen = generator(R)
    hidden = torch.randint(-2, 3, (R, 64), generator=gen, device=DEV).to(BF16)
    weight = (torch.randint(-2, 3, (V, 64), generator=gen, device=DEV) / 16).to(BF16)
    targets = torch.randint(0, V, (R,), generator=gen, device=DEV)
    targets[::2] = (hidden[::2].float() @ weight.float().T).argmax(-1)
    ids, log_q = tokens(R, V, 5, gen, DEV)
    check_linear(hidden, weight, targets, temperature=temperature)
    check_linear(hidden, weight, ids=ids, log_q=log_q, temperature=temperature, reduction="none")


def test_more_than_2_to_the_31_elements():
    """Logits whose offsets pass 32 bits, and a weight whose offsets do: the last rows as by
    themselves."""
    log("vocabulary losses, long offsets")
    R, V = 14200, 151936
    gen = generator(5)
    logits = torch.empty(R, V, dtype=BF16, device=DEV)
    for r in range(0, R, 1000):
        logits[r:r + 1000] = (2.5 * torch.randn(min(1000, R - r), V, generator=gen, device=DEV)).to(BF16)
    first = torch.randint(0, V - 9, (R, 1), generator=gen, device=DEV)
    ids, log_q = first + 3 * torch.arange(3, device=DEV), torch.full((R, 3), -1.5, device=DEV)
    x = logits.requires_grad_()
    loss = distillation_loss(x, ids, log_q, reduction="none")
    g, = torch.autograd.grad(loss, x, torch.ones(R, device=DEV))
    for part in (slice(0, 600), slice(R - 600, R)):
        y = logits.detach()[part].clone().requires_grad_()
        own = distillation_loss(y, ids[part], log_q[part], reduction="none")
        assert torch.equal(own, loss[part])
        assert torch.equal(torch.autograd.grad(own, y, torch.ones(600, device=DEV))[0], g[part])
    del x, logits, loss, g, y, own
    R, V, H = 70, 560001, 4096
    hidden = torch.randn(R, H, generator=gen, device=DEV).to(BF16)
    weight = torch.empty(V, H, dtype=BF16, device=DEV)
    for v in range(0, V, 80000):
        weight[v:v + 80000] = (0.03 * torch.randn(min(80000, V - v), H, generator=gen, device=DEV)).to(BF16)
    targets = torch.randint(0, V, (R,), generator=gen, device=DEV)
    targets[:4] = torch.tensor([V - 1, V - 2, 0, 524289], device=DEV)
    # the same tokens in another order: the vocabulary's second half first
    order = torch.arange(V, device=DEV).roll(V // 2)
    h, w = hidden.clone().requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets, reduction="none")
    gh, gw = torch.autograd.grad(loss, (h, w), torch.ones(R, device=DEV))
    other = weight.detach()[order].requires_grad_()
    h2 = hidden.clone().requires_grad_()
    loss2 = linear_cross_entropy(h2, other, (targets + V // 2) % V, reduction="none")
    gh2, gw2 = torch.autograd.grad(loss2, (h2, other), torch.ones(R, device=DEV))
    # sums in another order: the vocabulary's error, twice, and a rounding of the gradients
    assert bool(((loss - loss2).abs() <= 2 * (V / 256 + 60) * EPS * (1 + loss.abs())).all())
    assert float((gh.double() - gh2.double()).norm()) <= 2 * B * float(gh.double().norm())
    for v in range(0, V, 80000):
        a, b = gw[order[v:v + 80000]].float(), gw2[v:v + 80000].float()
        assert float((a - b).norm()) <= B * float(a.norm())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H", [1, 3, 12, 36, 65, 130])
def test_widths_of_no_whole_16_bytes(H, dtype):
    log(f"linear width {H} {dtype}")
    check_linear(*factors(70, 531, H, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V,H,K", [(1, 40, 8, 40), (9, 500, 64, 3), (70, 3001, 72, 20), (200, 700, 64, 256), (300, 120001, 64, 33),
                                     (515, 65601, 128, 130)])
def test_linear_distillation(R, V, H, K, dtype):
    if dtype == F32 and R * V * H > 1 << 31:
        R = 40
    log(f"linear distillation {R} x {V} x {H} known {K} {dtype}")
    gen = generator(R + K)
    hidden, weight, _ = factors(R, V, H, dtype)
    ids, log_q = tokens(R, V, K, gen, DEV)
    ids[:, 0] = torch.where(ids[:, 0] >= 0, ids[:, K - 1].clamp(min=0), -1)  # given twice, in most rows
    log_q = torch.where(log_q.isnan(), -5.0, log_q) - 0.7
    check_linear(hidden, weight, ids=ids, log_q=log_q)
    check_linear(hidden, weight, ids=ids, log_q=log_q, rest=False, temperature=2.0, reduction="sum", grads=(False, True))


@pytest.mark.parametrize("R,V", [(300, 120001), (90, 1003)])
def test_linear_targets_outside_and_nan(R, V):
    log(f"linear nan {R} x {V}")
    hidden, weight, targets = factors(R, V, 64, BF16)
    targets[:] = 7
    clean = linear_cross_entropy(hidden, weight, targets, reduction="none")
    targets[1], targets[2], targets[3] = V, -1, 2 ** 40
    hidden[80, 5] = math.nan
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    out = linear_cross_entropy(h, w, targets, reduction="none")
    bad = torch.zeros(R, dtype=torch.bool, device=DEV)
    bad[1:4] = bad[80] = True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad].detach(), clean[~bad])
    gh, gw = torch.autograd.grad(out, (h, w), torch.ones(R, device=DEV), retain_graph=True)
    assert torch.equal(gh.isnan().all(1), bad) and bool(gw.isnan().all())
    assert bool(gh[~bad].isfinite().all())
    # without part in the loss, a target outside the vocabulary leaves no trace
    hidden[80, 5] = 0.5
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    out = linear_cross_entropy(h, w, targets, reduction="none")
    gh, gw = torch.autograd.grad(out[4:].sum(), (h, w))
    assert not bool(gh[:4].any()) and bool(gh.isfinite().all()) and bool(gw.isfinite().all())
    mean = linear_cross_entropy(h, w, targets)
    assert bool(mean.isnan())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", [(70, 900), (300, 120000), (10, 40000)])
def test_linear_strides(R, V, dtype):
    """Rows of wider buffers, rows off every alignment, transposes: the bits of the
    contiguous call."""
    if dtype == F32 and R * V > 1 << 22:
        V = 3000
    log(f"linear strides {R} x {V} {dtype}")
    hidden, weight, targets = factors(R, V, 64, dtype)
    want, grads = check_linear(hidden, weight, targets)

    def off(x, by):
        wide = torch.zeros(x.shape[0], x.shape[1] + 2 * by, dtype=dtype, device=DEV)
        wide[:, by:by + x.shape[1]] = x
        return wide[:, by:by + x.shape[1]]
    for h, w in ((off(hidden, 8), off(weight, 16)), (off(hidden, 3), off(weight, 5)),
                 (hidden.t().contiguous().t(), weight.t().contiguous().t()),
                 (torch.stack((hidden, hidden), 1)[:, 1], torch.stack((weight, weight), 1)[:, 0])):
        assert not (h.is_contiguous() or w.is_contiguous())
        got, found = check_linear(h, w, targets)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(found, grads))
    other = torch.stack((targets, targets), 1)[:, 1]
    assert torch.equal(linear_cross_entropy(hidden, weight, other), want.detach())


@pytest.mark.parametrize("R,V,H,dtype", [(90, 1003, 72, BF16), (300, 120001, 64, BF16), (30, 777, 20, F32)])
def test_each_gradient_alone_and_twice(R, V, H, dtype):
    log(f"linear gradients {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets)
    both = torch.autograd.grad(loss, (h, w), retain_graph=True)
    again = torch.autograd.grad(loss, (h, w), retain_graph=True)
    alone = (torch.autograd.grad(loss, h, retain_graph=True)[0], torch.autograd.grad(loss, w)[0])
    for a, b, c in zip(both, again, alone):
        assert torch.equal(a, b) and torch.equal(a, c)
    frozen = linear_cross_entropy(h, w.detach(), targets)
    assert torch.equal(frozen, loss) and torch.equal(torch.autograd.grad(frozen, h)[0], both[0])
    frozen = linear_cross_entropy(h.detach(), w, targets)
    assert torch.equal(torch.autograd.grad(frozen, w)[0], both[1])
    # an upstream gradient of 0, and of another sign and size
    zero = torch.autograd.grad(linear_cross_entropy(h, w, targets) * 0.0, (h, w))
    assert not any(bool(g.any()) for g in zero)
    scaled = torch.autograd.grad(linear_cross_entropy(h, w, targets) * -4.0, (h, w))
    assert all(torch.equal(a, -4.0 * b) for a, b in zip(scaled, both))


def test_linear_against_differences():
    """As for distillation_loss: a direction d in the hidden states moves the logits by
    d W^T, of largest size L; the third derivative is at most 2 L^3 and rounding adds the
    losses' errors over h.  In the weight alike (both factors at once leave the products
    bilinear: each alone)."""
    log("linear differences")
    gen = generator(21)
    hidden, weight = torch.randn(6, 12, generator=gen, device=DEV), 0.5 * torch.randn(23, 12, generator=gen, device=DEV)
    ids, log_q = tokens(6, 23, 4, gen, DEV)
    f = lambda h, w: linear_distillation_loss(h, w, ids, log_q, reduction="none")
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    out = f(h, w)
    step = 2.0 ** -6
    for r in range(6):
        gh, gw = torch.autograd.grad(out[r], (h, w), retain_graph=True)
        dh = 2 * torch.rand(6, 12, generator=gen, device=DEV) - 1
        dw = 2 * torch.rand(23, 12, generator=gen, device=DEV) - 1
        for g, d, move, L in ((gh, dh, lambda t: f(hidden + t * dh, weight), (dh @ weight.T).abs().max()),
                              (gw, dw, lambda t: f(hidden, weight + t * dw), (hidden @ dw.T).abs().max())):
            slope = (move(step)[r] - move(-step)[r]) / (2 * step)
            off = float(((g * d).sum() - slope).abs())
            assert off <= step ** 2 / 6 * 2 * 2 * float(L) ** 3 + 300 * EPS * (1 + float(out[r].detach())) / step


def captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    return graph, outs


@pytest.mark.parametrize("R,V,H,dtype", [(300, 120001, 64, BF16), (90, 1003, 72, BF16), (10, 40000, 64, BF16), (30, 777, 20, F32)])
def test_linear_graph(R, V, H, dtype):
    """Captured forward and backward, replayed on changing inputs: the eager bits."""
    log(f"linear graph {R} x {V} x {H} {dtype}")
    hidden, weight, targets = factors(R, V, H, dtype)
    h, w, t = hidden.clone().requires_grad_(), weight.clone().requires_grad_(), targets.clone()

    def step():
        loss = linear_cross_entropy(h, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, (h, w))]
    graph, outs = captured(step)
    for i in range(3):
        with torch.no_grad():
            h.copy_(hidden.roll(i, 0))
            w.copy_(weight.roll(i, 0))
            t.copy_(targets.flip(0) if i else targets)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


@pytest.mark.parametrize("R,V,K,dtype", [(3, 151936, 20, BF16), (600, 4001, 70, F32)])
def test_distill_graph_and_streams(R, V, K, dtype):
    log(f"distill graph {R} x {V} {dtype}")
    logits, ids, log_q = make(R, V, K, dtype, seed=11)
    log_q = log_q.nan_to_num(-3.0)
    x, i, q = logits.clone().requires_grad_(), ids.clone(), log_q.clone()

    def step():
        loss = distillation_loss(x, i, q)
        return [loss.detach(), *torch.autograd.grad(loss, x)]
    graph, outs = captured(step)
    for n in range(3):
        with torch.no_grad():
            x.copy_(logits.roll(n, 1))
            i.copy_(ids.roll(n, 0))
            q.copy_(log_q.roll(n, 0))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), n
    streams = [torch.cuda.Stream() for _ in range(3)]
    want = distillation_loss(logits, ids, log_q, reduction="none")
    hidden, weight, targets = factors(200, 9001, 64, BF16)
    other = linear_cross_entropy(hidden, weight, targets)
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append((distillation_loss(logits, ids, log_q, reduction="none"),
                            linear_cross_entropy(hidden, weight, targets)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, want) and torch.equal(b, other) for a, b in got)


def test_no_second_derivative():
    log("vocabulary losses second derivative")
    hidden, weight, targets = factors(5, 40, 8, F32)
    h = hidden.requires_grad_()
    g, = torch.autograd.grad(linear_cross_entropy(h, weight, targets), h, torch.ones((), device=DEV, requires_grad=True),
                             create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_teacher_and_student_together(dtype):
    """A teacher's logits give its likeliest tokens, which a student learns from: from its
    logits and from its hidden states alike, and next to the cross entropy."""
    log(f"teacher and student {dtype}")
    R, V, H = 130, 4000, 128
    hidden, weight, targets = factors(R, V, H, dtype, seed=31)
    with torch.no_grad():
        teacher = token_log_probs((hidden.float() @ weight.float().T).roll(1, 0), targets, top=16, temperature=2.0)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    known = dict(ids=teacher.top_ids, log_q=teacher.top_log_prob)
    check_linear(h, w, temperature=2.0, **known)
    logits = h.float() @ w.float().T
    direct = distillation_loss(logits, teacher.top_ids, teacher.top_log_prob, temperature=2.0)
    fused = linear_distillation_loss(h, w, teacher.top_ids, teacher.top_log_prob, temperature=2.0)
    cross = linear_cross_entropy(h, w, targets)
    scored = token_log_probs(logits, targets).log_prob
    noise = (H / 32 + 8) * EPS * float(h.abs().max() * w.abs().sum(-1).max())
    size = 4 * (float(logits.abs().max()) + 1) * EPS
    assert abs(float(direct) - float(fused)) <= 8 * (noise + size) + 100 * EPS * float(direct)
    mean = -float(scored.double().sum()) / int((targets >= 0).sum())
    assert abs(float(cross) - mean) <= 8 * (noise + size) + 100 * EPS * mean
    total = (fused + 0.5 * cross).detach()
    gh, gw = torch.autograd.grad(fused + 0.5 * cross, (h, w))
    with torch.no_grad():  # a small step against the gradient lowers the loss by its square
        rate = 1e-3 / float(gh.double().square().sum() + gw.double().square().sum())
        h2, w2 = (x.float() - rate * g.float() for x, g in ((h, gh), (w, gw)))
        after = (linear_distillation_loss(h2, w2, teacher.top_ids, teacher.top_log_prob, temperature=2.0)
                 + 0.5 * linear_cross_entropy(h2, w2, targets))
    assert float(after) < float(total)
