"""token_log_probs against 64 bits: values, entropies, alternatives (order and ties),
gradients against the formula and against differences, rows without a target, masked
vocabularies, NaN, strides, both row regimes (many rows, few long ones), streams and
graphs.

Float32 tolerances: a logit over the temperature is rounded once (2^-24 of its size),
the exponentials and logarithms are a few units off, and a sum over V terms, taken in
parts of at most V / 256, adds at most (V / 256 + 10) 2^-24 of itself in the worst case;
an entropy takes the sum's error times its terms' size.  bf16 gradients are rounded to 8
bits: half a step, 2^-8 of the value."""

import math

import pytest
import torch

from alodlm_amd.credit import token_log_probs
from tests.helpers import log

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
EPS = 2.0 ** -24


def reference(logits, targets, top, temperature):
    x = logits.double() / temperature
    lp = x.log_softmax(-1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    picked = lp.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    picked = torch.where(targets == -100, 0.0, picked)
    # the values' order, the lower index first among equal ones
    ids = torch.sort(logits.float().cpu(), dim=-1, descending=True, stable=True)[1][:, :top].to(logits.device)
    return lp, entropy, picked, ids


def gradient(lp, entropy, targets, ids, g_lp, g_h, g_top, temperature):
    g = torch.zeros_like(lp)
    given = targets != -100
    g.scatter_add_(1, targets.clamp(min=0)[:, None], (g_lp.double() * given)[:, None])
    if ids.shape[1]:
        g.scatter_add_(1, ids, g_top.double())
    p = lp.exp()
    return (g - p * g.sum(-1, keepdim=True) - g_h.double()[:, None]
            * torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)) / temperature


def check(logits, targets, top, temperature=1.0, grad=True, seed=0):
    R, V = logits.shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    lp, entropy, picked, ids = reference(logits.detach(), targets, top, temperature)
    x = logits.detach().requires_grad_(grad)
    out = token_log_probs(x, targets, top=top, temperature=temperature)
    assert torch.equal(x.detach(), logits.detach())
    size = (logits.double().abs().where(logits.abs() < 1e30, 0).amax(-1) / temperature + 1)
    tol = (3 * size + V / 256 + 20) * EPS
    assert bool(((out.log_prob.double() - picked).abs() <= tol + EPS * picked.abs()).all())
    spread = (lp.exp() * torch.where(lp > -math.inf, lp.abs(), 0.0)).sum(-1) + 1
    assert bool(((out.entropy.double() - entropy).abs() <= 4 * tol * spread).all())
    assert torch.equal(out.top_ids, ids)
    if top:
        want = lp.gather(1, ids)
        fine = want > -math.inf
        assert torch.equal(out.top_log_prob > -math.inf, fine)
        off = (out.top_log_prob.double() - want).where(fine, 0.0).abs()
        assert bool((off <= tol[:, None] + EPS * want.where(fine, 0.0).abs()).all())
    if not grad:
        return out
    up = [torch.randn(R, generator=g, device=DEV), torch.randn(R, generator=g, device=DEV),
          torch.randn(R, top, generator=g, device=DEV)]
    got = torch.autograd.grad(out[:3], x, up)[0]
    assert got.dtype == logits.dtype and got.shape == logits.shape
    ref = gradient(lp, entropy, targets, ids, *up, temperature)
    p = lp.exp()
    terms = (up[0].abs() + up[2].abs().sum(-1) + up[1].abs() * (spread + entropy)).double()[:, None]
    # each term of a gradient is off by its factors' errors; p by that of lp
    err = (8 * tol[:, None] * (p * (terms + up[1].abs()[:, None] * lp.abs().where(lp > -math.inf, 0.0)))
           + 4 * EPS * ref.abs() + 1e-30) / min(temperature, 1.0)
    at = torch.cat((targets.clamp(min=0)[:, None], ids), 1)
    err = err.scatter_add(1, at, (4 * EPS * terms / temperature).expand(R, at.shape[1]).contiguous())
    if logits.dtype == BF16:
        err = err + 2.0 ** -8 * ref.abs()
    assert bool(((got.double() - ref).abs() <= err).all())
    return out


def make(R, V, dtype, seed=0, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed + R + V)
    logits = (scale * torch.randn(R, V, generator=g, device=DEV)).to(dtype)
    targets = torch.randint(0, V, (R,), generator=g, device=DEV)
    targets[::7] = -100
    return logits, targets


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (3, 2, 0), (5, 11, 4), (2, 64, 64), (300, 1003, 5),
                                     (17, 8192, 20), (9, 10007, 33), (4, 151936, 20), (2, 151936, 64),
                                     (1, 151937, 1), (600, 4099, 0), (2, 300001, 7), (1030, 515, 64)])
def test_against_64_bits(R, V, top, dtype):
    log(f"token_log_probs {R} x {V} top {top} {dtype}")
    check(*make(R, V, dtype), top)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_temperature(temperature, dtype):
    log(f"token_log_probs temperature {temperature} {dtype}")
    check(*make(40, 2000, dtype, seed=2), 5, temperature)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", [(5, 700), (3, 40000), (2, 151936), (300, 1003)])
def test_ties(R, V, dtype):
    """Whole rows of one value, a few values, equal largest ones far apart, zeros of
    both signs: the lower index first."""
    log(f"token_log_probs ties {R} x {V} {dtype}")
    _, targets = make(R, V, dtype)
    g = torch.Generator(device=DEV).manual_seed(1)
    few = torch.randint(0, 3, (R, V), generator=g, device=DEV).to(dtype)
    far = torch.randn(R, V, generator=g, device=DEV).clamp(max=2).to(dtype)
    far[:, V - 1] = far[:, 5] = far[:, V // 2] = 9.0
    zeros = torch.zeros(R, V, dtype=dtype, device=DEV)
    zeros[:, ::3] = -0.0
    for logits in (torch.full((R, V), 1.5, dtype=dtype, device=DEV), few, far, zeros):
        check(logits, targets, 40, grad=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", [(4, 900), (3, 151936), (300, 2001)])
def test_masked_vocabularies(R, V, dtype):
    """Rows of which few tokens can be (-inf or the type's lowest value elsewhere),
    fewer than the alternatives asked for, and rows of none."""
    log(f"token_log_probs masked {R} x {V} {dtype}")
    for low in (-math.inf, torch.finfo(dtype).min):
        logits, targets = make(R, V, dtype, seed=4)
        keep = torch.zeros(R, V, dtype=torch.bool, device=DEV)
        keep[:, [3, V // 3, V - 2]] = True
        targets = torch.where(targets == -100, -100, torch.full_like(targets, V // 3))
        check(torch.where(keep, logits, low), targets, 8)
    logits = torch.full((R, V), -math.inf, dtype=dtype, device=DEV).requires_grad_()
    out = token_log_probs(logits, targets, top=5)
    assert torch.equal(out.log_prob.detach(), torch.where(targets == -100, 0.0, -math.inf))
    assert not bool(out.entropy.any()) and bool((out.top_log_prob == -math.inf).all())
    assert torch.equal(out.top_ids, torch.arange(5, device=DEV).expand(R, 5))
    grad = torch.autograd.grad(out[:3], logits, [torch.ones_like(t) for t in out[:3]])[0]
    assert not bool(grad.any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_inf_and_bad_targets(dtype):
    log(f"token_log_probs nan {dtype}")
    logits, targets = make(8, 5000, dtype, seed=3)
    targets[:] = 17
    clean = token_log_probs(logits, targets, top=3)
    logits[1, 4000] = math.nan
    logits[2, 9] = math.inf
    targets[4], targets[5], targets[6] = 5000, -1, -100
    out = token_log_probs(logits, targets, top=3)
    assert out.log_prob.isnan().tolist() == [False, True, True, False, True, True, False, False]
    assert out.entropy.isnan().tolist() == [False, True, True] + [False] * 5
    assert bool(out.top_log_prob[1].isnan().all()) and float(out.log_prob[6]) == 0.0
    for r in (0, 3, 7):
        assert all(torch.equal(a[r], b[r]) for a, b in zip(out, clean))
    assert bool(((out.top_ids >= 0) & (out.top_ids < 5000)).all())
    logits[1, :] = math.nan  # ids still name tokens, each once
    logits[2, 5:] = math.nan
    ids = token_log_probs(logits, targets, top=9).top_ids
    assert bool(((ids >= 0) & (ids < 5000)).all())
    assert all(len(set(row)) == 9 for row in ids.tolist())
    x = logits.clone().requires_grad_()
    out = token_log_probs(x, targets)
    grad = torch.autograd.grad(out.log_prob.nan_to_num().sum() + out.entropy.nan_to_num().sum(), x)[0]
    assert bool(grad[[0, 3, 7]].isfinite().all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_bad_targets(dtype):
    """NaN where a log probability that is NaN takes part, else the other outputs' own."""
    log(f"token_log_probs bad targets' gradient {dtype}")
    logits, targets = make(5, 700, dtype, seed=8)
    targets[:] = torch.tensor([3, 700, -1, -100, 699])
    x = logits.clone().requires_grad_()
    out = token_log_probs(x, targets)
    every, = torch.autograd.grad(out.log_prob.sum(), x, retain_graph=True)
    assert every.isnan().all(1).tolist() == [False, True, True, False, False]
    assert bool(every[[0, 3, 4]].isfinite().all()) and not bool(every[3].any())
    known = (targets >= 0) & (targets < 700)
    some, = torch.autograd.grad(torch.where(known, out.log_prob, 0).sum() + out.entropy.sum(), x, retain_graph=True)
    entropy, = torch.autograd.grad(out.entropy.sum(), x)
    assert bool(some.isfinite().all()) and torch.equal(some[[1, 2, 3]], entropy[[1, 2, 3]])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    """A slice of a wider buffer, a row start off every alignment, a transpose."""
    log(f"token_log_probs strides {dtype}")
    wide, targets = make(6, 3001, dtype, seed=6)
    for view in (wide[:, 1:2050], wide[:, :2048], wide[::2], wide[:, 7:],
                 wide[:, :1000].t().contiguous().t(), wide[:1].expand(6, 3001)):
        t = targets[:view.shape[0]].clamp(max=view.shape[1] - 1)
        got, want = (token_log_probs(x, t, top=4) for x in (view, view.contiguous()))
        assert torch.equal(got.top_ids, want.top_ids)
        for a, b in zip(got[:3], want[:3]):  # the order of the sums goes by the alignment
            assert bool(((a - b).abs() <= 60 * EPS * (1 + b.abs())).all())
        check(view, t, 4)
    check(wide[::2][:, ::3], targets[:3] % 1000, 3)
    for view in (wide.as_strided((1, 3001), (0, 1)), wide.as_strided((1, 1), (0, 0)), wide[:, 5:6],
                 wide[2:3, 1:4]):
        check(view, targets[:view.shape[0]].clamp(max=view.shape[1] - 1), 1)


def test_no_second_derivative():
    log("token_log_probs second derivative")
    logits, targets = make(3, 40, F32)
    x = logits.requires_grad_()
    up = torch.ones(3, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(token_log_probs(x, targets).entropy, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_rows_and_targets_left_alone():
    log("token_log_probs no rows")
    out = token_log_probs(torch.zeros(0, 50, device=DEV).requires_grad_(),
                          torch.zeros(0, dtype=torch.int64, device=DEV), top=2)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 2), (0, 2)]
    logits, _ = make(5, 800, F32)
    check(logits, torch.full((5,), -100, device=DEV), 0)
    x = logits.requires_grad_()
    out = token_log_probs(x, torch.zeros(5, dtype=torch.int64, device=DEV), top=3)
    for part in (out.log_prob, out.entropy, out.top_log_prob):  # one output's gradient alone
        g = torch.autograd.grad(part.sum(), x, retain_graph=True)[0]
        assert bool(g.isfinite().all()) and bool(g.any())
    assert not out.top_ids.requires_grad
    twice = [torch.autograd.grad(out.entropy.sum(), x, retain_graph=True)[0] for _ in range(2)]
    assert torch.equal(*twice)


def test_gradient_against_differences():
    """Central differences of the kernel's own float32 results along random
    directions of largest size 1, step h.  The third derivative of a log probability
    along such a direction is a third central moment of values in [-1, 1], at most 2 in
    size; of the entropy, with |lp| up to L, at most 8 L + 16.  Rounding adds the
    results' 2^-24 relative errors (32 of them allowed) over h."""
    log("token_log_probs differences")
    g = torch.Generator(device=DEV).manual_seed(12)
    R, V, h = 6, 13, 2.0 ** -6
    logits = (2 * torch.randn(R, V, generator=g, device=DEV))
    targets = torch.randint(0, V, (R,), generator=g, device=DEV)
    x = logits.clone().requires_grad_()
    out = token_log_probs(x, targets, top=2)
    grads = [torch.autograd.grad(t.sum(), x, retain_graph=True)[0]
             for t in (out.log_prob, out.entropy, out.top_log_prob[:, 1])]
    size = float(logits.double().log_softmax(-1).abs().max())
    for _ in range(5):
        d = 2 * torch.rand(R, V, generator=g, device=DEV) - 1
        lo, hi = (token_log_probs(logits + s * h * d, targets) for s in (-1, 1))
        second = [(logits + s * h * d).double().log_softmax(-1).gather(1, out.top_ids[:, 1:])[:, 0] for s in (-1, 1)]
        slopes = [(hi.log_prob - lo.log_prob) / (2 * h), (hi.entropy - lo.entropy) / (2 * h),
                  ((second[1] - second[0]) / (2 * h)).float()]
        for grad, slope, third in zip(grads, slopes, (2.0, 8 * size + 16, 2.0)):
            tol = h * h / 6 * third + 32 * EPS * (size + 1) / h
            assert bool((((grad * d).sum(-1) - slope).abs() <= tol).all())


def test_streams_and_graph():
    """Two streams at once and a captured call, forward and backward, replayed on
    changing logits: the eager bits."""
    log("token_log_probs streams, graph")
    data = [make(*shape, BF16, seed=s) for s, shape in enumerate([(3, 151936), (400, 5001), (2, 90001)])]
    want = [token_log_probs(*d, top=10) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(3):
        got = []
        for d, s in zip(data, streams):
            with torch.cuda.stream(s):
                got.append(token_log_probs(*d, top=10))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    for (logits, targets), n in zip(data, (3, 400, 2)):
        x = logits.clone().requires_grad_()
        up = torch.ones(n, device=DEV)

        def step():
            out = token_log_probs(x, targets, top=10)
            return [*out, *torch.autograd.grad([out.log_prob, out.entropy], x, [up, up])]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for i in range(3):
            with torch.no_grad():
                x.copy_(logits.roll(i, 1))
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i
