"""token_log_probs at the places where its kernels' ranges meet, and in rows without a
token: the gradient of every column beside a border, whatever the row's alignment."""

import math

import pytest
import torch

from alodlm_amd.credit import token_log_probs
from tests.helpers import log
from tests.test_token_log_probs_gpu import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def border_columns(V, dtype):
    """The last nine columns, and those around every 16 KiB of a row (a workgroup's
    share of the gradient), as far as a row's alignment moves them."""
    step = 8192 if dtype == BF16 else 4096
    near = {c for k in range(step, V, step) for c in range(k - 9, k + 10)} | set(range(V - 9, V))
    return sorted(c for c in near if 0 <= c < V)


@pytest.mark.parametrize("dtype,V", [(BF16, 8193), (BF16, 8195), (BF16, 8199), (BF16, 16387), (BF16, 32769),
                                     (F32, 4097), (F32, 4098), (F32, 8193), (F32, 12291), (BF16, 8192), (F32, 4099)])
@pytest.mark.parametrize("own", ["target", "alternative"])
def test_gradient_beside_borders(dtype, V, own):
    """Nine rows, so that they start at every offset from a 16-byte boundary; a target,
    or the likeliest token, in each column beside a border."""
    log(f"token_log_probs borders {V} {dtype} {own}")
    R = 9
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.randn(R, V, generator=g, device=DEV).to(dtype)
    for c in border_columns(V, dtype):
        x = logits.clone()
        targets = torch.full((R,), c, device=DEV)
        if own == "alternative":
            x[:, c] = 9.0
            targets[:] = 1
        check(x, targets, 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_no_token_and_bad_targets(dtype):
    """Rows of -inf: the gradient is NaN where the log probability is (a target outside
    the vocabulary that takes part), else zero."""
    log(f"token_log_probs rows of no token {dtype}")
    targets = torch.tensor([3, 700, -1, -100, 699], device=DEV)
    bad = [False, True, True, False, False]
    x = torch.full((5, 700), -math.inf, dtype=dtype, device=DEV).requires_grad_()
    out = token_log_probs(x, targets, top=2)
    assert out.log_prob.isnan().tolist() == bad
    every, = torch.autograd.grad(out.log_prob.sum() + out.entropy.sum(), x, retain_graph=True)
    assert every.isnan().all(1).tolist() == bad and not bool(every[[0, 3, 4]].any())
    known = (targets >= 0) & (targets < 700)
    some, = torch.autograd.grad(torch.where(known, out.log_prob, 0).sum() + out.entropy.sum(), x)
    assert not bool(some.any())
