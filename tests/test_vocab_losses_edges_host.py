"""The vocabulary losses' edges without a GPU: forward-mode derivatives are refused."""

import pytest
import torch
from torch.autograd import forward_ad

from alodlm_amd.loss import distillation_loss, linear_cross_entropy, linear_distillation_loss

F32, I64 = torch.float32, torch.int64


def calls(hidden, weight, logits, log_q):
    targets, ids = torch.zeros(4, dtype=I64), torch.zeros(4, 3, dtype=I64)
    return {"cross": lambda: linear_cross_entropy(hidden, weight, targets),
            "distill": lambda: distillation_loss(logits, ids, log_q),
            "linear": lambda: linear_distillation_loss(hidden, weight, ids, log_q)}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call,dual", [("cross", 0), ("cross", 1), ("distill", 2), ("distill", 3), ("linear", 0),
                                       ("linear", 1), ("linear", 3)])
def test_tangents_are_refused(call, dual, grad):
    """With or without a gradient wanted, and under no_grad, which leaves tangents in force."""
    args = [torch.randn(4, 8), torch.randn(9, 8), torch.randn(4, 9), torch.full((4, 3), -2.0)]
    args[:3] = [x.requires_grad_(grad) for x in args[:3]]
    with forward_ad.dual_level():
        args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode, pytest.raises(NotImplementedError, match="forward-mode"):
                calls(*args)[call]()
        # where they are not in force, the call goes on to ask for a GPU
        with torch.inference_mode(), pytest.raises(ValueError, match="GPU|device"):
            calls(*args)[call]()
        args[dual] = forward_ad.unpack_dual(args[dual]).primal.detach()
        with pytest.raises(ValueError, match="GPU|device"):
            calls(*args)[call]()
