"""token_log_probs without a GPU: forward-mode derivatives and ignored ids that do not fit
the library's integers are refused."""

import pytest
import torch
from torch.autograd import forward_ad

from alodlm_amd.credit import token_log_probs


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    """With or without a gradient wanted, and under no_grad, which leaves tangents in force."""
    logits, targets = torch.randn(4, 9, requires_grad=grad), torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(logits, torch.ones(4, 9))
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode, pytest.raises(NotImplementedError, match="forward-mode"):
                token_log_probs(dual, targets, top=2)
        # where they are not in force, the call goes on to ask for a GPU
        with torch.inference_mode(), pytest.raises(ValueError, match="GPU|device"):
            token_log_probs(dual, targets, top=2)


@pytest.mark.parametrize("ignore", [2 ** 63, 2 ** 64, 2 ** 64 + 5, -2 ** 63 - 1])
def test_ignored_ids_past_64_bits(ignore):
    """2^64 + 5 would be 5 to the library, a token."""
    with pytest.raises(ValueError, match="ignore_index"):
        token_log_probs(torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64), ignore_index=ignore)
