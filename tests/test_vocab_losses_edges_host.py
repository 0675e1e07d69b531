"""The vocabulary losses' edges without a GPU: forward-mode derivatives and ignored ids
that do not fit the library's integers are refused, the backward's workspace is bounded
whatever the rows are."""

import pytest
import torch
from torch.autograd import forward_ad

from alodlm_amd import _lib
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


@pytest.mark.parametrize("ignore", [2 ** 63, 2 ** 64, 2 ** 64 + 5, -2 ** 63 - 1])
def test_ignored_ids_past_64_bits(ignore):
    """2^64 + 5 would be 5 to the library, a token."""
    with pytest.raises(ValueError, match="ignore_index"):
        linear_cross_entropy(torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=I64), ignore_index=ignore)
    for largest in (2 ** 63 - 1, -2 ** 63):
        with pytest.raises(ValueError, match="GPU|device"):
            linear_cross_entropy(torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=I64), ignore_index=largest)


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2)])
@pytest.mark.parametrize("H", [64, 2000, 2048, 4096])
@pytest.mark.parametrize("R", [1000, 4096, 8192, 16384, 32768, 65536, 131072])
def test_backward_workspace(R, H, dtype, size):
    """In bytes: what is held of the vocabulary at a time (half a GiB of the logits or their
    gradient; as much of a weight whose rows are copied), the sums of d_hidden (1 GiB or one
    float32 plane) and a quarter of a GiB for products that split their sums.  A plane for
    each piece would take 38 GiB for 65536 rows of width 4096, twice the logits' size."""
    if not _lib.LIBRARY.exists():
        pytest.skip("library not built (run python -m alodlm_amd.build)")
    GIB, V = 1 << 30, 151936
    for d_hidden, d_weight in ((1, 1), (1, 0), (0, 1)):
        used = 4 * _lib.query("alodlm_linear_loss_bwd_workspace", R, V, H, 0, d_hidden, d_weight, dtype)
        deep = -(-H // 64) * 64
        copies = 0 if dtype == 0 else (GIB // 2 if H % 64 else 0) + 2 * (R + 31) * deep
        assert used <= GIB // 2 + (max(GIB, 4 * R * H) if d_hidden else 0) + copies + GIB // 4
        if R >= 16384:
            assert used <= R * V * size // 2 + copies
