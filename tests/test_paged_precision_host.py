"""The bound of tests/paged_precision.py, on the CPU: probabilities of 16 bits keep it, and
ones whose second part is lost or belongs to other keys do not."""

import pytest
import torch

from tests.paged_oracle import attend
from tests.paged_precision import cancelling_values, fine_tolerance, product


@pytest.mark.parametrize("keys", [20, 45, 200, 700])
@pytest.mark.parametrize("dh", [64, 128])
def test_bound_tells_16_bits_from_8(keys, dh):
    g = torch.Generator().manual_seed(keys)
    v = cancelling_values(keys, 1, dh, g, torch.bfloat16)
    k = torch.randn(keys, 1, dh, generator=g).bfloat16()
    q = (0.5 * torch.randn(16, 1, dh, generator=g)).bfloat16()
    out, mag, size = attend(q, k.double(), v.double(), [keys] * 16, dh ** -0.5)
    tol = fine_tolerance(out, mag, size, keys, dh)
    worst = {}
    for low in ("kept", "lost", "moved"):
        got = torch.stack([product(k[:, 0].double() @ q[i, 0].double() * dh ** -0.5, v[:, 0], low)
                           for i in range(16)])[:, None]
        worst[low] = float(((got.double() - out).abs() / tol).max())
    assert worst["kept"] <= 1.0
    assert worst["lost"] > 1.5 and worst["moved"] > 1.5, worst
