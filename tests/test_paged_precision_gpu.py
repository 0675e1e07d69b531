"""Attention over pages with few columns a sequence: the probabilities of the second product
have 16 bits, which the bound of tests/paged_precision.py tells from 8."""

import pytest
import torch

from alodlm_amd.paged import paged_attention
from tests.helpers import log
from tests.paged_oracle import attend
from tests.paged_precision import cancelling_values, fine_tolerance
from tests.test_paged_gpu import Run

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.mark.parametrize("dh,page", [(128, 64), (64, 16), (128, 16), (64, 128)])
@pytest.mark.parametrize("eight_bit,rows", [
    (True, 1), (True, 13),  # the keys over the waves
    (True, 17), (True, 32),  # 16 columns a wave
    (False, 1), (False, 8), (False, 9), (False, 32)])
@pytest.mark.parametrize("tokens", [12, 37, 192, 660])
@pytest.mark.parametrize("final", [True, False])
def test_probabilities_of_16_bits(dh, page, eight_bit, rows, tokens, final):
    """Two heads a key/value head; whole tiles, tiles that not every row sees, open pages."""
    log(f"paged precision {dh} {page} {eight_bit} {rows} {tokens} {final}")
    run = Run(2, 4, 2, dh, BF16, page, eight_bit, tokens=tokens + 70, window=40, seed=tokens + rows)
    held = [tokens, tokens // 2]
    keys = [n + rows for n in held]
    k = [run.randn(n, 2, dh) for n in keys]
    v = [cancelling_values(n, 2, dh, run.g, BF16) for n in keys]
    old, new = ([torch.cat([t[part] for t, part in zip(x, parts)]).to(DEV) for x in (k, v)]
                for parts in ([slice(0, n) for n in held], [slice(n, None) for n in held]))
    run.cache.append(*old, run.batch(held))
    run.lengths = held
    batch = run.batch([rows, rows], final=final)
    run.cache.append(*new, batch)
    q = run.randn(2 * rows, 4, dh, scale=0.5)
    got = paged_attention(q.to(DEV), run.cache, batch).cpu()
    for b, n in enumerate(held):
        kept = keys[b] if final else n
        run.plain.k[b], run.plain.v[b] = list(k[b][:kept]), list(v[b][:kept])
        K, V = run.plain.tokens(b, list(k[b][kept:]), list(v[b][kept:]))
        mine = slice(b * rows, (b + 1) * rows)
        out, mag, size = attend(q[mine], K, V, [n + i + 1 for i in range(rows)], dh ** -0.5)
        off = ((got[mine].double() - out).abs() / fine_tolerance(out, mag, size, keys[b], dh)).max()
        assert float(off) <= 1.0, f"{float(off)} times the tolerance"
