"""The paged cache and its attention where little else goes: inf among the values of
tiles that every row sees, rows that no sequence is given, probabilities of more than 8
bits."""

import math

import pytest
import torch

from alodlm_amd.paged import PagedBatch, paged_attention
from tests.helpers import log
from tests.paged_oracle import attend, attention_tolerance
from tests.test_paged_gpu import Run

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32

# rows of a sequence that take each kernel with 2 heads a key/value head: keys over the
# waves, 16 columns a wave, 32 columns a wave
KERNEL_ROWS = [1, 8, 20, 32, 33, 70]


@pytest.mark.parametrize("shape", [(4, 2, 128, BF16, 64, False), (4, 2, 64, BF16, 16, False),
                                   (4, 2, 128, F32, 64, False), (4, 2, 40, BF16, 32, False)])
@pytest.mark.parametrize("rows", KERNEL_ROWS)
@pytest.mark.parametrize("tokens", [330, 2100])
def test_infinite_values(shape, rows, tokens):
    """inf in a value that every row sees, first tiles and last, one chunk of keys and
    several: inf of its sign in its column, NaN where both signs or a NaN meet, the
    other columns as they are without it, whichever kernel takes the call."""
    log(f"paged inf {shape} {rows} {tokens}")
    heads, kv, dh, dtype = shape[:4]
    run = Run(2, *shape, tokens=tokens + 80)
    counts = [tokens, 100]
    k, v = (run.randn(sum(counts), kv, dh) for _ in range(2))
    v[5, :, 1] = math.inf
    v[130, :, 2] = -math.inf
    v[200, 0, 3], v[70, 0, 3] = math.inf, -math.inf
    v[tokens - 2, :, 4] = math.inf
    v[150, :, 5], v[7, :, 6], v[300, :, 6] = math.nan, math.inf, math.inf
    v[150, 1, 6] = math.nan
    run.cache.append(k.to(DEV), v.to(DEV), run.batch(counts))
    run.lengths = counts
    run.plain.k, run.plain.v = [list(k[:tokens]), list(k[tokens:])], [list(v[:tokens]), list(v[tokens:])]
    batch = run.batch([rows, rows])
    q, more_k, more_v = (run.randn(2 * rows, n, dh) for n in (heads, kv, kv))
    run.cache.append(more_k.to(DEV), more_v.to(DEV), batch)
    got = paged_attention(q.to(DEV), run.cache, batch).cpu().double()
    for b, n in enumerate(counts):
        mine = slice(b * rows, (b + 1) * rows)
        run.plain.k[b] += list(more_k[mine])
        run.plain.v[b] += list(more_v[mine])
        K, V = run.plain.tokens(b)
        limits = [n + i + 1 for i in range(rows)]
        # the columns with inf or NaN: plain sums have them too, the weights being positive
        ref, mag, size = attend(q[mine], K, V, limits, dh ** -0.5)
        fine = ref.isfinite()
        assert bool((~fine).any()) == (b == 0)
        assert torch.equal(got[mine].isnan(), ref.isnan())
        assert torch.equal(got[mine].isinf(), ref.isinf())
        assert torch.equal(got[mine].where(ref.isinf(), 0.0), ref.where(ref.isinf(), 0.0))
        tol = attention_tolerance(ref, mag, size, max(limits), dtype, dh)
        assert bool(((got[mine] - ref).abs() <= tol)[fine].all())


@pytest.mark.parametrize("shape,tokens,limit", [
    ((4, 2, 128, BF16, 64, True), 300, 1), ((4, 2, 128, BF16, 64, True), 300, 20), ((4, 2, 64, BF16, 16, False), 90, 70),
    ((4, 2, 128, F32, 64, False), 300, 5), ((4, 2, 128, F32, 64, True), 40, 40), ((2, 1, 24, BF16, 64, True), 300, 3),
    ((4, 2, 128, BF16, 64, True), 6000, 1), ((4, 2, 128, F32, 64, False), 6000, 2)])
def test_rows_that_no_sequence_is_given(shape, tokens, limit):
    """Rows before the first sequence, past max_rows and behind the last one: zero in a
    fresh result, left alone in a caller's."""
    log(f"paged rows of nobody {shape} {tokens} {limit}")
    heads, kv, dh, dtype = shape[:4]
    run = Run(4, *shape, tokens=tokens + 100)
    held = [tokens, 1, 0, tokens]
    T = sum(held)
    k, v = (run.randn(T, kv, dh).to(DEV) for _ in range(2))
    run.cache.append(k, v, run.batch(held))
    counts = [limit + 7, limit, 0, limit + 300]
    offsets = [3]
    for n in counts:
        offsets.append(offsets[-1] + n)
    rows = offsets[-1] + 5
    q, k, v = (run.randn(rows, n, dh).to(DEV) for n in (heads, kv, kv))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    batch = PagedBatch(run.table, ints(held), ints(offsets), rows=rows, max_rows=limit, slots=run.slots)
    run.cache.append(k, v, batch)
    mine = torch.zeros(rows, dtype=torch.bool)
    for at, n in zip(offsets, counts):
        mine[at:at + min(n, limit)] = True
    out = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    paged_attention(q, run.cache, batch, out=out)
    assert bool((out[~mine] == 7.0).all()) and bool((out[mine] != 7.0).any(-1).any(-1).all())
    for _ in range(3):
        # a fresh result tends to lie where the last tensor of its size was
        used = torch.full(q.shape, math.nan, dtype=dtype, device=DEV)
        del used
        fresh = paged_attention(q, run.cache, batch)
        assert not bool(fresh[~mine].any()) and torch.equal(fresh[mine], out[mine])
        fresh = paged_attention(q, run.cache, PagedBatch(run.table, ints(held), ints([rows] * 5), rows=rows,
                                                         max_rows=limit, slots=run.slots))
        assert not bool(fresh.any())
