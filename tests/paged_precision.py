"""How exact the attention over pages is where its probabilities have 16 bits: values
under which their roundings show, the bound, and the second product written plainly."""

import torch

UNIT = 2.0 ** -23  # of a float32 sum: a matrix instruction need not round to nearest


def cancelling_values(tokens, kv_heads, dh, g, dtype):
    """[tokens, kv_heads, dh]: 1 and -1 in two tokens of each dimension, else 0.  A row is
    the difference of two of its probabilities, in which their roundings stay."""
    v = torch.zeros(tokens, kv_heads, dh)
    for h in range(kv_heads):
        for d in range(dh):
            a, b = torch.randperm(tokens, generator=g)[:2]
            v[a, h, d], v[b, h, d] = 1.0, -1.0
    return v.to(dtype)


def fine_tolerance(out, mag, size, keys, dh):
    """For ``cancelling_values`` (mag: the sum of p |v|; size: the largest scaled sum of
    |q k|).  A bf16 is within half a step, 2^-8, of its number, so a probability in two parts
    is within 2^-8 of 2^-8: 2^-16.  A score's dh exact products are summed in as many
    steps; its scaling, the exponential's argument and the factors that bring waves, chunks
    and earlier maxima to one reference (their arguments are differences of scores) are 16
    more: that, relative to the probabilities.  Sums run over two parts a key, and over a
    step in 16 of rescaling: 3 a key bounds them; two keys have values, and all are in the
    denominator.  The output's own rounding is 2^-8 of it."""
    score = 2.0 ** -16 + (dh + 16) * UNIT * size
    return 2.0 ** -8 * out.abs() + (2 * score + (3 * keys + 6 + 64) * UNIT) * 1.01 * mag + 1e-30


def product(s, v, low, scale=1.0):
    """The kernels' second product for scores s [keys] (in base e) and values v [keys, dh]
    on the CPU, the sums in 64 bits: probabilities in bf16, with their rounding errors as
    bf16 (``low`` "kept"), without ("lost"), or with those of keys 8 further on ("moved")."""
    e = (s - s.max()).exp().float()
    hi = e.bfloat16()
    part = (e - hi.float()).bfloat16()
    if low == "lost":
        part = torch.zeros_like(part)
    elif low == "moved":
        part = part.roll(8)
    p = hi.double() + part.double()
    return (p @ v.double() / p.sum()).bfloat16()
