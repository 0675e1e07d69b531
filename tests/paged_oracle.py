"""A paged cache and its attention written plainly: every sequence is a list of tokens;
pages, codes and attention (in 64 bits) are derived from it."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def rotate(x, cos, sin):
    """x * cos + rotate_half(x) * sin in float32, every product and the sum rounded,
    then once to x's type."""
    if cos is None:
        return x
    a, b = x.float().chunk(2, -1)
    c, s = cos.to(x.dtype).float()[:, None], sin.to(x.dtype).float()[:, None]
    return (x.float() * c + torch.cat((-b, a), -1) * s).to(x.dtype)


def quantise(block):
    """[tokens, dh] -> (codes as float64, exponent) of a page and head."""
    x = block.double()
    finite = x[x.isfinite()]
    largest = float(finite.abs().max()) if finite.numel() else 0.0
    e = -100
    if largest > 0:
        e = max(math.ceil(math.log2(largest / 448.0) - 1e-9), -100)
        while largest > 448.0 * 2.0 ** e:
            e += 1
        while e > -100 and largest <= 448.0 * 2.0 ** (e - 1):
            e -= 1
    y = (x * 2.0 ** -e).float()  # exact: a power of two
    y = torch.where(x.isfinite(), y, torch.nan)
    return y.to(E4M3).double(), e


class OracleCache:
    """Token lists per slot-like sequence id; ``kept`` tokens are final."""

    def __init__(self, sequences, page, eight_bit):
        self.page, self.eight_bit = page, eight_bit
        self.k = [[] for _ in range(sequences)]  # kept tokens, [kv_heads, dh] in the model's type
        self.v = [[] for _ in range(sequences)]

    def tokens(self, b, extra_k=(), extra_v=()):
        """(K, V) float64 [tokens, kv_heads, dh] as the cache holds them: the kept
        tokens' whole pages in 8 bits, the others as they are."""
        kept = len(self.k[b])
        K, V = list(self.k[b]) + list(extra_k), list(self.v[b]) + list(extra_v)
        if not K:
            return None, None
        K, V = torch.stack(K).double(), torch.stack(V).double()
        if self.eight_bit:
            for p in range(kept // self.page):
                rows = slice(p * self.page, (p + 1) * self.page)
                for x in (K, V):
                    for h in range(x.shape[1]):
                        codes, e = quantise(x[rows, h])
                        x[rows, h] = codes * 2.0 ** e
        return K, V


def attend(q, K, V, limits, scale):
    """float64 attention of rows q [n, heads, dh] over tokens K, V [t, kv_heads, dh],
    row i seeing the first limits[i]; also sum p |v| and the largest sum |q k| and |s|
    (for the tolerances).  Hidden tokens take no part, whatever they hold."""
    n, heads, dh = q.shape
    out = torch.zeros(n, heads, dh, dtype=torch.float64)
    mag = torch.zeros_like(out)
    size = torch.zeros(n, heads, 1, dtype=torch.float64)
    for i in range(n):
        t = limits[i]
        if t <= 0 or K is None:
            continue
        group = heads // K.shape[1]
        for h in range(heads):
            k, v = K[:t, h // group], V[:t, h // group]
            s = (k @ q[i, h].double()) * scale
            p = (s - s.max()).softmax(0)
            out[i, h] = p @ v
            mag[i, h] = p @ v.abs()
            size[i, h] = scale * (k.abs() @ q[i, h].double().abs()).max()
    return out, mag, size


def attention_tolerance(out, mag, size, keys, dtype, dh):
    """A score is off by at most dh + 2 roundings to float32 of the sum of its
    products' magnitudes, which is the relative error of a probability, beside the
    exponential's few units; the sums over the keys add keys * 2^-24 each.  In bf16 the
    probabilities (above and below the fraction line) and the output are rounded to 8
    bits: half a step, 2^-8 each."""
    eps = 2.0 ** -24
    delta = (dh + 2) * eps * size + (16 + keys) * eps
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * out.abs() + 2 * (2.0 ** -8 + delta) * mag + 1e-30
    return eps * out.abs() + 2 * delta * mag + 1e-30
