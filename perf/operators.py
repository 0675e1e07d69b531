"""Serving many requests at once: the paged key/value cache, the attention that reads
it, and the log probabilities of the tokens a model answered with.

* ``append`` - a step's keys and values of B sequences, rotated on the way, into their
  pages; the queries rotated beside them.  Pages are held in 8 bits (e4m3, one
  power-of-two scale per page, head and side; a page is sealed when its last token
  comes, younger tokens stay in open pages in the model's type) or in the model's type.
* ``attend`` - grouped-query attention of each sequence's new rows over its pages,
  causal among the new rows: one row per sequence (a decoding step), a window of rows
  that may be dropped again, or whole prompts of different lengths.
* ``logprob`` - log probabilities of given tokens, the entropy and the top
  alternatives of logits over the vocabulary, and the gradient in the logits.

Layouts: keys [pages, kv_heads, page, head_dim], values [pages, kv_heads, head_dim,
page] (tokens contiguous), exponents int8 [pages, 2 (keys, values), kv_heads], open
pages the same with [slots, open pages] in front; page p of a sequence, while open, is
open page p mod (open pages) of its slot.
"""

import math
import random
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda"
VOCAB, THETA = 151936, 1e6
# query heads, key/value heads, head_dim: the two configurations of bench.py
SHAPES = {"1.7b": (16, 8, 128), "8b": (32, 8, 128)}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
LOWEST = -100  # the smallest scale's exponent (and that of a page of zeros)


def listed():
    return [
        # a decoding step of 64 requests, one token each
        _paged("append_step", "append", "8b", 64, (100, 2000), (1, 1)),
        # the prompts of eight requests that came in together
        _paged("append_prompts", "append", "1.7b", 8, (0, 0), (300, 4000)),
        # decoding windows (committed and masked rows) behind prefixes kept in bf16
        _paged("append_windows", "append", "1.7b", 16, (50, 3000), (16, 32), store="bf16",
               final=False),
        # one request's decoding step early in its answer
        _paged("attend_one", "attend", "1.7b", 1, (299, 299), (1, 1)),
        # a decoding step of 64 requests of very different ages
        _paged("attend_step", "attend", "8b", 64, (200, 8000), (1, 1)),
        # one request with a very long context
        _paged("attend_long", "attend", "1.7b", 1, (130001, 130001), (1, 1)),
        # decoding windows of 16 requests, rows that the next pass rewrites
        _paged("attend_windows", "attend", "8b", 16, (300, 3100), (16, 27), final=False),
        # four prompts, attended to as they are written
        _paged("attend_prompts", "attend", "1.7b", 4, (0, 0), (700, 4100)),
        # a float32 model (the precision checkpoints are loaded in by default)
        _paged("attend_f32", "attend", "1.7b", 5, (30, 900), (1, 3), store="f32", dtype="f32"),
        # a decoding step's readout: eight rows, the tokens chosen and 20 alternatives
        _logprob("logprob_step", 8, VOCAB, 20, "bf16", False),
        # scoring and reinforcing answers: two 2048-token packs
        _logprob("logprob_train", 4096, VOCAB, 0, "bf16", True),
        # a small float32 vocabulary of odd size, gradients through the alternatives too
        _logprob("logprob_f32", 700, 10007, 5, "f32", True),
    ]


def _paged(name, kind, shape, sequences, lengths, rows, store="e4m3", dtype="bf16", final=True,
           page=64, ragged=1):
    nq, nkv, dh = SHAPES[shape] if isinstance(shape, str) else shape
    return {"name": name, "kind": kind, "heads": nq, "kv_heads": nkv, "head_dim": dh,
            "sequences": sequences, "shortest": lengths[0], "longest": lengths[1],
            "least_rows": rows[0], "most_rows": rows[1], "store": store, "dtype": dtype,
            "final": final, "page": page, "ragged": ragged}


def _logprob(name, rows, vocab, top, dtype, grad, temperature=1.0):
    return {"name": name, "kind": "logprob", "rows": rows, "vocab": vocab, "top": top,
            "dtype": dtype, "grad": grad, "temperature": temperature}


def draw(rng):
    """One more case of the listed ones' ranges."""
    log_int = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["append", "attend", "attend", "logprob"])
    if kind == "logprob":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        vocab = rng.choice([VOCAB, log_int(50, 150000)])
        most = (4096 if dtype == "bf16" else 1000) * VOCAB // vocab
        case = _logprob("", log_int(1, min(most, 8192)), vocab, rng.choice([0, 1, 5, rng.randint(1, 40)]),
                        dtype, rng.random() < 0.5, rng.choice([1.0, 1.0, 0.7, 1.6]))
    else:
        store, dtype = rng.choice([("e4m3", "bf16")] * 4 + [("bf16", "bf16"), ("e4m3", "f32"),
                                                            ("f32", "f32")])
        shape = rng.choice(["1.7b", "8b", (14, 2, 64), (8, 1, 128), (6, 6, 64)])
        page = rng.choice([16, 32, 64, 64, 128])
        form = rng.choice(["step", "step", "window", "prompt", "chunk"])
        far = log_int(20, 3000 if dtype == "f32" else 40000)
        if form == "step":
            n = log_int(1, max(1, min(96, 500000 // far)))
            case = _paged("", kind, shape, n, (rng.randint(0, far), far), (1, 1), store, dtype,
                          True, page)
        elif form == "window":
            n = log_int(1, max(1, min(24, 60000 // far)))
            case = _paged("", kind, shape, n, (rng.randint(0, far), far), (2, rng.randint(2, 40)),
                          store, dtype, rng.random() < 0.5, page)
        else:  # prompts, and chunks of prompts behind what is cached
            most = log_int(20, 600 if dtype == "f32" else 3000)
            before = (0, 0) if form == "prompt" else (0, log_int(1, 2000))
            case = _paged("", kind, shape, log_int(1, 6), before, (max(1, most // 8), most),
                          store, dtype, True, page)
        case["ragged"] = rng.randint(1, 10 ** 6)
    case.pop("name")
    return case


# ----------------------------------------------------------------------------
# What a case holds: lengths and rows of its sequences
# ----------------------------------------------------------------------------

def _open_pages(case):
    """Open pages of a slot: the page being filled and, for rows that may be dropped
    again, as many as a window reaches into."""
    rows = 1 if case["final"] else case["most_rows"]
    return max(2, (case["page"] - 1 + rows + case["page"] - 1) // case["page"])


def _sequences(case):
    """Tokens held before the step and rows of the step, per sequence.  The pages that
    a prompt fills are no multiple of the open pages, so that its last rows do not
    take the place of those it found open: a pass can be repeated on its state."""
    r = random.Random(case["ragged"])
    page, lengths, rows = case["page"], [], []
    for _ in range(case["sequences"]):
        lengths.append(r.randint(case["shortest"], case["longest"]))
        rows.append(r.randint(case["least_rows"], case["most_rows"]))
    lengths[-1], rows[0] = case["longest"], case["most_rows"]
    if case["kind"] == "append" and case["store"] == "e4m3" and case["final"]:
        for i, (length, n) in enumerate(zip(lengths, rows)):
            filled = (length + n) // page - length // page
            if filled and filled % _open_pages(case) == 0:
                rows[i] = n - page if n > page else n
    return lengths, rows


def _offsets(rows):
    offsets = [0]
    for n in rows:
        offsets.append(offsets[-1] + n)
    return offsets


# ----------------------------------------------------------------------------
# Inputs (from the seed alone)
# ----------------------------------------------------------------------------

def _pages(count, case, gen):
    """A pool of pages as ``append`` leaves them: normal keys and values, in 8 bits with
    the smallest power-of-two scale that holds a page's largest value."""
    nkv, dh, page = case["kv_heads"], case["head_dim"], case["page"]
    pool, exponents = [], []
    for shape in ((count, nkv, page, dh), (count, nkv, dh, page)):
        x = torch.randn(shape, generator=gen, device=DEVICE)
        if case["store"] == "e4m3":
            e = _exponent(x.abs().amax((-1, -2)))
            x = x.mul_(torch.exp2(-e.float())[..., None, None]).to(E4M3)
            exponents.append(e.to(torch.int8))
        else:
            x = x.to(DTYPES[case["store"]])
        pool.append(x)
    return (*pool, torch.stack(exponents, 1) if exponents else None)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case)
    if case["kind"] == "logprob":
        R, V = case["rows"], case["vocab"]
        s.logits = (2.5 * torch.randn(R, V, generator=gen, device=DEVICE)).to(dtype)
        s.targets = torch.randint(0, V, (R,), generator=gen, device=DEVICE)
        # an answer's own tokens are mostly likely ones; some rows carry no target
        likely = torch.rand(R, generator=gen, device=DEVICE) < 0.8
        s.targets = torch.where(likely, s.logits.argmax(-1), s.targets)
        s.targets[torch.rand(R, generator=gen, device=DEVICE) < 0.05] = -100
        s.d_log_prob = torch.randn(R, generator=gen, device=DEVICE)
        s.d_entropy = 0.01 * torch.randn(R, generator=gen, device=DEVICE)
        s.d_top = 0.1 * torch.randn(R, case["top"], generator=gen, device=DEVICE)
        s.logits.requires_grad_(case["grad"])
        return s
    nq, nkv, dh, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    lengths, rows = _sequences(case)
    s.most_rows, s.most_keys = max(rows), max(a + b for a, b in zip(lengths, rows))
    B, T, width = len(rows), sum(rows), -(-s.most_keys // page)
    used = [-(-(a + b) // page) for a, b in zip(lengths, rows)]
    s.keys, s.values, s.exponents = _pages(sum(used) + 3, case, gen)
    order = torch.randperm(sum(used) + 3, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    places = [(b, p) for b in range(B) for p in range(used[b])]
    at = torch.tensor(places, device=DEVICE)
    s.table = table.to(DEVICE)
    s.table[at[:, 0], at[:, 1]] = order[:len(places)]
    s.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    s.offsets = torch.tensor(_offsets(rows), dtype=torch.int32, device=DEVICE)
    s.open_keys = s.open_values = s.slots = None
    if case["store"] == "e4m3":
        shape = (B + 2, _open_pages(case), nkv)
        s.open_keys = torch.randn(*shape, page, dh, generator=gen, device=DEVICE).to(dtype)
        s.open_values = torch.randn(*shape, dh, page, generator=gen, device=DEVICE).to(dtype)
        s.slots = torch.randperm(B + 2, generator=gen, device=DEVICE)[:B].to(torch.int32)
    s.q = (2.0 * torch.randn(T, nq, dh, generator=gen, device=DEVICE)).to(dtype)
    if case["kind"] == "append":
        s.k = torch.randn(T, nkv, dh, generator=gen, device=DEVICE).to(dtype)
        s.v = torch.randn(T, nkv, dh, generator=gen, device=DEVICE).to(dtype)
        inverse = THETA ** (-torch.arange(0, dh, 2, device=DEVICE).double() / dh)
        angles = _positions(s)[1].double()[:, None] * torch.cat((inverse, inverse))
        s.cos, s.sin = angles.cos().to(dtype), angles.sin().to(dtype)
    if own:  # the handles that a program keeps: the cache, and a step's batch for all layers
        from alodlm_amd.paged import PagedBatch, PagedCache
        s.cache = PagedCache(s.keys, s.values, s.exponents, s.open_keys, s.open_values)
        s.batch = PagedBatch(s.table, s.lengths, s.offsets, max_rows=s.most_rows, slots=s.slots,
                             final=case["final"])
    return s


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------

def run(s):
    kind = s.case["kind"]
    if kind == "append":
        if own:
            q = s.cache.append(s.k, s.v, s.batch, cos=s.cos, sin=s.sin, q=s.q)
        else:
            q = _append(s)
        return [x for x in (q, s.keys, s.values, s.exponents, s.open_keys, s.open_values)
                if x is not None]
    if kind == "attend":
        if own:
            from alodlm_amd.paged import paged_attention
            return paged_attention(s.q, s.cache, s.batch)
        return _attend(s)
    if own:
        from alodlm_amd.credit import token_log_probs
        r = token_log_probs(s.logits, s.targets, top=s.case["top"],
                            temperature=s.case["temperature"])
        outs = [r.log_prob, r.entropy] + ([r.top_log_prob, r.top_ids] if s.case["top"] else [])
        if s.case["grad"]:
            down = [s.d_log_prob, s.d_entropy] + ([s.d_top] if s.case["top"] else [])
            outs += torch.autograd.grad(outs[:len(down)], s.logits, down)
        return [x.detach() for x in outs]
    return _log_probs(s)


# ----------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------

def _exponent(largest):
    """The smallest e >= LOWEST with largest <= 448 * 2^e (448 = 0.875 * 2^9)."""
    mantissa, e = torch.frexp(largest)
    e = torch.where(mantissa <= 0.875, e - 9, e - 8)
    return torch.where(largest > 0, e, LOWEST).clamp(min=LOWEST)


def _positions(s):
    """Sequence and position of every row."""
    T = s.q.shape[0]
    row = torch.arange(T, device=DEVICE)
    seq = torch.bucketize(row, s.offsets[1:].long(), right=True)
    return seq, s.lengths.long()[seq] + row - s.offsets.long()[seq]


def _rotated(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return (x.float() * cos.float()[:, None] + torch.cat((-b, a), -1) * sin.float()[:, None]).to(x.dtype)


def _append(s):
    page = s.case["page"]
    q, k = _rotated(s.q, s.cos, s.sin), _rotated(s.k, s.cos, s.sin)
    seq, pos = _positions(s)
    if s.case["store"] != "e4m3":
        at = s.table.long()[seq, pos // page]
        s.keys[at, :, pos % page] = k
        s.values[at, :, :, pos % page] = s.v
        return q
    B, slots, cap = s.table.shape[0], s.slots.long(), s.open_keys.shape[1]
    first = s.lengths.long() // page
    total = s.lengths.long() + s.offsets.long().diff()
    sealed = total // page if s.case["final"] else first
    touched = (page - 1 + s.most_rows + page - 1) // page
    # the touched pages of every sequence: what its first one holds already, then the new rows
    K = s.k.new_zeros(B, touched, s.k.shape[1], page, s.k.shape[2])
    V = s.v.new_zeros(B, touched, s.v.shape[1], s.v.shape[2], page)
    K[:, 0], V[:, 0] = s.open_keys[slots, first % cap], s.open_values[slots, first % cap]
    index = pos // page - first[seq]
    K[seq, index, :, pos % page] = k
    V[seq, index, :, :, pos % page] = s.v
    number = first[:, None] + torch.arange(touched, device=DEVICE)
    b, i = torch.nonzero(number < sealed[:, None], as_tuple=True)
    at = s.table.long()[b, number[b, i]]
    for pool, full, side in ((s.keys, K, 0), (s.values, V, 1)):
        full = full[b, i].float()
        e = _exponent(full.abs().amax((-1, -2)))
        pool.view(torch.uint8)[at] = (full * torch.exp2(-e.float())[..., None, None]).to(E4M3).view(torch.uint8)
        s.exponents[at, side] = e.to(torch.int8)
    stay = torch.nonzero(pos >= sealed[seq] * page).flatten()
    slot, ring, place = slots[seq[stay]], pos[stay] // page % cap, pos[stay] % page
    s.open_keys[slot, ring, :, place] = k[stay]
    s.open_values[slot, ring, :, :, place] = s.v[stay]
    return q


def _attend(s):
    c = s.case
    page, nq, nkv, dh = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    rows = s.offsets.long().diff()
    total, B, n, group = s.lengths.long() + rows, rows.numel(), s.most_rows, nq // nkv
    at = s.table.long().clamp(min=0)
    P = at.shape[1]
    if c["store"] == "e4m3":
        scale = torch.exp2(s.exponents.float())[at]  # [B, P, 2, nkv]
        K = s.keys.view(torch.uint8)[at].view(E4M3).float() * scale[:, :, 0, :, None, None]
        V = s.values.view(torch.uint8)[at].view(E4M3).float() * scale[:, :, 1, :, None, None]
        number = torch.arange(P, device=DEVICE)
        closed = (number < ((total if c["final"] else s.lengths.long()) // page)[:, None])[..., None, None, None]
        ring = number % s.open_keys.shape[1]
        slots = s.slots.long()
        K = torch.where(closed, K, s.open_keys[slots[:, None], ring].float())
        V = torch.where(closed, V, s.open_values[slots[:, None], ring].float())
    else:
        K, V = s.keys[at].float(), s.values[at].float()
    K = K.transpose(1, 2).reshape(B, nkv, P * page, dh)
    V = V.permute(0, 2, 1, 4, 3).reshape(B, nkv, P * page, dh)
    i = torch.arange(n, device=DEVICE)
    row = (s.offsets.long()[:-1, None] + i).clamp(max=s.q.shape[0] - 1)  # [B, n]
    Q = s.q.float()[row].view(B, n, nkv, group, dh).permute(0, 2, 1, 3, 4).reshape(B, nkv, n * group, dh)
    S = Q @ K.transpose(-1, -2) * dh ** -0.5
    seen = torch.arange(P * page, device=DEVICE) < (s.lengths.long()[:, None] + i + 1)[..., None]  # [B, n, keys]
    S = S.view(B, nkv, n, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf).view(B, nkv, n * group, -1)
    S = torch.exp(S.sub_(S.amax(-1, keepdim=True)))
    O = (S @ V) / S.sum(-1, keepdim=True)
    O = O.view(B, nkv, n, group, dh).permute(0, 2, 1, 3, 4).reshape(B, n, nq, dh)
    seq, pos = _positions(s)
    return O[seq, pos - s.lengths.long()[seq]].to(s.q.dtype)


def _log_probs(s):
    c, R, V = s.case, s.case["rows"], s.case["vocab"]
    logits = s.logits.detach()
    x = logits.float() * (1.0 / c["temperature"])
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    lp = x - total.log()
    p = e / total
    entropy = -(p * lp).sum(-1)
    given = s.targets >= 0
    target = s.targets.clamp(min=0)
    log_prob = lp.gather(1, target[:, None])[:, 0] * given
    outs = [log_prob, entropy]
    if c["top"]:
        # values in order, the lower index first among equal ones: one whole number per logit
        bits = (logits.float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * 2 ** 32 + (V - 1 - torch.arange(V, device=DEVICE))
        ids = V - 1 - order.topk(c["top"], -1)[0] % 2 ** 32
        outs += [lp.gather(1, ids), ids]
    if c["grad"]:
        d_target = s.d_log_prob * given
        grad = p * (-(d_target + s.d_top.sum(-1)))[:, None] - p * (lp + entropy[:, None]) * s.d_entropy[:, None]
        grad.scatter_add_(1, target[:, None], d_target[:, None])
        if c["top"]:
            grad.scatter_add_(1, ids, s.d_top)
        outs.append((grad * (1.0 / c["temperature"])).to(logits.dtype))
    return outs


# ----------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "f32": 4, "e4m3": 1}
    es = size[case["dtype"]]
    if case["kind"] == "logprob":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * es * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top"]),
                "flops": n * (12 if case["grad"] else 6)}
    lengths, rows = _sequences(case)
    nq, nkv, dh, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    side = 2 * nkv * dh  # values of a token's key and value
    if case["kind"] == "append":
        moved = 2 * nq * dh * es + side * es + 2 * dh * es
        total = sum(rows) * moved
        for length, n in zip(lengths, rows):
            sealed = ((length + n) // page if case["final"] else length // page) * page
            if case["store"] != "e4m3" or sealed <= length:
                total += n * side * es
            else:  # the open rows of the first page are read, whole pages written
                total += side * (length % page * es + (sealed - length // page * page) + (length + n - sealed) * es)
        return {"bytes": total, "flops": sum(rows) * 3 * (nq + nkv) * dh}
    total = pairs = 0
    for length, n in zip(lengths, rows):
        keys = length + n
        sealed = (keys if case["final"] else length) // page * page if case["store"] == "e4m3" else 0
        total += side * (sealed + (keys - sealed) * es) + 2 * n * nq * dh * es
        pairs += n * length + n * (n + 1) // 2
    return {"bytes": total, "flops": 4 * nq * dh * pairs}


# ----------------------------------------------------------------------------
# The definitions in 64 bits
# ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprob":
        return _exact_log_probs(s)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["heads"] * s.most_rows * s.most_keys > 2 ** 31:
        return None
    return _exact_attend(s)


def _half_turn(x, cos, sin):
    h = x.shape[-1] // 2
    lo, hi, c, n = x[..., :h], x[..., h:], cos[:, None].double(), sin[:, None].double()
    return torch.cat((lo * c[..., :h] - hi * n[..., :h], hi * c[..., h:] + lo * n[..., h:]), -1)


def _exact_append(s):
    """A sealed page's values are those its rows have before they are rounded to 8 bits,
    over the page's scale."""
    page, e4m3 = s.case["page"], s.case["store"] == "e4m3"
    q, k, v = _half_turn(s.q.double(), s.cos, s.sin), _half_turn(s.k.double(), s.cos, s.sin), s.v.double()
    keys, values = s.keys.to(torch.float32).double(), s.values.to(torch.float32).double()
    lengths, offsets, table = s.lengths.tolist(), s.offsets.tolist(), s.table.tolist()
    opened = [s.open_keys.double(), s.open_values.double()] if e4m3 else None
    for b, length in enumerate(lengths):
        n = offsets[b + 1] - offsets[b]
        end, start = length + n, length // page * page
        K, V = k[offsets[b]:offsets[b + 1]], v[offsets[b]:offsets[b + 1]]
        if not e4m3:
            for at in range(length, end):
                keys[table[b][at // page], :, at % page] = K[at - length]
                values[table[b][at // page], :, :, at % page] = V[at - length]
            continue
        slot, cap = int(s.slots[b]), s.open_keys.shape[1]
        before = start // page % cap
        K = torch.cat((opened[0][slot, before, :, :length - start].transpose(0, 1), K))
        V = torch.cat((opened[1][slot, before, :, :, :length - start].permute(2, 0, 1), V))
        sealed = (end if s.case["final"] else length) // page * page
        for p in range(start, sealed, page):
            for x, pool, axes in ((K, keys, (1, 0, 2)), (V, values, (1, 2, 0))):
                block = x[p - start:p - start + page]
                largest = block.to(s.k.dtype).double().abs().amax((0, 2))
                e = torch.ceil(torch.log2(largest / 448.0)).clamp(min=LOWEST)
                pool[table[b][p // page]] = block.permute(*axes) * torch.exp2(-e)[:, None, None]
        for at in range(max(sealed, length), end):
            opened[0][slot, at // page % cap, :, at % page] = K[at - start]
            opened[1][slot, at // page % cap, :, :, at % page] = V[at - start]
    return [q, keys, values, None, *opened] if e4m3 else [q, keys, values]


def _exact_attend(s):
    c = s.case
    page, nkv, dh = c["page"], c["kv_heads"], c["head_dim"]
    group = c["heads"] // nkv
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    lengths, offsets, table = s.lengths.tolist(), s.offsets.tolist(), s.table.tolist()
    for b, length in enumerate(lengths):
        r0, r1 = offsets[b], offsets[b + 1]
        end = length + r1 - r0
        count = -(-end // page)
        sealed = (end if c["final"] else length) // page if c["store"] == "e4m3" else count
        ids = torch.tensor(table[b][:count], device=DEVICE).long()
        K = s.keys.to(torch.float32)[ids].double()
        V = s.values.to(torch.float32)[ids].double()
        if c["store"] == "e4m3":
            K *= 2.0 ** s.exponents[ids, 0].double()[:, :, None, None]
            V *= 2.0 ** s.exponents[ids, 1].double()[:, :, None, None]
            for p in range(sealed, count):
                K[p] = s.open_keys[s.slots[b], p % s.open_keys.shape[1]].double()
                V[p] = s.open_values[s.slots[b], p % s.open_keys.shape[1]].double()
        K = K.transpose(0, 1).reshape(nkv, -1, dh)[:, :end]
        V = V.permute(1, 2, 0, 3).reshape(nkv, dh, -1)[:, :, :end]
        hidden = torch.arange(end, device=DEVICE) > length + torch.arange(r1 - r0, device=DEVICE)[:, None]
        for h in range(c["heads"]):
            scores = s.q[r0:r1, h].double() @ K[h // group].T / math.sqrt(dh)
            p = scores.masked_fill(hidden, -math.inf).softmax(-1)
            out[r0:r1, h] = p @ V[h // group].T
    return out


def _exact_log_probs(s):
    c = s.case
    top, rows = c["top"], s.logits.shape[0]
    parts = []
    for r in range(0, rows, 512):
        logits = s.logits.detach()[r:r + 512].double()
        lp = (logits / c["temperature"]).log_softmax(-1)
        entropy = -(lp.exp() * lp).sum(-1)
        target = s.targets[r:r + 512]
        picked = torch.where(target >= 0, lp.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0)
        part = [picked, entropy]
        ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top] if top else None
        if top:
            part += [lp.gather(1, ids)]
        if c["grad"]:
            up, d = s.d_entropy[r:r + 512, None].double(), s.d_log_prob[r:r + 512].double() * (target >= 0)
            down = torch.zeros_like(lp)
            down.scatter_add_(1, target.clamp(min=0)[:, None], d[:, None])
            if top:
                down.scatter_add_(1, ids, s.d_top[r:r + 512].double())
            p = lp.exp()
            part.append((down - p * down.sum(-1, keepdim=True) - up * p * (lp + entropy[:, None])) / c["temperature"])
        parts.append(part)
    outs = [torch.cat(x) for x in zip(*parts)]
    return outs[:3] + [None] + outs[3:] if top else outs
