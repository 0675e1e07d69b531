"""A key/value cache of many sequences in pages, and the attention over it.

``inference.PrefixCache`` holds one request's prefix; this is the cache of a program
that serves many at once.  One ``PagedCache`` per layer (per layer and depth for
recurrent layers, as ``PrefixCache.key`` has it) holds pages that the program hands
out to sequences; one ``PagedBatch`` per step says which rows belong to which
sequence and where their pages are, for every layer of the step::

    batch = PagedBatch(table, lengths, offsets, max_rows=1)
    for layer in layers:
        ...                                          # q, k, v of the new rows
        q = cache[layer].append(k, v, batch, cos=cos, sin=sin, q=q)
        o = paged_attention(q, cache[layer], batch)

In 8 bits a page is sealed when its last token is kept: e4m3 codes with one
power-of-two scale per page, head and side (keys, values), so a value is rounded once
and is exact in bfloat16.  Younger tokens stay in the model's type in their sequence's
open pages.  What a token is cached as does not depend on how its sequence was split
into calls.  A decoding window, whose rows the next pass rewrites, is a batch with
``final=False``; ``retire`` keeps the first of its rows, as
``PrefixCache.retire`` does.

No call reads the device from the host (only a batch made without ``rows`` does, and
``PagedBatch.check``), and every call can be captured into a graph; the batch's tensors
are read when a call runs, so a program may change them in place between replays.  The
kernels follow no entry that is out of range: such tokens are neither written nor
attended to (``check`` finds them, for debugging).  Sequences may share whole pages (a
common prefix); a page that is still being written, and a slot, belong to one.
"""

import ctypes

import torch

from . import _lib
from ._lib import call_on, ptr, query
from .layers import table

PAGE_SIZES = (16, 32, 64, 128)
E4M3 = torch.float8_e4m3fn


class _CacheStruct(ctypes.Structure):
    """ctypes mirror of alodlm_paged_cache (include/alodlm_hip.h)."""
    _fields_ = ([(name, ctypes.c_void_p) for name in
                 ("keys", "values", "exponents", "open_keys", "open_values")]
                + [(name, ctypes.c_int64) for name in
                   ("pages", "page_size", "kv_heads", "head_dim", "slots", "open_pages")]
                + [("dtype", ctypes.c_int32), ("eight_bit", ctypes.c_int32)])


class _BatchStruct(ctypes.Structure):
    """ctypes mirror of alodlm_paged_batch (include/alodlm_hip.h)."""
    _fields_ = ([(name, ctypes.c_void_p) for name in ("table", "lengths", "offsets", "slots")]
                + [(name, ctypes.c_int64) for name in
                   ("sequences", "width", "rows", "max_rows", "max_keys")]
                + [("final_rows", ctypes.c_int32), ("reserved", ctypes.c_int32)])


def _need(condition, message):
    if not condition:
        raise ValueError(message)


class _Fixed:
    """An object whose fields stay what ``__init__`` made of its arguments: the kernels
    are given a struct of them, which would not follow."""
    _fixed = frozenset()

    def _fix(self):
        object.__setattr__(self, "_fixed", frozenset(vars(self)))

    def _free(self, name):
        if name in self._fixed:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: change a tensor in place, "
                                 f"or make another {type(self).__name__}")

    def __setattr__(self, name, value):
        self._free(name)
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        self._free(name)
        object.__delattr__(self, name)


class PagedCache(_Fixed):
    """One layer's pages.

    ``keys`` [pages, kv_heads, page_size, head_dim] and ``values`` [pages, kv_heads,
    head_dim, page_size] are float32 or bfloat16, or float8_e4m3fn with ``exponents``
    int8 [pages, 2, kv_heads] and the open pages ``open_keys`` [slots, open_pages,
    kv_heads, page_size, head_dim] and ``open_values`` (the last two dimensions
    exchanged) in float32 or bfloat16, the type of the rows that are appended.
    ``allocate`` makes them.  The fields are fixed; the tensors' contents are not."""

    def __init__(self, keys, values, exponents=None, open_keys=None, open_values=None):
        _need(keys.ndim == 4 and values.ndim == 4, "keys and values must have four dimensions")
        pages, heads, page, dh = keys.shape
        _need(tuple(values.shape) == (pages, heads, dh, page),
              f"values must be {[pages, heads, dh, page]} beside keys {list(keys.shape)}, "
              f"got {list(values.shape)}")
        _need(page in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {page}")
        _need(8 <= dh <= 256 and dh % 8 == 0, f"head_dim must be a multiple of 8 up to 256, got {dh}")
        self.eight_bit = keys.dtype == E4M3
        tensors = [keys, values]
        if self.eight_bit:
            _need(page * dh <= 16384, "8-bit pages hold at most 16384 values a head")
            _need(None not in (exponents, open_keys, open_values),
                  "an 8-bit cache needs exponents and open pages")
            _need(exponents.dtype == torch.int8 and tuple(exponents.shape) == (pages, 2, heads),
                  f"exponents must be int8 {[pages, 2, heads]}")
            _need(open_keys.ndim == 5 and tuple(open_keys.shape[2:]) == (heads, page, dh)
                  and tuple(open_values.shape) == (*open_keys.shape[:2], heads, dh, page)
                  and open_keys.numel() > 0,
                  "open pages must be [slots, open_pages, ...] of the pages' shapes")
            _need(open_values.dtype == open_keys.dtype, "open keys and values differ in dtype")
            self.dtype = open_keys.dtype
            tensors += [exponents, open_keys, open_values]
        else:
            _need(exponents is None and open_keys is None and open_values is None,
                  "exponents and open pages belong to 8-bit pages")
            self.dtype = keys.dtype
        code = _lib.dtype_code(self.dtype)
        _need(values.dtype == keys.dtype, "keys and values differ in dtype")
        _need(pages > 0, "a cache needs pages")
        for t in tensors:
            _need(t.is_contiguous() and t.device == keys.device, "the cache's tensors must be "
                  "contiguous and on one device")
            _need(t is exponents or t.data_ptr() % 16 == 0, "the cache's tensors must be 16-byte aligned")
        self.keys, self.values, self.exponents = keys, values, exponents
        self.open_keys, self.open_values = open_keys, open_values
        self.device, self.kv_heads, self.head_dim, self.page_size = keys.device, heads, dh, page
        slots, opened = open_keys.shape[:2] if self.eight_bit else (0, 0)
        self._struct = _CacheStruct(ptr(keys), ptr(values), ptr(exponents), ptr(open_keys),
                                    ptr(open_values), pages, page, heads, dh, slots, opened, code,
                                    int(self.eight_bit))
        self._ref = ctypes.byref(self._struct)
        self._fix()

    @classmethod
    def allocate(cls, pages, kv_heads, head_dim, dtype, device, page_size=64, eight_bit=True,
                 slots=1, window=1):
        """A cache of ``pages`` pages.  In 8 bits, ``slots`` sequences can have open
        pages at a time, with room for windows of up to ``window`` rows that are not
        final (see ``PagedBatch``)."""
        store = E4M3 if eight_bit else dtype
        keys = torch.zeros(pages, kv_heads, page_size, head_dim, dtype=store, device=device)
        values = torch.zeros(pages, kv_heads, head_dim, page_size, dtype=store, device=device)
        if not eight_bit:
            return cls(keys, values)
        opened = max(1, -(-(page_size - 1 + window) // page_size))
        exponents = torch.full((pages, 2, kv_heads), -100, dtype=torch.int8, device=device)
        shape = (slots, opened, kv_heads)
        return cls(keys, values, exponents,
                   torch.zeros(*shape, page_size, head_dim, dtype=dtype, device=device),
                   torch.zeros(*shape, head_dim, page_size, dtype=dtype, device=device))

    # ------------------------------------------------------------------ calls
    def _rows(self, t, heads, batch, what):
        """``t`` as the kernels read it, and its row stride: rows [heads, head_dim], the
        stride free, 16-byte aligned (copied where it is not)."""
        if t.dtype != self.dtype:
            raise ValueError(f"{what} must be {self.dtype}, got {t.dtype}")
        if t.device != self.device:
            raise ValueError(f"{what} must be on {self.device}")
        shape, dh = t.shape, self.head_dim
        if (len(shape) != 3 or shape[0] != batch.rows or shape[2] != dh
                or (shape[1] != heads and heads is not None)):
            raise ValueError(f"{what} must be [{batch.rows}, {heads or 'heads'}, {dh}], "
                             f"got {list(shape)}")
        row, head, dim = t.stride()
        if shape[0] < 2:  # one row's stride says nothing
            row = shape[1] * dh
        if (dim != 1 or head != dh or row < shape[1] * dh or row * t.element_size() % 16
                or t.data_ptr() % 16):
            t = t.contiguous() if t.data_ptr() % 16 == 0 or not t.is_contiguous() else t.clone()
            row = shape[1] * dh
        return t, row

    def _table(self, t, batch, like):
        """A rotary table as the kernels read it (``layers.table``), 16-byte aligned."""
        if (t.dtype != like.dtype or t.device != like.device or t.shape != (batch.rows, self.head_dim)
                or not t.is_contiguous()):
            t = table(t, batch.rows, self.head_dim, like)
        return t.clone() if t.data_ptr() % 16 else t

    def _check(self, batch):
        if self.device.type != "cuda":
            raise ValueError("the paged cache runs on the HIP kernels; allocate it on a CUDA (ROCm) "
                             "device")
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        if self.eight_bit and batch.slots is None and batch.sequences > self.open_keys.shape[0]:
            raise ValueError(f"{batch.sequences} sequences without slots of their own, and "
                             f"{self.open_keys.shape[0]} slots")

    def append(self, k, v, batch, cos=None, sin=None, q=None):
        """Writes the rows' keys and values [rows, kv_heads, head_dim] behind their
        sequences.  With ``cos``/``sin`` [rows, head_dim] the keys are rotated on the
        way (x * cos + rotate_half(x) * sin, in float32 and rounded once), and so are
        the queries ``q`` [rows, heads, head_dim], which are returned."""
        self._check(batch)
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin belong together")
        if q is not None and cos is None:
            raise ValueError("q is given to be rotated: cos and sin are missing")
        k, ldk = self._rows(k, self.kv_heads, batch, "k")
        v, ldv = self._rows(v, self.kv_heads, batch, "v")
        if cos is not None:
            cos, sin = self._table(cos, batch, k), self._table(sin, batch, k)
        out, heads, ldq = None, 0, 0
        if q is not None:
            q, ldq = self._rows(q, None, batch, "q")
            heads = q.shape[1]
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        call_on(self.device, "alodlm_paged_append", self._ref, batch.ref(self), ptr(k), ldk,
                ptr(v), ldv, ptr(q), ldq, ptr(out), heads, ptr(cos), ptr(sin))
        return out

    def retire(self, batch, counts):
        """Keeps the first ``counts[b]`` rows (int32 [sequences]) of a batch that is
        not final; the program then adds them to its lengths."""
        self._check(batch)
        _need(not batch.final, "the batch's rows are kept already")
        counts = batch.per_sequence(counts, "counts")
        call_on(self.device, "alodlm_paged_retire", self._ref, batch.ref(self), ptr(counts))


class PagedBatch(_Fixed):
    """One step's rows.

    ``table`` int32 [sequences, width]: the pages of each sequence in order;
    ``lengths`` int32 [sequences]: the tokens it holds before the step; ``offsets``
    int32 [sequences + 1]: sequence b has the rows [offsets[b], offsets[b + 1]).
    ``slots`` int32 [sequences]: the slot of its open pages (8 bits; default: b).
    ``rows`` (default: offsets[-1], read from the device) is the number of rows that
    the step's tensors have; rows before the first sequence and behind the last one are
    padding.  ``max_rows`` bounds a sequence's rows (default: ``rows``) and ``max_keys``
    its tokens with them (default: what the table holds): they size the launches, so a
    table much wider than its tokens wants ``max_keys``.  A sequence's rows past max_rows
    are padding too, and its tokens past max_keys are not attended to.  ``final``: the rows
    are kept, else they are a window that ``retire`` shortens.  The fields are fixed: a
    step with other tensors or bounds is another batch; the tensors' contents may change."""

    def __init__(self, table, lengths, offsets, rows=None, max_rows=None, max_keys=None, slots=None,
                 final=True):
        _need(table.ndim == 2 and table.shape[1] > 0, "table must be [sequences, width]")
        self.sequences, self.width, self.device = table.shape[0], table.shape[1], table.device
        self.table = self._ints(table, tuple(table.shape), "table")
        self.lengths = self.per_sequence(lengths, "lengths")
        self.offsets = self._ints(offsets, (self.sequences + 1,), "offsets")
        self.slots = None if slots is None else self.per_sequence(slots, "slots")
        self.rows = int(self.offsets[-1]) if rows is None else int(rows)
        self.max_rows = self.rows if max_rows is None else min(int(max_rows), self.rows)
        self.max_keys = max_keys
        self.final = bool(final)
        _need(self.rows >= 0 and self.max_rows >= 0 and (max_keys is None or max_keys >= 0),
              "rows, max_rows and max_keys must not be negative")
        self._refs = {}
        self._fix()

    def _ints(self, t, shape, what):
        if (t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != self.device
                or not t.is_contiguous()):
            raise ValueError(f"{what} must be contiguous int32 {list(shape)} on {self.device}, got "
                             f"{t.dtype} {list(t.shape)} on {t.device}")
        return t

    def per_sequence(self, t, what):
        return self._ints(t, (self.sequences,), what)

    def ref(self, cache):
        """The C struct of this batch on a cache (they differ in the page size)."""
        entry = self._refs.get(cache.page_size)
        if entry is None:
            room = self.width * cache.page_size
            struct = _BatchStruct(ptr(self.table), ptr(self.lengths), ptr(self.offsets),
                                  ptr(self.slots), self.sequences, self.width, self.rows,
                                  self.max_rows, room if self.max_keys is None else min(self.max_keys, room),
                                  int(self.final), 0)
            entry = self._refs[cache.page_size] = (ctypes.byref(struct), struct)
        return entry[0]

    def check(self, cache):
        """Raises ValueError for entries out of range.  Reads the device: for
        debugging, not for a step."""
        page = cache.page_size
        lengths, offsets = self.lengths.tolist(), self.offsets.tolist()
        counts = [b - a for a, b in zip(offsets, offsets[1:])]
        _need(not offsets or offsets[0] >= 0, "offsets start below zero")
        _need(all(n >= 0 for n in counts), "offsets must be nondecreasing")
        _need(offsets[-1] <= self.rows, "offsets exceed the rows")
        _need(all(n <= self.max_rows for n in counts), "a sequence has more than max_rows rows")
        _need(all(n >= 0 for n in lengths), "lengths must not be negative")
        bound = self.width * page if self.max_keys is None else min(self.max_keys, self.width * page)
        _need(all(a + n <= bound for a, n in zip(lengths, counts)),
              "a sequence's tokens exceed its table or max_keys")
        pages = cache.keys.shape[0]
        for b, (row, length, n) in enumerate(zip(self.table.tolist(), lengths, counts)):
            used = row[:-(-(length + n) // page)]
            _need(all(0 <= p < pages for p in used), f"sequence {b} names a page outside the cache")
        if cache.eight_bit:
            slots = range(self.sequences) if self.slots is None else self.slots.tolist()
            _need(all(0 <= s < cache.open_keys.shape[0] for s in slots),
                  "a sequence names a slot outside the cache")
            _need(len(set(slots)) == self.sequences, "two sequences name one slot")


def paged_attention(q, cache, batch, scale=None, out=None):
    """Softmax attention of the batch's rows over their sequences' cached tokens: q
    [rows, heads, head_dim] (grouped-query heads), result [rows, heads, head_dim].
    Row i of sequence b sees the first lengths[b] + i + 1 tokens; ``append`` has
    written the batch's own.  ``scale`` is head_dim^-0.5 unless given.  A row that
    sees no token is zero.  Rows that are padding are zero, or left as they were in a
    caller's ``out``.  Weights are summed relative to 2^-8 of the row's largest or more: a
    result is finite while the tokens times the largest value stay below 2^119.  No
    gradient: this is the decoder's side."""
    cache._check(batch)
    q, ldq = cache._rows(q, None, batch, "q")
    heads = q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads do not share {cache.kv_heads} key/value heads")
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    fresh = out is None
    if fresh:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (out.dtype != q.dtype or out.shape != q.shape or out.device != q.device
          or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError(f"out must be a contiguous, 16-byte aligned {q.dtype} tensor of q's shape")
    ref = batch.ref(cache)
    need = query("alodlm_paged_attention_workspace", cache._ref, ref, heads)
    workspace = torch.empty(need, dtype=torch.float32, device=q.device) if need else None
    call_on(q.device, "alodlm_paged_attention", cache._ref, ref, ptr(q), ldq, ptr(out), heads,
            scale, int(fresh), ptr(workspace))
    return out
