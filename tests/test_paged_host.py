"""The paged cache without a GPU: struct layouts, refusals of shapes, types and sizes
(the library's own too), the batch's checks and the tolerance of the plain cache."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from alodlm_amd import _lib
from alodlm_amd.credit import token_log_probs
from alodlm_amd.paged import (E4M3, PagedBatch, PagedCache, _BatchStruct, _CacheStruct,
                              paged_attention)
from tests.paged_oracle import quantise

BF16 = torch.bfloat16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def cache(pages=8, kv_heads=2, head_dim=16, dtype=BF16, page_size=16, **more):
    return PagedCache.allocate(pages, kv_heads, head_dim, dtype, "cpu", page_size=page_size, **more)


def batch(table=((0, 1), (2, 3)), lengths=(5, 0), offsets=(0, 1, 3), **more):
    return PagedBatch(torch.tensor(table, dtype=torch.int32), ints(*lengths), ints(*offsets), **more)


@pytest.mark.parametrize("struct,name", [(_CacheStruct, "alodlm_paged_cache"),
                                         (_BatchStruct, "alodlm_paged_batch")])
def test_structs_match_header(tmp_path, struct, name):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    include = Path(__file__).resolve().parents[1] / "include"
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "probe.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"alodlm_hip.h\"\nint main(void) {\n"
                   + "".join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
    subprocess.run([gcc, "-I", str(include), str(src), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout
    assert [int(v) for v in out.split()] == [getattr(struct, f).offset for f in fields] + [
        ctypes.sizeof(struct)]


def test_allocated_shapes():
    c = cache(pages=8, page_size=16, slots=3, window=18)
    assert c.eight_bit and c.keys.dtype == E4M3 and c.dtype == BF16
    assert tuple(c.open_keys.shape) == (3, 3, 2, 16, 16)  # 15 open tokens and 18 rows: 3 pages
    assert tuple(cache(window=1).open_keys.shape)[:2] == (1, 1)
    plain = cache(eight_bit=False, dtype=torch.float32)
    assert not plain.eight_bit and plain.exponents is None and plain.dtype == torch.float32


def test_cache_refusals():
    c = cache(slots=2)
    parts = [c.keys, c.values, c.exponents, c.open_keys, c.open_values]
    PagedCache(*parts)
    with pytest.raises(ValueError, match="page size"):
        cache(page_size=48)
    with pytest.raises(ValueError, match="head_dim"):
        cache(head_dim=12)
    with pytest.raises(ValueError, match="head_dim"):
        cache(head_dim=264)
    with pytest.raises(ValueError, match="16384"):
        cache(head_dim=256, page_size=128)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        cache(dtype=torch.float16)
    with pytest.raises(ValueError, match="open pages"):
        PagedCache(*parts[:2])
    with pytest.raises(ValueError, match="exponents"):
        PagedCache(*parts[:2], c.exponents.to(torch.int32), *parts[3:])
    with pytest.raises(ValueError, match="values must be"):
        PagedCache(c.keys, c.keys[:, :, :8], *parts[2:])
    with pytest.raises(ValueError, match="open pages"):
        PagedCache(*parts[:3], c.open_keys[:, :, :1], c.open_values)
    with pytest.raises(ValueError, match="belong to 8-bit"):
        PagedCache(torch.zeros(2, 1, 16, 16), torch.zeros(2, 1, 16, 16), c.exponents)
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache(torch.zeros(2, 1, 16, 32)[..., ::2], torch.zeros(2, 1, 16, 16))


def test_batch_refusals():
    with pytest.raises(ValueError, match="lengths"):
        batch(lengths=(5, 0, 1))
    with pytest.raises(ValueError, match="offsets"):
        batch(offsets=(0, 1))
    with pytest.raises(ValueError, match="int32"):
        PagedBatch(torch.zeros(2, 2, dtype=torch.int64), ints(1, 1), ints(0, 1, 2))
    with pytest.raises(ValueError, match="slots"):
        batch(slots=ints(0))
    with pytest.raises(ValueError, match="negative"):
        batch(rows=-1)
    with pytest.raises(ValueError, match="contiguous"):  # a copy would not follow changes in place
        batch(slots=torch.arange(4, dtype=torch.int32)[::2])
    b = batch()
    assert (b.rows, b.max_rows, b.sequences, b.width) == (3, 3, 2, 2)
    assert batch(rows=7, max_rows=9).max_rows == 7


def test_checks_find_entries_out_of_range():
    c = cache(slots=2)
    batch().check(c)
    for bad in (dict(table=((0, 8), (2, 3)), lengths=(16, 0)), dict(table=((-1, 0), (2, 3))),
                dict(lengths=(-1, 0)), dict(lengths=(32, 0)), dict(offsets=(0, 3, 1), rows=3),
                dict(offsets=(0, 1, 3), rows=2), dict(max_rows=1), dict(max_keys=5),
                dict(slots=ints(0, 2)), dict(slots=ints(-1, 0)), dict(slots=ints(1, 1)), dict(offsets=(-1, 1, 3))):
        with pytest.raises(ValueError):
            batch(**bad).check(c)
    # a page that no token lies in may be named anyhow
    batch(table=((0, 99), (2, -5))).check(c)


def test_calls_need_the_gpu():
    c, b = cache(slots=2), batch()
    rows = torch.zeros(3, 2, 16, dtype=BF16)
    for run in (lambda: c.append(rows, rows, b), lambda: paged_attention(rows, c, b),
                lambda: c.retire(batch(final=False), ints(0, 0)),
                lambda: token_log_probs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="HIP kernels"):
            run()


def structs(c, b, **changes):
    cs = _CacheStruct.from_buffer_copy(c._struct)
    b.ref(c)
    bs = _BatchStruct.from_buffer_copy(b._refs[c.page_size][1])
    for key, value in changes.items():
        setattr(cs if hasattr(cs, key) else bs, key, value)
    return ctypes.byref(cs), ctypes.byref(bs)


def library():
    if not _lib.LIBRARY.exists():
        pytest.skip("library not built")


@pytest.mark.parametrize("change,match", [
    (dict(page_size=24), "page size"), (dict(head_dim=20), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=512), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"),
    (dict(dtype=7), "dtype"), (dict(slots=0), "slots"), (dict(sequences=-1), "sequences"),
    (dict(rows=-1), "rows"), (dict(max_rows=4), "max_rows"), (dict(width=0), "width"),
    (dict(width=1 << 28), "width"), (dict(keys=None), "lacks"), (dict(exponents=None), "lacks"),
    (dict(offsets=None), "lacks"), (dict(table=None), "lacks"), (dict(max_keys=33), "max_keys"),
    (dict(final_rows=0, max_rows=3, open_pages=1), "window")])
def test_library_refuses_structs(change, match):
    """Host checks of the C entry points: nothing is launched."""
    library()
    c, b = structs(cache(slots=2), batch(), **change)
    with pytest.raises(ValueError, match=match):
        _lib.call("alodlm_paged_append", c, b, None, 32, None, 32, None, 0, None, 0, None, None, None)
    with pytest.raises(ValueError, match=match):
        _lib.call("alodlm_paged_attention", c, b, None, 32, None, 2, 0.25, 0, None, None)
    assert _lib.query("alodlm_paged_attention_workspace", c, b, 2) == 0


def test_library_refuses_arguments():
    library()
    c, b = structs(cache(slots=2), batch())
    append = lambda k=None, ldk=32, q=None, ldq=0, cos=None, sin=None: _lib.call(
        "alodlm_paged_append", c, b, k, ldk, None, 32, q, ldq, None, 2, cos, sin, None)
    attend = lambda q=None, ldq=32, heads=2, scale=0.25: _lib.call(
        "alodlm_paged_attention", c, b, q, ldq, None, heads, scale, 0, None, None)
    for run, match in ((lambda: append(ldk=31), "strides"), (lambda: append(cos=16), "cos"),
                       (lambda: append(q=16, ldq=32), "rotated"), (lambda: append(k=8), "aligned"),
                       (lambda: append(ldk=36), "aligned"), (lambda: attend(ldq=16), "stride"),
                       (lambda: attend(heads=3, ldq=64), "heads"), (lambda: attend(heads=0), "heads"),
                       (lambda: attend(scale=0.0), "scale"), (lambda: attend(scale=float("nan")), "scale"),
                       (lambda: attend(q=8), "aligned"), (lambda: append(), "no rows"),
                       (lambda: attend(), "no rows"),
                       (lambda: _lib.call("alodlm_paged_retire", c, b, None, None), "kept already")):
        with pytest.raises(ValueError, match=match):
            run()


@pytest.mark.parametrize("args,match", [
    ((None, 4, None, 1, 5, 0, 1.0), "stride"), ((None, 5, None, -1, 5, 0, 1.0), "rows"),
    ((None, 5, None, 1, 0, 0, 1.0), "vocabulary"), ((None, 5, None, 1, 5, 6, 1.0), "top"),
    ((None, 500, None, 1, 500, 65, 1.0), "top"), ((None, 5, None, 1, 5, 0, 0.0), "temperature"),
    ((None, 5, None, 1, 5, 2, 1.0), "alternatives")])
def test_library_refuses_log_prob_arguments(args, match):
    library()
    with pytest.raises(ValueError, match=match):
        _lib.call("alodlm_token_log_probs", *args, -100, None, None, None, None, None, None, 1, None)


def test_log_prob_refusals():
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.int64)
    for args, kwargs, match in (((x[0], t), {}, "rows, vocabulary"), ((x, t.int()), {}, "int64"),
                                ((x, t[:2]), {}, "one per row"), ((x, t), dict(top=8), "top"),
                                ((x, t), dict(top=-1), "top"), ((x, t), dict(temperature=0.0), "temperature"),
                                ((x, t), dict(temperature=float("inf")), "temperature"),
                                ((x, t), dict(temperature=float("nan")), "temperature"),
                                ((x.half(), t), {}, "float32 or bfloat16")):
        with pytest.raises(ValueError, match=match):
            token_log_probs(*args, **kwargs)


def test_plain_page_scales():
    """The page's exponent is the smallest that holds its largest value, and a code is
    off by half a step of three mantissa bits: 2^-4 of its value."""
    for largest, e in ((448.0, 0), (449.0, 1), (224.0, -1), (1.0, -8), (1.75, -8), (1.76, -7), (0.0, -100),
                       (1e-38, -100)):
        x = torch.linspace(-largest, largest / 3, 33)
        codes, got = quantise(x)
        assert got == e, largest
        if largest > 1e-30:
            small = 2.0 ** (e - 10)  # half the subnormals' step
            assert bool(((codes * 2.0 ** e - x.double()).abs()
                         <= (2.0 ** -4 * x.double().abs()).clamp(min=small)).all())
    assert quantise(torch.tensor([1.0, float("inf"), float("nan")]))[0].isnan().tolist() == [False, True, True]
