"""What a paged cache and its batch refuse besides shapes and types, without a GPU."""

import ctypes

import pytest
import torch

from alodlm_amd import _lib
from tests.test_paged_host import batch, cache, ints, library, structs


def test_fields_are_fixed():
    """The kernels take what a cache and a batch were made of: another tensor, bound or
    flag needs another object; tensors may change in place."""
    c, b = cache(slots=2), batch()
    made = ctypes.string_at(b.ref(c), ctypes.sizeof(b._refs[c.page_size][1]))
    for name, value in (("table", b.table.clone()), ("lengths", ints(7, 7)), ("offsets", ints(0, 0, 0)),
                        ("slots", ints(1, 0)), ("rows", 2), ("max_rows", 1), ("max_keys", 3), ("final", False),
                        ("sequences", 1), ("width", 1)):
        before = getattr(b, name)
        with pytest.raises(AttributeError, match=name):
            setattr(b, name, value)
        with pytest.raises(AttributeError, match=name):
            delattr(b, name)
        assert getattr(b, name) is before
    for name in ("keys", "values", "exponents", "open_keys", "open_values"):
        before = getattr(c, name)
        with pytest.raises(AttributeError, match=name):
            setattr(c, name, before.clone())
        assert getattr(c, name) is before
    for name, value in (("page_size", 32), ("kv_heads", 1), ("head_dim", 8), ("eight_bit", False),
                        ("dtype", torch.float32), ("device", torch.device("cpu"))):
        with pytest.raises(AttributeError, match=name):
            setattr(c, name, value)
    b.lengths.copy_(ints(9, 9))
    assert ctypes.string_at(b.ref(c), len(made)) == made
    c.layer = 3  # a program's own names are free
    c.layer = b.step = 4
    assert c.layer == b.step == 4


@pytest.mark.parametrize("page,head_dim", [(16, 64), (128, 64), (64, 24)])
def test_key_counts_next_to_2_to_the_31(page, head_dim):
    """The kernels count keys in 32 bits, a chunk and a few tiles past the last: tables of
    2^31 - 2^20 keys or more are refused."""
    library()
    c, b = cache(pages=2, page_size=page, head_dim=head_dim, slots=2), batch()
    for width, fine in (((2 ** 31 - 2 ** 20) // page - 1, True), ((2 ** 31 - 2 ** 20) // page, False),
                        (2 ** 31 // page - 2, False)):
        cs, bs = structs(c, b, width=width, max_keys=width * page)
        # nothing is launched: the rows are missing
        with pytest.raises(ValueError, match="no rows" if fine else "width"):
            _lib.call("alodlm_paged_attention", cs, bs, None, 2 * head_dim, None, 2, 0.25, 0, None, None)
        with pytest.raises(ValueError, match="no rows" if fine else "width"):
            _lib.call("alodlm_paged_append", cs, bs, None, 2 * head_dim, None, 2 * head_dim, None, 0, None, 0,
                      None, None, None)


def test_temperatures_whose_base_2_form_is_infinite():
    """The exponentials are in base 2: a temperature whose inverse log2 e takes past float32
    is refused.  The calls lack arrays: nothing is launched."""
    library()
    for inverse, match in ((3.4028234e38 * 0.6931471, "alternatives"), (2.4e38, "temperature"),
                           (3.4e38, "temperature")):
        with pytest.raises(ValueError, match=match):
            _lib.call("alodlm_token_log_probs", None, 5, None, 1, 5, 2, inverse, -100, None, None, None, None, None,
                      None, 1, None)
        upstream = 16  # of the alternatives, whose ids are missing
        with pytest.raises(ValueError, match=match):
            _lib.call("alodlm_token_log_probs_bwd", None, 5, None, None, None, None, None, None, upstream, 1, 5, 2,
                      inverse, -100, None, 1, None)


def test_scales_whose_base_2_form_is_infinite():
    """The same for the attention's scale."""
    library()
    c, b = structs(cache(slots=2), batch())
    for scale, match in ((3.4028234e38 * 0.6931471, "no rows"), (2.4e38, "scale")):
        with pytest.raises(ValueError, match=match):
            _lib.call("alodlm_paged_attention", c, b, None, 32, None, 2, scale, 0, None, None)


@pytest.mark.parametrize("missing", ["logits", "targets", "log_prob", "entropy", "stats"])
def test_log_probabilities_need_their_arrays(missing):
    """The library's own checks: a missing array is refused before anything is launched."""
    library()
    at = {name: None if name == missing else 16 for name in ("logits", "targets", "log_prob", "entropy", "stats")}
    with pytest.raises(ValueError, match="lacks"):
        _lib.call("alodlm_token_log_probs", at["logits"], 5, at["targets"], 1, 5, 0, 1.0, -100, at["log_prob"],
                  at["entropy"], at["stats"], None, None, None, 1, None)
    at["dlogits"] = at.pop("log_prob")
    with pytest.raises(ValueError, match="lacks"):
        _lib.call("alodlm_token_log_probs_bwd", at["logits"], 5, at["targets"], None, at["stats"], at["entropy"], None,
                  None, None, 1, 5, 0, 1.0, -100, at["dlogits"], 1, None)
