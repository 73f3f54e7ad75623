"""The paged operators' host side without a GPU: the struct's mirror, the C entry points' checks, the helpers."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def struct(**change):
    """A layer that passes the checks (its addresses are never followed: every call below is refused before that)."""
    from retrievalattention_b200 import _lib

    p = _lib.Paged(2, 4, 7, 16, 100, 8, _lib.RI_BF16, 0, 4 * 16 * 128, 4 * 16 * 128, 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24,
                   1 << 25, 1 << 26)
    for name, value in change.items():
        setattr(p, name, value)
    return p


def test_struct_mirror_matches_header_field_order():
    from retrievalattention_b200 import _lib

    text = open(os.path.join(ROOT, "include", "ri_b200.h")).read()
    body = text[text.index("typedef struct ri_paged {"):text.index("} ri_paged;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [n for line in re.findall(r"[^;{]+;", body[body.index("{") + 1:]) for n in re.findall(r"\b([a-z_0-9]+)\s*(?=[,;])", line)]
    assert fields == [f[0] for f in _lib.Paged._fields_]


@pytest.mark.parametrize("change,words", [
    (dict(batch=0), b"batch=0"), (dict(kv_heads=0), b"kv_heads=0"), (dict(batch=70000), b"batch=70000"),
    (dict(page_size=4), b"page_size=4"), (dict(page_size=24), b"page_size=24"), (dict(page_size=2048), b"page_size=2048"),
    (dict(n_pages=0), b"n_pages=0"), (dict(table_stride=0), b"table_stride=0"), (dict(table_stride=1 << 28), b"too far"),
    (dict(dtype=7), b"dtype=7"), (dict(key_page_stride=4 * 16 * 128 - 8), b"overlap"), (dict(value_page_stride=4 * 16 * 128 + 4), b"odd places"),
    (dict(d_keys=(1 << 20) + 8), b"aligned"), (dict(d_lengths=None), b"null"), (dict(d_table=None), b"null"), (dict(d_status=None), b"null"),
])
def test_layers_that_are_refused(change, words):
    from retrievalattention_b200 import _lib

    p = C.byref(struct(**change))
    for size in (_lib.lib.ri_paged_decode_scratch_bytes(p), _lib.lib.ri_paged_observe_scratch_bytes(p),
                 _lib.lib.ri_paged_evict_scratch_bytes(p, 10)):
        assert size == -1 and words in _lib.lib.ri_last_error()


def test_workspaces_follow_what_is_asked():
    from retrievalattention_b200 import _lib

    with_weights, without = struct(), struct(d_weight=None)
    a, b = (_lib.lib.ri_paged_decode_scratch_bytes(C.byref(p)) for p in (with_weights, without))
    steps = 2 * 4 * (8 * 16 // 16)
    assert a - b == 16 + steps * 7 * 16 * 4 and b > 0          # a score for every slot and query head
    assert _lib.lib.ri_paged_decode_scratch_bytes(C.byref(struct(group_size=9))) == -1
    assert _lib.lib.ri_paged_evict_scratch_bytes(C.byref(with_weights), 0) == -1
    few, many = (_lib.lib.ri_paged_evict_scratch_bytes(C.byref(with_weights), keep) for keep in (1, 64))
    assert many - few == 2 * 4 * 63 * 8                         # at most min(keep, slots - keep) moves a group


@pytest.mark.parametrize("entry,args", [
    ("ri_paged_decode", lambda: (1 << 20, 128 * 27, 1 << 21, None, 0.1, 1 << 22, None)),               # queries overlap
    ("ri_paged_decode", lambda: (1 << 20, 128 * 28, None, None, 0.1, 1 << 22, None)),
    ("ri_paged_decode", lambda: (1 << 20, 128 * 28, 1 << 21, None, float("nan"), 1 << 22, None)),
    ("ri_paged_observe", lambda: (1 << 20, 0, 0.1, 1 << 22, None)),
    ("ri_paged_observe", lambda: (1 << 20, 1 << 20, 0.1, 1 << 22, None)),                             # 7 << 20 rows
    ("ri_paged_evict", lambda: (1 << 20, 10, 6, 5, 1 << 22, None)),                                   # 11 protected of 10
    ("ri_paged_evict", lambda: (None, 10, 4, 5, 1 << 22, None)),
    ("ri_rope_paged_append", lambda: (1 << 20, 128 * 36, 1 << 21, 50, 1 << 22, bytes([3] * 64), 3, 2, None, 1 << 23, 1 << 24, None, None, None)),
    ("ri_rope_paged_append", lambda: (1 << 20, 128 * 36, 1 << 21, 50, 1 << 22, bytes(64), 1, 3, None, 1 << 23, 1 << 24, None, None, None)),
    ("ri_rope_paged_append", lambda: (1 << 20, 128 * 35, 1 << 21, 50, 1 << 22, bytes(64), 1, 2, None, 1 << 23, 1 << 24, None, None, None)),
])
def test_calls_that_are_refused(entry, args):
    from retrievalattention_b200 import _lib

    assert getattr(_lib.lib, entry)(C.byref(struct()), *args()) == -1
    assert entry.encode() in _lib.lib.ri_last_error()


def test_axes_of_the_frequencies():
    from retrievalattention_b200 import paged

    assert paged.rope_sections(64) == (0,) * 64
    assert paged.rope_sections(16, 24, 24) == (0,) * 16 + (1,) * 24 + (2,) * 24
    dealt = paged.rope_interleaved(24, 20, 20)
    assert len(dealt) == 64 and dealt[:7] == (0, 1, 2, 0, 1, 2, 0) and [dealt.count(a) for a in range(3)] == [24, 20, 20]
    for bad in ((0.5,) * 64, (-1,) * 64, ("a",) * 64):
        with pytest.raises(ValueError):
            paged._axes(bad)


def test_binding_checks_before_it_touches_a_device():
    import importlib.util

    import torch

    from retrievalattention_b200 import paged

    spec = importlib.util.spec_from_file_location("_paged_binding", paged._BINDING)      # not connected: that needs a GPU
    native = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(native)
    pages, table, lengths = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on a GPU"):
        native.decode(q, pages, pages, table, lengths, None, None, None, 0.1)
    with pytest.raises(ValueError, match="q_heads a multiple"):
        native.decode(q[:, :, :7], pages, pages, table, lengths, None, None, None, 0.1)
    with pytest.raises(TypeError):
        native.decode("q", pages, pages, table, lengths, None, None, None, 0.1)
