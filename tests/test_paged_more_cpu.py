"""The C entry points for norms, windows, prompts and shared prefixes without a GPU: what they refuse, and their workspaces."""
import ctypes as C

import pytest

from test_paged_cpu import struct


def lib():
    from retrievalattention_b200 import _lib

    return _lib.lib


@pytest.mark.parametrize("entry,args,words", [
    ("ri_paged_decode_window", lambda: (1 << 20, 128 * 28, 0, 4, 1 << 21, None, 0.1, 1 << 22, None), b"window=0"),
    ("ri_paged_decode_window", lambda: (1 << 20, 128 * 28, 5, -1, 1 << 21, None, 0.1, 1 << 22, None), b"sink=-1"),
    ("ri_paged_decode_window", lambda: (1 << 20, 128 * 27, 5, 0, 1 << 21, None, 0.1, 1 << 22, None), b"overlap"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, 0, 1 << 21, 5, 0, 1 << 22, None, 0.1, 1 << 23, None), b"rows=0"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, 9, 1 << 21, -5, 0, 1 << 22, None, 0.1, 1 << 23, None), b"window=-5"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, 9, 1 << 21, 5, -1, 1 << 22, None, 0.1, 1 << 23, None), b"sink=-1"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, 9, None, 5, 0, 1 << 22, None, 0.1, 1 << 23, None), b"null"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 27, 9, 1 << 21, 5, 0, 1 << 22, None, 0.1, 1 << 23, None), b"overlap"),
    ("ri_paged_prompt", lambda: ((1 << 20) + 8, 128 * 28, 9, 1 << 21, 5, 0, 1 << 22, None, 0.1, 1 << 23, None), b"aligned"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, 9, 1 << 21, 5, 0, 1 << 22, None, 0.0, 1 << 23, None), b"scale"),
    ("ri_paged_prompt", lambda: (1 << 20, 128 * 28, (1 << 31) - 1, 1 << 21, 0, 0, 1 << 22, None, 0.1, 1 << 23, None), b"too large"),
    ("ri_paged_shared_decode", lambda: (1 << 20, 128 * 28, 1 << 21, 0, 1 << 22, 1 << 23, None, 0.1, 1 << 24, None), b"groups=0"),
    ("ri_paged_shared_decode", lambda: (1 << 20, 128 * 28, 1 << 21, 3, 1 << 22, 1 << 23, None, 0.1, 1 << 24, None), b"groups=3"),
    ("ri_paged_shared_decode", lambda: (1 << 20, 128 * 28, 1 << 21, 1, None, 1 << 23, None, 0.1, 1 << 24, None), b"null"),
    ("ri_paged_shared_decode", lambda: (1 << 20, 128 * 28, None, 1, 1 << 22, 1 << 23, None, 0.1, 1 << 24, None), b"null"),
    ("ri_paged_shared_decode", lambda: (1 << 20, 128 * 28, 1 << 21, 1, 1 << 22, 1 << 23, None, float("nan"), 1 << 24, None), b"scale"),
])
def test_calls_that_are_refused(entry, args, words):
    wide = dict(table_stride=1 << 17) if words == b"too large" else {}
    assert getattr(lib(), entry)(C.byref(struct(d_weight=None, **wide)), *args()) == -1
    assert words in lib().ri_last_error()


def test_weights_are_refused():
    assert lib().ri_paged_decode_window(C.byref(struct()), 1 << 20, 128 * 28, 5, 0, 1 << 21, None, 0.1, 1 << 22, None) == -1
    assert b"weights" in lib().ri_last_error()
    assert lib().ri_paged_shared_decode(C.byref(struct()), 1 << 20, 128 * 28, 1 << 21, 1, 1 << 22, 1 << 23, None, 0.1, 1 << 24, None) == -1
    assert b"weights" in lib().ri_last_error()


def norm_args(q=1 << 23, k=1 << 24, q_heads=1, k_heads=1, eps=1e-6):
    return (1 << 20, 128 * 36, 1 << 21, 50, 1 << 22, bytes(64), 1, 2, None, None, q, k, q_heads, k_heads, eps, 1 << 25, None, None, None)


@pytest.mark.parametrize("change,words", [
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(q=(1 << 23) + 8), b"aligned"), (dict(q_heads=2), b"weights of 2"),
    (dict(k_heads=28), b"and 28 heads"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"),
])
def test_norms_that_are_refused(change, words):
    assert lib().ri_rope_paged_append_norm(C.byref(struct(d_token=None)), *norm_args(**change)) == -1
    assert words in lib().ri_last_error()


def test_split_norms_that_are_refused():
    good = dict(q=1 << 23, k=1 << 24, q_heads=1, k_heads=1, eps=1e-6)
    for change in (dict(q=None), dict(k=(1 << 24) + 8), dict(q_heads=3), dict(k_heads=8), dict(eps=-1.0)):
        a = {**good, **change}
        assert lib().ri_rope_split_norm(1 << 20, 1 << 21, 1 << 22, a["q"], a["k"], a["q_heads"], a["k_heads"], a["eps"], 1 << 25, 1 << 26, 1 << 27,
                                        2, 8, 2, 50, 0, None) == -1


def test_workspaces():
    """A prompt needs one where an item may be cut: more than eight steps of 128 slots."""
    size = lambda width, rows, window=0, sink=0: lib().ri_paged_prompt_scratch_bytes(C.byref(struct(table_stride=width)), rows, window, sink)  # noqa: E731
    assert size(64, 500) == 0 and size(65, 500) > 0            # 1024 and 1040 slots
    assert size(6000, 500, 800, 4) == 0 and size(6000, 500, 2000, 4) == size(65, 500)
    assert size(6000, 1, 2000, 4) < size(6000, 500, 2000, 4)
    assert lib().ri_paged_prompt_scratch_bytes(C.byref(struct(batch=16385, kv_heads=1)), 5, 0, 0) == -1
    shared = lambda width: lib().ri_paged_shared_decode_scratch_bytes(C.byref(struct(table_stride=width)), 1)  # noqa: E731
    assert 0 < shared(8) < shared(1 << 15)                     # few slots are attended one by one
