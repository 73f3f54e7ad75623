"""``cache_hub.paged_cache`` on the host: what it refuses, its lengths and pages.  The pools lie on the CPU here; no kernel runs."""
import types

import pytest
import torch


@pytest.fixture
def make(monkeypatch):
    from retrievalattention_b200.cache_hub import paged_cache

    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda device: types.SimpleNamespace(total_memory=1 << 37))
    monkeypatch.setattr(paged_cache, "_to_device", lambda self, values: torch.tensor(values, dtype=torch.int32))

    def build(**change):
        args = dict(layer_num=1, batch_size=2, max_length=100, num_key_value_heads=2, num_heads=8, head_dim=128, dtype=torch.bfloat16,
                    layer_mapping={"0": "cpu"}, num_gpus=1, model_size=1)
        return paged_cache(**{**args, **change})

    return build


@pytest.mark.parametrize("change,words", [
    (dict(num_heads=18), "18 query heads"), (dict(num_heads=32), "32 query heads"), (dict(num_heads=7), "7 query heads"),
    (dict(num_heads=1), "1 query heads"), (dict(num_key_value_heads=0), "0 KV heads"),
    (dict(page_size=4), "page_size=4"), (dict(page_size=24), "page_size=24"), (dict(page_size=2048), "page_size=2048"), (dict(page_size=0), "page_size=0"),
    (dict(dtype=torch.float32), "float32"), (dict(head_dim=64), "head_dim"), (dict(batch_size=0), "or more"), (dict(max_length=0), "or more"),
    (dict(num_pages=0), "or more"), (dict(keep=0, sink=0, recent=0), "keep=0"), (dict(keep=10), "keep=10"), (dict(keep=80, sink=-1), "keep=80"),
    (dict(keep=80, slack=-1), "slack=-1"),
])
def test_what_no_call_would_take_is_refused_at_once(make, change, words):
    with pytest.raises(ValueError, match=words):
        make(**change)


def test_limits_are_the_kernels(make):
    """The largest group and the page sizes that the constructor takes are those of the C entry points."""
    import ctypes as C

    from retrievalattention_b200 import _lib, paged

    for group, page, ok in ((1, 8, True), (paged.MAX_GROUP, 1024, True), (paged.MAX_GROUP + 1, 16, False), (1, 4, False), (1, 2048, False)):
        p = _lib.Paged(2, 2, group, page, 100, 8, _lib.RI_BF16, 0, 2 * page * 128, 2 * page * 128, 1 << 20, 1 << 21, 1 << 22, 1 << 23,
                       1 << 24, 1 << 25, 1 << 26)
        assert (_lib.lib.ri_paged_decode_scratch_bytes(C.byref(p)) > 0) == ok
        if ok:
            make(num_heads=2 * group, page_size=page)
        else:
            with pytest.raises(ValueError):
                make(num_heads=2 * group, page_size=page)


@pytest.fixture
def evictions(monkeypatch):
    """Lengths of the requests at every call of the eviction kernel."""
    from retrievalattention_b200 import paged

    seen = []
    monkeypatch.setattr(paged, "paged_evict", lambda *a: seen.append(a[5].tolist()))
    return seen


def generate(cache, steps):
    for _ in range(steps):
        cache.begin(1)
        cache.evict()


@pytest.mark.parametrize("max_length", [65, 66, 80, 128])
def test_generation_goes_on_where_max_length_is_near_keep(make, evictions, max_length):
    """With slack=64 no request ever gets to keep + slack."""
    cache = make(keep=64, sink=2, recent=12, max_length=max_length, slack=64)
    generate(cache, 300)
    assert max(cache.length_of) <= max_length and cache.lengths.tolist() == cache.length_of and cache.seen_after.tolist() == [300, 300]
    assert evictions and all(max(n) > 64 for n in evictions)
    assert [len(p) for p in cache._pages] == [-(-n // 16) for n in cache.length_of]


def test_generation_goes_on_in_a_pool_sized_for_keep(make, evictions):
    """Two requests of 64 slots, and the page that each needs for one more."""
    cache = make(keep=64, sink=2, recent=12, max_length=400, slack=64, num_pages=10)
    generate(cache, 300)
    assert max(cache.length_of) <= 64 + 16 and len(evictions) > 10
    assert sorted(cache._free + sum(cache._pages, [])) == list(range(10))


def test_requests_run_to_the_slack_where_there_is_room(make, evictions):
    cache = make(keep=32, sink=2, recent=12, max_length=400, slack=20)
    generate(cache, 53)
    assert evictions == [[53, 53]] and cache.length_of == [32, 32]
    cache.begin([3, 0])
    assert not cache.evict() and cache.evict(slack=0) and not cache.evict(slack=0)


def test_nothing_to_evict_is_still_an_error(make, evictions):
    cache = make(keep=32, sink=2, recent=12, max_length=32)
    generate(cache, 32)
    with pytest.raises(RuntimeError, match="more than max_length"):
        cache.begin(1)
    cache = make(keep=32, sink=2, recent=12, num_pages=3)
    generate(cache, 16)
    with pytest.raises(RuntimeError, match="pool has 1 pages left"):
        cache.begin(1)
    assert not evictions


def test_table_width_bounds_the_workspaces():
    import ctypes as C

    from retrievalattention_b200 import _lib

    def sizes(stride, width):
        p = _lib.Paged(2, 4, 7, 16, 100, stride, _lib.RI_BF16, width, 4 * 16 * 128, 4 * 16 * 128, 1 << 20, 1 << 21, 1 << 22, 1 << 23,
                       1 << 24, 1 << 25, 1 << 26)
        return [_lib.lib.ri_paged_decode_scratch_bytes(C.byref(p)), _lib.lib.ri_paged_observe_scratch_bytes(C.byref(p)),
                _lib.lib.ri_paged_evict_scratch_bytes(C.byref(p), 100)]

    assert sizes(8000, 40) == sizes(40, 0) == sizes(40, 40) != sizes(8000, 0)
    assert min(sizes(1 << 28, 40)) > 0                            # where a row begins does not count
    for width in (-1, 41):
        assert sizes(40, width) == [-1] * 3 and b"table_width" in _lib.lib.ri_last_error()


def test_axes_that_are_no_list_of_them():
    from retrievalattention_b200 import paged

    assert paged._axes((1,) * 64) == paged._axes(bytes([1] * 64)) == paged._axes(torch.ones(64, dtype=torch.int64)) == bytes([1] * 64)
    for bad in (64, 64.0, None, torch.tensor(64), "0" * 64, [256] * 64):
        with pytest.raises(ValueError, match="axis_of"):
            paged._axes(bad)


@pytest.mark.timeout(20)
def test_sections_that_are_no_numbers_of_frequencies():
    from retrievalattention_b200 import paged

    assert paged.rope_interleaved() == paged.rope_sections() == () and paged.rope_interleaved(0, 2) == (1, 1)
    for make_axes in (paged.rope_sections, paged.rope_interleaved):
        for bad in ((-1,), (65, -1), (32.5, 31.5)):
            with pytest.raises(ValueError, match="sections"):
                make_axes(*bad)


def test_windows(make):
    cache = make(layer_num=2, layer_mapping={"0": "cpu", "1": "cpu"}, attn_window=[None, 30], attn_sink=4)
    assert cache.attn_window == [None, 30] and make(attn_window=30).attn_window == [30]
    for bad in (dict(attn_window=0), dict(attn_window=[3, 4]), dict(attn_window=3, attn_sink=-1), dict(attn_window=3, keep=80)):
        with pytest.raises(ValueError):
            make(**bad)


def test_shared_pages_and_their_groups(make):
    cache = make(batch_size=5, page_size=16, num_pages=30)
    cache.begin([50, 0, 0, 20, 0])
    assert cache.share(0, [1, 2]) == 48                       # whole pages
    assert cache.length_of == [50, 48, 48, 20, 0] and cache.lengths.tolist() == cache.length_of == cache.seen_after.tolist()
    assert (cache.page_table[:3, :3] == cache.page_table[0, :3]).all() and cache.free_pages == 30 - 4 - 2
    groups = lambda: (cache._group_start.tolist(), cache._group_shared.tolist())  # noqa: E731
    assert cache._alike and groups() == ([0, 3, 4, 5, 5, 5], [48, 0, 0, 0, 0])      # filled up with empty ones
    cache.begin([1, 1, 1, 1, 0])                              # request 0 goes on in its last page, the others on pages of their own
    assert cache.free_pages == 30 - 4 - 2 - 2
    assert len({int(cache.page_table[b, 3]) for b in range(3)}) == 3
    assert cache.share(1, [4], slots=33) == 32
    assert groups() == ([0, 3, 4, 5, 5, 5], [48, 0, 0, 0, 0])
    cache.release(0)                                          # what others begin with stays
    assert cache.free_pages == 30 - 4 - 2 - 2 + 1 and groups() == ([0, 1, 3, 4, 5, 5], [0, 48, 0, 0, 0])
    cache.release(2)
    cache.release(4)
    assert not cache._alike
    cache.release(1)
    cache.release(3)
    assert cache.free_pages == 30 and not cache._sharers and sorted(cache._free) == list(range(30))


def test_what_cannot_be_shared_is_refused(make):
    cache = make(batch_size=3)
    cache.begin([40, 3, 0])
    for of, requests, slots in ((0, [0], None), (0, [1], None), (0, [2, 2], None), (0, [3], None), (0, [2], 41), (0, [2], -1)):
        with pytest.raises(ValueError):
            cache.share(of, requests, slots)
    assert cache.share(1, [2]) == 0 and cache.length_of == [40, 3, 0]
    cache = make(keep=80)
    cache.begin([40, 0])
    with pytest.raises(ValueError, match="evicted"):
        cache.share(0, [1])
