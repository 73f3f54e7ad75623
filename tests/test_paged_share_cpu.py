"""``share`` of ``paged_cache`` and ``PagedDecoder`` on the host: whatever the requests come in, and whose prompt it is."""
import pytest
import torch

from test_paged_cache_cpu import make  # noqa: F401


def test_requests_in_anything_that_can_be_gone_through(make):  # noqa: F811
    from retrievalattention_b200.decode_layer import ModelShape, PagedDecoder

    for requests in ([1, 2], (1, 2), torch.tensor([1, 2]), iter([1, 2]), (b for b in (1, 2)), map(int, "12")):
        cache = make(batch_size=4, page_size=16)
        model = PagedDecoder(ModelShape(64, 64, 50, 1, 8, 2), cache, 4, 200, "cpu")
        cache.begin([40, 0, 0, 3])
        assert model.share(0, requests) == 32
        assert cache.length_of == [40, 32, 32, 3] and model._next_position == [0, 32, 32, 0]
        assert model.positions.tolist() == [[0, 32, 32, 0]]


@pytest.mark.parametrize("of", [-1, -3, 3, 100])
def test_requests_that_are_none(make, of):  # noqa: F811
    cache = make(batch_size=3)
    cache.begin([0, 0, 40])
    with pytest.raises(ValueError, match="of 3"):
        cache.share(of, [0])
    assert cache.length_of == [0, 0, 40] and not cache._sharers


def test_windows_that_are_no_numbers_of_slots(make):  # noqa: F811
    import math

    for bad in (dict(attn_window=2.5), dict(attn_window=[2.5]), dict(attn_window=30, attn_sink=0.5)):
        with pytest.raises(ValueError, match="attn_window"):
            make(**bad)
    for bad in (math.inf, math.nan):                            # no window is None
        with pytest.raises((ValueError, OverflowError)):
            make(attn_window=bad)
    cache = make(attn_window=30.0, attn_sink=4.0)
    assert cache.attn_window == [30] and all(type(x) is int for x in cache.attn_window + [cache.attn_sink])
