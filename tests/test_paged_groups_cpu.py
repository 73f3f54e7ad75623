"""``cache_hub.paged_cache`` on the host: which requests are attended together, over how many slots."""
import itertools
import random

from test_paged_cache_cpu import make  # noqa: F401


def groups(cache):
    return cache._group_start.tolist(), cache._group_shared.tolist()


def test_the_longest_common_prompt_is_not_lost(make):  # noqa: F811
    """A system prompt of a page, a document behind it, questions about the document."""
    cache = make(batch_size=5, max_length=4000, page_size=16, num_pages=600)
    cache.begin([16, 0, 0, 0, 0])
    assert cache.share(0, [1]) == 16
    cache.begin([3, 1600, 0, 0, 0])
    assert cache.share(1, [2, 3, 4]) == 1616
    cache.begin([1, 1, 5, 6, 7])
    starts, shared = groups(cache)
    assert starts == [0, 1, 5, 5, 5, 5] and shared == [0, 1616, 0, 0, 0]
    cache.release(0)
    assert groups(cache)[1][:2] == [0, 1616]


def test_the_fewest_slots_are_read(make):  # noqa: F811
    """Against every way to cut requests into runs."""
    rng = random.Random(4)
    cache = make(batch_size=7, max_length=4000)
    for _ in range(60):
        tree = [[]]
        while len(tree) < 7:                                    # each begins as one of those before it does
            like = rng.choice(tree)
            tree.append(like[:rng.randint(0, len(like))] + [rng.random() for _ in range(rng.randint(0, 4))])
        cache._pages = [tree[i] for i in rng.sample(range(7), 7)]
        alike = lambda a, b: next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))  # noqa: E731
        most = 0
        for cuts in itertools.product((False, True), repeat=6):
            ends = [i + 1 for i, c in enumerate(cuts) if c] + [7]
            total = 0
            for i, j in zip([0] + ends, ends):
                total += (j - i - 1) * min((alike(cache._pages[i], cache._pages[x]) for x in range(i + 1, j)), default=0)
            most = max(most, total)
        starts, shared = cache._in_common(range(7))
        assert starts[0] == 0 and starts[-1] == 7 and all(i < j for i, j in zip(starts, starts[1:])) and len(shared) == len(starts) - 1
        assert sum((j - i - 1) * n for i, j, n in zip(starts, starts[1:], shared)) == most * cache.page_size
        for i, j, n in zip(starts, starts[1:], shared):
            assert all(cache._pages[x][:n // cache.page_size] == cache._pages[i][:n // cache.page_size] for x in range(i, j))


def called(cache, monkeypatch):
    """What `attend` calls, with the groups it hands over."""
    from retrievalattention_b200 import paged

    calls = []
    monkeypatch.setattr(paged, "paged_decode", lambda q, *args, **rest: calls.append(None))
    monkeypatch.setattr(paged, "paged_shared_decode", lambda q, k, v, table, lengths, starts, shared, **rest: calls.append((starts.tolist(), shared.tolist())))
    return calls


def test_some_of_the_requests_are_grouped_too(make, monkeypatch):  # noqa: F811
    """One of those that begin alike is done: the others still read once what they have in common."""
    cache = make(batch_size=5, max_length=40000, page_size=16, num_pages=2600, num_key_value_heads=8, num_heads=32)
    calls = called(cache, monkeypatch)
    for name in ("_PAYS_MB", "_PAYS_MB_EACH"):                  # whatever it saves
        monkeypatch.setattr(cache, name, 0, raising=False)
    cache.begin([32768, 0, 0, 0, 40])
    assert cache.share(0, [1, 2, 3]) == 32768
    cache.release(2)
    for step in range(2):
        cache.begin([1, 1, 0, 1, 1])
        cache.attend(None, 0, requests=[0, 1, 3, 4])
        assert calls.pop() == ([0, 3, 4], [32768, 0])
        cache.attend(None, 0, requests=(4, 3, 1))               # in the order of their queries
        assert calls.pop() == ([0, 1, 3], [0, 32768])
        cache.attend(None, 0, requests=[4])
        cache.attend(None, 0, requests=[3, 4])
        assert calls == [None, None] and not calls.clear()
    cache.release(0)                                            # groups of before are not gone by
    cache.begin([1, 1, 0, 1, 1])
    cache.attend(None, 0, requests=[0, 1, 3, 4])
    assert calls.pop() == ([0, 1, 3, 4], [0, 32768, 0])
    cache.release(1)
    cache.begin([0, 0, 0, 1, 1])
    cache.attend(None, 0, requests=[3, 4])
    assert calls.pop() is None


def test_little_in_common_is_not_worth_a_kernel(make, monkeypatch):  # noqa: F811
    """A page in common in front of long requests: one by one, all of them or some; a captured call goes by the groups all the same, which
    may have more in common when it is replayed."""
    args = dict(batch_size=3, max_length=70000, page_size=16, num_pages=9000, num_key_value_heads=8, num_heads=32)
    cache = make(**args)
    calls = called(cache, monkeypatch)
    cache.begin([30, 0, 30000])
    cache.share(0, [1])
    cache.begin([30000, 30000, 1])
    cache.attend(None, 0)
    cache.attend(None, 0, requests=[0, 1])
    assert calls == [None, None] and cache._alike
    monkeypatch.setattr(cache, "_captures", lambda: True)
    cache.attend(None, 0)
    assert calls.pop() == ([0, 2, 3, 3], [16, 0, 0])
    monkeypatch.setattr(cache, "_captures", lambda: False)
    cache = make(**args)                                        # 265 MB (of 2^20) of keys and values in common
    cache.begin([68010, 0, 1])
    cache.share(0, [1], 68000)
    cache.attend(None, 0, requests=[0, 1])                      # 256 and 4 for each of two requests
    assert calls.pop() == ([0, 2], [68000])
    cache.attend(None, 0)                                       # of three
    assert calls.pop() is None
