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
