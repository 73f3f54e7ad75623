"""``cache_hub.paged_cache`` on the host: whose a step's rows are stays in one place from step to step, as captured calls need it."""
from test_paged_cache_cpu import make  # noqa: F401


def test_rows_of_every_step_lie_in_one_place(make, monkeypatch):  # noqa: F811
    from retrievalattention_b200 import paged

    cache, handed = make(batch_size=3), []
    monkeypatch.setattr(paged, "paged_prompt", lambda q, k, v, table, lengths, starts, **rest: handed.append(starts))
    monkeypatch.setattr(paged, "rope_paged_append", lambda *args, **rest: handed.append(args[9]))
    monkeypatch.setattr(cache, "_captures", lambda: True, raising=False)
    where = set()
    for counts, starts in (([5, 0, 7], [0, 5, 5, 12]), (1, [0, 1, 2, 3]), (1, [0, 1, 2, 3]), ([0, 2, 1], [0, 0, 2, 3]), ([1, 1, 1], [0, 1, 2, 3]),
                           (2, [0, 2, 4, 6]), (1, [0, 1, 2, 3])):
        cache.begin(counts)
        handed.clear()
        cache.append(0, *[None] * 5)
        cache.prompt(None, 0)
        assert [x.tolist() for x in handed] == [starts, starts], counts
        where |= {x.data_ptr() for x in handed}
    assert len(where) == 1
