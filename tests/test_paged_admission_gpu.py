"""Requests that come and go: a prompt in a released place beside running requests, and steps of some of the requests."""
import pytest
import torch

from paged_helpers import DIM, attend

pytestmark = pytest.mark.gpu

HK, GROUP, PAGE = 2, 4, 16


def make(batch, keep=None, **more):
    from retrievalattention_b200.cache_hub import paged_cache

    args = dict(page_size=PAGE, keep=keep, sink=2, recent=12, slack=8)
    return paged_cache(1, batch, 600, HK, HK * GROUP, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1, **{**args, **more})


def feed(cache, counts, gen):
    """A step of `counts` tokens: random rows appended, and the queries of all of them."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.decode_layer import cos_sin_cache

    rows = sum(counts)
    qkv = torch.randn((rows, (HK * GROUP + 2 * HK) * DIM), generator=gen).bfloat16().cuda()
    q = torch.empty((rows, HK * GROUP, DIM), dtype=torch.bfloat16, device="cuda")
    cache.begin(counts)
    positions = torch.cat([torch.arange(int(s), int(s) + n) for s, n in zip(cache.seen.tolist(), counts)])
    cache.append(0, qkv, cos_sin_cache(2000, DIM, 1e4, "cuda"), positions.cuda(), paged.rope_sections(64), q)
    return q


def slots(cache, pool, b):
    ids = cache.page_table[b, :-(-cache.length_of[b] // PAGE)].long()
    return pool[ids].transpose(0, 1).flatten(1, 2)[:, :cache.length_of[b]].cpu().double()


def last_queries(q, n, window):
    x = torch.zeros((1, window, HK * GROUP, DIM), dtype=q.dtype, device="cuda")
    w = min(n, window)
    x[0, window - w:] = q[-w:]
    return x


def given(cache, b, queries):
    """What the last queries of request b give its slots, in 64 bits."""
    n, window = cache.length_of[b], queries.shape[1]
    last = n - window + torch.arange(window)
    rows = torch.where((last >= 0)[:, None, None], queries[0].cpu().double(), 0.0).view(window, HK, GROUP, DIM).transpose(0, 1)
    allowed = (torch.arange(n) <= last[:, None]).repeat_interleave(GROUP, 0)
    return attend(rows.reshape(HK, -1, DIM), slots(cache, cache.key_pages[0], b), slots(cache, cache.value_pages[0], b), allowed)[2].sum(1)


@pytest.mark.parametrize("evicted", [False, True])
def test_a_prompt_in_a_released_place(evicted):
    """Its slots get the weights of its own queries, nobody else's change, and eviction goes by them."""
    keep = 40
    cache, gen = make(3, keep=keep), torch.Generator().manual_seed(5)
    counts = [100, 70, 30] if evicted else [38, 20, 30]
    q = feed(cache, counts, gen)
    cache.observe(torch.cat([last_queries(x, x.shape[0], 16) for x in q.split(counts)]), 0)
    assert cache.evict(slack=0) == evicted
    feed(cache, [1, 1, 1], gen)
    cache.release(1)
    others = {b: slots(cache, cache.weight[0], b) for b in (0, 2)}
    q = feed(cache, [0, 90, 0], gen)
    with pytest.raises(RuntimeError if evicted else ValueError, match="evicted" if evicted else "no tokens in this step"):
        cache.observe(torch.zeros((3, 16, HK * GROUP, DIM), dtype=q.dtype, device="cuda"), 0)
    queries = last_queries(q, 90, 16)
    cache.observe(queries, 0, requests=[1])
    for b, w in others.items():
        assert torch.equal(slots(cache, cache.weight[0], b), w)
    want = given(cache, 1, queries)
    assert ((slots(cache, cache.weight[0], 1) - want).abs() <= 1e-4 * want + 1e-12).all()

    # what stays: the first two and last twelve tokens, then the largest weights
    weight, token = slots(cache, cache.weight[0], 1), slots(cache, cache.token[0], 1)
    assert cache.evict(slack=0) and cache.length_of[1] == keep
    for h in range(HK):
        safe = (token[h] < 2) | (token[h] >= 90 - 12)
        order = sorted(range(90), key=lambda j: (not safe[j], -weight[h, j].item(), j))
        assert set(slots(cache, cache.token[0], 1)[h].tolist()) == {token[h, j].item() for j in order[:keep]}
    with pytest.raises(RuntimeError, match="request 1 were evicted"):
        cache.observe(queries, 0, requests=[1])
    cache.release(1)                                             # and the place is as good as new
    q = feed(cache, [0, 17, 0], gen)
    cache.observe(last_queries(q, 17, 16), 0, requests=[1])
    want = given(cache, 1, last_queries(q, 17, 16))
    assert ((slots(cache, cache.weight[0], 1) - want).abs() <= 1e-4 * want + 1e-12).all()


def test_steps_of_some_requests_in_their_order():
    cache, gen = make(4, keep=64), torch.Generator().manual_seed(6)
    feed(cache, [33, 5, 60, 20], gen)
    cache.release(1)
    before = {b: slots(cache, cache.weight[0], b) for b in (0, 2, 3)}
    feed(cache, [1, 0, 0, 1], gen)
    assert cache.length_of == [34, 0, 60, 21] == cache.lengths.tolist()
    q = torch.randn((2, 1, HK * GROUP, DIM), generator=gen).bfloat16().cuda()
    lse = torch.empty((2, HK * GROUP), device="cuda")
    out = cache.attend(q, 0, lse=lse, requests=[3, 0])
    for i, b in enumerate((3, 0)):
        want, want_lse, p = attend(q[i, 0].cpu().double().view(HK, GROUP, DIM), slots(cache, cache.key_pages[0], b), slots(cache, cache.value_pages[0], b))
        assert ((out[i, 0].cpu().double().view_as(want) - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * 5).all()
        assert ((lse[i].cpu().double().view_as(want_lse) - want_lse).abs() <= 3e-5).all()
        old = torch.cat([before[b], torch.zeros(HK, 1)], 1)      # and the new slot
        assert ((slots(cache, cache.weight[0], b) - old - p.sum(1)).abs() <= 6e-5 * p.sum(1) + 2.0 ** -22).all()
    assert torch.equal(slots(cache, cache.weight[0], 2), before[2])
    for bad in ([], [0, 0], [4], [-1]):
        with pytest.raises(ValueError, match="different requests"):
            cache.attend(q, 0, requests=bad)


def test_prompts_of_several_steps_are_observed_at_once():
    """A request whose prompt ended a step before the others' is observed with them."""
    cache, gen = make(2, keep=400), torch.Generator().manual_seed(7)
    first = feed(cache, [70, 90], gen)[70:]
    q = feed(cache, [50, 0], gen)
    queries = torch.cat([last_queries(x, x.shape[0], 16) for x in (q, first)])
    cache.observe(queries, 0)
    cache.evict(slack=0)
    for b in range(2):
        want = given(cache, b, queries[b:b + 1])
        assert ((slots(cache, cache.weight[0], b) - want).abs() <= 1e-4 * want + 1e-12).all()
    feed(cache, [9, 0], gen)
    with pytest.raises(ValueError, match="request 1 had no tokens"):
        cache.observe(queries, 0)
