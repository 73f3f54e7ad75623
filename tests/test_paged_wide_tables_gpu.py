"""Page tables with rows that lie apart, and caches whose max_length is far beyond what their requests hold."""
import pytest
import torch

from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu


def widened(layer, more, seed=0):
    """The layer's table as the front columns of a wider one, whose other entries name no page."""
    wide = torch.full((layer.table.shape[0], layer.table.shape[1] + more), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, :layer.table.shape[1]] = layer.table
    return wide[:, :layer.table.shape[1]]


@pytest.mark.parametrize("lengths", [(300, 0, 77), (5000, 3, 900)])
def test_the_same_results_to_the_bit(lengths):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors
    from retrievalattention_b200.decode_layer import cos_sin_cache

    results = []
    for more in (0, 1000):
        layer = Layer(lengths, 2, 16, torch.bfloat16, seed=71, room=16)
        table = widened(layer, more)
        assert table.is_contiguous() == (more == 0)
        q = torch.randn((3, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
        late = torch.randn((3, 12, 8, DIM), generator=layer.gen).bfloat16().cuda()
        qkv = torch.randn((3, 12 * DIM), generator=layer.gen).bfloat16().cuda()
        lse = torch.empty((3, 8), device="cuda")
        out = paged.paged_decode(q, layer.keys, layer.values, table, layer.lengths, lse=lse, weight=layer.weight)
        paged.paged_observe(late, layer.keys, table, layer.lengths, layer.weight)
        rows = torch.empty((3, 8, DIM), dtype=torch.bfloat16, device="cuda")
        paged.rope_paged_append(qkv, cos_sin_cache(100, DIM, 1e4, "cuda"), torch.arange(3, device="cuda"), paged.rope_sections(64), rows, layer.keys,
                                layer.values, table, layer.lengths, weight=layer.weight, token=layer.token, seen=layer.lengths)
        paged.paged_evict(layer.keys, layer.values, layer.weight, layer.token, table, layer.lengths + 1, layer.lengths + 1, 64, 4, 16)
        check_prefill_errors()
        results.append((out, lse, rows, layer.keys, layer.values, layer.weight, layer.token))
    for a, b in zip(*results):
        kind = torch.int16 if a.element_size() == 2 else torch.int32
        assert torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


def test_one_request_and_rows_that_overlap():
    from retrievalattention_b200 import paged

    layer = Layer((300,), 2, 16, torch.bfloat16, seed=72)
    q = torch.randn((1, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    want = paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths)
    assert torch.equal(paged.paged_decode(q, layer.keys, layer.values, widened(layer, 7), layer.lengths), want)
    two = torch.cat([q, q])
    with pytest.raises(ValueError, match="overlap"):
        paged.paged_decode(two, layer.keys, layer.values, layer.table.expand(2, -1), layer.lengths.expand(2).contiguous())
    with pytest.raises(ValueError, match="dense rows"):
        paged.paged_decode(q, layer.keys, layer.values, torch.cat([layer.table] * 2, 1)[:, ::2], layer.lengths)


def test_workspaces_follow_the_slots_in_use():
    """16 requests of 512 slots in a cache that would take 128K of each: a step's decode needs a score for every slot in use and query
    head (1 MB) and the partial results (some 5 MB), not one for every slot that there might be (268 MB)."""
    from retrievalattention_b200.cache_hub import paged_cache

    cache = paged_cache(1, 16, 131072, 8, 32, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1, num_pages=16 * 36, keep=512, sink=4, recent=64)
    cache.begin(512)
    q = torch.randn((16, 1, 32, DIM), device="cuda").bfloat16()
    out = torch.empty_like(q)
    cache.attend(q, 0, out=out)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    cache.attend(q, 0, out=out)
    assert torch.cuda.max_memory_allocated() - before <= 16 << 20
    cache.begin(1)
    assert cache.evict(slack=0)
    assert torch.cuda.max_memory_allocated() - before <= 16 << 20


def test_an_eviction_and_a_longer_request_are_followed():
    from paged_helpers import attend
    from retrievalattention_b200.cache_hub import paged_cache

    gen = torch.Generator().manual_seed(73)
    cache = paged_cache(1, 2, 10000, 1, 4, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1, page_size=8, keep=64, sink=4, recent=16)
    for pool in (cache.key_pages[0], cache.value_pages[0]):
        pool.copy_(torch.randn(pool.shape, generator=gen).bfloat16())

    def check():
        q = torch.randn((2, 1, 4, DIM), generator=gen).bfloat16().cuda()
        out = cache.attend(q, 0)
        for b in range(2):
            ids = cache.page_table[b, :-(-cache.length_of[b] // 8)].long()
            k, v = (p[ids, 0].flatten(0, 1)[:cache.length_of[b]].cpu().double()[None] for p in (cache.key_pages[0], cache.value_pages[0]))
            want = attend(q[b, 0].cpu().double()[None], k, v)[0][0]
            assert ((out[b, 0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * 5).all()

    cache.begin([100, 20])
    check()
    cache.evict(slack=0)
    check()
    cache.begin([1, 5000])
    check()
    cache.release(1)
    cache.begin([30, 1])
    check()


def test_a_captured_step_follows_requests_that_grow():
    from paged_helpers import attend
    from retrievalattention_b200.cache_hub import paged_cache

    gen = torch.Generator().manual_seed(74)
    cache = paged_cache(1, 2, 6000, 1, 4, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1, page_size=8, keep=5000, sink=4, recent=16)
    for pool in (cache.key_pages[0], cache.value_pages[0]):
        pool.copy_(torch.randn(pool.shape, generator=gen).bfloat16())
    q = torch.randn((2, 1, 4, DIM), generator=gen).bfloat16().cuda()
    cache.begin([30, 7])
    cache.attend(q, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, 0)
        with pytest.raises(RuntimeError, match="captured"):
            cache.attend(q, 0, requests=[0])
    for more in (1, [700, 40], [1, 4500]):
        cache.begin(more)
        graph.replay()
        for b in range(2):
            ids = cache.page_table[b, :-(-cache.length_of[b] // 8)].long()
            k, v = (p[ids, 0].flatten(0, 1)[:cache.length_of[b]].cpu().double()[None] for p in (cache.key_pages[0], cache.value_pages[0]))
            want = attend(q[b, 0].cpu().double()[None], k, v)[0][0]
            assert ((out[b, 0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * 5).all()
