"""``paged.paged_observe`` against softmax in 64 bits.

Tolerance: as for ``paged_decode`` a probability is within 6e-5 of its own size; the sum over the query rows adds their rounding
(2^-24 a term, at most 2^9 terms here: 3e-5), and the slot's old weight its own."""
import pytest
import torch

from paged_helpers import DIM, Layer, attend

pytestmark = pytest.mark.gpu


def given(layer, q, scale=DIM ** -0.5):
    """What every slot is given, per request [kv_heads, slots] in 64 bits."""
    b, window, hq, _ = q.shape
    sums = []
    for i, n in enumerate(layer.lengths_list):
        gs = hq // layer.hk
        rows = q[i].cpu().double().view(window, layer.hk, gs, DIM).transpose(0, 1)
        last = n - window + torch.arange(window)
        rows = torch.where((last >= 0)[None, :, None, None], rows, torch.zeros_like(rows)).reshape(layer.hk, window * gs, DIM)
        allowed = (torch.arange(n) <= last[:, None]).repeat_interleave(gs, 0)
        sums.append(attend(rows, layer.k[i], layer.v[i], allowed, scale)[2].sum(1))
    return sums


def check(layer, q, scale=None, calls=1):
    from retrievalattention_b200 import paged

    untouched = layer.weight.clone()
    for _ in range(calls):
        paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight, scale=scale)
    mine = torch.zeros_like(untouched, dtype=torch.bool)
    for i, add in enumerate(given(layer, q, DIM ** -0.5 if scale is None else scale)):
        n = layer.lengths_list[i]
        layer.scatter(mine, i, torch.ones((layer.hk, n), dtype=torch.bool))
        got, want = layer.gather(layer.weight, i).double(), layer.w[i] + calls * add
        assert ((got - want).abs() <= calls * 9e-5 * add + calls * 2.0 ** -23 * want + 1e-12).all(), i
    assert torch.equal(layer.weight.view(torch.int32)[~mine], untouched.view(torch.int32)[~mine])


@pytest.mark.parametrize("lengths,kv_heads,group,window,page,dtype", [
    ((1,), 1, 1, 1, 8, torch.bfloat16),                              # one slot, one row
    ((0,), 1, 4, 4, 16, torch.bfloat16),                             # nothing
    ((0, 3, 127, 128, 129, 0), 2, 3, 5, 8, torch.float16),           # windows longer than the request; edges of a tile
    ((1001,), 8, 4, 16, 16, torch.bfloat16),
    ((300, 77, 513), 2, 4, 32, 32, torch.bfloat16),                  # 128 rows: one tile of them
    ((300, 77, 513), 2, 3, 43, 64, torch.float16),                   # 129 rows: two
    ((2000, 100), 1, 8, 32, 128, torch.bfloat16),                    # 256 rows
    ((700, 30), 2, 8, 33, 256, torch.bfloat16),                      # 264 rows: 256 and then 8
    ((900,), 1, 5, 110, 1024, torch.float16),                        # 550 rows
    ((40,) * 50, 4, 2, 7, 16, torch.bfloat16),                       # more groups than SMs
    ((9001, 1), 2, 7, 9, 8, torch.bfloat16),                         # 63 rows; one group over many SMs
    ((390, 7, 8, 9), 2, 6, 40, 8, torch.float16),                    # 240 rows, the smallest pages
])
def test_against_64_bits(lengths, kv_heads, group, window, page, dtype):
    layer = Layer(lengths, kv_heads, page, dtype, seed=31)
    q = torch.randn((len(lengths), window, kv_heads * group, DIM), generator=layer.gen).to(dtype)
    for i, n in enumerate(lengths):
        q[i, :max(0, window - n)] = float("nan")                     # rows in front of a short request may hold anything
    check(layer, q.cuda())


def test_scale_pages_apart_and_two_calls():
    layer = Layer((500, 3), 2, 16, torch.bfloat16, seed=32, apart=True)
    q = torch.randn((2, 8, 8, DIM), generator=layer.gen).bfloat16().cuda()
    check(layer, q, scale=0.05, calls=2)


def test_scores_that_grow_along_the_cache():
    layer = Layer((2000,), 1, 32, torch.float16, seed=33)
    k = (torch.randn((1, 2000, DIM), generator=layer.gen) * torch.linspace(0.1, 8, 2000)[None, :, None]).half()
    layer.fill(0, k, layer.v[0].half(), layer.w[0].float(), layer.t[0])
    q = torch.randn((1, 16, 4, DIM), generator=layer.gen).half().cuda()
    from retrievalattention_b200 import paged

    paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight)
    add = given(layer, q)[0]
    got = layer.gather(layer.weight, 0).double() - layer.w[0]
    assert ((got - add).abs() <= 8 * 9e-5 * add + 2.0 ** -23 * (layer.w[0] + add) + 1e-12).all()     # products eight times as large


def test_one_query_is_what_decode_gives():
    from retrievalattention_b200 import paged

    layer = Layer((333, 20), 2, 16, torch.bfloat16, seed=34)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    other = layer.weight.clone()
    paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight)
    paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths, weight=other)
    for i in range(2):
        a, b = layer.gather(layer.weight, i), layer.gather(other, i)
        assert ((a - b).abs() <= 1.2e-4 * b).all()


def test_repeats_to_the_bit_and_in_a_captured_call():
    from retrievalattention_b200 import paged

    layer = Layer((3000, 700, 1), 2, 16, torch.bfloat16, seed=35)
    start = layer.weight.clone()
    q = torch.randn((3, 20, 8, DIM), generator=layer.gen).bfloat16().cuda()
    paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight)
    first = layer.weight.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight)
    for _ in range(2):
        layer.weight.copy_(start)
        graph.replay()
        assert torch.equal(layer.weight.view(torch.int32), first.view(torch.int32))


def test_offsets_past_32_bits():
    page, hk = 128, 8
    first = (1 << 31) // (hk * page * DIM) + 3
    layer = Layer((700, 260), hk, page, torch.bfloat16, seed=36, first_page=first)
    assert layer.keys.numel() > 1 << 31
    check(layer, torch.randn((2, 4, 16, DIM), generator=layer.gen).bfloat16().cuda())


def test_page_number_outside_the_pool_is_reported():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer((100, 40), 1, 16, torch.bfloat16, seed=37, spare=0)
    q = torch.randn((2, 3, 2, DIM), generator=layer.gen).bfloat16().cuda()
    table = layer.table.clone()
    table[0, 2] = layer.keys.shape[0]
    with pytest.raises(RuntimeError, match="names no page"):
        paged.paged_observe(q, layer.keys, table, layer.lengths, layer.weight)
        check_prefill_errors()
    got, add = layer.gather(layer.weight, 1).double(), given(layer, q)[1]
    assert ((got - layer.w[1] - add).abs() <= 1e-4 * add + 2.0 ** -23 * (layer.w[1] + add)).all()


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer((100, 40), 2, 16, torch.bfloat16, seed=38)
    q = torch.randn((2, 5, 8, DIM), generator=layer.gen).bfloat16().cuda()
    good = dict(q=q, key_pages=layer.keys, page_table=layer.table, lengths=layer.lengths, weight=layer.weight)
    for change in (dict(q=q[:, :, :7]), dict(q=q.half()), dict(q=q[:1]), dict(q=q[:, :0]), dict(q=q.transpose(1, 2)), dict(q=q.cpu()),
                   dict(q=q.clone().requires_grad_()), dict(weight=None), dict(weight=layer.weight.double()),
                   dict(key_pages=layer.keys[0]), dict(lengths=layer.lengths.long())):
        with pytest.raises(ValueError):
            paged.paged_observe(**{**good, **change})
    with pytest.raises(RuntimeError, match="scale"):
        paged.paged_observe(**good, scale=0.0)
