"""``paged.paged_decode`` against attention in 64 bits: outputs, log-sum-exp and accumulated weights.

Tolerances.  A score is a sum of 128 products that are exact in 32 bits; their magnitudes times the scale add up to about 8 here, and
32-bit sums of that, in whatever order, are within 32 roundings of 2^-24 of it: 1.6e-5.  Hence lse within 3e-5 and a probability
within 6e-5 of its own size.  The output is a sum of probabilities (two 16-bit parts: 2^-16) times values plus its own rounding."""
import pytest
import torch

from paged_helpers import DIM, Layer, attend, rounding

pytestmark = pytest.mark.gpu


def call(layer, q, **more):
    from retrievalattention_b200 import paged

    return paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths, **more)


def check(layer, q, out, lse=None, before=None, scale=DIM ** -0.5):
    b, _, hq, _ = q.shape
    half, tiny = rounding(q.dtype)
    for i in range(b):
        want, want_lse, p = attend(q[i, 0].cpu().double().view(layer.hk, hq // layer.hk, DIM), layer.k[i], layer.v[i], scale=scale)
        got = out[i, 0].cpu().double().view_as(want)
        most = layer.v[i].abs().max() if layer.v[i].numel() else 0.0
        assert ((got - want).abs() <= half * want.abs() + 1e-4 * most + tiny).all(), (i, (got - want).abs().max())
        if lse is not None:
            got = lse[i].cpu().double().view_as(want_lse)
            assert torch.equal(torch.isinf(got), torch.isinf(want_lse))
            assert ((got - want_lse).abs()[torch.isfinite(want_lse)] <= 3e-5).all()
        if before is not None:
            n = layer.lengths_list[i]
            given = p.sum(1)
            got = layer.gather(layer.weight, i).double()
            assert got.shape == given.shape == (layer.hk, n)
            assert ((got - (before[i] + given)).abs() <= 6e-5 * given + 2.0 ** -23 * (before[i] + given) + 1e-12).all()


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("lengths,kv_heads,group,page,dtype", [
    ((1,), 1, 1, 16, torch.bfloat16),                          # one slot
    ((0,), 2, 4, 16, torch.bfloat16),                          # none
    ((0, 7, 8, 9, 0), 2, 3, 8, torch.float16),                 # pages of half a step
    ((0, 15, 16, 17, 31, 33), 2, 3, 16, torch.float16),        # edges of a step
    ((0, 0, 1), 1, 8, 32, torch.bfloat16),                     # requests without slots in front
    ((2047, 0, 130), 3, 5, 64, torch.float16),                 # a CTA's range over several groups
    ((4095,), 1, 7, 8, torch.bfloat16),                        # one group over the whole chip
    ((9001, 1), 2, 8, 256, torch.bfloat16),
    ((37,) * 90, 8, 2, 16, torch.bfloat16),                    # more groups than warps
    ((129, 640, 1023), 8, 4, 1024, torch.bfloat16),            # the largest pages
    ((980, 0, 31) * 5, 4, 7, 16, torch.float16),               # two CTAs to a group
    ((100, 5) * 8, 8, 1, 8, torch.bfloat16),                   # one
    ((2100,) * 3, 8, 2, 32, torch.bfloat16),                   # longer than a group's CTAs take: an even split over the chip
])
def test_against_64_bits(lengths, kv_heads, group, page, dtype, weights):
    layer = Layer(lengths, kv_heads, page, dtype, seed=3)
    q = torch.randn((len(lengths), 1, kv_heads * group, DIM), generator=layer.gen).to(dtype).cuda()
    lse = torch.full((len(lengths), kv_heads * group), 7.0, device="cuda")
    untouched = layer.weight.clone()
    out = call(layer, q, lse=lse, weight=layer.weight if weights else None)
    check(layer, q, out, lse, layer.w if weights else None)
    # slots that no request uses keep what they held; so does everything without weights
    mine = torch.zeros_like(untouched, dtype=torch.bool)
    for b, n in enumerate(lengths if weights else ()):
        layer.scatter(mine, b, torch.ones((kv_heads, n), dtype=torch.bool))
    assert torch.equal(layer.weight.view(torch.int32)[~mine], untouched.view(torch.int32)[~mine])


def test_weights_add_up_over_steps_and_repeat_to_the_bit():
    layer = Layer((300, 77), 2, 16, torch.bfloat16, seed=5)
    start = layer.weight.clone()
    total = [w.clone() for w in layer.w]
    qs = [torch.randn((2, 1, 8, DIM), generator=layer.gen).bfloat16().cuda() for _ in range(3)]
    for q in qs:
        call(layer, q, weight=layer.weight)
    for i in range(2):
        for q in qs:
            total[i] += attend(q[i, 0].cpu().double().view(2, 4, DIM), layer.k[i], layer.v[i])[2].sum(1)
        assert ((layer.gather(layer.weight, i).double() - total[i]).abs() <= 1e-4 * total[i]).all()
    first = layer.weight.clone()
    layer.weight.copy_(start)
    for q in qs:
        call(layer, q, weight=layer.weight)
    assert torch.equal(layer.weight.view(torch.int32), first.view(torch.int32))


def test_strided_queries_pages_apart_scale_and_given_output():
    layer = Layer((500, 3, 0), 2, 16, torch.bfloat16, seed=6, apart=True)
    assert layer.keys.stride(0) == 2 * layer.keys[0].numel()
    wide = torch.randn((3, 1, 12 + 4, DIM), generator=layer.gen).bfloat16().cuda()       # a slice of a fused projection
    q = wide[:, :, :12]
    out = torch.empty((3, 1, 12, DIM), dtype=q.dtype, device="cuda")
    assert call(layer, q, out=out, scale=0.05) is out
    check(layer, q, out, scale=0.05)


def test_scores_that_grow_along_the_cache():
    """The running maximum moves at nearly every step; probabilities in front vanish."""
    layer = Layer((2000,), 1, 32, torch.float16, seed=7)
    k = (torch.randn((1, 2000, DIM), generator=layer.gen) * torch.linspace(0.1, 8, 2000)[None, :, None]).half()
    layer.fill(0, k, layer.v[0].half(), layer.w[0].float(), layer.t[0])
    q = torch.randn((1, 1, 4, DIM), generator=layer.gen).half().cuda()
    lse = torch.empty((1, 4), device="cuda")
    out = call(layer, q, lse=lse, weight=layer.weight)
    want, want_lse, p = attend(q[0, 0].cpu().double()[None], layer.k[0], layer.v[0])
    # magnitudes of the products are eight times those above
    assert ((lse[0].cpu().double() - want_lse[0]).abs() <= 8 * 3e-5).all()
    assert ((out[0, 0].cpu().double() - want[0]).abs() <= 2.0 ** -11 * want[0].abs() + 8 * 1e-4 * layer.v[0].abs().max()).all()
    given = p.sum(1)
    assert ((layer.gather(layer.weight, 0).double() - layer.w[0] - given).abs() <= 8 * 6e-5 * given + 2.0 ** -23 * (1 + given)).all()


def test_infinite_values_come_out_as_infinities():
    layer = Layer((100,), 1, 16, torch.bfloat16, seed=8)
    v = layer.v[0].clone()
    v[0, 40, 5], v[0, 99, 6] = float("inf"), float("-inf")
    layer.fill(0, layer.k[0].bfloat16(), v.bfloat16(), layer.w[0].float(), layer.t[0])
    out = call(layer, torch.randn((1, 1, 2, DIM), generator=layer.gen).bfloat16().cuda())
    assert (out[0, 0, :, 5] == float("inf")).all() and (out[0, 0, :, 6] == float("-inf")).all()
    keep = [c for c in range(DIM) if c not in (5, 6)]
    assert torch.isfinite(out[0, 0][:, keep]).all()


def test_offsets_past_32_bits():
    """Pages behind 2^31 elements of the pools, weights included."""
    page, hk = 128, 8
    first = (1 << 31) // (hk * page * DIM) + 3
    layer = Layer((700, 260), hk, page, torch.bfloat16, seed=9, first_page=first)
    assert layer.keys.numel() > 1 << 31
    q = torch.randn((2, 1, 16, DIM), generator=layer.gen).bfloat16().cuda()
    out = call(layer, q, weight=layer.weight)
    check(layer, q, out, before=layer.w)


def test_captured_call_follows_lengths_and_pages():
    layer = Layer((64, 200), 2, 16, torch.bfloat16, seed=10)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    call(layer, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(layer, q)
    layer.table.copy_(layer.table.flip(0))                    # the requests change places, and one of them length
    layer.lengths.copy_(torch.tensor([200, 33], dtype=torch.int32))
    graph.replay()
    for x in (layer.k, layer.v):
        x.reverse()
        x[1] = x[1][:, :33]
    check(layer, q, out)


def test_another_stream():
    layer = Layer((1000,), 2, 16, torch.bfloat16, seed=11)
    q = torch.randn((1, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [call(layer, q) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for out in outs:
        check(layer, q, out)


def test_page_number_outside_the_pool_is_reported():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer((100, 40), 1, 16, torch.bfloat16, seed=12, spare=0)
    q = torch.randn((2, 1, 2, DIM), generator=layer.gen).bfloat16().cuda()
    for bad in (-1, layer.keys.shape[0], 1 << 30):
        table = layer.table.clone()
        table[0, 2] = bad
        out, weight = torch.empty_like(q), layer.weight.clone()
        check_prefill_errors()
        with pytest.raises(RuntimeError, match="names no page"):       # by the call itself, if the kernel is done by then
            paged.paged_decode(q, layer.keys, layer.values, table, layer.lengths, out=out, weight=weight)
            check_prefill_errors()
        want, _, p = attend(q[1, 0].cpu().double()[None], layer.k[1], layer.v[1])       # the other request is served
        assert ((out[1, 0].cpu().double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 1e-3).all()
        assert ((layer.gather(weight, 1).double() - layer.w[1] - p.sum(1)).abs() <= 1e-4 * p.sum(1) + 2.0 ** -22).all()


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer((100, 40), 2, 16, torch.bfloat16, seed=13)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    good = dict(q=q, key_pages=layer.keys, value_pages=layer.values, page_table=layer.table, lengths=layer.lengths)
    paged.paged_decode(**good)
    ints = torch.zeros(2, dtype=torch.int64, device="cuda")
    for change in (dict(q=q[:, :, :7]), dict(q=q.half()), dict(q=q[..., :64]), dict(q=q[:1]), dict(q=q.transpose(2, 3)),
                   dict(q=q.cpu()), dict(q=q.clone().requires_grad_()), dict(q=torch.cat([q, q], 1)),
                   dict(key_pages=layer.keys[..., :64]), dict(key_pages=layer.keys.transpose(1, 2)), dict(value_pages=None),
                   dict(value_pages=layer.values[:-1]), dict(value_pages=layer.values.half()), dict(key_pages=layer.keys.cpu()),
                   dict(page_table=layer.table.long()), dict(page_table=layer.table.t()), dict(page_table=layer.table.cpu()),
                   dict(lengths=ints), dict(lengths=layer.lengths[:1]), dict(lengths=layer.lengths.cpu()),
                   dict(weight=layer.weight.double()), dict(weight=layer.weight[:-1]), dict(weight=layer.weight.transpose(1, 2)),
                   dict(weight=layer.weight.clone().requires_grad_()),
                   dict(lse=torch.empty((2, 7), device="cuda")), dict(lse=torch.empty((2, 8))),
                   dict(out=torch.empty((2, 1, 8, DIM), device="cuda"))):
        with pytest.raises(ValueError):
            paged.paged_decode(**{**good, **change})
    with pytest.raises(TypeError):
        paged.paged_decode(**{**good, "q": q.float(), "key_pages": layer.keys.float(), "value_pages": layer.values.float()})
    odd = torch.zeros((4, 2, 24, DIM), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="page_size"):
        paged.paged_decode(**{**good, "key_pages": odd, "value_pages": odd})
    with pytest.raises(RuntimeError, match="group_size"):
        paged.paged_decode(**{**good, "q": torch.cat([q, q, q], 2)})
    with pytest.raises(RuntimeError, match="aligned"):
        raw = torch.zeros(q.numel() + 4, dtype=q.dtype, device="cuda")[4:].view(q.shape)
        paged.paged_decode(**{**good, "q": raw})
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            paged.paged_decode(**good, scale=scale)
