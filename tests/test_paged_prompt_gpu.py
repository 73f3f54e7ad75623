"""``paged.paged_prompt`` against attention in 64 bits: prompts and pieces of prompts over pages, windows, first slots."""
import pytest
import torch

from attend_helpers import attend_rows, close, visible
from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu
INF = float("inf")


def expected(layer, b, q, n, window, sink):
    """Rows q [n, heads, 128] of request b's last n tokens, with the allowances."""
    length = layer.lengths_list[b]
    own = torch.arange(length - n, length)
    seen = visible(own, length, window, sink)
    return attend_rows(q.cpu().double(), layer.k[b], layer.v[b], seen)


def run(layer, counts, group, window=None, sink=0, seed=0, apart=0, front=0, behind=0, scale=None):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    gen = torch.Generator().manual_seed(seed + 100)
    hq, rows = layer.hk * group, front + sum(counts) + behind
    wide = torch.randn((rows, hq * DIM + apart), generator=gen).to(layer.dtype).cuda()
    q = wide[:, :hq * DIM].unflatten(1, (hq, DIM))
    starts = torch.tensor([front] + list(counts)).cumsum(0).to(torch.int32).cuda()
    out = torch.full((rows, hq, DIM), 7.0, dtype=layer.dtype, device="cuda")
    lse = torch.full((rows, hq), 7.0, device="cuda")
    got = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink, out=out, lse=lse)
    check_prefill_errors()
    assert got.data_ptr() == out.data_ptr()
    at = front
    for b, n in enumerate(counts):
        if n:
            r = slice(at, at + n)
            want = expected(layer, b, q[r], n, window, sink)
            assert close(out[r], lse[r], *want), (b, n, float((out[r].cpu().double() - want[0]).abs().max()))
        at += n
    assert (out[:front] == 7).all() and (out[at:] == 7).all() and (lse[:front] == 7).all() and (lse[at:] == 7).all()
    return q, starts, out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,held,hk,group,page,window,sink", [
    ((1,), 0, 1, 1, 16, None, 0),                       # one token, the only one
    ((1, 1, 1), 300, 2, 4, 8, 100, 3),                  # single tokens behind what is cached
    ((5, 0, 77), 0, 2, 4, 16, None, 0),                 # a request without rows
    ((130,), 0, 1, 7, 16, None, 0),                     # 18 tokens a tile
    ((333, 40), 129, 2, 4, 32, None, 0),
    ((300, 20), 100, 2, 2, 64, 64, 4),
    ((257,), 700, 1, 8, 128, 128, 0),
    ((200,), 512, 1, 4, 256, 130, 200),                 # more first slots than a tile
    ((90, 600), 0, 1, 3, 8, 1, 0),                      # every token sees itself alone
    ((90, 600), 0, 1, 5, 16, 1, 1),
    ((400,), 0, 2, 6, 16, 250, 300),                    # first slots that overlap the window
    ((64,), 64, 4, 1, 1024, 5000, 9),                   # a window wider than the request
])
def test_against_64_bits(dtype, counts, held, hk, group, page, window, sink):
    layer = Layer([n + held for n in counts], hk, page, dtype, seed=len(counts) + page)
    run(layer, counts, group, window, sink)


@pytest.mark.parametrize("page", [8, 64])
def test_items_that_fall_to_several_ctas(page):
    """Few rows over many slots: partial results, two tiles and one."""
    for counts, held, group in (((70, 3), 9000, 4), ((40,), 20000, 1), ((33, 1, 0, 9), 5000, 7)):
        layer = Layer([n + held for n in counts], 1, page, torch.bfloat16, seed=group)
        run(layer, counts, group)
        run(layer, counts, group, window=4000, sink=5)


@pytest.mark.parametrize("group", [4, 7])
def test_many_requests(group):
    """Items of one tile and of two, in no order, many to a CTA."""
    gen = torch.Generator().manual_seed(group)
    counts = torch.randint(0, 75, (600,), generator=gen).tolist()
    held = torch.randint(0, 300, (600,), generator=gen).tolist()
    layer = Layer([n + h for n, h in zip(counts, held)], 2, 16, torch.bfloat16, seed=9)
    run(layer, counts, group)
    run(layer, counts, group, window=70, sink=3)


def test_rows_apart_and_rows_of_nobody():
    layer = Layer([50, 200], 2, 16, torch.bfloat16, apart=True)
    run(layer, (50, 37), 4, window=60, sink=2, apart=128, front=3, behind=5)


def test_more_rows_than_slots():
    """Rows in front of a request's first slot see nothing."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([3, 0], 2, 16, torch.bfloat16)
    q = torch.randn(5 + 4, 8, DIM, device="cuda").to(torch.bfloat16)
    starts, lse = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda"), torch.empty(9, 8, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, lse=lse)
    check_prefill_errors()
    want = expected(layer, 0, q[2:5], 3, None, 0)
    assert close(out[2:5], lse[2:5], *want)
    for r in (0, 1, 5, 6, 7, 8):
        assert (out[r] == 0).all() and (lse[r] == -INF).all()


@pytest.mark.parametrize("window,sink", [(None, 0), (90, 3)])
@pytest.mark.parametrize("count,held", [(150, 0), (20, 5000)])
def test_infinite_and_nan_values_that_a_row_does_not_see(count, held, window, sink):
    """Keys and values of later tokens, and of those in front of the window, take no part, whatever they hold."""
    n = count + held
    layer = Layer([n], 2, 16, torch.bfloat16, seed=5)
    late = n - 7                                        # the last seven tokens are seen by themselves and those behind them
    k, v, w, t = layer.k[0].clone(), layer.v[0].clone(), layer.w[0], layer.t[0]
    v[:, late, 5], v[:, late, 77], k[0, late + 3] = INF, float("nan"), float("nan")
    if window is not None:
        v[:, held // 2 + 4, 9] = float("nan")
    layer.fill(0, k.float(), v.float(), w.float(), t)
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    q = torch.randn((count, 8, DIM), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    starts, lse = torch.tensor([0, count], dtype=torch.int32, device="cuda"), torch.empty(count, 8, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink, lse=lse)
    check_prefill_errors()
    seen = visible(torch.arange(held, n), n, window, sink)
    clean = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    want, lse_want, spread, score = attend_rows(q.cpu().double(), clean, v, seen)
    p_nan = seen[:, late + 3]                            # rows (of the first KV head's group) that see the NaN key
    want[p_nan, :4], lse_want[p_nan, :4] = float("nan"), float("nan")
    inf_rows = seen[:, late]
    got, got_lse = out.cpu().double(), lse.cpu().double()
    assert torch.isnan(got[p_nan, :4]).all() and torch.isnan(got_lse[p_nan, :4]).all()
    for rows, heads in ((~p_nan, slice(0, 4)), (torch.ones_like(p_nan), slice(4, 8))):
        ok = torch.ones(DIM, dtype=torch.bool)
        ok[[5, 77, 9]] = False
        r = torch.nonzero(rows)[:, 0]
        assert close(out[r][:, heads][..., ok], lse[r][:, heads], want[r][:, heads][..., ok], lse_want[r][:, heads], spread[r][:, heads][..., ok],
                     score[r][:, heads])
        blind, sees = torch.nonzero(rows & ~inf_rows)[:, 0], torch.nonzero(rows & inf_rows)[:, 0]
        ch = [5, 77]
        assert close(out[blind][:, heads][..., ch], None, want[blind][:, heads][..., ch], lse_want[blind][:, heads], spread[blind][:, heads][..., ch],
                     score[blind][:, heads])
        assert (got[sees][:, heads, 5] == INF).all() and torch.isnan(got[sees][:, heads, 77]).all()
        if window is not None:
            nan9 = seen[:, held // 2 + 4]
            assert torch.equal(torch.isnan(got[r][:, heads, 9]), nan9[r, None].expand(-1, 4))


def test_infinities_of_both_signs_and_a_slot_that_counts_nothing():
    """+infinity and -infinity in a channel make NaN of it, one of them itself; a slot of score -infinity hands on nothing."""
    from retrievalattention_b200 import paged

    for held in (0, 4000):
        n = 100 + held
        layer = Layer([n], 1, 16, torch.bfloat16, seed=8)
        k, v = layer.k[0].clone(), layer.v[0].clone()
        at = held // 2 + 3
        v[:, at, 0], v[:, at + 1, 0] = INF, -INF
        v[:, at, 1], v[:, at + 2, 2] = INF, -INF
        k[:, at + 4], k[:, at + 4, 0] = 0.0, -INF
        v[:, at + 4, 3], v[:, at + 4, 4] = INF, float("nan")
        layer.fill(0, k.float(), v.float(), layer.w[0].float(), layer.t[0])
        q = torch.randn((100, 4, DIM), generator=torch.Generator().manual_seed(1)).abs().to(torch.bfloat16).cuda()
        out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, torch.tensor([0, 100], dtype=torch.int32, device="cuda"))
        own = torch.arange(held, n)
        late = own >= at + 4
        assert torch.isnan(out[late][..., 0]).all() and (out[late][..., 1] == INF).all() and (out[late][..., 2] == -INF).all()
        finite = torch.isfinite(k).all(-1)[0] & torch.isfinite(v).all(-1)[0] | (torch.arange(n) == at) | (torch.arange(n) == at + 1) | (torch.arange(n) == at + 2)
        seen = visible(own, n, None, 0) & finite
        kc = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
        want = attend_rows(q.cpu().double(), kc, v, seen)
        assert close(out[..., 3:], None, *(x[..., 3:] if x.dim() == 3 else x for x in want))


def test_scores_of_minus_infinity():
    """Keys that no finite query goes with: such slots count nothing, a row of nothing else is zeros."""
    layer = Layer([140], 1, 16, torch.bfloat16, seed=8)
    k = layer.k[0].clone()
    k[:, :40] = 0.0
    k[:, :40, 0] = -INF
    layer.fill(0, k.float(), layer.v[0].float(), layer.w[0].float(), layer.t[0])
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    q = torch.randn(140, 4, DIM, device="cuda").abs().to(torch.bfloat16)
    starts, lse = torch.tensor([0, 140], dtype=torch.int32, device="cuda"), torch.empty(140, 4, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, lse=lse)
    check_prefill_errors()
    assert (out[:40] == 0).all() and (lse[:40] == -INF).all()
    seen = visible(torch.arange(140), 140, None, 0) & (torch.arange(140) >= 40)
    k = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    want = attend_rows(q.cpu().double(), k, layer.v[0], seen)
    assert close(out, lse, *want)


def test_growing_scores():
    """Maxima that rise along the request, so that accumulators are rescaled again and again."""
    layer = Layer([1500], 1, 32, torch.bfloat16, seed=4)
    k = (layer.k[0] * torch.linspace(0.1, 12.0, 1500, dtype=torch.float64)[:, None]).to(torch.bfloat16)
    layer.fill(0, k, layer.v[0].float(), layer.w[0].float(), layer.t[0])
    run(layer, (700,), 4)
    run(layer, (700,), 4, window=600, sink=2)


def test_pages_that_no_row_sees_are_left_alone():
    """Page numbers between the first slots and the window may name no page."""
    layer = Layer([4000], 2, 16, torch.bfloat16, seed=2)
    layer.table[0, 1:200] = -5                         # slots 16 to 3199; the earliest row's window begins at 3201
    run(layer, (300,), 4, window=500, sink=10)


def test_pools_past_two_to_the_31_elements():
    """Rows that lie behind 2^31 elements of a pool, read by the copies and where a row is done again."""
    first = (1 << 31) // (2 * 64 * DIM) + 5
    layer = Layer([1500, 300], 2, 64, torch.bfloat16, seed=3, first_page=first)
    run(layer, (700, 20), 4)
    v = layer.v[0].clone()
    v[:, 1400, 3] = float("nan")                        # rows in front of it are done again
    layer.fill(0, layer.k[0].float(), v.float(), layer.w[0].float(), layer.t[0])
    from retrievalattention_b200 import paged

    q = torch.randn(100, 8, DIM, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, 100, 100], dtype=torch.int32, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, torch.tensor([1450, 0], dtype=torch.int32, device="cuda"), starts)
    clean = torch.nan_to_num(v, nan=0.0)
    want = attend_rows(q.cpu().double(), layer.k[0][:, :1450], clean[:, :1450], visible(torch.arange(1350, 1450), 1450, None, 0))
    assert torch.isnan(out[50:, :, 3]).all()
    out[50:, :, 3], want[0][50:, :, 3], want[2][50:, :, 3] = 0.0, 0.0, 0.0
    assert close(out, None, *want)


def test_scale_and_wide_tables():
    from retrievalattention_b200 import paged

    layer = Layer([100], 1, 16, torch.float16, seed=2)
    wide = torch.full((1, 5000), -1, dtype=torch.int32, device="cuda")
    wide[:, :layer.table.shape[1]] = layer.table
    q = torch.randn(20, 4, DIM, device="cuda").half()
    starts = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, wide, layer.lengths, starts, scale=0.3)
    want = attend_rows(q.cpu().double(), layer.k[0], layer.v[0], visible(torch.arange(80, 100), 100, None, 0), scale=0.3)
    assert close(out, None, *want)


def test_a_captured_call_follows_lengths_and_rows():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([900, 2000], 2, 16, torch.bfloat16, seed=6)
    q = torch.randn(64, 8, DIM, device="cuda").to(torch.bfloat16)
    starts, lengths = torch.tensor([0, 30, 64], dtype=torch.int32, device="cuda"), layer.lengths.clone()
    out, lse = torch.empty_like(q), torch.empty(64, 8, device="cuda")
    call = lambda: paged.paged_prompt(q, layer.keys, layer.values, layer.table, lengths, starts, window=700, sink=4, out=out, lse=lse)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n0, n1, split in ((900, 2000, 30), (64, 1200, 64), (500, 40, 40)):
        lengths.copy_(torch.tensor([n0, n1], dtype=torch.int32))
        starts[1] = split
        graph.replay()
        check_prefill_errors()
        for b, (lo, hi, n) in enumerate(((0, split, n0), (split, 64, n1))):
            if hi > lo:
                seen = visible(torch.arange(n - (hi - lo), n), n, 700, 4)
                assert close(out[lo:hi], lse[lo:hi], *attend_rows(q[lo:hi].cpu().double(), layer.k[b][:, :n], layer.v[b][:, :n], seen))


def test_results_repeat_and_follow_the_stream():
    from retrievalattention_b200 import paged

    layer = Layer([6000], 2, 16, torch.bfloat16, seed=6)
    q = torch.randn(100, 8, DIM, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    args = layer.keys, layer.values, layer.table, layer.lengths, starts
    first = paged.paged_prompt(q, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        for _ in range(20):
            late.copy_(q)
        again = paged.paged_prompt(late, *args)
    side.synchronize()
    assert torch.equal(first, again)


@pytest.mark.parametrize("group", [3, 5, 7])
def test_results_repeat_whatever_ran_before(group):
    """Rows that fill up a tile hold what another call left in shared memory: nothing of it reaches the rounding of the others."""
    from retrievalattention_b200 import paged

    layer = Layer([1727, 1606], 2, 64, torch.bfloat16, seed=6)
    gen = torch.Generator().manual_seed(group)
    q = torch.randn(2000, 2 * group, DIM, generator=gen).to(torch.bfloat16).cuda()
    starts = torch.tensor([0, 1000, 2000], dtype=torch.int32, device="cuda")
    call = lambda x: paged.paged_prompt(x, layer.keys, layer.values, layer.table, layer.lengths, starts, window=1, sink=1)  # noqa: E731
    want = call(q)
    for i in range(8):
        call(q * (100.0 * i))                           # something else in the rows
        assert torch.equal(call(q), want)


def test_two_calls_at_once():
    """On two streams, prompts and shared prefixes beside each other: each result is what it is alone."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([3000, 2900, 2800], 2, 16, torch.bfloat16, seed=6)
    layer.table[1:, :128] = layer.table[0, :128]
    wide = torch.full((3, 150000), -1, dtype=torch.int32, device="cuda")
    wide[:, :layer.table.shape[1]] = layer.table
    q, one = torch.randn(400, 8, DIM, device="cuda").to(torch.bfloat16), torch.randn(3, 1, 8, DIM, device="cuda").to(torch.bfloat16)
    starts, groups, common = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 300, 310, 400], [0, 3], [2048]))
    calls = [lambda: paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=500, sink=4),
             lambda: paged.paged_shared_decode(one, layer.keys, layer.values, wide, layer.lengths, groups, common),
             lambda: paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts)]
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    results = [[] for _ in calls]
    for _ in range(10):
        for call, stream, got in zip(calls, streams, results):
            with torch.cuda.stream(stream):
                got.append(call())
    torch.cuda.synchronize()
    check_prefill_errors()
    for got, want in zip(results, alone):
        assert all(torch.equal(x, want) for x in got)


def test_outputs_on_any_boundary_of_16_bytes():
    from retrievalattention_b200 import paged

    layer = Layer([200], 2, 16, torch.bfloat16, seed=6)
    q = torch.randn(100, 8, DIM, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    args = layer.keys, layer.values, layer.table, layer.lengths, starts
    want = paged.paged_prompt(q, *args)
    for off in (8, 16):
        flat = torch.zeros(q.numel() + 64, dtype=torch.bfloat16, device="cuda")
        out = flat[off:off + q.numel()].view(q.shape)
        paged.paged_prompt(q, *args, out=out)
        assert torch.equal(out, want) and (flat[:off] == 0).all() and (flat[off + q.numel():] == 0).all()


def test_bad_page_numbers_are_reported():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([100], 2, 16, torch.bfloat16)
    layer.table[0, 3] = 10 ** 6
    q = torch.zeros(4, 8, DIM, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="names no page"):
        paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
        check_prefill_errors()


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer([40, 50], 2, 16, torch.bfloat16)
    q = torch.zeros(6, 8, DIM, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    good = dict(q=q, keys=layer.keys, values=layer.values, table=layer.table, lengths=layer.lengths, starts=starts)

    def call(window=None, sink=0, out=None, lse=None, scale=None, **change):
        x = {**good, **change}
        return paged.paged_prompt(x["q"], x["keys"], x["values"], x["table"], x["lengths"], x["starts"], window=window, sink=sink, out=out, lse=lse,
                                  scale=scale)

    call()
    assert call(q=q[:0], starts=torch.zeros_like(starts)).shape == (0, 8, DIM)
    for bad in (dict(q=q[:, :7]), dict(q=q.half()), dict(q=q.cpu()), dict(q=q[..., :64]), dict(q=q.repeat(1, 3, 1)), dict(q=q.transpose(0, 1)),
                dict(starts=starts[:2]), dict(starts=starts.long()), dict(starts=starts.cpu()), dict(values=None),
                dict(window=0), dict(window=-3), dict(window=4, sink=-1), dict(lse=torch.empty(6, 7, device="cuda")),
                dict(out=torch.empty_like(q)[:, ::2]), dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(RuntimeError):
            call(**bad)
