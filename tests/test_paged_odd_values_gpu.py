"""Infinite and NaN values anywhere among the slots of ``paged_prompt`` and ``paged_shared_decode``: every row gets what the slots that it
sees give it, and the call takes no more than a few times as long."""
import pytest
import torch

from attend_helpers import attend_rows, close, visible
from paged_helpers import DIM, Layer
from test_paged_shared_gpu import begin_alike, roomy

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def check(out, lse, q, k, v, seen):
    """Rows of a request against the sums over finite values, and where they are not: a channel is infinite or NaN where a slot that the row
    sees is, NaN where infinities of both signs meet."""
    want, want_lse, spread, score = attend_rows(q.cpu().double(), k, torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0), seen)
    group = q.shape[1] // k.shape[0]
    plus, minus = ((torch.einsum("rs,hsd->rhd", seen.float(), x.float()) > 0).repeat_interleave(group, 1)
                   for x in ((v == INF) | v.isnan(), (v == -INF) | v.isnan()))
    got = out.cpu().double()
    assert torch.equal(got.isnan(), plus & minus)
    assert torch.equal(got == INF, plus & ~minus) and torch.equal(got == -INF, minus & ~plus)
    odd = plus | minus
    got[odd], want[odd] = 0.0, 0.0
    assert close(got.to(out.dtype), lse, want, want_lse, spread, score)


def put(layer, b, places):
    """Values of request b: {(slot or slots, channel or channels): value}, of every head."""
    v = layer.v[b].clone()
    for (slot, channel), x in places.items():
        v[:, slot, channel] = x
    layer.fill(b, layer.k[b].float(), v.float(), layer.w[b].float(), layer.t[b])


def prompt(layer, counts, group, window=None, sink=0):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    rows, hq = sum(counts), layer.hk * group
    q = torch.randn((rows, hq, DIM), generator=torch.Generator().manual_seed(rows)).to(layer.dtype).cuda()
    starts, lse = torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32).cuda(), torch.empty(rows, hq, device="cuda")
    out = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink, lse=lse)
    again = paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink)
    check_prefill_errors()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    at = 0
    for b, n in enumerate(counts):
        length, r = layer.lengths_list[b], slice(at, at + n)
        check(out[r], lse[r], q[r], layer.k[b], layer.v[b], visible(torch.arange(length - n, length), length, window, sink))
        at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sink", [(None, 0), (90, 3), (700, 40)])
@pytest.mark.parametrize("counts,held,hk,group,page", [
    ((600,), 0, 2, 4, 16),                               # a whole prompt: items of two tiles
    ((20, 300), 1500, 1, 7, 64),                         # pieces: items of one tile and of two
    ((40,), 6000, 1, 4, 128),                            # an item that many CTAs share
    ((3, 1, 2), 2500, 2, 8, 8),                          # one tile, its steps in turn for two groups
])
def test_anywhere(dtype, counts, held, hk, group, page, window, sink):
    for where in (0.0, 0.5, 0.97):
        layer = Layer([n + held for n in counts], hk, page, dtype, seed=page)
        for b, n in enumerate(layer.lengths_list):
            at = min(int(where * n), n - 1)
            put(layer, b, {(at, 5): NAN, (max(0, at - 1), 77): INF, (min(at + 1, n - 1), 126): -INF, (at // 2, 40): INF, (at, 40): -INF})
        prompt(layer, counts, group, window, sink)


@pytest.mark.parametrize("window", [None, 300])
def test_nothing_but_odd_values(window):
    """All of a page, all of a channel, and the last token's whole value."""
    for counts, held in (((400,), 0), ((30,), 3000)):
        layer = Layer([n + held for n in counts], 1, 64, torch.bfloat16, seed=3)
        n = layer.lengths_list[0]
        put(layer, 0, {(slice(None), 9): INF, (slice(n // 2, n // 2 + 64), slice(None)): NAN, (n - 1, slice(None)): -INF})
        prompt(layer, counts, 4, window, 2)


def test_slots_beside_the_first_ones():
    """What lies behind the first slots in their page is seen by no row whose window lies behind."""
    layer = Layer([2000], 2, 64, torch.bfloat16, seed=4)
    put(layer, 0, {(slice(4, 64), slice(None)): NAN})
    prompt(layer, (1200,), 4, 200, 4)
    prompt(layer, (30,), 4, 200, 4)


def test_a_slot_that_hardly_counts():
    """Probabilities that vanish beside the row's largest still hand on an infinite value; a score of -infinity does not."""
    for counts, held in (((300,), 0), ((40,), 5000)):
        layer = Layer([n + held for n in counts], 1, 16, torch.bfloat16, seed=4)
        n = layer.lengths_list[0]
        k = layer.k[0].clone()
        k[:, n // 3], k[:, n // 4] = 0.0, 0.0
        k[:, n // 3, 0], k[:, n // 4, 0] = -3e4, -INF
        v = layer.v[0].clone()
        v[:, n // 3, 7], v[:, n // 4, 8] = INF, INF
        layer.fill(0, k.float(), v.float(), layer.w[0].float(), layer.t[0])
        from retrievalattention_b200 import paged

        rows = counts[0]
        q = torch.randn((rows, 4, DIM), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        q[..., 0] = 1.0
        starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        out = paged.paged_prompt(q.cuda(), layer.keys, layer.values, layer.table, layer.lengths, starts).cpu()
        own = torch.arange(n - rows, n)
        sees = (own >= n // 3)[:, None].expand(-1, 4)
        assert torch.equal(out[..., 7] == INF, sees) and torch.isfinite(out[..., [6, 8, 9]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_prefixes(dtype):
    """A request that is shorter than what the others have in common does not see what lies behind its end."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    for lengths, group in (((1500, 900, 1600, 1), 4), ((1100,) * 40 + (700, 3), 8)):
        layer = Layer(lengths, 1, 16, dtype, seed=6)
        v = layer.v[0].clone()
        v[:, 1000, 3], v[:, 1001, 4], v[:, 2, 5], v[:, 800, 6] = NAN, INF, -INF, INF
        layer.fill(0, layer.k[0].float(), v.float(), layer.w[0].float(), layer.t[0])
        begin_alike(layer, ((0, len(lengths), 1024 // 16),))
        q = torch.randn((len(lengths), 1, group, DIM), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        lse = torch.empty(len(lengths), group, device="cuda")
        out = paged.paged_shared_decode(q, layer.keys, layer.values, roomy(layer.table), layer.lengths,
                                        torch.tensor([0, len(lengths)], dtype=torch.int32, device="cuda"),
                                        torch.tensor([1024], dtype=torch.int32, device="cuda"), lse=lse)
        check_prefill_errors()
        for b, n in enumerate(lengths):
            check(out[b], lse[b:b + 1], q[b], layer.k[b], layer.v[b], torch.ones(1, n, dtype=torch.bool))


@pytest.mark.parametrize("places", [{(4000, 5): NAN}, {(8100, 5): NAN}, {(slice(4, 64), 5): INF}, {(slice(None), slice(None)): NAN},
                                    {(slice(None), 9): INF}, {(slice(None), 9): INF, (8000, 8): NAN}])
def test_they_take_no_more_than_a_few_times_as_long(places):
    """8192 tokens: every segment once more, over tiles that one warp has cleaned, and looked up.  (A row after the other over the slots it
    sees: hundreds of times.)"""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer, window, sink = Layer([8192], 8, 64, torch.bfloat16, seed=2), None, 0
    if (slice(4, 64), 5) in places:
        window, sink = 1024, 4
    q = torch.randn(8192, 32, DIM, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, 8192], dtype=torch.int32, device="cuda")

    def once():
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        paged.paged_prompt(q, layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink)
        end.record()
        end.synchronize()
        return begin.elapsed_time(end)

    def least():
        return min(once() for _ in range(5))

    plain = least()
    put(layer, 0, places)
    odd = least()
    check_prefill_errors()
    print(f"{plain:.3f} -> {odd:.3f} ms")
    assert odd <= 12 * plain, (plain, odd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix", [256, 12800])
@pytest.mark.parametrize("own_above", [True, False])
def test_an_infinite_value_far_below_the_other_part(own_above, prefix, dtype):
    """Scores in common and a request's own lie 120 apart (2^-173, nothing in 32 bits); an infinite value of the lower ones is handed on
    whichever part comes first."""
    from retrievalattention_b200 import paged

    layer = Layer([prefix + 100, prefix + 9, prefix + 40], 1, 16, dtype, seed=6)
    begin_alike(layer, ((0, 3, prefix // 16),))
    for b, n in enumerate(layer.lengths_list):
        k, v = layer.k[b] * 0.05, layer.v[b].clone()
        k[:, :, 0] = 0.0
        k[:, prefix:, 0] = (120.0 if own_above else -120.0) * DIM ** 0.5 / 16
        if own_above:
            v[:, prefix // 3, 5], v[:, prefix - 1, 6] = INF, -INF
        else:
            v[:, prefix + 3, 5], v[:, n - 1, 6] = INF, -INF
        layer.fill(b, k.float(), v.float(), layer.w[b].float(), layer.t[b])
    q = torch.randn((3, 1, 4, DIM), generator=torch.Generator().manual_seed(2)) * 0.1
    q[..., 0] = 16
    out = paged.paged_shared_decode(q.to(dtype).cuda(), layer.keys, layer.values, roomy(layer.table), layer.lengths,
                                    torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([prefix], dtype=torch.int32, device="cuda"))
    out = out.float().cpu()
    assert (out[..., 5] == INF).all() and (out[..., 6] == -INF).all(), out[:, 0, :, 5:7]
    assert torch.isfinite(out[..., [c for c in range(DIM) if c not in (5, 6)]]).all()
