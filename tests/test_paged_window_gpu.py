"""``paged.paged_decode`` with a window and a few first slots, against attention in 64 bits."""
import pytest
import torch

from attend_helpers import attend_rows, close, visible
from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu
INF = float("inf")


def run(layer, group, window, sink, seed=0):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    batch, hq = len(layer.lengths_list), layer.hk * group
    q = torch.randn((batch, 1, hq, DIM), generator=torch.Generator().manual_seed(seed + 60)).to(layer.dtype).cuda()
    lse = torch.full((batch, hq), 7.0, device="cuda")
    out = paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths, lse=lse, window=window, sink=sink)
    check_prefill_errors()
    for b, n in enumerate(layer.lengths_list):
        want = attend_rows(q[b].cpu().double(), layer.k[b], layer.v[b], visible([n - 1], n, window, sink))
        assert close(out[b], lse[b:b + 1], *want), (b, n, float((out[b].cpu().double() - want[0]).abs().max()))
    return q, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("lengths,hk,group,window,sink", [
    ((0, 1, 2, 17), 2, 4, 1, 0),
    ((0, 1, 2, 17, 40), 2, 4, 1, 1),
    ((100, 31, 32, 33), 1, 8, 16, 4),
    ((100, 20, 47), 2, 7, 15, 17),                     # first slots that end inside a step, and in the window's first one
    ((300, 5, 29), 1, 1, 20, 300),                     # more first slots than there are
    ((2000, 999), 2, 4, 500, 33),
    ((50, 60), 2, 2, 1 << 40, 0),                      # a window wider than anything
])
def test_against_64_bits(dtype, page, lengths, hk, group, window, sink):
    run(Layer(lengths, hk, page, dtype, seed=len(lengths) + page), group, window, sink)


@pytest.mark.parametrize("page", [8, 128])
def test_long_windows(page):
    """Windows that many CTAs share, and sums in two levels."""
    run(Layer((30000, 9000, 100), 2, page, torch.bfloat16, seed=1), 4, 8000, 4)
    run(Layer((150000,), 1, page, torch.bfloat16, seed=1), 4, 140000, 4)
    run(Layer((40000,) * 20, 1, page, torch.float16, seed=2), 2, 6000, 0)


def test_what_is_not_seen_may_hold_anything():
    for first in range(0, 40, 7):
        n, window, sink = 200 + first, 50, 5
        layer = Layer([n], 2, 16, torch.bfloat16, seed=first)
        k, v = layer.k[0].clone(), layer.v[0].clone()
        k[:, sink:n - window], v[:, sink:n - window] = float("nan"), INF
        layer.fill(0, k.float(), v.float(), layer.w[0].float(), layer.t[0])
        layer.k[0], layer.v[0] = torch.nan_to_num(k, nan=0.0), torch.nan_to_num(v, posinf=0.0)
        run(layer, 4, window, sink)


def test_first_slots_that_end_inside_the_window_s_first_step():
    layer = Layer([90], 1, 16, torch.bfloat16, seed=3)
    k, v = layer.k[0].clone(), layer.v[0].clone()
    v[:, 18:20] = INF                                  # between sink 18 and low 20, both in the second step
    layer.fill(0, k.float(), v.float(), layer.w[0].float(), layer.t[0])
    layer.v[0] = torch.nan_to_num(v, posinf=0.0)
    run(layer, 4, 70, 18)


def test_steps_that_are_not_seen_are_not_looked_up():
    layer = Layer([4000], 2, 16, torch.bfloat16, seed=2)
    layer.table[0, 1:200] = -5                         # slots 16 to 3199
    run(layer, 4, 800, 10)


def test_a_captured_call_follows_lengths():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([3000, 2000], 2, 16, torch.bfloat16, seed=6)
    q, out, lengths = torch.randn(2, 1, 8, DIM, device="cuda").to(torch.bfloat16), None, layer.lengths.clone()
    out, lse = torch.empty_like(q), torch.empty(2, 8, device="cuda")
    call = lambda: paged.paged_decode(q, layer.keys, layer.values, layer.table, lengths, out=out, lse=lse, window=700, sink=4)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for ns in ((3000, 2000), (703, 704), (1, 0), (720, 1999)):
        lengths.copy_(torch.tensor(ns, dtype=torch.int32))
        graph.replay()
        check_prefill_errors()
        for b, n in enumerate(ns):
            assert close(out[b], lse[b:b + 1], *attend_rows(q[b].cpu().double(), layer.k[b][:, :n], layer.v[b][:, :n], visible([n - 1], n, 700, 4)))


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer([40, 50], 2, 16, torch.bfloat16)
    q = torch.zeros(2, 1, 8, DIM, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(window=0), dict(window=-1), dict(window=5, sink=-1), dict(window=5, weight=layer.weight)):
        with pytest.raises(ValueError):
            paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths, **bad)
