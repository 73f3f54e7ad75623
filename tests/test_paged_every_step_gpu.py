"""Long windows, prompts and shared prefixes whose every step of 16 slots shows in the outputs: a value lies in one channel out of 128, another
one from step to step, so that a step that is lost, or read in another's place, moves a channel by more than it may be off.

All values are positive, so an output is off by what `attend_rows` allows relative to itself: two roundings to 16 bits (2^-7 of it in bf16,
2^-10 in fp16) and 2e-4.  A channel has at most 70 steps of nearly the same weight.  The host checks that `close` turns down outputs with a step
left out, with the next one's values in its place, and with a step counted twice."""
import pytest
import torch

from attend_helpers import attend_rows, close, visible
from paged_helpers import DIM, Layer
from test_paged_shared_gpu import begin_alike, roomy

pytestmark = pytest.mark.gpu
STEP = 16


def mark(layer, b, seed=1):
    """Request b's slots: flat scores, and marked values."""
    n, gen = layer.lengths_list[b], torch.Generator().manual_seed(seed)
    slot = torch.arange(n)
    v = torch.zeros(layer.hk, n, DIM)
    v[:, slot, slot // STEP % DIM] = 1 + 0.25 * torch.rand(layer.hk, n, generator=gen)
    layer.fill(b, (layer.k[b] * 0.1).to(layer.dtype).float(), v.to(layer.dtype).float(), layer.w[b].float(), layer.t[b])


def turned_down(q, k, v, seen, dtype):
    """Of the steps that all rows see: first, last, and some between."""
    whole = seen.all(0)[:seen.shape[1] // STEP * STEP].view(-1, STEP).all(1).nonzero()[:, 0].tolist()
    right = attend_rows(q, k, v, seen)
    assert close(right[0].to(dtype), right[1].float(), *right)
    for step in [whole[0], whole[-2]] + whole[1:-1:max(1, len(whole) // 3)]:
        rows = slice(step * STEP, (step + 1) * STEP)
        for other in (torch.zeros_like(v[:, rows]), v[:, rows].roll(1, -1), 2 * v[:, rows]):
            wrong = v.clone()
            wrong[:, rows] = other
            out = attend_rows(q, k, wrong, seen)[0].to(dtype)
            assert not close(out, None, *right), step


@pytest.mark.parametrize("lengths,hk,page,dtype,group,window,sink", [
    ((30000, 9000, 100), 2, 8, torch.bfloat16, 4, 8000, 4),
    ((30000, 9000, 100), 2, 128, torch.bfloat16, 7, 8000, 40),
    ((150000,), 1, 16, torch.bfloat16, 4, 140000, 4),
    ((40000,) * 12, 1, 64, torch.float16, 2, 6000, 0),
])
def test_windows(lengths, hk, page, dtype, group, window, sink):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer(lengths, hk, page, dtype, seed=1)
    for b in range(len(lengths)):
        mark(layer, b)
    batch = len(lengths)
    q = torch.randn((batch, 1, hk * group, DIM), generator=torch.Generator().manual_seed(60)).to(dtype)
    lse = torch.empty(batch, hk * group, device="cuda")
    out = paged.paged_decode(q.cuda(), layer.keys, layer.values, layer.table, layer.lengths, lse=lse, window=window, sink=sink)
    check_prefill_errors()
    for b, n in enumerate(lengths):
        seen = visible([n - 1], n, window, sink)
        assert close(out[b], lse[b:b + 1], *attend_rows(q[b].double(), layer.k[b], layer.v[b], seen)), b
    turned_down(q[0].double(), layer.k[0], layer.v[0], visible([lengths[0] - 1], lengths[0], window, sink), dtype)


@pytest.mark.parametrize("counts,held,group,page,window,sink", [
    ((70, 3), 9000, 4, 64, None, 0), ((70, 3), 9000, 4, 8, 4000, 5), ((33,), 20000, 1, 128, None, 0), ((500,), 6000, 7, 16, 5000, 40),
])
def test_prompts(counts, held, group, page, window, sink):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([n + held for n in counts], 1, page, torch.bfloat16, seed=2)
    for b in range(len(counts)):
        mark(layer, b)
    q = torch.randn((sum(counts), group, DIM), generator=torch.Generator().manual_seed(61)).to(torch.bfloat16)
    starts, lse = torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32).cuda(), torch.empty(sum(counts), group, device="cuda")
    out = paged.paged_prompt(q.cuda(), layer.keys, layer.values, layer.table, layer.lengths, starts, window=window, sink=sink, lse=lse)
    check_prefill_errors()
    at = 0
    for b, n in enumerate(counts):
        length, r = layer.lengths_list[b], slice(at, at + n)
        seen = visible(torch.arange(length - n, length), length, window, sink)
        assert close(out[r], lse[r], *attend_rows(q[r].double(), layer.k[b], layer.v[b], seen)), b
        at += n
    length = layer.lengths_list[0]
    seen = visible(torch.arange(length - 2, length), length, window, sink)
    turned_down(q[counts[0] - 2:counts[0]].double(), layer.k[0], layer.v[0], seen, torch.bfloat16)


@pytest.mark.parametrize("page,dtype", [(8, torch.bfloat16), (64, torch.bfloat16), (256, torch.float16)])
def test_shared_prefixes(page, dtype):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer((13000, 12900, 12801, 20000), 2, page, dtype, seed=3)
    for b in range(4):
        mark(layer, b, seed=b)
    begin_alike(layer, ((0, 4, 12800 // page),))
    q = torch.randn((4, 1, 8, DIM), generator=torch.Generator().manual_seed(62)).to(dtype)
    lse = torch.empty(4, 8, device="cuda")
    out = paged.paged_shared_decode(q.cuda(), layer.keys, layer.values, roomy(layer.table), layer.lengths,
                                    torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.tensor([12800], dtype=torch.int32, device="cuda"), lse=lse)
    check_prefill_errors()
    for b, n in enumerate(layer.lengths_list):
        assert close(out[b], lse[b:b + 1], *attend_rows(q[b].double(), layer.k[b], layer.v[b], torch.ones(1, n, dtype=torch.bool))), b
    turned_down(q[3].double(), layer.k[3], layer.v[3], torch.ones(1, 20000, dtype=torch.bool), dtype)


@pytest.mark.parametrize("dtype,part", [(torch.float16, 0.02), (torch.bfloat16, 0.01)])
@pytest.mark.parametrize("lengths,kv_heads,group,page,window,sink", [((5003, 2500, 0, 77), 4, 7, 8, 1000, 20), ((60000, 9001), 2, 8, 256, 30000, 4)])
def test_window_outputs_are_the_rounded_ones(lengths, kv_heads, group, page, window, sink, dtype, part):
    """An error e, relative, moves at most 2 e / 2^-11 of fp16 outputs over a rounding edge, 2 e / 2^-8 of bf16 ones.  Scores and sums
    4e-6, bf16's probabilities of 16 bits 2^-16 more: 1.6 and 1 %."""
    from retrievalattention_b200 import paged

    layer = Layer(lengths, kv_heads, page, dtype, seed=5)
    q = torch.randn((len(lengths), 1, kv_heads * group, DIM), generator=layer.gen).to(dtype)
    out = paged.paged_decode(q.cuda(), layer.keys, layer.values, layer.table, layer.lengths, window=window, sink=sink).cpu()
    wrong = total = 0
    for b, n in enumerate(lengths):
        if n:
            want = attend_rows(q[b].double(), layer.k[b], layer.v[b], visible([n - 1], n, window, sink))[0]
            wrong += (out[b] != want.to(dtype)).sum().item()
            total += want.numel()
    assert wrong <= part * total, wrong / total
