"""Captured calls and calls on other streams, for the operators over a paged cache that write to it; and the weights of many requests of
uneven lengths, on the smallest pages with few query rows."""
import pytest
import torch

from paged_helpers import DIM, Layer
from test_paged_append_gpu import near, rotated, sections, table_of
from test_paged_evict_gpu import moves_of
from test_paged_observe_gpu import check, given

pytestmark = pytest.mark.gpu


def bits(x):
    return x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.int32)


class Append:
    """Rows for a layer; `check` after a call that found `held` slots in the requests."""

    def __init__(self, layer, counts, group, seed):
        gen = torch.Generator().manual_seed(seed)
        self.layer, self.counts, self.axis_of, self.cos_sin = layer, counts, sections(16, 24, 24), table_of(600)
        self.hq, rows = layer.hk * group, sum(counts)
        self.qkv = torch.randn((rows, (self.hq + 2 * layer.hk) * DIM), generator=gen).to(layer.dtype).cuda()
        self.positions = torch.randint(0, 600, (3, rows), generator=gen).cuda()
        self.row_start = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
        self.seen = torch.randint(0, 1000, (len(counts),), generator=gen).to(torch.int32).cuda()
        self.q = torch.empty((rows, self.hq, DIM), dtype=layer.dtype, device="cuda")

    def __call__(self):
        from retrievalattention_b200 import paged

        paged.rope_paged_append(self.qkv, self.cos_sin, self.positions, self.axis_of, self.q, self.layer.keys, self.layer.values,
                                self.layer.table, self.layer.lengths, self.row_start, weight=self.layer.weight, token=self.layer.token,
                                seen=self.seen)

    def check(self, held):
        layer, hq, hk = self.layer, self.hq, self.layer.hk
        x = self.qkv.cpu().double().view(-1, hq + 2 * hk, DIM)
        want = rotated(x[:, :hq + hk], self.cos_sin, self.positions, self.axis_of)
        assert near(self.q, want[:, :hq], x[:, :hq])
        at = 0
        for b, n in enumerate(self.counts):
            upto = held[b] + n
            new = lambda pool: layer.gather(pool, b, upto)[:, held[b]:].transpose(0, 1)  # noqa: E731
            rows = slice(at, at + n)
            assert near(new(layer.keys), want[rows, hq:], x[rows, hq:hq + hk])
            assert torch.equal(new(layer.values).double(), x[rows, hq + hk:])
            assert (new(layer.weight) == 0).all()
            assert (new(layer.token) == (int(self.seen[b]) + torch.arange(n))[:, None]).all()
            at += n


def test_captured_append_follows_lengths_and_positions():
    layer = Layer((5, 30), 2, 16, torch.bfloat16, seed=81, room=40)
    call = Append(layer, [9, 3], 4, 1)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    layer.lengths.copy_(torch.tensor([14, 33], dtype=torch.int32))
    call.positions.add_(7).remainder_(600)
    call.qkv.neg_()
    call.seen.add_(9)
    graph.replay()
    call.check([14, 33])


def evicted(layer, lengths, keep, sink, recent):
    """The pools after an eviction of the first `lengths[b]` slots."""
    pools = {n: getattr(layer, n).cpu().clone() for n in ("keys", "values", "weight", "token")}
    moved = 0
    for b, n in enumerate(lengths):
        ids = torch.tensor(layer.pages_of[b])
        for h in range(layer.hk if n > keep else 0):
            holes, fillers = moves_of(pools["weight"][ids, h].reshape(-1)[:n], pools["token"][ids, h].reshape(-1)[:n], keep, sink, recent, n)
            to, of = (torch.tensor(x, dtype=torch.long) for x in (holes, fillers))
            moved += len(holes)
            for p in pools.values():
                p[ids[to // layer.page], h, to % layer.page] = p[ids[of // layer.page], h, of % layer.page].clone()
    return pools, moved


def evict(layer, keep):
    from retrievalattention_b200 import paged

    paged.paged_evict(layer.keys, layer.values, layer.weight, layer.token, layer.table, layer.lengths, layer.lengths, keep, 4, 16)


@pytest.mark.parametrize("keep,lengths", [(64, (300, 100)), (900, (4000, 1000))])
def test_captured_evict_follows_lengths_and_weights(keep, lengths):
    """With few moves the selection's clusters do them, with many a second kernel."""
    layer = Layer(lengths, 2, 16, torch.float16, seed=82)
    graph = torch.cuda.CUDAGraph()
    layer.lengths.zero_()
    evict(layer, keep)                                            # nothing to do
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        evict(layer, keep)
    now = [lengths[0] - 7, keep - 1]
    layer.lengths.copy_(torch.tensor(now, dtype=torch.int32))
    layer.weight.copy_(torch.rand(layer.weight.shape, generator=layer.gen))
    want, moved = evicted(layer, now, keep, 4, 16)
    assert moved > 0
    graph.replay()
    for name, p in want.items():
        assert torch.equal(bits(getattr(layer, name)).cpu(), bits(p)), name


def test_another_stream():
    """Inputs made on the current stream, calls on a side stream one behind the other, results read on the current one."""
    layer = Layer((700, 90), 2, 16, torch.bfloat16, seed=83, room=20)
    late = torch.randn((2, 10, 8, DIM), generator=layer.gen).bfloat16().cuda()
    expected = [w + g for w, g in zip(layer.w, given(layer, late))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        from retrievalattention_b200 import paged

        paged.paged_observe(late, layer.keys, layer.table, layer.lengths, layer.weight)
    torch.cuda.current_stream().wait_stream(side)
    for b in range(2):
        got = layer.gather(layer.weight, b).double()
        assert ((got - expected[b]).abs() <= 9e-5 * expected[b] + 1e-12).all()

    call = Append(layer, [9, 20], 4, 2)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    call.check([700, 90])

    lengths = [709, 110]
    layer.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    want, moved = evicted(layer, lengths, 100, 4, 16)
    assert moved > 0
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        evict(layer, 100)
    torch.cuda.current_stream().wait_stream(side)
    for name, p in want.items():
        assert torch.equal(bits(getattr(layer, name)).cpu(), bits(p)), name


@pytest.mark.parametrize("kv_heads,group,window", [(1, 1, 7), (2, 3, 3), (4, 5, 4), (2, 8, 8), (2, 8, 12)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_observe_uneven_requests_on_the_smallest_pages(kv_heads, group, window, dtype):
    """A CTA's range runs over several groups; 7 to 96 query rows; ends of pages, tiles and windows in every place."""
    lengths = [1, 0, 129, 8, 640, 127, 7, 255, 0, 1030, 9, 128, 64, 513, 16, 3] * 3
    layer = Layer(lengths, kv_heads, 8, dtype, seed=84)
    q = torch.randn((len(lengths), window, kv_heads * group, DIM), generator=layer.gen).to(dtype)
    for i, n in enumerate(lengths):
        q[i, :max(0, window - n)] = float("nan")
    check(layer, q.cuda())
