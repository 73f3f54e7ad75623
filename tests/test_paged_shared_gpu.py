"""``paged.paged_shared_decode`` against attention of every request by itself, in 64 bits."""
import pytest
import torch

from attend_helpers import attend_rows, close
from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu
INF = float("inf")


def begin_alike(layer, groups):
    """Requests first .. last - 1 of every (first, last, pages) take the first one's pages, and what is in them."""
    for first, last, pages in groups:
        n = pages * layer.page
        for b in range(first + 1, last):
            layer.table[b, :pages] = layer.table[first, :pages]
            layer.pages_of[b][:pages] = layer.pages_of[first][:pages]
            m = min(n, layer.lengths_list[b], layer.lengths_list[first])
            for x in (layer.k, layer.v):
                x[b][:, :m] = x[first][:, :m]


def roomy(table):
    """The same table with room for more than a million slots a request: with few, requests are attended one by one."""
    wide = torch.full((table.shape[0], 150000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return wide


def run(layer, starts, shared, group, seed=0, lse=True, stride=0):
    run_with(layer, layer.table, starts, shared, group, seed, lse, stride)
    return run_with(layer, roomy(layer.table), starts, shared, group, seed, lse, stride)


def run_with(layer, table, starts, shared, group, seed, lse, stride):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    batch, hq = len(layer.lengths_list), layer.hk * group
    gen = torch.Generator().manual_seed(seed + 50)
    q = torch.randn((batch, hq * DIM + stride), generator=gen).to(layer.dtype).cuda()[:, :hq * DIM].view(batch, 1, hq, DIM) if not stride else \
        torch.randn((batch, hq * DIM + stride), generator=gen).to(layer.dtype).cuda()[:, :hq * DIM].unflatten(1, (1, hq, DIM))
    sums = torch.full((batch, hq), 7.0, device="cuda") if lse else None
    out = paged.paged_shared_decode(q, layer.keys, layer.values, table, layer.lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                    torch.tensor(shared, dtype=torch.int32, device="cuda"), lse=sums)
    check_prefill_errors()
    for b, n in enumerate(layer.lengths_list):
        want = attend_rows(q[b].cpu().double(), layer.k[b], layer.v[b], torch.ones(1, n, dtype=torch.bool))
        assert close(out[b], sums[b:b + 1] if lse else None, *want), (b, n, float((out[b].cpu().double() - want[0]).abs().max()))
    return q, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,groups,hk,group,page,cut", [
    ((300, 280), ((0, 2, 16),), 2, 4, 16, 0),
    ((33, 20, 16), ((0, 3, 1),), 1, 7, 16, 0),                    # the third has no slot of its own
    ((500, 130, 400, 1, 0, 90), ((0, 2, 8), (2, 3, 3)), 2, 4, 16, 0),      # requests of no group, one without slots
    ((700,) * 40, ((0, 40, 4),), 1, 8, 128, 0),                   # 320 rows: a pair of tiles and one more
    ((260,) * 20, ((0, 9, 16), (9, 20, 8)), 2, 5, 16, 0),         # 45 and 55 rows
    ((300, 310, 305), ((0, 3, 16),), 2, 2, 16, 9),                # not all that the pages have in common
    ((80, 3, 60), ((0, 3, 4),), 2, 4, 16, 0),                     # one shorter than what the others have in common
])
def test_against_64_bits(dtype, lengths, groups, hk, group, page, cut):
    layer = Layer(lengths, hk, page, dtype, seed=len(lengths))
    begin_alike(layer, groups)
    starts = [groups[0][0]] + [last for _, last, _ in groups]
    run(layer, starts, [pages * page - cut for *_, pages in groups], group)


def test_many_requests():
    """Items of one tile and of two, and own slots, many to a CTA."""
    gen = torch.Generator().manual_seed(1)
    lengths = (600 + torch.randint(0, 300, (300,), generator=gen)).tolist()
    layer = Layer(lengths, 2, 16, torch.bfloat16, seed=9)
    starts = [0, 3, 90, 110, 111, 200, 290]
    begin_alike(layer, [(i, j, 37) for i, j in zip(starts, starts[1:])])
    run(layer, starts, [592] * 6, 4)


@pytest.mark.parametrize("page", [8, 64, 256])
def test_long_prefix(page):
    """A group's item falls to many CTAs."""
    pages = 12800 // page
    layer = Layer((13000, 12900, 12801, 14000), 2, page, torch.bfloat16, seed=3)
    begin_alike(layer, ((0, 4, pages),))
    run(layer, [0, 4], [12800], 4)


def test_groups_in_the_middle_and_groups_without_slots():
    layer = Layer((50, 200, 210, 220, 60), 2, 16, torch.bfloat16, seed=4)
    begin_alike(layer, ((1, 4, 12),))
    run(layer, [1, 4], [192], 4)
    run(layer, [1, 1, 4], [100, 192], 4)                # an empty group
    run(layer, [0, 1, 4, 5], [0, 192, 0], 4, stride=256)


def test_as_paged_decode():
    from retrievalattention_b200 import paged

    layer = Layer((3000, 2500, 2100), 2, 16, torch.bfloat16, seed=4)
    begin_alike(layer, ((0, 3, 125),))
    q, out = run(layer, [0, 3], [2000], 4)
    other = paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths)
    # either is off by at most two half steps of what it adds up
    assert ((out.float() - other.float()).abs() <= 2.0 ** -6 * (other.float().abs() + 0.2)).all()


def test_infinite_and_nan_slots():
    """What one request's own slots hold concerns no other; what is in common concerns all that see it."""
    layer = Layer((300, 280, 270), 1, 16, torch.bfloat16, seed=7)
    begin_alike(layer, ((0, 3, 16),))
    for b, slot, channel, x in ((0, 290, 3, float("nan")), (1, 270, 4, INF), (2, 100, 5, INF)):
        id, at = layer.pages_of[b][slot // 16], slot % 16
        layer.values[id, 0, at, channel] = x
    from retrievalattention_b200 import paged

    q = torch.randn(3, 1, 4, DIM, device="cuda").to(torch.bfloat16)
    out = paged.paged_shared_decode(q, layer.keys, layer.values, roomy(layer.table), layer.lengths, torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                                    torch.tensor([256], dtype=torch.int32, device="cuda"))[:, 0]
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, :, 3] = want[1, :, 4] = want[:, :, 5] = True
    assert torch.equal(bad, want) and torch.isnan(out[0, :, 3]).all() and (out[1, :, 4] == INF).all() and (out[:, :, 5] == INF).all()


def test_a_captured_call_follows_lengths():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer((900, 850, 800), 2, 16, torch.bfloat16, seed=6)
    begin_alike(layer, ((0, 3, 48),))
    q = torch.randn(3, 1, 8, DIM, device="cuda").to(torch.bfloat16)
    starts, shared = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [768]))
    out, lse, lengths = torch.empty_like(q), torch.empty(3, 8, device="cuda"), layer.lengths.clone()
    table = roomy(layer.table)
    call = lambda: paged.paged_shared_decode(q, layer.keys, layer.values, table, lengths, starts, shared, out=out, lse=lse)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for ns, common in (((900, 850, 800), 768), ((768, 769, 780), 768), ((900, 10, 790), 500), ((0, 0, 0), 16)):
        lengths.copy_(torch.tensor(ns, dtype=torch.int32))
        shared.fill_(common)
        graph.replay()
        check_prefill_errors()
        for b, n in enumerate(ns):
            assert close(out[b], lse[b:b + 1], *attend_rows(q[b].cpu().double(), layer.k[b][:, :n], layer.v[b][:, :n], torch.ones(1, n, dtype=torch.bool)))


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer([40, 50], 2, 16, torch.bfloat16)
    q = torch.zeros(2, 1, 8, DIM, dtype=torch.bfloat16, device="cuda")
    starts, shared = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([32], dtype=torch.int32, device="cuda")
    good = dict(q=q, starts=starts, shared=shared, out=None, lse=None)

    def call(**change):
        x = {**good, **change}
        return paged.paged_shared_decode(x["q"], layer.keys, layer.values, layer.table, layer.lengths, x["starts"], x["shared"], out=x["out"],
                                         lse=x["lse"])

    call()
    for bad in (dict(q=q[:1]), dict(q=q.half()), dict(q=q[:, :, :7]), dict(q=q.repeat(1, 1, 3, 1)), dict(starts=starts[:1]), dict(starts=starts.long()),
                dict(shared=shared.cpu()), dict(shared=shared[:0], starts=starts[:1]), dict(shared=shared.repeat(3), starts=starts.repeat(2)),
                dict(out=torch.empty_like(q).half()), dict(lse=torch.empty(2, 7, device="cuda")), dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call(**bad)
