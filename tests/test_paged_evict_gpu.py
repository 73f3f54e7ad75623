"""``paged.paged_evict`` against a sort: which slots stay, where they go, and everything that must not change.  All of it exact."""
import pytest
import torch

from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu


def moves_of(w, t, keep, sink, recent, seen):
    """(holes, fillers) of one head, both ascending: weights and token numbers of its slots, on the CPU."""
    n = w.numel()
    safe = [(x < sink or x >= seen - recent) for x in t.tolist()]
    weight = w.tolist()
    rank = sorted(range(n), key=lambda j: (not safe[j], 0.0 if safe[j] else (float("inf") if weight[j] != weight[j] else -weight[j]),
                                           (not safe[j]) and weight[j] != weight[j], j))
    stay = set(rank[:keep])
    return [j for j in range(keep) if j not in stay], sorted(j for j in stay if j >= keep)


def run(layer, keep, sink, recent, seen=None):
    from retrievalattention_b200 import paged

    seen = list(layer.lengths_list) if seen is None else seen
    pools = dict(keys=layer.keys, values=layer.values, weight=layer.weight, token=layer.token)
    want = {n: p.cpu().clone() for n, p in pools.items()}
    moved = 0
    for b, n in enumerate(layer.lengths_list):
        if n <= keep:
            continue
        ids = torch.tensor(layer.pages_of[b])
        for h in range(layer.hk):
            w = want["weight"][ids, h].reshape(-1)[:n]
            t = want["token"][ids, h].reshape(-1)[:n]
            holes, fillers = moves_of(w, t, keep, sink, recent, seen[b])
            assert len(holes) == len(fillers)
            moved += len(holes)
            to, of = torch.tensor(holes, dtype=torch.long), torch.tensor(fillers, dtype=torch.long)
            for p in want.values():
                p[ids[to // layer.page], h, to % layer.page] = p[ids[of // layer.page], h, of % layer.page].clone()
    paged.paged_evict(layer.keys, layer.values, layer.weight, layer.token, layer.table, layer.lengths,
                      torch.tensor(seen, dtype=torch.int32, device="cuda"), keep, sink, recent)
    for name, p in pools.items():
        kind = torch.int16 if p.element_size() == 2 else torch.int32
        assert torch.equal(p.cpu().contiguous().view(kind), want[name].contiguous().view(kind)), name
    return moved


@pytest.mark.parametrize("lengths,kv_heads,page,dtype,keep,sink,recent", [
    ((0, 1, 2), 1, 8, torch.bfloat16, 1, 0, 0),                       # one slot stays
    ((0, 9, 100, 17), 2, 16, torch.float16, 16, 0, 0),                # one request of one slot more
    ((100, 64, 333), 3, 8, torch.bfloat16, 64, 4, 16),
    ((1001,), 8, 16, torch.bfloat16, 512, 4, 64),                     # clusters of eight CTAs
    ((700, 650), 2, 32, torch.float16, 649, 4, 64),                   # nearly everything stays
    ((300,) * 20, 8, 64, torch.bfloat16, 100, 100, 0),                # one CTA a group; the first tokens fill it
    ((300,) * 3, 2, 256, torch.bfloat16, 100, 0, 100),                # the last ones do
    ((700,) * 19, 8, 16, torch.bfloat16, 300, 4, 16),                 # the same, and more moves than it does itself
    ((20000, 3000), 2, 128, torch.bfloat16, 5000, 4, 64),             # slots left over after one digit and after two
    ((513, 12), 4, 1024, torch.bfloat16, 12, 5, 7),
    ((4160, 4160), 4, 32, torch.float16, 4096, 4, 64),
])
def test_which_slots_stay_and_where_they_go(lengths, kv_heads, page, dtype, keep, sink, recent):
    moved = run(Layer(lengths, kv_heads, page, dtype, seed=21), keep, sink, recent)
    assert moved > 0 or sink + recent == keep or max(lengths) <= keep + 1


def put(layer, w, t=None):
    for b, n in enumerate(layer.lengths_list):
        layer.fill(b, layer.k[b].to(layer.dtype), layer.v[b].to(layer.dtype), w[b], layer.t[b] if t is None else t[b])


@pytest.mark.parametrize("kind", ["all equal", "two values", "zeros of both signs", "extremes", "negative", "tiny"])
def test_ties_and_strange_weights(kind):
    lengths = (777, 130)
    layer = Layer(lengths, 2, 16, torch.bfloat16, seed=22)
    gen = torch.Generator().manual_seed(1)
    made = []
    for n in lengths:
        r = torch.randint(0, 6, (2, n), generator=gen)
        made.append({"all equal": torch.full((2, n), 0.25), "two values": (r > 3).float(),
                     "zeros of both signs": torch.where(r > 2, 0.0, -0.0),
                     "extremes": torch.tensor([float("inf"), float("-inf"), float("nan"), 3.4e38, -3.4e38, 0.0])[r],
                     "negative": -torch.rand((2, n), generator=gen), "tiny": torch.rand((2, n), generator=gen) * 1e-44}[kind])
    put(layer, made)
    run(layer, 100, 4, 16)


def test_after_an_earlier_eviction():
    """Tokens out of order: protection goes by token numbers, not by slots."""
    layer = Layer((500, 222), 2, 16, torch.bfloat16, seed=23)
    gen = torch.Generator().manual_seed(2)
    order = [torch.stack([torch.randperm(900, generator=gen)[:n] for _ in range(2)]).to(torch.int32) for n in (500, 222)]
    put(layer, [torch.rand((2, n), generator=gen) for n in (500, 222)], order)
    assert run(layer, 200, 8, 30, seen=[900, 900]) > 0


@pytest.mark.parametrize("kv_heads,batch,tokens,keep", [(1, 1, 400000, 100000), (8, 19, 43000, 20000)])
def test_more_slots_than_shared_memory_holds(kv_heads, batch, tokens, keep):
    layer = Layer((1,) * batch, kv_heads, 64, torch.bfloat16, seed=24, room=tokens)
    n = [tokens - 7 * b for b in range(batch)]
    layer.lengths_list = n
    layer.lengths.copy_(torch.tensor(n, dtype=torch.int32))
    gen = torch.Generator().manual_seed(3)
    layer.weight.copy_(torch.randint(0, 5000, layer.weight.shape, generator=gen).float())
    layer.token.copy_(torch.randint(0, tokens, layer.token.shape, generator=gen))
    for pool in (layer.keys, layer.values):
        pool.copy_(torch.arange(pool.numel() // DIM, device="cuda").remainder(251).view(*pool.shape[:3], 1).expand_as(pool))
    assert run(layer, keep, 4, 64) > 0


def test_twice_is_once():
    from retrievalattention_b200 import paged

    layer = Layer((300, 90), 2, 16, torch.bfloat16, seed=25)
    run(layer, 64, 4, 16)
    layer.lengths.clamp_(max=64)
    before = [x.clone() for x in (layer.keys, layer.values, layer.weight, layer.token)]
    paged.paged_evict(layer.keys, layer.values, layer.weight, layer.token, layer.table, layer.lengths,
                      torch.tensor([300, 90], dtype=torch.int32, device="cuda"), 64, 4, 16)
    for x, y in zip(before, (layer.keys, layer.values, layer.weight, layer.token)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_pages_apart_and_room_for_no_more():
    run(Layer((100, 80), 2, 16, torch.bfloat16, seed=26, apart=True), 30, 2, 8)
    run(Layer((100, 80), 2, 16, torch.bfloat16, seed=26), 4000, 2, 8)           # no table reaches that far


def test_attention_after_eviction_is_that_of_the_slots_that_stayed():
    from paged_helpers import attend
    from retrievalattention_b200 import paged

    layer = Layer((260, 70), 2, 16, torch.bfloat16, seed=27)
    kept = []
    for b, n in enumerate((260, 70)):
        kept.append([])
        for h in range(2):
            holes, fillers = moves_of(layer.w[b][h], layer.t[b][h], 64, 4, 16, n)
            kept[b].append(sorted((set(range(64)) - set(holes)) | set(fillers)))
    run(layer, 64, 4, 16)
    layer.lengths.clamp_(max=64)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen).bfloat16().cuda()
    out = paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths)
    for b in range(2):
        k, v = (torch.stack([x[b][h, kept[b][h]] for h in range(2)]) for x in (layer.k, layer.v))
        want = attend(q[b, 0].cpu().double().view(2, 4, DIM), k, v)[0].view(8, DIM)
        assert ((out[b, 0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * v.abs().max()).all()


def test_page_number_outside_the_pool_is_reported_and_other_requests_are_served():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer((100, 90), 2, 16, torch.bfloat16, seed=29, spare=0)
    want = Layer((100, 90), 2, 16, torch.bfloat16, seed=29, spare=0)
    run(want, 40, 2, 8)
    for entry in (0, 4):                                                 # a hole's page, a filler's
        table = layer.table.clone()
        table[0, entry] = layer.keys.shape[0] + 5
        with pytest.raises(RuntimeError, match="names no page"):
            paged.paged_evict(layer.keys, layer.values, layer.weight, layer.token, table, layer.lengths,
                              torch.tensor([100, 90], dtype=torch.int32, device="cuda"), 40, 2, 8)
            check_prefill_errors()
        for name in ("keys", "values", "weight", "token"):
            a, b = layer.gather(getattr(layer, name), 1), want.gather(getattr(want, name), 1)
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), name
        layer = Layer((100, 90), 2, 16, torch.bfloat16, seed=29, spare=0)


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer((100, 40), 2, 16, torch.bfloat16, seed=28)
    good = dict(key_pages=layer.keys, value_pages=layer.values, weight=layer.weight, token=layer.token, page_table=layer.table,
                lengths=layer.lengths, seen=layer.lengths, keep=30, n_sink=4, n_recent=10)
    for change in (dict(value_pages=None), dict(weight=None), dict(token=None), dict(token=layer.token.long()),
                   dict(weight=layer.weight.half()), dict(seen=layer.lengths.long()), dict(seen=layer.lengths[:1]),
                   dict(seen=layer.lengths.cpu())):
        with pytest.raises(ValueError):
            paged.paged_evict(**{**good, **change})
    for change in (dict(keep=0), dict(keep=13), dict(n_sink=-1), dict(n_recent=-1), dict(n_sink=2 ** 31 - 1, n_recent=2 ** 31 - 1)):
        with pytest.raises(RuntimeError, match="keep"):
            paged.paged_evict(**{**good, **change})
    odd = torch.zeros(layer.weight.numel() + 1, device="cuda")[1:].view(layer.weight.shape)
    with pytest.raises(RuntimeError, match="aligned"):
        paged.paged_evict(**{**good, "weight": odd})
