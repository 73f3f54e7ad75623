"""Infinite and NaN keys, queries and scores in ``paged.paged_decode`` and ``paged.paged_observe``.

A score of -infinity is a slot that gets nothing; a NaN or +infinity makes the softmax of its query row NaN, as the definition does:
that head's output and log-sum-exp, and the weights of the slots that the row sees.  Everything else is as without it."""
import pytest
import torch

from paged_helpers import DIM, Layer, attend, rounding

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
SHORT, LONG = (300, 77), (9001, 70)            # a cluster of CTAs per group; an even split over the chip


def prepared(lengths, kv_heads, dtype, seed, at, value, slot, channel=5):
    """A layer whose request 0 has `value` in one channel of the key of `slot` of KV head `at`, and its keys before."""
    layer = Layer(lengths, kv_heads, 16, dtype, seed=seed)
    k = layer.k[0].clone()
    k[at, slot, channel] = value
    layer.fill(0, k.to(dtype), layer.v[0].to(dtype), layer.w[0].float(), layer.t[0])
    return layer


def decode(layer, q):
    from retrievalattention_b200 import paged

    lse = torch.zeros((q.shape[0], q.shape[2]), device="cuda")
    out = paged.paged_decode(q, layer.keys, layer.values, layer.table, layer.lengths, lse=lse, weight=layer.weight)
    return out, lse


def check_decode(layer, q, out, lse, dead=()):
    """Heads of `dead`, of request 0, are NaN, and so are the weights of their KV heads; everything else as defined."""
    half, tiny = rounding(layer.dtype)
    group = q.shape[2] // layer.hk
    for b in range(q.shape[0]):
        want, want_lse, p = attend(q[b, 0].cpu().double().view(layer.hk, group, DIM), layer.k[b], layer.v[b])
        got_w = layer.gather(layer.weight, b).double()
        for h in range(layer.hk):
            heads = range(h * group, (h + 1) * group)
            lost = [b == 0 and x in dead for x in heads]
            for i, x in enumerate(heads):
                got, got_lse = out[b, 0, x].cpu().double(), lse[b, x].item()
                if lost[i]:
                    assert got.isnan().all() and got_lse != got_lse, (b, x)
                else:
                    assert ((got - want[h, i]).abs() <= half * want[h, i].abs() + 1e-4 * 6 + tiny).all(), (b, x)
                    assert abs(got_lse - want_lse[h, i].item()) <= 3e-5
            if any(lost):
                assert got_w[h].isnan().all(), (b, h)
            else:
                given = p[h].sum(0)
                assert ((got_w[h] - layer.w[b][h] - given).abs() <= 6e-5 * given + 2.0 ** -23 * (1 + given)).all(), (b, h)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [SHORT, LONG])
@pytest.mark.parametrize("slot", [0, 40, -1])
def test_decode_nan_key(lengths, dtype, slot):
    layer = prepared(lengths, 2, dtype, 61, 1, NAN, slot)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen).to(dtype).cuda()
    check_decode(layer, q, *decode(layer, q), dead=range(4, 8))


@pytest.mark.parametrize("lengths", [SHORT, LONG])
def test_decode_infinite_key(lengths):
    """-infinity for heads whose query is positive in the channel, +infinity for the others."""
    layer = prepared(lengths, 2, torch.float16, 62, 0, -INF, 33)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen)
    q[0, 0, :4, 5] = torch.tensor([0.5, 1.0, 2.0, 0.25])
    whole = q.half().cuda()
    check_decode(layer, whole, *decode(layer, whole))
    layer = prepared(lengths, 2, torch.float16, 62, 0, -INF, 33)
    q[0, 0, 2, 5] = -1.0
    q = q.half().cuda()
    check_decode(layer, q, *decode(layer, q), dead=(2,))


@pytest.mark.parametrize("lengths", [SHORT, LONG])
def test_decode_nan_query(lengths):
    layer = Layer(lengths, 2, 16, torch.bfloat16, seed=63)
    q = torch.randn((2, 1, 8, DIM), generator=layer.gen)
    q[0, 0, 5, 100] = NAN
    q = q.bfloat16().cuda()
    check_decode(layer, q, *decode(layer, q), dead=(5,))


@pytest.mark.parametrize("lengths", [SHORT, LONG])
def test_decode_only_minus_infinity(lengths):
    """A head all of whose scores are -infinity is as one without slots."""
    layer = Layer(lengths, 1, 16, torch.bfloat16, seed=64)
    k = layer.k[0].clone()
    k[:, :, 7] = -INF
    layer.fill(0, k.bfloat16(), layer.v[0].bfloat16(), layer.w[0].float(), layer.t[0])
    q = torch.randn((2, 1, 2, DIM), generator=layer.gen)
    q[0, 0, :, 7] = 1.0
    out, lse = decode(layer, q.bfloat16().cuda())
    assert (out[0] == 0).all() and (lse[0] == -INF).all() and torch.isfinite(out[1].float()).all()
    assert torch.equal(layer.gather(layer.weight, 0).double(), layer.w[0])


def observe(layer, q):
    from retrievalattention_b200 import paged

    paged.paged_observe(q, layer.keys, layer.table, layer.lengths, layer.weight)
    return [layer.gather(layer.weight, b).double() - layer.w[b] for b in range(q.shape[0])]


def given(layer, q, b):
    window, gs, n = q.shape[1], q.shape[2] // layer.hk, layer.lengths_list[b]
    rows = q[b].cpu().double().view(window, layer.hk, gs, DIM).transpose(0, 1).reshape(layer.hk, window * gs, DIM)
    allowed = (torch.arange(n) <= (n - window + torch.arange(window))[:, None]).repeat_interleave(gs, 0)
    s = (rows @ layer.k[b].transpose(1, 2)) * DIM ** -0.5
    return torch.where(allowed, torch.softmax(s.masked_fill(~allowed, -INF), -1), 0.0).sum(1)


def check_observe(layer, q, got):
    for b in range(q.shape[0]):
        want = given(layer, q, b)
        assert torch.equal(got[b].isnan(), want.isnan()), b
        ok = ~want.isnan()
        assert ((got[b] - want).abs()[ok] <= 9e-5 * want[ok] + 2.0 ** -23 * (layer.w[b][ok] + want[ok]) + 1e-12).all(), b


ROWS = [(1, 1), (10, 2), (11, 3), (16, 4), (35, 2), (43, 3), (50, 5)]           # window, heads to a KV head: 1 to 250 rows


@pytest.mark.parametrize("window,group", ROWS)
@pytest.mark.parametrize("slot", [0, 100, 512, -60, -1])
def test_observe_minus_infinity(window, group, slot):
    """No row gives the slot anything, rows that fill up a tile included; the last slot is alone in its part of a tile."""
    layer = prepared((577, 90), 2, torch.float16, 65, 1, -INF, slot)
    q = torch.randn((2, window, 2 * group, DIM), generator=layer.gen)
    q[0, :, :, 5] = q[0, :, :, 5].abs() + 0.1
    q = q.half().cuda()
    got = observe(layer, q)
    check_observe(layer, q, got)
    assert got[0][1, slot] == 0


@pytest.mark.parametrize("window,group", ROWS)
@pytest.mark.parametrize("slot,value", [(0, NAN), (64, NAN), (576, NAN), (200, INF), (576, INF)])
def test_observe_nan_and_plus_infinity(window, group, slot, value):
    """577 slots: the last one is alone in its part of a tile."""
    layer = prepared((577, 90), 2, torch.bfloat16, 66, 0, value, slot)
    q = torch.randn((2, window, 2 * group, DIM), generator=layer.gen)
    q[0, :, :, 5] = q[0, :, :, 5].abs() + 0.1
    q = q.bfloat16().cuda()
    got = observe(layer, q)
    assert got[0][0].isnan().all() and torch.isfinite(got[0][1]).all()
    check_observe(layer, q, got)


@pytest.mark.parametrize("window,group", ROWS)
def test_observe_nan_query(window, group):
    """Slots that the row does not see keep what they have."""
    layer = Layer((577, 90), 2, 16, torch.bfloat16, seed=67)
    q = torch.randn((2, window, 2 * group, DIM), generator=layer.gen)
    q[0, window // 2, group, 9] = NAN
    q = q.bfloat16().cuda()
    got = observe(layer, q)
    last = 577 - window + window // 2
    assert got[0][1, :last + 1].isnan().all() and torch.isfinite(got[0][1, last + 1:]).all() and torch.isfinite(got[0][0]).all()
    check_observe(layer, q, got)


def test_observe_only_minus_infinity():
    """Rows all of whose scores are -infinity are as rows that see no slot."""
    layer = Layer((300, 77), 1, 16, torch.bfloat16, seed=68)
    k = layer.k[0].clone()
    k[:, :, 7] = -INF
    layer.fill(0, k.bfloat16(), layer.v[0].bfloat16(), layer.w[0].float(), layer.t[0])
    q = torch.randn((2, 9, 3, DIM), generator=layer.gen)
    q[0, :, :, 7] = 1.0
    got = observe(layer, q.bfloat16().cuda())
    assert (got[0] == 0).all() and torch.isfinite(got[1]).all() and (got[1][0, :60] > 0).all()


@pytest.mark.parametrize("slots", [range(64, 128), range(0, 577, 2), range(0, 576)])
def test_observe_many_minus_infinity(slots):
    """Whole parts of tiles of them, and every second slot."""
    layer = Layer((577, 90), 1, 16, torch.bfloat16, seed=69)
    k = layer.k[0].clone()
    k[:, list(slots), 7] = -INF
    layer.fill(0, k.bfloat16(), layer.v[0].bfloat16(), layer.w[0].float(), layer.t[0])
    q = torch.randn((2, 9, 3, DIM), generator=layer.gen)
    q[0, :, :, 7] = 1.0
    q = q.bfloat16().cuda()
    rows = q[0].cpu().double().reshape(27, DIM)
    s = (rows @ layer.k[0][0].t()) * DIM ** -0.5
    allowed = (torch.arange(577) <= (577 - 9 + torch.arange(9))[:, None]).repeat_interleave(3, 0)
    p = torch.softmax(s.masked_fill(~allowed, -INF), -1)
    want = torch.where(p.isnan(), 0.0, p).sum(0)                  # NaN: every slot that the row sees is at -infinity
    got = observe(layer, q)[0][0]
    assert (got[list(slots)] == 0).all()
    assert ((got - want).abs() <= 9e-5 * want + 2.0 ** -23 * (layer.w[0][0] + want) + 1e-12).all()
