"""Norms of query and key heads in the pass that rotates them: ``paged.rope_paged_append`` and ``decode_layer.rope_split``.

Tolerance: the sum of 128 squares, its root and four products in 32 bits are off by at most 16 * 2^-24 of the two parts of a rotated
channel (1e-6), and the result is rounded once."""
import pytest
import torch

from paged_helpers import DIM, Layer, rounding

pytestmark = pytest.mark.gpu


def normed(x, weight, eps):
    """x [rows, heads, 128] in 64 bits."""
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.cpu().double()


def turned(x, cos_sin, positions, axis_of):
    """(rotated heads, sum of the sizes of the two parts)."""
    t, pos = cos_sin.cpu().double(), positions.cpu()
    c = torch.stack([t[pos[a], i] for i, a in enumerate(axis_of)], 1)[:, None]
    s = torch.stack([t[pos[a], 64 + i] for i, a in enumerate(axis_of)], 1)[:, None]
    a, b = x[..., :64], x[..., 64:]
    size = a.abs() + b.abs()
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([size, size], -1)


def near(got, want, size):
    half, tiny = rounding(got.dtype)
    return bool(((got.cpu().double() - want).abs() <= half * want.abs() * 1.01 + 1e-6 * size + tiny).all())


def weights(heads, per_head, dtype, gen):
    return (1 + 0.5 * torch.randn((heads, DIM) if per_head else (DIM,), generator=gen)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,hk,group,page,per_head,axes,eps", [
    ((1, 1, 1), 2, 4, 16, False, 1, 1e-6),               # a decode step
    ((7, 0, 130), 1, 3, 8, True, 3, 1e-5),               # an odd number of heads
    ((900, 600), 2, 1, 16, False, 1, 0.0),               # short rows, several to a unit
    ((900, 601), 1, 1, 16, True, 2, 1e-6),
    ((40,), 8, 8, 32, True, 1, 1e-6),                    # rows in two parts
])
def test_append_against_64_bits(dtype, counts, hk, group, page, per_head, axes, eps):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors
    from retrievalattention_b200.decode_layer import cos_sin_cache

    gen = torch.Generator().manual_seed(len(counts))
    held = [3 + 5 * b for b in range(len(counts))]
    layer = Layer(held, hk, page, dtype, room=max(counts))
    hq, rows = hk * group, sum(counts)
    x = torch.randn((rows, hq + 2 * hk, DIM), generator=gen) * torch.rand((rows, hq + 2 * hk, 1), generator=gen).exp2() ** 8
    x[0, 0] = 0.0                                        # a head of zeros stays one (eps 0: 0 / 0)
    qkv = x.to(dtype).flatten(1).cuda()
    axis_of = paged.rope_sections(64) if axes == 1 else paged.rope_interleaved(*([64 // axes] * (axes - 1) + [64 - 64 // axes * (axes - 1)]))
    positions, cos_sin = torch.randint(0, 500, (axes, rows), generator=gen).cuda(), cos_sin_cache(500, DIM, 1e4, "cuda")
    starts = torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32).cuda()
    q_norm, k_norm = weights(hq, per_head, dtype, gen), weights(hk, per_head, dtype, gen)
    q = torch.empty((rows, hq, DIM), dtype=dtype, device="cuda")
    k, v = torch.empty((rows, hk, DIM), dtype=dtype, device="cuda"), torch.empty((rows, hk, DIM), dtype=dtype, device="cuda")
    paged.rope_paged_append(qkv, cos_sin, positions, axis_of, q, layer.keys, layer.values, layer.table, layer.lengths, starts, keys=k, values=v,
                            q_norm=q_norm, k_norm=k_norm, eps=eps)
    check_prefill_errors()
    x = qkv.cpu().double().unflatten(1, (-1, DIM))
    want_q, size_q = turned(normed(x[:, :hq], q_norm, eps), cos_sin, positions, axis_of)
    want_k, size_k = turned(normed(x[:, hq:hq + hk], k_norm, eps), cos_sin, positions, axis_of)
    if eps == 0.0:
        assert torch.isnan(q[0, 0]).all()
        want_q[0, 0], size_q[0, 0], q[0, 0] = 0.0, 0.0, 0.0
    else:
        assert (q[0, 0] == 0).all()
    assert near(q, want_q, size_q) and near(k, want_k, size_k) and torch.equal(v, qkv.unflatten(1, (-1, DIM))[:, hq + hk:])
    at = 0
    for b, n in enumerate(counts):
        for j in range(n):
            id, inside = layer.pages_of[b][(held[b] + j) // page], (held[b] + j) % page
            assert torch.equal(layer.keys[id, :, inside], k[at + j]) and torch.equal(layer.values[id, :, inside], v[at + j])
        at += n


def test_without_norms_nothing_changes():
    """Weights of one over heads whose mean square is one give what the rotation alone gives, but for the norm's own roundings."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.decode_layer import cos_sin_cache

    layer = Layer([0], 1, 16, torch.bfloat16, room=40)
    x = torch.where(torch.rand(40, 3, DIM, device="cuda") < 0.5, -1.0, 1.0)
    qkv, ones = x.to(torch.bfloat16).flatten(1), torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
    positions, cos_sin = torch.arange(40, device="cuda"), cos_sin_cache(100, DIM, 1e4, "cuda")
    starts = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    got = []
    for norm in ({}, dict(q_norm=ones, k_norm=ones, eps=0.0)):
        q = torch.empty((40, 1, DIM), dtype=torch.bfloat16, device="cuda")
        paged.rope_paged_append(qkv, cos_sin, positions, (0,) * 64, q, layer.keys, layer.values, layer.table, layer.lengths, starts, **norm)
        got.append(q.float())
    assert ((got[0] - got[1]).abs() <= 2.0 ** -7 * got[0].abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hq,hk,per_head", [(1, 8, 2, False), (5, 7, 1, True), (33, 32, 8, False)])
def test_rope_split_against_64_bits(dtype, rows, hq, hk, per_head):
    from retrievalattention_b200.decode_layer import cos_sin_cache, rope_split

    gen = torch.Generator().manual_seed(rows)
    qkv = (torch.randn((rows, (hq + 2 * hk) * DIM), generator=gen) * 3).to(dtype).cuda()
    positions, cos_sin = torch.randint(0, 500, (rows,), generator=gen).cuda(), cos_sin_cache(500, DIM, 1e4, "cuda")
    q_norm, k_norm = weights(hq, per_head, dtype, gen), weights(hk, per_head, dtype, gen)
    q, k, v = (torch.empty((rows, 1, h, DIM), dtype=dtype, device="cuda") for h in (hq, hk, hk))
    rope_split(qkv, cos_sin, positions, q, k, v, q_norm=q_norm, k_norm=k_norm, eps=1e-6)
    x = qkv.cpu().double().unflatten(1, (-1, DIM))
    for got, part, w in ((q, x[:, :hq], q_norm), (k, x[:, hq:hq + hk], k_norm)):
        assert near(got[:, 0], *turned(normed(part, w, 1e-6), cos_sin, positions[None], (0,) * 64))
    assert torch.equal(v[:, 0], qkv.unflatten(1, (-1, DIM))[:, hq + hk:])


def test_refusals():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.decode_layer import cos_sin_cache, rope_split

    layer = Layer([0], 2, 16, torch.bfloat16, room=4)
    qkv, q = torch.zeros(1, 12 * DIM, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 8, DIM, dtype=torch.bfloat16, device="cuda")
    cos_sin, positions = cos_sin_cache(10, DIM, 1e4, "cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    w = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(1, 2, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for bad in (dict(q_norm=w), dict(k_norm=w), dict(q_norm=w.float(), k_norm=w), dict(q_norm=w[:64], k_norm=w), dict(q_norm=w.expand(2, DIM), k_norm=w),
                dict(q_norm=w, k_norm=w.cpu()), dict(q_norm=w, k_norm=w, eps=-1.0), dict(q_norm=w, k_norm=w, eps=float("nan")),
                dict(q_norm=w, k_norm=w.repeat(8, 1)), dict(q_norm=w.clone().requires_grad_(), k_norm=w)):
        with pytest.raises(ValueError):
            paged.rope_paged_append(qkv, cos_sin, positions, (0,) * 64, q, layer.keys, layer.values, layer.table, layer.lengths, **bad)
        with pytest.raises(ValueError):
            rope_split(qkv, cos_sin, positions, q, k, v, **bad)
