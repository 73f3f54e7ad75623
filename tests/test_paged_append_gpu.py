"""``paged.rope_paged_append`` against the rotation in 64 bits, and the rows' places in the cache.

Tolerance of a rotated channel: two products and a sum in 32 bits (3 * 2^-24 of |x| + |y|, 2e-7) and the rounding of the result.
Values and places are exact."""
import pytest
import torch

from paged_helpers import DIM, Layer, rounding

pytestmark = pytest.mark.gpu


def table_of(n, theta=1e4):
    from retrievalattention_b200.decode_layer import cos_sin_cache

    return cos_sin_cache(n, DIM, theta, "cuda")


def rotated(x, cos_sin, positions, axis_of):
    """x [rows, heads, 128] in 64 bits."""
    t = cos_sin.cpu().double()
    pos = positions.cpu().clamp(0, t.shape[0] - 1)
    pos = pos if pos.dim() == 2 else pos[None]
    c = torch.stack([t[pos[a], i] for i, a in enumerate(axis_of)], 1)[:, None]
    s = torch.stack([t[pos[a], 64 + i] for i, a in enumerate(axis_of)], 1)[:, None]
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def near(got, want, x):
    half, tiny = rounding(got.dtype)
    size = x[..., :64].abs() + x[..., 64:].abs()
    return ((got.cpu().double() - want).abs() <= half * want.abs() + 2e-7 * torch.cat([size, size], -1) + tiny).all()


def run(layer, counts, hq, axis_of, seed=0, fused=0, extra=True, starts=True, first_row=0, trailing=0, clip=0, error=None):
    """Append counts[b] rows to request b and check everything.  `clip` rows of each are left out of the cache, and `error` reported."""
    from contextlib import nullcontext

    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    gen = torch.Generator().manual_seed(seed)
    hk, rows, axes = layer.hk, first_row + sum(counts) + trailing, max(axis_of) + 1
    wide = torch.randn((rows, (hq + 2 * hk) * DIM + fused), generator=gen).to(layer.dtype).cuda()
    qkv = wide[:, :(hq + 2 * hk) * DIM]
    positions = torch.randint(-3, 605, (axes, rows), generator=gen).cuda()            # a few outside the table
    cos_sin = table_of(600)
    if axes == 1:
        positions = positions[0].contiguous()
    row_start = torch.tensor([first_row] + counts).cumsum(0).to(torch.int32).cuda()
    seen = torch.randint(0, 1000, (len(counts),), generator=gen).to(torch.int32)
    q = torch.full((rows, hq, DIM), 9.0, dtype=layer.dtype, device="cuda")
    k, v = (torch.full((rows, hk, DIM), 9.0, dtype=layer.dtype, device="cuda") for _ in range(2)) if extra else (None, None)
    pools = dict(keys=layer.keys, values=layer.values, weight=layer.weight, token=layer.token)
    before = {n: p.clone() for n, p in pools.items()}
    with pytest.raises(RuntimeError, match=error) if error else nullcontext():       # by the call itself, if the kernel is done by then
        paged.rope_paged_append(qkv, cos_sin, positions, axis_of, q, layer.keys, layer.values, layer.table, layer.lengths,
                                row_start if starts else None, weight=layer.weight, token=layer.token, seen=seen.cuda(), keys=k,
                                values=v)
        check_prefill_errors()
    x = qkv.cpu().double().view(rows, hq + 2 * hk, DIM)
    want = rotated(x[:, :hq + hk], cos_sin, positions, axis_of)
    assert near(q, want[:, :hq], x[:, :hq])
    dense_v = qkv.view(rows, hq + 2 * hk, DIM)[:, hq + hk:] if not fused else qkv.reshape(rows, hq + 2 * hk, DIM)[:, hq + hk:]
    if extra:
        assert near(k, want[:, hq:], x[:, hq:hq + hk]) and torch.equal(v, dense_v)
    at = first_row
    mine = torch.zeros(layer.weight.shape, dtype=torch.bool, device="cuda")
    for b, n in enumerate(counts):
        held, kept = layer.lengths_list[b], n - clip
        for j in range(kept):
            slot = held + j
            id, inside = layer.pages_of[b][slot // layer.page], slot % layer.page
            mine[id, :, inside] = True
            assert near(layer.keys[id, :, inside], want[at + j, hq:], x[at + j, hq:hq + hk])
            assert torch.equal(layer.values[id, :, inside], dense_v[at + j])
            assert (layer.weight[id, :, inside] == 0).all() and (layer.token[id, :, inside] == int(seen[b]) + j).all()
        at += n
    for name, p in pools.items():                            # every other slot is as it was
        kind = torch.int16 if p.element_size() == 2 else torch.int32
        assert torch.equal(p.contiguous().view(kind)[~mine], before[name].contiguous().view(kind)[~mine]), name


def sections(*n):
    from retrievalattention_b200.paged import rope_sections

    return rope_sections(*n)


@pytest.mark.parametrize("lengths,counts,kv_heads,group,page,dtype,axes", [
    ((0,), [1], 1, 1, 8, torch.bfloat16, (64,)),
    ((0, 5, 15, 16), [1, 1, 1, 1], 2, 4, 16, torch.bfloat16, (16, 24, 24)),
    ((7, 0, 8, 33), [9, 1, 0, 40], 3, 5, 8, torch.float16, (16, 24, 24)),           # a request without rows
    ((0, 0, 0), [0, 0, 30], 4, 7, 32, torch.float16, (32, 32)),                     # the first requests without rows
    ((100,), [130], 8, 8, 64, torch.bfloat16, (10, 20, 30, 4)),                     # 80 heads: two rounds of a CTA
    ((3,) * 40, [1] * 40, 1, 8, 16, torch.bfloat16, (16, 24, 24)),                  # more requests than lanes
    ((1,) * 64, [2] * 64, 1, 1, 8, torch.float16, (64,)),                           # two full rounds of requests
    ((333, 9, 0), [1501, 77, 40], 2, 3, 32, torch.float16, (16, 24, 24)),           # several rows to a CTA
    ((64, 1), [700, 1], 8, 4, 16, torch.bfloat16, (24, 20, 20)),
    ((3, 0, 77) * 3, [700, 1, 2, 0, 3, 555, 700, 1, 40], 1, 8, 32, torch.bfloat16, (16, 24, 24)),      # four rows to a unit, of several requests
    ((3, 9), [2001, 700], 2, 5, 16, torch.float16, (24, 20, 20)),                   # three
    ((5,) * 70, [31] * 70, 2, 8, 8, torch.bfloat16, (64,)),                         # two, more requests than lanes
    ((0,), [1333], 8, 8, 128, torch.bfloat16, (64,)),                               # the same with two rounds a row
])
def test_rows_and_places(lengths, counts, kv_heads, group, page, dtype, axes):
    layer = Layer(lengths, kv_heads, page, dtype, seed=1, room=max(counts))
    run(layer, counts, kv_heads * group, sections(*axes))


def test_interleaved_axes_strided_projection_pages_apart():
    from retrievalattention_b200.paged import rope_interleaved

    axis_of = rope_interleaved(24, 20, 20)
    assert len(axis_of) == 64 and axis_of[:6] == (0, 1, 2, 0, 1, 2) and axis_of[-4:] == (0, 0, 0, 0)
    run(Layer((5, 21), 2, 16, torch.bfloat16, seed=2, room=9, apart=True), [9, 4], 8, axis_of, fused=64)


def test_one_row_per_request_without_row_start_and_without_copies():
    run(Layer((5, 16, 0), 2, 16, torch.float16, seed=3, room=1), [1, 1, 1], 6, sections(64), starts=False, extra=False)


def test_rows_of_no_request_are_rotated_only():
    run(Layer((5, 16), 2, 16, torch.bfloat16, seed=4, room=5), [3, 5], 4, sections(16, 24, 24), first_row=2, trailing=3)


def test_rows_that_do_not_fit_are_reported():
    layer = Layer((30,), 2, 16, torch.bfloat16, seed=5)
    layer.table = layer.table[:, :2].contiguous()              # 32 slots, four rows
    run(layer, [4], 4, sections(64), clip=2, error="did not fit the pages")
    layer = Layer((16,), 2, 16, torch.bfloat16, seed=5)        # the table's second entry is -1
    layer.pages_of[0] = layer.pages_of[0][:1]
    run(layer, [1], 4, sections(64), clip=1, error="names no page")


def test_no_rows():
    run(Layer((3,), 1, 8, torch.bfloat16, seed=6, room=1), [0], 2, sections(64))


def test_refusals():
    from retrievalattention_b200 import paged

    layer = Layer((5, 9), 2, 16, torch.bfloat16, seed=7, room=4)
    rows, hq = 5, 8
    good = dict(qkv=torch.zeros((rows, (hq + 4) * DIM), dtype=torch.bfloat16, device="cuda"), cos_sin=table_of(50),
                positions=torch.zeros((3, rows), dtype=torch.int64, device="cuda"), axis_of=sections(16, 24, 24),
                q=torch.zeros((rows, hq, DIM), dtype=torch.bfloat16, device="cuda"), key_pages=layer.keys, value_pages=layer.values,
                page_table=layer.table, lengths=layer.lengths, row_start=torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda"))
    paged.rope_paged_append(**good)
    for change in (dict(qkv=good["qkv"][:, 1:]), dict(qkv=good["qkv"].half()), dict(qkv=good["qkv"].t()),
                   dict(q=good["q"][:, :7]), dict(q=good["q"].transpose(0, 1)), dict(cos_sin=good["cos_sin"].double()),
                   dict(cos_sin=good["cos_sin"][:, :64]), dict(positions=good["positions"].int()),
                   dict(positions=good["positions"][:, :4]), dict(positions=good["positions"].cpu()),
                   dict(axis_of=(0,) * 63), dict(axis_of=(0,) * 63 + (-1,)), dict(axis_of=(0.0,) * 64),
                   dict(row_start=good["row_start"][:2]), dict(row_start=good["row_start"].long()),
                   dict(keys=good["q"]), dict(token=layer.token), dict(seen=good["row_start"]),
                   dict(qkv=good["qkv"].clone().requires_grad_()), dict(value_pages=None)):
        with pytest.raises(ValueError):
            paged.rope_paged_append(**{**good, **change})
    with pytest.raises(RuntimeError, match="follows axis 3 of 3"):
        paged.rope_paged_append(**{**good, "axis_of": (3,) * 64})
    with pytest.raises(RuntimeError, match="need row_start"):
        paged.rope_paged_append(**{**good, "row_start": None})
    odd = torch.zeros(good["qkv"].numel() + 4, dtype=torch.bfloat16, device="cuda")[4:].view(good["qkv"].shape)
    with pytest.raises(RuntimeError, match="aligned"):
        paged.rope_paged_append(**{**good, "qkv": odd})
