"""The operators over a paged cache together: a small model that takes prompts with images and generates, against the same model in
32 bits recomputed over the whole sequence; and what eviction does to its cache."""
import pytest
import torch

from paged_helpers import DIM

pytestmark = pytest.mark.gpu


def small(window=16, keep=None, slack=8, page=16, pages=None, batch=3, layers=2, max_length=600):
    from retrievalattention_b200.cache_hub import paged_cache
    from retrievalattention_b200.decode_layer import ModelShape, PagedDecoder
    from retrievalattention_b200.paged import rope_sections

    shape = ModelShape(256, 512, 1000, layers, 8, 2, rope_theta=1e4)
    cache = paged_cache(layers, batch, max_length, 2, 8, DIM, torch.bfloat16, {str(i): "cuda:0" for i in range(layers)}, 1, 1,
                        page_size=page, num_pages=pages, keep=keep, sink=2, recent=12, slack=slack)
    return PagedDecoder(shape, cache, batch, 2000, "cuda", seed=3, std=0.05, axis_of=rope_sections(16, 24, 24), window=window)


def with_image(n):
    """Positions of n tokens, an image of 4 x 5 patches from token 6 on where there is room."""
    p = torch.arange(n).expand(3, n).clone()
    if n > 26:
        p[:, 6:26] = torch.stack([torch.full((20,), 6), 6 + torch.arange(20) // 5, 6 + torch.arange(20) % 5])
        p[:, 26:] -= 15
    return p.cuda()


def in_32_bits(model, ids, positions):
    """Logits of the last token, everything recomputed."""
    s = model.shape
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.rms_eps) * w.float()  # noqa: E731
    axis = torch.tensor(model.axis_of, device="cuda")
    i = torch.arange(64, device="cuda")
    angle = model.cos_sin[positions]
    c, z = angle[axis, :, i].t()[:, None], angle[axis, :, 64 + i].t()[:, None]
    x = model.embed[ids].float()
    for L in model.layers:
        heads = (norm(x, L["norm1"]) @ L["wqkv"].float().t()).view(len(ids), -1, DIM)
        a, b = heads[:, :10, :64], heads[:, :10, 64:]
        turned = torch.cat([a * c - b * z, b * c + a * z], -1)
        q, k = turned[:, :8].transpose(0, 1), turned[:, 8:].transpose(0, 1).repeat_interleave(4, 0)
        v = heads[:, 10:].transpose(0, 1).repeat_interleave(4, 0)
        w = (q @ k.transpose(1, 2)) * DIM ** -0.5
        w = w.masked_fill(torch.ones_like(w[0], dtype=torch.bool).triu(1), float("-inf")).softmax(-1)
        x = x + (w @ v).transpose(0, 1).reshape(len(ids), -1) @ L["wo"].float().t()
        g, u = (norm(x, L["norm2"]) @ L["gate_up"].float().t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ L["down"].float().t()
    return (norm(x, model.final_norm) @ model.lm_head.float().t())[-1]


def test_prompts_and_steps_against_32_bits():
    model = small()
    gen = torch.Generator().manual_seed(1)
    counts = (37, 5, 90)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).cuda() for n in counts]
    positions = [with_image(n) for n in counts]
    logits = model.prefill_forward(prompts, positions)
    ids = [list(p) for p in prompts]
    for step in range(20):
        for b in range(3):
            want = in_32_bits(model, torch.stack(ids[b]), positions[b])
            # 16-bit activations of two layers: 2^-8 a rounding, a dozen of them one behind the other
            assert (logits[b] - want).norm() <= 0.05 * want.norm(), (step, b)
            ids[b].append(model.input_ids[b].clone())
            positions[b] = torch.cat([positions[b], (positions[b].max() + 1).expand(3, 1)], 1)
        logits = model.decode_forward()
    assert model.cache.lengths.tolist() == [n + 20 for n in counts] == model.cache.length_of
    assert model.cache.free_pages == model.cache.num_pages - sum(-(-(n + 20) // 16) for n in counts)


def test_eviction_holds_requests_to_their_slots_and_gives_pages_back():
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    keep, slack = 40, 8
    model = small(keep=keep, slack=slack)
    cache, counts = model.cache, (37, 5, 200)
    gen = torch.Generator().manual_seed(2)
    model.prefill_forward([torch.randint(0, 1000, (n,), generator=gen).cuda() for n in counts])
    assert cache.lengths.tolist() == [37, 5, keep] == cache.length_of
    assert cache.free_pages == cache.num_pages - (3 + 1 + 3)
    evicted = 0
    for step in range(60):
        logits = model.decode_forward()
        assert torch.isfinite(logits).all()
        assert cache.lengths.tolist() == cache.length_of and max(cache.length_of) <= keep + slack
        seen = [n + step + 1 for n in counts]
        assert cache.seen_after.tolist() == seen
        for b in range(3):
            n = cache.length_of[b]
            ids = cache.page_table[b, :-(-n // 16)].long()
            assert ids.tolist() == cache._pages[b]
            for layer in range(2):
                tokens = cache.token[layer][ids].transpose(0, 1).reshape(2, -1)[:, :n]
                weight = cache.weight[layer][ids].transpose(0, 1).reshape(2, -1)[:, :n]
                for h in range(2):
                    have = set(tokens[h].tolist())
                    assert len(have) == n and have <= set(range(seen[b]))
                    assert set(range(min(2, seen[b]))) <= have and set(range(max(0, seen[b] - 12), seen[b])) <= have
                assert (weight >= 0).all() and (weight[:, 0] > 0).all()
        evicted += max(cache.length_of) <= keep
    assert evicted >= 5
    check_prefill_errors()


def test_a_place_is_taken_by_another_request():
    model = small(batch=2, pages=12)
    gen = torch.Generator().manual_seed(3)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    model.prefill_forward([prompt(100), prompt(60)])
    assert model.cache.free_pages == 12 - 7 - 4
    with pytest.raises(RuntimeError, match="pool has 1 pages left"):
        model.cache.begin([20, 20])
    assert model.cache.length_of == [100, 60]                 # nothing was taken
    model.cache.release(0)
    assert model.cache.free_pages == 8 and model.cache.length_of == [0, 60]
    model.cache.begin([5, 1])
    assert model.cache.lengths.tolist() == [5, 61] and model.cache.held.tolist() == [0, 60]
    with pytest.raises(RuntimeError, match="more than"):
        model.cache.begin([600, 0])


def test_decode_entry_point_reads_the_cache():
    from paged_helpers import attend
    from retrievalattention_b200.attn_hub import paged_decode_attn

    model = small(batch=2, keep=40)
    cache, gen = model.cache, torch.Generator().manual_seed(4)
    model.prefill_forward([torch.randint(0, 1000, (n,), generator=gen).cuda() for n in (30, 9)])
    q = torch.randn((2, 1, 8, DIM), generator=gen).bfloat16().cuda()
    before = cache.weight[1].clone()
    out = paged_decode_attn(q, None, None, 1, cache)
    for b, n in enumerate((30, 9)):
        ids = cache.page_table[b, :-(-n // 16)].long()
        k, v, old, new = (p[ids].transpose(0, 1).flatten(1, 2)[:, :n].cpu().double()
                          for p in (cache.key_pages[1], cache.value_pages[1], before, cache.weight[1]))
        want, _, p = attend(q[b, 0].cpu().double().view(2, 4, DIM), k, v)
        assert ((out[b, 0].cpu().double() - want.view(8, DIM)).abs() <= 2.0 ** -8 * want.view(8, DIM).abs() + 1e-4 * v.abs().max()).all()
        assert ((new - old - p.sum(1)).abs() <= 1e-4 * p.sum(1) + 2.0 ** -22 * new).all()


def test_refusals():
    from retrievalattention_b200.cache_hub import paged_cache

    one = {"0": "cuda:0"}
    with pytest.raises(ValueError, match="head_dim"):
        paged_cache(1, 1, 100, 2, 8, 64, torch.bfloat16, one, 1, 1)
    with pytest.raises(ValueError, match="keep"):
        paged_cache(1, 1, 100, 2, 8, 128, torch.bfloat16, one, 1, 1, keep=10)
    with pytest.raises(ValueError, match="one GPU"):
        paged_cache(2, 1, 100, 2, 8, 128, torch.bfloat16, {"0": "cuda:0", "1": "cuda:1"}, 1, 1)
    cache = paged_cache(1, 2, 100, 2, 8, 128, torch.bfloat16, one, 1, 1)
    with pytest.raises(ValueError, match="every request"):
        cache.begin([1])


@pytest.mark.parametrize("keep", [None, 500])
def test_prompts_take_the_places_of_requests_that_are_done(keep):
    """Three places, five requests, against 32 bits."""
    model = small(keep=keep, slack=8)
    gen = torch.Generator().manual_seed(7)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    ids, positions = {}, {}

    def admit(prompts, requests=None):
        where = [with_image(p.numel()) for p in prompts]
        logits = model.prefill_forward(prompts, where, requests)
        for i, b in enumerate(range(3) if requests is None else requests):
            ids[b], positions[b] = list(prompts[i]), where[i]
        return logits

    def check(logits, requests):
        assert logits.shape[0] == len(requests)
        for i, b in enumerate(requests):
            want = in_32_bits(model, torch.stack(ids[b]), positions[b])
            assert (logits[i] - want).norm() <= 0.05 * want.norm(), b
            ids[b].append(model.input_ids[b].clone())
            assert ids[b][-1] == logits[i].argmax()
            positions[b] = torch.cat([positions[b], (positions[b].max() + 1).expand(3, 1)], 1)

    check(admit([prompt(37), prompt(5), prompt(90)]), range(3))
    check(model.decode_forward(), range(3))
    model.release(1)
    for _ in range(3):
        check(model.decode_forward(), (0, 2))
    free = model.cache.free_pages
    check(admit([prompt(61)], [1]), (1,))
    assert model.cache.free_pages == free - 4
    for _ in range(2):
        check(model.decode_forward(), range(3))
    model.release(0)
    model.release(2)
    check(model.decode_forward(), (1,))
    check(admit([prompt(3), prompt(40)], [0, 2]), (0, 2))
    check(model.decode_forward(), range(3))
    assert model.cache.length_of == [4, 61 + 4, 41] == model.cache.lengths.tolist()
    for bad in ([1], [0, 0], [3], [-1]):
        with pytest.raises(ValueError):
            model.prefill_forward([prompt(4)] * len(bad), requests=bad)
    for b in range(3):
        model.release(b)
    with pytest.raises(ValueError, match="no request"):
        model.decode_forward()
    assert model.cache.free_pages == model.cache.num_pages


def test_steps_from_an_empty_cache():
    model = small()
    ids = [[model.input_ids[b].clone()] for b in range(3)]
    for step in range(4):
        logits = model.decode_forward()
        for b in range(3):
            want = in_32_bits(model, torch.stack(ids[b]), torch.arange(step + 1, device="cuda").expand(3, -1))
            assert (logits[b] - want).norm() <= 0.05 * want.norm()
            ids[b].append(model.input_ids[b].clone())


def test_generation_ends_where_the_positions_do():
    """Eviction holds the slots, not the positions; and nothing was taken by the call that raises."""
    model = small(keep=40)
    model.cos_sin = model.cos_sin[:120].contiguous()
    gen = torch.Generator().manual_seed(8)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    with pytest.raises(ValueError, match="0 to 119"):
        model.prefill_forward([prompt(4), prompt(121), prompt(4)])
    for far in (120, -1):
        where = [torch.arange(4).expand(3, 4).cuda() for _ in range(3)]
        where[1] = where[1].clone()
        where[1][2, 1] = far
        with pytest.raises(ValueError, match="the table has"):
            model.prefill_forward([prompt(4)] * 3, where)
    with pytest.raises(ValueError, match="positions"):
        model.prefill_forward([prompt(4)] * 3, [torch.zeros(2, 4, dtype=torch.int64).cuda()] * 3)
    assert model.cache.length_of == [0, 0, 0]
    model.prefill_forward([prompt(100), prompt(110), prompt(20)], [with_image(100), with_image(110), with_image(20)])
    assert model.positions.tolist() == [[85, 95, 20]] * 3         # an image takes 5 positions for its 20 tokens
    for _ in range(25):
        model.decode_forward()
    with pytest.raises(RuntimeError, match=r"requests \[1\] are at the end"):
        model.decode_forward()
    seen = model.cache.seen_after.tolist()
    assert seen == [125, 135, 45] and model.positions[0].tolist() == [110, 120, 45]
    model.release(1)
    for _ in range(10):
        model.decode_forward()                                    # the others go on
    assert model.positions[0].tolist() == [120, 120, 55]
    with pytest.raises(RuntimeError, match=r"requests \[0\] are at the end"):
        model.decode_forward()
