"""A small model whose queries and keys are normalised, one of whose layers looks back over a window, and whose requests begin alike,
against the same model in 32 bits recomputed over the whole sequence: norms, prompts, steps and shared prefixes together."""
import pytest
import torch

from paged_helpers import DIM

pytestmark = pytest.mark.gpu


def small(window=(None, 24), sink=3, qk_norm=True, batch=3, page=16, max_length=600, keep=None):
    from retrievalattention_b200.cache_hub import paged_cache
    from retrievalattention_b200.decode_layer import ModelShape, PagedDecoder

    layers = len(window)
    shape = ModelShape(256, 512, 1000, layers, 8, 2, rope_theta=1e4, qk_norm=qk_norm)
    cache = paged_cache(layers, batch, max_length, 2, 8, DIM, torch.bfloat16, {str(i): "cuda:0" for i in range(layers)}, 1, 1,
                        page_size=page, attn_window=list(window), attn_sink=sink, keep=keep)
    return PagedDecoder(shape, cache, batch, 2000, "cuda", seed=3, std=0.05)


def in_32_bits(model, ids):
    """Logits of the last token, everything recomputed."""
    s, cache, n = model.shape, model.cache, len(ids)
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.rms_eps) * w.float()  # noqa: E731
    angle = model.cos_sin[torch.arange(n, device="cuda")]
    c, z = angle[:, None, :64], angle[:, None, 64:]
    i = torch.arange(n, device="cuda")
    x = model.embed[ids].float()
    for L, window in zip(model.layers, cache.attn_window):
        heads = (norm(x, L["norm1"]) @ L["wqkv"].float().t()).view(n, -1, DIM)
        q, k, v = heads[:, :8], heads[:, 8:10], heads[:, 10:]
        if s.qk_norm:
            q, k = norm(q, L["q_norm"]), norm(k, L["k_norm"])
        turn = lambda h: torch.cat([h[..., :64] * c - h[..., 64:] * z, h[..., 64:] * c + h[..., :64] * z], -1)  # noqa: E731
        q, k = turn(q).transpose(0, 1), turn(k).transpose(0, 1).repeat_interleave(4, 0)
        w = (q @ k.transpose(1, 2)) * DIM ** -0.5
        seen = i <= i[:, None]
        if window is not None:
            seen &= (i > i[:, None] - window) | (i < cache.attn_sink)
        w = w.masked_fill(~seen, float("-inf")).softmax(-1)
        x = x + (w @ v.transpose(0, 1).repeat_interleave(4, 0)).transpose(0, 1).reshape(n, -1) @ L["wo"].float().t()
        g, u = (norm(x, L["norm2"]) @ L["gate_up"].float().t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ L["down"].float().t()
    return (norm(x, model.final_norm) @ model.lm_head.float().t())[-1]


def check(model, logits, ids, requests):
    for row, b in zip(logits, requests):
        want = in_32_bits(model, torch.stack(ids[b]))
        # 16-bit activations of two layers: 2^-8 a rounding, a dozen of them one behind the other
        assert (row - want).norm() <= 0.05 * want.norm(), b
        ids[b].append(model.input_ids[b].clone())


@pytest.mark.parametrize("window,sink,qk_norm", [((None, 24), 3, True), ((17, 40), 0, False), ((None, None), 0, True)])
def test_prompts_steps_and_more_tokens(window, sink, qk_norm):
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    model = small(window, sink, qk_norm)
    gen = torch.Generator().manual_seed(1)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    prompts = [prompt(n) for n in (90, 5, 41)]
    ids = [list(p) for p in prompts]
    check(model, model.prefill_forward(prompts), ids, range(3))
    for _ in range(3):
        check(model, model.decode_forward(), ids, range(3))
    # more of two conversations: the token that was not fed yet, and what the user says next
    more = [torch.cat([ids[b][-1:][0][None], prompt(n)]) for b, n in ((0, 30), (2, 1))]
    for b, p in zip((0, 2), more):
        ids[b] = ids[b][:-1] + list(p)
    check(model, model.extend_forward(more, requests=[0, 2]), ids, (0, 2))
    model.release(1)                                          # its place's next tokens are another request's first
    ids[1] = list(prompt(7))
    check(model, model.extend_forward([torch.stack(ids[1])], requests=[1]), ids, (1,))
    for _ in range(3):
        check(model, model.decode_forward(), ids, range(3))
    check_prefill_errors()


@pytest.mark.parametrize("window", [(None, 24), (None, None)])
def test_requests_that_begin_alike(window):
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    model = small(window, batch=4)
    gen = torch.Generator().manual_seed(2)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    begin = prompt(75)
    for b in (1, 2, 3):
        model.release(b)
    ids = [list(begin), None, None, None]
    check(model, model.prefill_forward([begin], requests=[0]), ids, (0,))
    assert model.share(0, [1, 2]) == 64
    rest = [torch.cat([begin[64:], prompt(n)]) for n in (3, 20)]
    for b, p in zip((1, 2), rest):
        ids[b] = list(begin[:64]) + list(p)
    check(model, model.extend_forward(rest, requests=[1, 2]), ids, (1, 2))
    assert model.cache._alike and model.cache._group_shared.tolist()[0] == 64
    for step in range(4):
        check(model, model.decode_forward(), ids, (0, 1, 2))
    model.release(0)                                          # the pages that the others begin with stay
    other = prompt(33)
    ids[0], ids[3] = list(other), list(other)
    check(model, model.prefill_forward([other, other], requests=[0, 3]), ids, (0, 3))
    for step in range(3):
        check(model, model.decode_forward(), ids, range(4))
    for b in range(4):
        model.release(b)
    assert model.cache.free_pages == model.cache.num_pages
    check_prefill_errors()


def test_captured_attention_of_requests_that_begin_alike():
    """A captured call goes by the whole page table, whose room is what decides between the kernels: the same sums either way."""
    from retrievalattention_b200.attn_hub import paged_decode_attn
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    model = small((None,), batch=3, max_length=120000, page=64)
    cache, gen = model.cache, torch.Generator().manual_seed(4)
    model.release(1)
    model.release(2)
    model.prefill_forward([torch.randint(0, 1000, (200,), generator=gen).cuda()], requests=[0])
    assert model.share(0, [1, 2], 150) == 128
    model.extend_forward([torch.randint(0, 1000, (n,), generator=gen).cuda() for n in (9, 1)], requests=[1, 2])
    q, out, lse, other = (torch.randn(3, 1, 8, DIM, device="cuda").to(torch.bfloat16), torch.empty(3, 1, 8, DIM, device="cuda", dtype=torch.bfloat16),
                          torch.empty(3, 8, device="cuda"), torch.empty(3, 8, device="cuda"))
    paged_decode_attn(q, None, None, 0, cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, 0, out=out, lse=lse)
    graph.replay()
    eager = cache.attend(q, 0, lse=other)
    check_prefill_errors()
    # probabilities and outputs are rounded to 16 bits, half a step of 2^-7 each, on either side
    same = lambda: ((out.float() - eager.float()).abs() <= 2.0 ** -6 * (eager.float().abs() + 0.2)).all() and (lse - other).abs().max() <= 1e-4  # noqa: E731
    assert same()
    # requests that come and go: the captured call finds the new groups
    model.release(1)
    model.prefill_forward([torch.randint(0, 1000, (70,), generator=gen).cuda()], requests=[1])
    graph.replay()
    eager = cache.attend(q, 0, lse=other)
    assert same()
    check_prefill_errors()


def test_refusals():
    model = small(window=(None,), batch=2, keep=40 + 64, sink=0)
    with pytest.raises(ValueError, match="eviction"):
        model.extend_forward([torch.zeros(3, dtype=torch.int64, device="cuda")], requests=[0])
    with pytest.raises(ValueError, match="evicted"):
        model.share(0, [1])


def test_decoder_over_the_wave_index_takes_norms():
    """``SyntheticDecoder`` with norms: its queries and keys are what ``rope_split`` makes of them."""
    from retrievalattention_b200.decode_layer import ModelShape, SyntheticDecoder

    class Cache:
        context = 7

        def decode_update_kv_cache(self, k, v, layer):
            self.k = k.clone()

        def compute(self, q, layer, out):
            self.q = q.clone()
            return out.zero_()

    shape = ModelShape(256, 512, 1000, 1, 8, 2, qk_norm=True)
    model = SyntheticDecoder(shape, Cache(), 2, 100, "cuda", std=0.05)
    model.decode_forward()
    x = model.embed[torch.zeros(2, dtype=torch.int64, device="cuda")].float()
    L = model.layers[0]
    x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + shape.rms_eps) * L["norm1"].float()).to(torch.bfloat16)
    heads = torch.nn.functional.linear(x, L["wqkv"]).float().view(2, 12, DIM)
    angle = model.cos_sin[7]
    for got, part, w in ((model.cache.q, heads[:, :8], L["q_norm"]), (model.cache.k, heads[:, 8:10], L["k_norm"])):
        h = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + shape.rms_eps) * w.float()
        want = torch.cat([h[..., :64] * angle[:64] - h[..., 64:] * angle[64:], h[..., 64:] * angle[:64] + h[..., :64] * angle[64:]], -1)
        # the projection's 16-bit rows are the library's on both sides; norm of the row before may round one step apart
        assert (got[:, 0].float() - want).norm() <= 2.0 ** -7 * want.norm()
