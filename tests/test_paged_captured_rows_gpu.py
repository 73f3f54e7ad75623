"""Captured ``append`` and ``prompt`` of a ``paged_cache``, replayed in later steps whose rows are shared out otherwise."""
import pytest
import torch

from paged_helpers import DIM

pytestmark = pytest.mark.gpu


def test_a_captured_prompt_follows_the_rows_of_later_steps():
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors
    from retrievalattention_b200.cache_hub import paged_cache
    from retrievalattention_b200.decode_layer import cos_sin_cache

    gen = torch.Generator().manual_seed(3)
    steps = [[20, 0, 4], [3, 11, 10], [8, 8, 8], [0, 24, 0]]           # 24 rows each
    rows = [torch.randn(24, 12 * DIM, generator=gen).to(torch.bfloat16).cuda() for _ in steps]
    cos_sin, axis_of = cos_sin_cache(200, DIM, 1e4, "cuda"), paged.rope_sections(64)
    results = []
    for captured in (False, True):
        cache = paged_cache(1, 3, 100, 2, 8, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1)
        qkv, positions = torch.zeros_like(rows[0]), torch.zeros(24, dtype=torch.int64, device="cuda")
        q = torch.zeros(24, 8, DIM, dtype=torch.bfloat16, device="cuda")
        out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()

        def layer():
            cache.append(0, qkv, cos_sin, positions, axis_of, q)
            cache.prompt(q, 0, out=out)

        got = []
        for i, (counts, x) in enumerate(zip(steps, rows)):
            at = list(cache.length_of)
            cache.begin(counts)
            qkv.copy_(x)
            positions.copy_(torch.cat([torch.arange(a, a + n) for a, n in zip(at, counts)]))
            if not captured or i == 0:
                layer()
            if captured and i == 0:
                with torch.cuda.graph(graph):
                    layer()
            if captured:
                graph.replay()
                junk = [torch.full((4,), 1 << 20, dtype=torch.int32, device="cuda") for _ in range(200)]      # takes the place of what is freed
                del junk
            got.append(out.clone())
        check_prefill_errors()
        results.append(got)
    for eager, replayed in zip(*results):
        # the whole page table instead of the columns in use may cut items elsewhere: two roundings to 16 bits, half a step of 2^-7 each
        assert ((eager.float() - replayed.float()).abs() <= 2.0 ** -6 * (eager.float().abs() + 0.2)).all()
