"""``paged.paged_decode`` over long caches: what the sums over hundreds of steps and the 16-bit parts of the probabilities cost.

Requests share their pages here (nothing is written to them), so that a warp gets thousands of slots from a small pool."""

import pytest
import torch

from paged_helpers import DIM

pytestmark = pytest.mark.gpu


def shared(k, v, batch, page=32):
    """Slots [n, 128] as the one KV head of `batch` requests: pools, table, lengths."""
    n = k.shape[0]
    pages = -(-n // page)
    pools = []
    for x in (k, v):
        pool = torch.zeros((pages * page, DIM), dtype=x.dtype, device="cuda")
        pool[:n] = x
        pools.append(pool.view(pages, 1, page, DIM))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, pages).contiguous()
    return (*pools, table, torch.full((batch,), n, dtype=torch.int32, device="cuda"))


def in_64_bits(q, k, v):
    return torch.softmax(q[:, 0].double() @ k.double().t() * DIM ** -0.5, -1) @ v.double()


def test_long_sums_are_rounded_to_nearest():
    """400 steps a warp, fp16.  Against the output in 64 bits an error e, relative, moves a value over a rounding edge with a
    probability of at most 2 e / 2^-11.  32-bit sums that round to nearest stay within 4e-6: sqrt(400) 2^-24 for the chain of steps, the
    probabilities' 22 bits, 1e-6 from the scores.  That is 1.6 % of the values; sums that are cut off at each step lose 400 * 2^-24
    and more, always towards zero."""
    from retrievalattention_b200 import paged

    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    batch, n, group = 128, 60000, 4
    q = torch.randn((batch, 1, group, DIM), generator=gen, device="cuda").half()
    k, v = (torch.randn((n, DIM), generator=gen, device="cuda").half() for _ in range(2))
    out = paged.paged_decode(q, *shared(k, v, batch))[:, 0]
    want = in_64_bits(q, k, v)
    wrong = (out != want.half()).double().mean().item()
    assert wrong <= 0.02, wrong
    assert ((out.double() - want).abs() <= (2.0 ** -11 + 2e-5) * want.abs() + 2.0 ** -25 + 1e-8).all()


def with_sinks(below, dtype, n, every, batch, group, seed):
    """Queries and slots: every `every`-th slot's score is `below` above the others' in every head, and its value is zero."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    q = torch.randn((batch, 1, group, DIM), generator=gen, device="cuda")
    q[..., 0] = 16
    k = torch.randn((n, DIM), generator=gen, device="cuda") * 0.05
    k[:, 0] = 0
    v = torch.rand((n, DIM), generator=gen, device="cuda") * 64 + 32
    k[::every], v[::every] = 0, 0
    k[::every, 0] = below * DIM ** 0.5 / 16
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("below", [14.0, 15.0, 17.0, 20.0])
@pytest.mark.parametrize("n,every,batch", [(60000, 1000, 64), (3000, 1000, 5), (40, 1000, 3)])
def test_slots_far_below_the_largest(n, every, batch, below, dtype):
    """Slots without a value take nearly all of the probability, and what is left decides the output.

    All values are positive, so the output is off by as much, relative, as its terms: a score of 20 is off by at most
    32 roundings of 2^-24 of it, 4e-5, twice (slot and log-sum-exp), the 16 bits of bf16's probabilities by 2^-16, the sums by
    2^-20; then its own rounding."""
    from retrievalattention_b200 import paged

    q, k, v = with_sinks(below, dtype, n, every, batch, 4, seed=2)
    out = paged.paged_decode(q, *shared(k, v, batch))[:, 0].double()
    want = in_64_bits(q, k, v)
    half, tiny = (2.0 ** -8, 0.0) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    assert ((out - want).abs() <= (half + 2e-4) * want.abs() + tiny).all(), ((out - want).abs() / want.abs()).max().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 6000])
def test_infinite_values_of_slots_far_below(n, dtype):
    """30 below the largest: 2^-43."""
    from retrievalattention_b200 import paged

    q, k, v = with_sinks(30.0, dtype, n, 1000, 3, 4, seed=3)
    v[3, 5], v[n - 9, 77] = float("inf"), -float("inf")          # beside the slot of the largest score, and away from it
    out = paged.paged_decode(q, *shared(k, v, 3))[:, 0]
    assert (out[..., 5] == float("inf")).all() and (out[..., 77] == -float("inf")).all()
    rest = [c for c in range(DIM) if c not in (5, 77)]
    assert torch.isfinite(out[..., rest]).all()


def test_scores_that_fall_along_the_cache():
    """Scores fall by 4 (in nats) a step: the reference follows them down as far as it may, and what they give vanishes beside the
    first ones."""
    from retrievalattention_b200 import paged

    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    q = torch.randn((2, 1, 4, DIM), generator=gen, device="cuda").half()
    q[..., 0] = 16
    k = (torch.randn((4000, DIM), generator=gen, device="cuda") * 0.05).half()
    k[:, 0] = torch.linspace(0, -1000, 4000).cuda() * DIM ** 0.5 / 16
    v = torch.randn((4000, DIM), generator=gen, device="cuda").half()
    lse = torch.empty((2, 4), device="cuda")
    out = paged.paged_decode(q, *shared(k, v, 2), lse=lse)[:, 0].double()
    want = in_64_bits(q, k, v)
    # the first dozen slots count: scores of at most 3 in magnitude, 1e-5 off, on values of at most 4
    assert ((out - want).abs() <= 2.0 ** -11 * want.abs() + 1e-4).all()
    scores = q[:, 0].double() @ k.double().t() * DIM ** -0.5
    assert ((lse.double() - torch.logsumexp(scores, -1)).abs() <= 3e-5).all()


@pytest.mark.parametrize("dtype,part", [(torch.float16, 0.02), (torch.bfloat16, 0.01)])
@pytest.mark.parametrize("lengths,kv_heads,group,page", [((777, 0, 300), 8, 4, 16), ((9001, 1), 2, 8, 256), ((5003, 2500, 0, 77), 4, 7, 8)])
def test_outputs_are_the_rounded_ones(lengths, kv_heads, group, page, dtype, part):
    """An error e, relative, moves at most 2 e / 2^-11 of fp16 outputs over a rounding edge, 2 e / 2^-8 of bf16 ones.  Scores and sums
    4e-6, bf16's probabilities of 16 bits 2^-16 more: 1.6 and 1 %."""
    from paged_helpers import Layer
    from retrievalattention_b200 import paged

    layer = Layer(lengths, kv_heads, page, dtype, seed=5)
    q = torch.randn((len(lengths), 1, kv_heads * group, DIM), generator=layer.gen).to(dtype)
    out = paged.paged_decode(q.cuda(), layer.keys, layer.values, layer.table, layer.lengths).cpu()
    wrong = total = 0
    for b, n in enumerate(lengths):
        if n:
            s = q[b, 0].double().view(kv_heads, group, DIM) @ layer.k[b].transpose(1, 2) * DIM ** -0.5
            want = (torch.softmax(s, -1) @ layer.v[b]).view(-1, DIM)
            wrong += (out[b, 0] != want.to(dtype)).sum().item()
            total += want.numel()
    assert wrong <= part * total, wrong / total
