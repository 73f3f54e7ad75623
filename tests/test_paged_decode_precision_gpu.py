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
