"""``paged.paged_shared_decode``: outputs are those of ``paged_decode`` in precision, whichever kernels the room of the page table asks for."""
import pytest
import torch

from paged_helpers import DIM, Layer
from test_paged_shared_gpu import begin_alike, roomy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("dtype,part", [(torch.float16, 0.02), (torch.bfloat16, 0.01)])
@pytest.mark.parametrize("lengths,groups,kv_heads,group,page", [
    ((13000, 12900, 12801, 14000), ((0, 4, 200),), 2, 4, 64),      # an item that many CTAs share
    ((700,) * 40, ((0, 40, 4),), 1, 8, 128),                        # items of two tiles and of one
    ((900, 850, 20, 1000), ((0, 2, 50), (2, 4, 1)), 2, 7, 16),
])
def test_outputs_are_the_rounded_ones(lengths, groups, kv_heads, group, page, dtype, part, room):
    """An error e, relative, moves at most 2 e / 2^-11 of fp16 outputs over a rounding edge, 2 e / 2^-8 of bf16 ones.  Scores and sums
    4e-6, bf16's probabilities of 16 bits (two parts of 8) 2^-16 more: 1.6 and 1 %, as for requests that are attended one by one.  One part
    of 8 bits would move every fourth and more."""
    from retrievalattention_b200 import paged

    layer = Layer(lengths, kv_heads, page, dtype, seed=5)
    begin_alike(layer, groups)
    starts, shared = [groups[0][0]] + [last for _, last, _ in groups], [pages * page for *_, pages in groups]
    q = torch.randn((len(lengths), 1, kv_heads * group, DIM), generator=layer.gen).to(dtype)
    out = paged.paged_shared_decode(q.cuda(), layer.keys, layer.values, roomy(layer.table) if room else layer.table, layer.lengths,
                                    torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                    torch.tensor(shared, dtype=torch.int32, device="cuda")).cpu()
    wrong = total = 0
    for b in range(len(lengths)):
        s = q[b, 0].double().view(kv_heads, group, DIM) @ layer.k[b].transpose(1, 2) * DIM ** -0.5
        want = (torch.softmax(s, -1) @ layer.v[b]).view(-1, DIM)
        wrong += (out[b, 0] != want.to(dtype)).sum().item()
        total += want.numel()
    assert wrong <= part * total, wrong / total
