"""``paged.paged_prompt`` with rows that several requests claim: reported, nothing written, and the next call is as ever."""
import pytest
import torch

from paged_helpers import DIM, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts", [[0, 6, 3, 9], [9, 0, 0, 9], [0, 9, 9, 4], [0, 1 << 30, -(1 << 30), 9]])
@pytest.mark.parametrize("held", [0, 3000])
def test_rows_that_do_not_ascend(starts, held):
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    layer = Layer([held + n for n in (20, 30, 9)], 2, 16, torch.bfloat16)
    q = torch.randn(9, 8, DIM, device="cuda").to(torch.bfloat16)
    right = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device="cuda")
    args = layer.keys, layer.values, layer.table, layer.lengths
    want = paged.paged_prompt(q, *args, right)
    check_prefill_errors()
    out, lse = torch.full_like(q, 7.0), torch.full((9, 8), 7.0, device="cuda")
    with pytest.raises(RuntimeError, match="row_start descends"):
        paged.paged_prompt(q, *args, torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out, lse=lse)
        check_prefill_errors()
    assert (out == 7).all() and (lse == 7).all()
    assert torch.equal(paged.paged_prompt(q, *args, right), want)
    check_prefill_errors()
