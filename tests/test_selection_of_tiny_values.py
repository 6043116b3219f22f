"""Block selection where squares of the inputs fall below the smallest fp32 number: the choice is still that of scores in
64 bits."""
import pytest
import torch

from ma_transformer_b200 import selected_attention as sel
from test_selected_attention import plain_select


@pytest.mark.gpu
@pytest.mark.parametrize("down_q, down_k", [(80, 0), (0, 80), (60, 60), (100, 20)])
@pytest.mark.parametrize("causal", [True, False])
def test_near_scores_of_tiny_values_are_ordered_in_64_bits(down_q, down_k, causal):
    """Blocks whose bounds differ in one column's last bit, which fp32 sums cannot tell apart, scaled by powers of two."""
    S, block, D = 1280, 16, 64
    g = torch.Generator().manual_seed(12)
    k = torch.randn(1, 1, 1, D, generator=g).bfloat16().expand(1, S, 1, D).contiguous() * 8
    for n in range(S // block):
        c = (n * 7) % D
        x = k[0, n * block, 0, c].float()
        k[0, n * block, 0, c] = (x + x.abs() * torch.finfo(torch.bfloat16).eps).bfloat16()
    q = torch.randn(1, S, 2, D, generator=g).bfloat16() * 1e-3
    q[..., 0] = 30
    q, k = q * 2.0 ** -down_q, k * 2.0 ** -down_k
    got = sel.select_blocks(q.cuda(), k.cuda(), block, 9, causal).cpu()
    assert torch.equal(got, plain_select(q, k, block, 9, causal))
