"""Block-selected attention at the largest sizes and over several groups of pairs."""
import pytest
import torch

from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import selected_attention as sel


@pytest.mark.gpu
def test_more_rows_than_lanes_count_in_32_bits():
    """512 query heads on one key head and 2^28 + 2^15 rows of 8 columns: lanes times rows pass 2^32.  The last block's rows
    read their own block only, so they and its gradients are those of the block alone, bit for bit."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 40 GiB")
    S, H, D, block = 2 ** 19 + 64, 512, 8, 64
    q = torch.empty(1, S, H, D, dtype=torch.bfloat16, device="cuda").normal_()
    k, v = (torch.empty(1, S, 1, D, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2))
    blocks = (torch.arange(S, device="cuda", dtype=torch.int32) // block).view(1, S, 1, 1)
    out, lse = sel.forward_selected(q, k, v, blocks, block)
    grads = sel.backward_selected(q, k, v, out, lse, q, blocks, block)
    ql, kl, vl = (t[:, -block:].contiguous() for t in (q, k, v))
    own = torch.zeros(1, block, 1, 1, dtype=torch.int32, device="cuda")
    out_l, lse_l = sel.forward_selected(ql, kl, vl, own, block)
    grads_l = sel.backward_selected(ql, kl, vl, out_l, lse_l, ql, own, block)
    for name, whole, last in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads), (out_l, lse_l, *grads_l)):
        assert torch.equal(whole[:, -block:], last), name


@pytest.mark.parametrize("change", [dict(S=2 ** 60), dict(S=2 ** 62 + 64), dict(B=2 ** 48, H=2 ** 16, Hkv=2 ** 16), dict(B=2 ** 15, H=2 ** 49, Hkv=2 ** 49),
                                    dict(H=2 ** 60), dict(H=2 ** 62), dict(S=2 ** 30, H=2 ** 4, topk=1)])
def test_sizes_whose_products_wrap_are_refused(change):
    a = dict(B=1, S=64, H=4, Hkv=2, D=64, dtype=nat.MAT_BF16, block=16, topk=16)
    a.update(change)
    shape, rest, p = (a["B"], a["S"], a["H"], a["Hkv"], a["D"], a["dtype"]), (a["block"], a["topk"]), 256
    assert nat.lib.mat_selected_attn_fwd_workspace_bytes(*shape, *rest) == 0
    assert nat.lib.mat_selected_attn_bwd_workspace_bytes(*shape, *rest) == 0
    assert nat.lib.mat_selected_attn_fwd(p, p, p, p, p, *shape, p, *rest, 1, 0.0, None, 0, None) in (1, 2)
    assert nat.lib.mat_selected_attn_bwd(p, p, p, p, p, p, p, p, p, *shape, p, *rest, 1, 0.0, None, 0, None) in (1, 2)
    if a["topk"] != 1:                       # the selection itself takes longer sequences
        assert nat.lib.mat_select_blocks_workspace_bytes(*shape, *rest) == 0
        assert nat.lib.mat_select_blocks(p, p, *shape, *rest, 1, p, None, 0, None) in (1, 2)
