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


@pytest.mark.parametrize("dtype", [nat.MAT_BF16, nat.MAT_F32])
@pytest.mark.parametrize("B, S, H, Hkv, D, block, topk", [
    (64, 2000, 16, 16, 128, 16, 1), (64, 2000, 16, 16, 128, 16, 4), (8, 8192, 32, 32, 128, 16, 1), (1, 2 ** 20, 8, 8, 64, 16, 2),
    (2, 4096, 64, 8, 128, 128, 8), (1, 131072, 4, 1, 128, 64, 16), (1, 100, 4, 2, 64, 16, 3), (4000, 64, 16, 16, 64, 64, 1)])
def test_workspaces_hold_1_gib_of_pairs_at_most(B, S, H, Hkv, D, block, topk, dtype):
    """Or one (batch, key head) pair where that takes more; the backward holds 4 bytes a row beside it."""
    for size, rest in ((nat.lib.mat_selected_attn_fwd_workspace_bytes, 0), (nat.lib.mat_selected_attn_bwd_workspace_bytes, 4 * B * S * H)):
        one = size(1, S, H // Hkv, 1, D, dtype, block, topk)
        assert one <= size(B, S, H, Hkv, D, dtype, block, topk) <= max(1 << 30, one) + rest + 8192


@pytest.mark.gpu
@pytest.mark.parametrize("B, S, H, Hkv, D, block, topk, dtype", [
    (1, 2048, 100, 100, 128, 32, 16, torch.bfloat16),
    (2, 4096, 200, 200, 64, 16, 1, torch.float16),          # delta from the tiles
    (1, 2048, 320, 160, 64, 96, 8, torch.float32)])
def test_groups_of_pairs_give_the_bits_of_their_parts(B, S, H, Hkv, D, block, topk, dtype):
    """Pairs that do not fit the workspace together go one group after the other, the last one short."""
    g = torch.Generator(device="cuda").manual_seed(41)
    q, do = (torch.randn(B, S, H, D, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    k, v = (torch.randn(B, S, Hkv, D, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    blocks = sel.select_blocks(q, k, block, topk)
    out, lse = sel.forward_selected(q, k, v, blocks, block)
    whole = (out, *sel.backward_selected(q, k, v, out, lse, do, blocks, block), lse)
    dt = {torch.bfloat16: nat.MAT_BF16, torch.float16: nat.MAT_F16, torch.float32: nat.MAT_F32}[dtype]
    size = nat.lib.mat_selected_attn_bwd_workspace_bytes
    part, G = 20, H // Hkv
    assert size(B, S, H, Hkv, D, dt, block, topk) < B * Hkv / part * size(1, S, part * G, part, D, dt, block, topk) - (64 << 20)      # groups
    assert size(1, S, part * G, part, D, dt, block, topk) > part * 0.9 * size(1, S, G, 1, D, dt, block, topk)          # one group
    for b in range(B):
        for h in list(range(0, Hkv, 3 * part)) + [Hkv - part]:
            cut = lambda t, n: t[b:b + 1, :, h * n:(h + part) * n].contiguous()  # noqa: E731
            x, y, kk, vv, bl = cut(q, G), cut(do, G), cut(k, 1), cut(v, 1), cut(blocks, 1)
            assert torch.equal(sel.select_blocks(x, kk, block, topk), bl)
            o, l = sel.forward_selected(x, kk, vv, bl, block)
            mine = (o, *sel.backward_selected(x, kk, vv, o, l, y, bl, block), l)
            for name, a, c, n in zip(("out", "dq", "dk", "dv", "lse"), whole, mine, (G, G, 1, 1, G)):
                assert torch.equal(cut(a, n), c), (name, b, h)
