"""Block-selected attention and its gradients against plain 64-bit code.

Tolerances count roundings, u half a step of the element type (finfo.eps / 2), P the weights, E = max sum |q k| scale:
  c = 2 * 2 D 2^-24 E + 2^-18        fp32 scores on both sides of exp(s - lse), the exponential, the sums
  out  u |out| + (w + c) P |v|       w = u where the weights are rounded for the tensor cores (16-bit types), else 0
  dv   u |dv|  + (w + c) P^T |do|
  dS   e = (w + c) |dS| + P (c |do| |v|^T + (u + c) |do| . |o|)     (delta comes from the rounded output)
  dq   u |dq|  + scale e |k|,  dk  u |dk| + scale e^T |q|
A sum of fp32 terms adds n 2^-24 of its absolute terms; n <= 4096 here: 2^-12 of it would be far off, but partial sums of
at most 128 terms join in pairs of chunks, and c's 2^-18 covers 64 roundings of 2^-24; fp32 cases stay below 700 keys a
row, and errors of rounding to nearest grow with the square root of n.
"""
import math

import pytest
import torch

import ma_transformer_b200 as mt
from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import paged_attention as paged
from ma_transformer_b200 import selected_attention as sel


def inputs(B, S, H, Hkv, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, S, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv, H))


def plain_select(q, k, block, topk, causal):
    """By the definition, in 64 bits, row by row of blocks."""
    B, S, H, D = q.shape
    Hkv = k.shape[2]
    nb = -(-S // block)
    lo = torch.stack([k[:, n * block:(n + 1) * block].double().amin(1) for n in range(nb)], 1)     # [B, nb, Hkv, D]
    hi = torch.stack([k[:, n * block:(n + 1) * block].double().amax(1) for n in range(nb)], 1)
    qg = q.double().view(B, S, Hkv, H // Hkv, D)
    score = torch.einsum("bshd,bnhd->bshn", qg.clamp(min=0).sum(3), hi) + torch.einsum("bshd,bnhd->bshn", qg.clamp(max=0).sum(3), lo)
    own = torch.arange(S) // block
    n = torch.arange(nb)
    if causal:
        score = score.masked_fill((n > own[:, None])[None, :, None], -math.inf)
    score.scatter_(3, own.view(1, S, 1, 1).expand(B, S, Hkv, 1), math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    index = torch.where(order.values[..., :topk] > -math.inf, order.indices[..., :topk], nb).sort(-1).values
    index = torch.nn.functional.pad(index, (0, max(0, topk - nb)), value=nb)
    return torch.where(index < nb, index, -1).int().contiguous()


def mask_of(blocks, S, block, causal):
    """[B, Hkv, S, S] truth values of the pairs that the lists give, entry by entry."""
    B, _, Hkv, T = blocks.shape
    nb = -(-S // block)
    keep = torch.zeros(B, Hkv, S, nb, dtype=torch.bool)
    rows = blocks.permute(0, 2, 1, 3).long()
    prev = torch.full(rows.shape[:3], -1)
    own = (torch.arange(S) // block)[None, None]
    for t in range(T):
        n = rows[..., t]
        counts = (n > prev) & (n < nb) & ((n <= own) if causal else True)
        prev = torch.maximum(prev, n)
        keep.scatter_(3, torch.where(counts, n, 0)[..., None], counts[..., None] | keep.gather(3, torch.where(counts, n, 0)[..., None]))
    keep = keep.repeat_interleave(block, 3)[..., :S]
    if causal:
        keep &= torch.ones(S, S, dtype=torch.bool).tril()
    return keep


def reference(q, k, v, do, blocks, block, causal, scale=None):
    """out, lse, dq, dk, dv in 64 bits and the allowance of each."""
    dtype, (B, S, H, D) = q.dtype, q.shape
    Hkv, G = k.shape[2], H // k.shape[2]
    scale = scale or 1 / math.sqrt(D)
    keep = mask_of(blocks, S, block, causal)[:, :, None]
    q, do = (t.double().view(B, S, Hkv, G, D).permute(0, 2, 3, 1, 4) for t in (q, do))
    k, v = (t.double().transpose(1, 2)[:, :, None] for t in (k, v))
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(s, -1)
    P = torch.where(keep, torch.exp(s - lse.masked_fill(lse == -math.inf, 0)[..., None]), 0.0)
    out = P @ v
    dP = do @ v.transpose(-1, -2)
    dS = P * (dP - (do * out).sum(-1, keepdim=True))
    dq, dk, dv = dS @ k * scale, (dS.transpose(-1, -2) @ q * scale).sum(2), (P.transpose(-1, -2) @ do).sum(2)
    u = torch.finfo(dtype).eps / 2
    w = 0 if dtype == torch.float32 else u
    E = float((q.abs() @ k.abs().transpose(-1, -2)).max()) * scale
    c = 2 * 2 * D * 2.0 ** -24 * E + 2.0 ** -18
    e = (w + c) * dS.abs() + P * (c * (do.abs() @ v.abs().transpose(-1, -2)) + (u + c) * (do * out).abs().sum(-1, keepdim=True))
    tol = (u * out.abs() + (w + c) * (P @ v.abs()), c * (1 + lse.abs()) , u * dq.abs() + scale * (e @ k.abs()),
           u * dk.abs() + scale * (e.transpose(-1, -2) @ q.abs()).sum(2), u * dv.abs() + (w + c) * (P.transpose(-1, -2) @ do.abs()).sum(2))
    rows = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, S, H, D)  # noqa: E731
    flat = lambda t: t.permute(0, 3, 1, 2).reshape(B, S, H)  # noqa: E731
    swap = lambda t: t.transpose(1, 2)  # noqa: E731
    f = (rows, flat, rows, swap, swap)
    return [g(t) for g, t in zip(f, (out, lse, dq, dk, dv))], [g(t) for g, t in zip(f, tol)]


def check(got, want, tol, names=("out", "lse", "dq", "dk", "dv")):
    for name, g, w, t in zip(names, got, want, tol):
        g = g.cpu().double()
        dead = w == -math.inf
        assert (g[dead] == -math.inf).all(), name
        err = (g - w).abs().masked_fill(dead, 0)
        t = t.masked_fill(dead, 1) + 1e-30
        assert not (~(err <= t)).any(), f"{name}: off by {float(err.max())}, {float((err / t).max())} of what is allowed"


def run_all(q, k, v, do, blocks, block, causal, scale=None):
    q, k, v, do, blocks = (t.cuda() for t in (q, k, v, do, blocks))
    out, lse = sel.forward_selected(q, k, v, blocks, block, causal, scale)
    return [out, lse, *sel.backward_selected(q, k, v, out, lse, do, blocks, block, causal, scale)]


CASES = [
    # B, S, H, Hkv, D, block, topk, causal, dtype
    (1, 1, 1, 1, 64, 16, 1, True, torch.bfloat16),
    (2, 100, 2, 2, 32, 16, 3, True, torch.float32),
    (1, 257, 4, 2, 64, 64, 2, True, torch.bfloat16),
    (1, 300, 4, 1, 64, 32, 4, False, torch.float16),
    (2, 130, 6, 3, 80, 16, 20, True, torch.float32),
    (1, 640, 8, 1, 128, 128, 2, True, torch.bfloat16),
    (1, 333, 3, 3, 128, 48, 3, False, torch.bfloat16),
    (1, 500, 2, 2, 8, 16, 5, True, torch.float16),
    (1, 260, 5, 1, 24, 112, 2, True, torch.float32),
    (1, 1100, 2, 1, 64, 16, 40, False, torch.bfloat16),
    (3, 64, 2, 2, 96, 64, 1, True, torch.float16),
    (1, 2100, 1, 1, 64, 64, 6, True, torch.bfloat16),
    (1, 700, 16, 1, 72, 64, 3, True, torch.bfloat16),
    (2, 500, 4, 2, 64, 16, 1, True, torch.bfloat16),
    (1, 553, 2, 1, 128, 128, 1, True, torch.bfloat16),
    (1, 400, 6, 2, 40, 32, 2, False, torch.float16),
    (1, 300, 2, 1, 128, 96, 1, False, torch.float16),
]


# ---- refusals (no GPU needed) ------------------------------------------------------------------------------

@pytest.mark.parametrize("change", [dict(B=0), dict(S=0), dict(H=3), dict(Hkv=0), dict(D=20), dict(D=136), dict(dtype=9), dict(block=8), dict(block=24),
                                    dict(block=256), dict(topk=0), dict(topk=2000), dict(B=70000), dict(q=0), dict(q=8), dict()])
def test_refusals(change):
    a = dict(B=1, S=64, H=4, Hkv=2, D=64, dtype=nat.MAT_BF16, block=16, topk=2, q=256)
    a.update(change)
    shape = (a["B"], a["S"], a["H"], a["Hkv"], a["D"], a["dtype"])
    p, q = 256, a["q"] or None
    codes = (nat.lib.mat_select_blocks(q, p, *shape, a["block"], a["topk"], 1, p, None, 0, None),
             nat.lib.mat_selected_attn_bwd(q, p, p, p, p, p, p, p, p, *shape, p, a["block"], a["topk"], 1, 0.0, None, 0, None))
    want = {4} if not change else {1, 2}
    assert set(codes) <= want and nat.lib.mat_last_error()
    if change:
        assert nat.lib.mat_selected_attn_fwd(q, p, p, p, p, *shape, p, a["block"], a["topk"], 1, 0.0, None, 0, None) in (1, 2)
    if change and "q" not in change:
        assert nat.lib.mat_select_blocks_workspace_bytes(*shape, a["block"], a["topk"]) == 0
        assert nat.lib.mat_selected_attn_bwd_workspace_bytes(*shape, a["block"], a["topk"]) == 0


def test_host_tensors_are_refused():
    q, k, v, _ = inputs(1, 32, 2, 2, 64, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sel.select_blocks(q, k, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        sel.selected_block_attention(q, k, v, 16, 2)


# ---- selection ----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_select_blocks(case):
    B, S, H, Hkv, D, block, topk, causal, dtype = case
    q, k, _, _ = inputs(B, S, H, Hkv, D, dtype)
    got = sel.select_blocks(q.cuda(), k.cuda(), block, topk, causal).cpu()
    assert torch.equal(got, plain_select(q, k, block, topk, causal))


@pytest.mark.gpu
def test_selection_of_equal_scores_takes_the_lower_block():
    S, block = 1600, 16
    q = torch.ones(1, S, 2, 64, dtype=torch.bfloat16)
    k = torch.ones(1, S, 1, 64, dtype=torch.bfloat16)
    k[:, 70 * block:71 * block] = 2
    for causal in (True, False):
        got = sel.select_blocks(q.cuda(), k.cuda(), block, 5, causal).cpu()
        assert torch.equal(got, plain_select(q, k, block, 5, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("S, Hkv, dtype", [(20000, 1, torch.float32), (20000, 1, torch.bfloat16), (16384, 4, torch.bfloat16), (6000, 2, torch.float16)])
@pytest.mark.parametrize("causal", [True, False])
def test_selection_of_many_blocks(S, Hkv, dtype, causal):
    """More blocks than one warp's registers hold, more score rows than are held at a time, every width of row."""
    q, k, _, _ = inputs(1, S, 2 * Hkv, Hkv, 16, dtype)
    got = sel.select_blocks(q.cuda(), k.cuda(), 16, 7, causal).cpu()
    nb = S // 16
    kb = k[0].double().view(nb, 16, Hkv, 16)
    lo, hi = kb.amin(1), kb.amax(1)
    for s in (0, 15, 16, 111, 112, 2047, 2048, 5000, 5999, S // 2, S - 17, S - 1):
        if s >= S:
            continue
        for h in range(Hkv):
            row = q[0, s, 2 * h:2 * h + 2].double()
            score = (row.clamp(min=0).sum(0) * hi[:, h] + row.clamp(max=0).sum(0) * lo[:, h]).sum(-1)
            own = s // 16
            last = own + 1 if causal else nb
            rank = sorted(range(last), key=lambda n: (n != own, -float(score[n]), n))[:7]
            assert got[0, s, h].tolist() == sorted(rank) + [-1] * (7 - len(rank)), (s, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_nearer_than_their_fp32_error_are_ordered_in_64_bits(dtype):
    """Blocks whose bounds differ in one column's last bit: fp32 sums cannot tell most of them apart."""
    S, block, D = 1280, 16, 64
    g = torch.Generator().manual_seed(11)
    k = torch.randn(1, 1, 1, D, generator=g).to(dtype).expand(1, S, 1, D).contiguous() * 8
    for n in range(S // block):                           # one element of a block a step larger, another column each
        c = (n * 7) % D
        x = k[0, n * block, 0, c].float()
        k[0, n * block, 0, c] = (x + x.abs() * torch.finfo(dtype).eps).to(dtype)
    q = torch.randn(1, S, 2, D, generator=g).to(dtype) * 1e-3
    q[..., 0] = 30
    got = sel.select_blocks(q.cuda(), k.cuda(), block, 9, True).cpu()
    assert torch.equal(got, plain_select(q, k, block, 9, True))


# ---- attention and gradients --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(case):
    B, S, H, Hkv, D, block, topk, causal, dtype = case
    q, k, v, do = inputs(B, S, H, Hkv, D, dtype, seed=1)
    blocks = plain_select(q, k, block, topk, causal)
    want, tol = reference(q, k, v, do, blocks, block, causal)
    check(run_all(q, k, v, do, blocks, block, causal), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_lists_of_any_content(dtype, causal):
    """Rows without a block, repeated entries, entries out of order, behind the query or outside the sequence."""
    B, S, H, Hkv, D, block = 1, 200, 4, 2, 64, 32
    q, k, v, do = inputs(B, S, H, Hkv, D, dtype, seed=2)
    g = torch.Generator().manual_seed(4)
    blocks = torch.randint(-3, 10, (B, S, Hkv, 6), generator=g).int()
    blocks[:, 3:9] = -1
    blocks[:, 50, :, 0] = 2 ** 31 - 1
    blocks[:, 51, :, 0] = -2 ** 31
    want, tol = reference(q, k, v, do, blocks, block, causal, scale=0.21)
    got = run_all(q, k, v, do, blocks, block, causal, scale=0.21)
    check(got, want, tol)
    assert (got[0][:, 3:9] == 0).all() and (got[2][:, 3:9] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_block_that_nobody_chose_gets_zero_gradients_and_everybodys_choice_all_of_them(dtype):
    B, S, H, Hkv, D, block = 1, 2000, 2, 1, 64, 64
    q, k, v, do = inputs(B, S, H, Hkv, D, dtype, seed=3)
    blocks = torch.zeros(B, S, Hkv, 2, dtype=torch.int32)
    blocks[..., 1] = -1
    want, tol = reference(q, k, v, do, blocks, block, False)
    got = run_all(q, k, v, do, blocks, block, False)
    check(got, want, tol)
    assert (got[3][:, block:] == 0).all() and (got[4][:, block:] == 0).all()


@pytest.mark.gpu
def test_large_scores_stay_finite():
    q, k, v, do = inputs(1, 150, 2, 2, 64, torch.float32, seed=5)
    q = q * 200
    blocks = plain_select(q, k, 16, 4, True)
    got = run_all(q, k, v, do, blocks, 16, True)
    assert all(torch.isfinite(t).all() for t in got)
    want, tol = reference(q, k, v, do, blocks, 16, True)
    check(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_keys_behind_the_query_may_hold_anything(dtype):
    """Padded tokens behind a row, infinite or not a number, change nothing for it, in the row's own block or later ones;
    rows that see them get what the formula gives."""
    B, S, H, Hkv, D, block = 1, 180, 4, 2, 72, 64
    q, k, v, do = inputs(B, S, H, Hkv, D, dtype, seed=10)
    blocks = plain_select(q, k, block, 2, True)
    want, tol = reference(q, k, v, do, blocks, block, True)
    k[:, 150:], v[:, 151], v[:, 152, :, 5], v[:, 160:] = float("nan"), float("nan"), float("inf"), -float("inf")
    out, lse = sel.forward_selected(*(t.cuda() for t in (q, k, v, blocks)), block)
    check([out[:, :150], lse[:, :150]], [w[:, :150] for w in want[:2]], [t[:, :150] for t in tol[:2]], ("out", "lse"))
    assert torch.isnan(out[:, 150:]).all()
    k = inputs(B, S, H, Hkv, D, dtype, seed=10)[1]
    out, _ = sel.forward_selected(*(t.cuda() for t in (q, k, v, blocks)), block)
    assert torch.isfinite(out[:, :151]).all() and torch.isnan(out[:, 151:153]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [CASES[2], CASES[4]], ids=str)
def test_the_same_every_time_in_graphs_and_on_another_stream(case):
    B, S, H, Hkv, D, block, topk, causal, dtype = case
    q, k, v, do = (t.cuda() for t in inputs(B, S, H, Hkv, D, dtype, seed=6))

    def step():
        blocks = sel.select_blocks(q, k, block, topk, causal)
        out, lse = sel.forward_selected(q, k, v, blocks, block, causal)
        return [blocks, out, lse, *sel.backward_selected(q, k, v, out, lse, do, blocks, block, causal)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    runs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        runs.append((graph, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for (graph, _), s in zip(runs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, res in runs:
        assert all(torch.equal(a, b) for a, b in zip(want, res))


@pytest.mark.gpu
def test_gradients_through_autograd_and_against_differences():
    B, S, H, Hkv, D, block, topk = 1, 70, 4, 2, 32, 16, 3
    q, k, v, do = inputs(B, S, H, Hkv, D, torch.float32, seed=7)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out = mt.selected_block_attention(*leaves, block, topk)
    out.backward(do.cuda())
    blocks = plain_select(q, k, block, topk, True)
    want, tol = reference(q, k, v, do, blocks, block, True)
    check([out.detach(), *(t.grad for t in leaves)], [want[0], *want[2:]], [tol[0], *tol[2:]], ("out", "dq", "dk", "dv"))
    # differences of the 64-bit formula with the lists held: a direction's slope is the gradient's product with it
    g = torch.Generator().manual_seed(8)
    for i in range(3):
        d = torch.randn((q, k, v)[i].shape, generator=g).double()
        at = lambda e: [t.double() + (e * d if j == i else 0) for j, t in enumerate((q, k, v))]  # noqa: E731
        loss = lambda e: float((reference(*at(e), do.double(), blocks, block, True)[0][0] * do.double()).sum())  # noqa: E731
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        product = float((leaves[i].grad.cpu().double() * d).sum())
        # the gradient's own allowance along d, and (1e-5)^2 of the third derivative (of the order of the slope's terms)
        assert abs(slope - product) <= float((tol[2 + i] * d.abs()).sum()) + 1e-6 * (1 + abs(slope))


@pytest.mark.gpu
def test_autograd_of_views_and_of_some_inputs():
    x = torch.randn(1, 80, 3, 2, 64, device="cuda", dtype=torch.bfloat16)
    q, k, v = (x[:, :, i] for i in range(3))             # strided views
    k = k.detach().requires_grad_(True)
    out = mt.selected_block_attention(q, k, v, 16, 2)
    out.sum().backward()                                 # an expanded gradient
    c = [t.detach().contiguous() for t in (q, k, v)]
    blocks = sel.select_blocks(c[0], c[1], 16, 2)
    o, lse = sel.forward_selected(*c, blocks, 16)
    _, dk, _ = sel.backward_selected(*c, o, lse, torch.ones_like(o), blocks, 16)
    assert torch.equal(o, out.detach()) and torch.equal(dk, k.grad)


# ---- together -----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_served_one_by_one_read_what_the_sequence_reads(dtype):
    """A prompt appended to a paged cache and further tokens one at a time: each new token's pages and output are the
    last row's of the whole sequence with blocks of the page's size."""
    S, prompt, H, Hkv, D, page, topk = 150, 130, 4, 2, 64, 16, 4
    q, k, v, _ = (t.cuda() for t in inputs(1, S, H, Hkv, D, dtype, seed=9))
    f = mt.rotary_frequencies(D)
    cache = mt.PagedKVCache(12, page, Hkv, D, dtype, key_bounds=True)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()[None]
    at = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    q_rot = [paged.append(cache, k[0, :prompt], v[0, :prompt], table, at(0), query=q[0, :prompt], inv_freq=f,
                          cu_seqlens=torch.tensor([0, prompt], dtype=torch.int32, device="cuda"))]
    for i in range(prompt, S):
        qi = paged.append(cache, k[0, i:i + 1], v[0, i:i + 1], table, at(i), query=q[0, i:i + 1], inv_freq=f)
        q_rot.append(qi)
        pages = paged.select_pages(qi, cache, table, at(i + 1), topk)
        out = paged.decode(qi, cache, table, at(i + 1), pages=pages)
        n = i + 1
        held = table[0, :-(-n // page)].long()
        keys, values = (x[held].flatten(0, 1)[None, :n].contiguous() for x in (cache.k, cache.v))
        queries = torch.cat(q_rot)[None].contiguous()
        blocks = sel.select_blocks(queries, keys, page, topk)
        assert torch.equal(blocks[0, -1], pages[0])
        if i % 7 == 0:
            want, tol = reference(queries.cpu(), keys.cpu(), values.cpu(), torch.zeros_like(queries).cpu(), blocks.cpu(), page, True)
            assert ((out[0].cpu().double() - want[0][0, -1]).abs() <= tol[0][0, -1]).all()
            whole, _ = sel.forward_selected(queries, keys, values, blocks, page)
            assert ((whole[0, -1].cpu().double() - want[0][0, -1]).abs() <= tol[0][0, -1]).all()
    assert nat.device_status() == 0
