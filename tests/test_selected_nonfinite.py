"""Block-selected attention where tokens hold infinities or NaN: pairs that do not see each other change nothing, pairs that
do get what the formula gives.  The plain form sums over the seen pairs only, row by row in 64 bits."""
import math

import pytest
import torch

from ma_transformer_b200 import selected_attention as sel
from test_selected_attention import inputs, mask_of, plain_select


def row_by_row(q, k, v, do, blocks, block, causal, E):
    """out, lse, dq, dk, dv and their allowances; E bounds the finite scores (sum |q k| scale)."""
    B, S, H, D = q.shape
    Hkv = k.shape[2]
    scale = 1 / math.sqrt(D)
    u = torch.finfo(q.dtype).eps / 2
    w = 0 if q.dtype == torch.float32 else u
    c = 2 * 2 * D * 2.0 ** -24 * E + 2.0 ** -18
    keep = mask_of(blocks, S, block, causal)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    want = [torch.zeros_like(q), torch.zeros(B, S, H).double(), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    tol = [torch.zeros_like(t) for t in want]
    for b in range(B):
        for h in range(H):
            n = h // (H // Hkv)
            for i in range(S):
                seen = keep[b, n, i].nonzero()[:, 0]
                x, y, kk, vv = q[b, i, h], do[b, i, h], k[b, seen, n], v[b, seen, n]
                s = kk @ x * scale
                P = torch.softmax(s, 0)
                o = P @ vv
                dS = P * (vv @ y - (y * o).sum())
                e = (w + c) * dS.abs() + P * (c * (vv.abs() @ y.abs()) + (u + c) * (y * o).abs().sum())
                for z, t, a, r in ((0, (b, i, h), o, u * o.abs() + (w + c) * (P @ vv.abs())), (1, (b, i, h), torch.logsumexp(s, 0), c * (1 + torch.logsumexp(s, 0).abs())),
                                   (2, (b, i, h), scale * dS @ kk, scale * e @ kk.abs()), (3, (b, seen, n), scale * dS[:, None] * x, scale * e[:, None] * x.abs()),
                                   (4, (b, seen, n), P[:, None] * y, (w + c) * P[:, None] * y.abs())):
                    want[z][t] += a
                    tol[z][t] += r
    return want, [t + (u * x.abs() if z >= 2 else 0) + 1e-30 for z, (x, t) in enumerate(zip(want, tol))]


def spoil(kind, q, k, v, do, blocks, block):
    nan, inf = float("nan"), float("inf")
    if "rows" not in kind:                    # the last tokens read their own block only
        blocks[:, 150:] = -1
        blocks[:, 150:, :, 0] = (torch.arange(150, q.shape[1]) // block).int()[None, :, None]
    if kind == "padding":                   # a batch whose last tokens were never filled
        for t in (q, k, v, do):
            t[:, 150:] = nan
    elif kind == "keys":
        k[:, 155, :, 3], k[:, 160, 0, 4], v[:, 165], v[:, 167, :, 2], k[:, 176] = inf, -inf, nan, inf, nan
    elif kind == "few rows":                # keys behind them in their block stay clean
        q[:, 130, 0], q[:, 133, 1, 2], do[:, 136, 0, 5], do[:, 137, 1, 6], do[:, 138, 1, 6] = nan, -inf, inf, inf, -inf
    else:                                   # queries and output gradients
        q[:, 130, 0], q[:, 150, 1, 2], do[:, 140, 0, 5], do[:, 145, 1, 6], do[:, 147, 1, 6], do[:, 160:, 0] = nan, inf, inf, -inf, inf, nan


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["padding", "keys", "rows", "few rows"])
@pytest.mark.parametrize("S, H, Hkv, D, block, topk, dtype", [
    (180, 4, 2, 64, 64, 2, torch.bfloat16),
    (180, 4, 2, 72, 64, 3, torch.float16),
    (200, 2, 2, 128, 128, 2, torch.bfloat16),           # two halves a block
    (180, 2, 1, 40, 16, 4, torch.bfloat16),             # few keys a row: delta from the tiles
    (200, 2, 1, 64, 96, 1, torch.float16),
    (180, 4, 2, 72, 64, 2, torch.float32),
    (200, 2, 1, 32, 112, 2, torch.float32)])
def test_pairs_that_do_not_see_each_other_change_nothing(S, H, Hkv, D, block, topk, dtype, kind):
    q, k, v, do = inputs(1, S, H, Hkv, D, dtype, seed=21)
    blocks = plain_select(q, k, block, topk, True)
    E = float((q.double().abs().transpose(1, 2) @ k.double().abs().repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)).max()) / math.sqrt(D)
    spoil(kind, q, k, v, do, blocks, block)
    want, tol = row_by_row(q, k, v, do, blocks, block, True, E)
    q, k, v, do, blocks = (t.cuda() for t in (q, k, v, do, blocks))
    out, lse = sel.forward_selected(q, k, v, blocks, block)
    got = [out, lse, *sel.backward_selected(q, k, v, out, lse, do, blocks, block)]
    for name, g, w, t in zip(("out", "lse", "dq", "dk", "dv"), got, want, tol):
        g, finite = g.cpu().double(), torch.isfinite(w)
        assert not finite.all() and (finite.any() or kind == "rows"), name        # in "rows" every key may be reached
        assert torch.equal(torch.isfinite(g), finite), f"{name}: {int((torch.isfinite(g) != finite).sum())} values"
        err = (g - w).abs().masked_fill(~finite, 0)
        assert (err <= t.masked_fill(~finite, 1)).all(), f"{name}: off by {float(err.max())}"


def choose(score, own, last, topk):
    """The own block and the best others of the first `last`, not-a-number scores last, equal ones by the lower index."""
    rank = sorted(range(last), key=lambda n: (n != own, math.isnan(score[n]), -score[n] if score[n] == score[n] else 0, n))[:topk]
    return sorted(rank) + [-1] * (topk - len(rank))


def block_scores(q, k, block, row):
    """Scores [Hkv, blocks] of one row by the definition, sum over heads and columns of max(q lo, q hi), in 64 bits."""
    S, Hkv = k.shape[1:3]
    parts = [k[0, n:n + block].double() for n in range(0, S, block)]
    lo, hi = torch.stack([x.amin(0) for x in parts], 1), torch.stack([x.amax(0) for x in parts], 1)        # [Hkv, blocks, D]
    heads = q[0, row].double().view(Hkv, -1, 1, q.shape[-1])
    return torch.maximum(heads * lo[:, None], heads * hi[:, None]).sum((1, 3))


def check_choice(q, k, block, topk, causal, rows):
    got = sel.select_blocks(q.cuda(), k.cuda(), block, topk, causal).cpu()
    nb = -(-k.shape[1] // block)
    for s in rows:
        score, own = block_scores(q, k, block, s).tolist(), s // block
        for h in range(k.shape[2]):
            assert got[0, s, h].tolist() == choose(score[h], own, own + 1 if causal else nb, topk), (s, h)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S, D, dtype", [(500, 64, torch.bfloat16), (500, 80, torch.float16), (500, 64, torch.float32), (16500, 8, torch.bfloat16)])
def test_blocks_with_a_key_that_is_not_a_number_are_chosen_last(S, D, dtype, causal):
    """One NaN in a block of keys makes its score NaN, whichever token, head or column holds it; the own block stays in."""
    q, k, _, _ = inputs(1, S, 4, 2, D, dtype, seed=22)
    k[0, 3, 0, 5], k[0, 47, 1, D - 1], k[0, 111, :, 0], k[0, S - 1, 0, 1] = float("nan"), -float("nan"), float("nan"), float("nan")
    k[0, 200:232] = float("nan")
    k[0, [3, 47, 111]] *= 4                               # without the NaN these blocks would be high
    rows = list(range(0, 240, 3)) + [S - 17, S - 2, S - 1]
    for topk in (4, 15):
        check_choice(q, k, 16, topk, causal, rows)
    if S < 1000:
        check_choice(q, k, 16, 40, causal, rows)          # more places than blocks that are numbers


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S, H, D, dtype", [(500, 2, 64, torch.bfloat16), (500, 6, 80, torch.float16), (500, 4, 64, torch.float32), (16500, 2, 8, torch.bfloat16)])
def test_blocks_with_infinite_keys_score_by_the_definition(S, H, D, dtype, causal):
    """An infinite bound counts for the heads whose sign takes it, and is not a number for a query of zero."""
    q, k, _, _ = inputs(1, S, H, 2, D, dtype, seed=23)
    inf = float("inf")
    k[0, 3, 0, 5], k[0, 47, 1, D - 1], k[0, 111, :, 0], k[0, 150, 0, 3], k[0, 151, 0, 3], k[0, 200:232, :, 6] = inf, -inf, inf, inf, -inf, -inf
    q[0, ::7, :, 5] = 0
    q[0, 1::7, 0, 6] = 0
    rows = list(range(0, 240, 3)) + [S - 17, S - 2, S - 1]
    for topk in (3, 14):
        check_choice(q, k, 16, topk, causal, rows)
