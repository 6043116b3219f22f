"""Page selection beside the forms that the paged attention's own tests reach: batches that fill the GPU, keys that are not
numbers."""
import math

import pytest
import torch

import ma_transformer_b200 as mt
from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import paged_attention as paged


def choose(score, own, topk):
    """The own page and the best others, not-a-number scores last, equal ones by the lower index."""
    rank = sorted(range(len(score)), key=lambda n: (n != own, math.isnan(score[n]), -score[n] if score[n] == score[n] else 0, n))[:topk]
    return sorted(rank) + [-1] * (topk - len(rank))


def scores(q, kb, pages, h, G):
    """By the definition, sum over heads and columns of max(q lo, q hi), in 64 bits."""
    lo, hi = kb[pages, 0, h].double(), kb[pages, 1, h].double()
    return sum(torch.maximum(r * lo, r * hi) for r in q[h * G:(h + 1) * G].double()).sum(-1).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 72), (torch.float32, 64), (torch.float32, 256)])
def test_keys_that_are_not_numbers_make_their_page_the_last_choice(dtype, D):
    """Appended one by one and as a prompt: a page's bounds are NaN in the columns where a key is."""
    N, H, Hkv, page, topk = 400, 4, 2, 16, 5
    g = torch.Generator().manual_seed(31)
    q, k, v = (torch.randn(N, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv))
    k[3, 0, 5], k[47, 1, D - 1], k[111, :, 0], k[200:232] = float("nan"), -float("nan"), float("nan"), float("nan")
    k[[3, 47, 111]] *= 4
    table = torch.randperm(25, generator=g).to(torch.int32)
    at = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    caches = [mt.PagedKVCache(25, page, Hkv, D, dtype, key_bounds=True) for _ in range(2)]
    kd, vd, td = k.cuda(), v.cuda(), table.cuda()[None]
    paged.append(caches[0], kd, vd, td, at(0), cu_seqlens=torch.tensor([0, N], dtype=torch.int32, device="cuda"))
    for i in range(N):
        paged.append(caches[1], kd[i:i + 1], vd[i:i + 1], td, at(i))
    held = k.view(25, page, Hkv, D)
    want = torch.full((25, 2, Hkv, D), 7.0, dtype=dtype)
    want[table.long(), 0], want[table.long(), 1] = held.float().amin(1).to(dtype), held.float().amax(1).to(dtype)
    for cache in caches:
        assert torch.equal(cache.key_bounds.cpu().isnan(), want.isnan()) and torch.equal(cache.key_bounds.cpu().nan_to_num(9), want.nan_to_num(9))
        for n in (130, 215, 400):
            for topk in (5, 23):
                pages = paged.select_pages(q[n - 1:n].cuda(), cache, td, at(n), topk).cpu()
                used = table[:-(-n // page)].long()
                for h in range(Hkv):
                    assert pages[0, h].tolist() == choose(scores(q[n - 1], want, used, h, H // Hkv), len(used) - 1, topk), (n, h, topk)
    assert nat.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, H, D", [(torch.bfloat16, 2, 64), (torch.float32, 6, 64)])
def test_pages_with_infinite_keys_score_by_the_definition(dtype, H, D):
    """An infinite bound counts for the heads whose sign takes it, and is not a number for a query of zero."""
    B, n_pages, page, Hkv = 4, 40, 8, 2
    g = torch.Generator().manual_seed(32)
    kb = torch.randn(n_pages, 2, Hkv, D, generator=g).sort(1).values.to(dtype)
    kb[3, 1, 0, 5], kb[7, 0, 1, 2], kb[9, 0, :, 4], kb[9, 1, :, 4], kb[20, 0, :, 1] = math.inf, -math.inf, -math.inf, math.inf, -math.inf
    q = torch.randn(B, H, D, generator=g).to(dtype)
    q[0, :, 5], q[1, 0, 4] = 0, 0
    k = torch.zeros(n_pages, page, Hkv, D, dtype=dtype, device="cuda")
    cache = mt.PagedKVCache.from_tensors(k, k.clone(), key_bounds=kb.cuda())
    table = torch.stack([torch.randperm(n_pages, generator=g) for _ in range(B)])
    n = torch.full((B,), n_pages * page, dtype=torch.int32)
    for topk in (2, 6, 38):
        pages = paged.select_pages(q.cuda(), cache, table.int().cuda(), n.cuda(), topk).cpu()
        for b in range(B):
            for h in range(Hkv):
                assert pages[b, h].tolist() == choose(scores(q[b], kb, table[b], h, H // Hkv), n_pages - 1, topk), (b, h, topk)
    assert nat.device_status() == 0


# Batches of 148 and more (sequence, key head) rows are scored and selected by one CTA a row; fewer rows are scored by all
# CTAs first.  Both are held to the definition, at every width that has a kernel of its own.

def serving_batch(lengths, H, Hkv, D, page, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lengths]
    n_pages = sum(used) + 1
    kb = torch.randn(n_pages, 2, Hkv, D, generator=g).sort(1).values.to(dtype)
    table = torch.full((len(lengths), max(used) + 2), -5, dtype=torch.int32)
    ids = torch.randperm(n_pages, generator=g).tolist()
    for b, n in enumerate(used):
        for w in range(n):
            table[b, w] = ids.pop()
    return kb, table, torch.randn(len(lengths), H, D, generator=g).to(dtype)


def check_pages(lengths, H, Hkv, page, kb, table, q, topks):
    k = torch.zeros(kb.shape[0], page, Hkv, kb.shape[3], dtype=kb.dtype, device="cuda")
    cache = mt.PagedKVCache.from_tensors(k, k, key_bounds=kb.cuda())
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = [[scores(q[b], kb, table[b, :-(-m // page)].long(), h, H // Hkv) for h in range(Hkv)] for b, m in enumerate(lengths)]
    for topk in topks:
        pages = paged.select_pages(q.cuda(), cache, table.cuda(), n, topk).cpu()
        for b, m in enumerate(lengths):
            for h in range(Hkv):
                assert pages[b, h].tolist() == choose(want[b][h], (m - 1) // page, topk), (b, h, topk)
    assert nat.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["many", "few"])
@pytest.mark.parametrize("D, dtype", [(8, torch.bfloat16), (32, torch.float16), (64, torch.bfloat16), (72, torch.float16), (128, torch.bfloat16), (200, torch.float16),
                                      (256, torch.bfloat16), (16, torch.float32), (24, torch.float32), (64, torch.float32), (80, torch.float32), (128, torch.float32),
                                      (256, torch.float32)])
def test_select_pages_of_batches(D, dtype, rows):
    """Mixed lengths, idle slots and single tokens among them."""
    lengths = [0, 1, 8, 9, 1500, 777, 64, 333, 2, 1201] * (4 if rows == "many" else 1)
    kb, table, q = serving_batch(lengths, 8, 4, D, 8, dtype, D)
    check_pages(lengths, 8, 4, 8, kb, table, q, (1, 4, 33))


@pytest.mark.gpu
@pytest.mark.parametrize("B, H, Hkv", [(150, 1, 1), (19, 40, 8)])
def test_select_pages_of_batches_with_equal_bounds_and_bounds_that_are_not_numbers(B, H, Hkv):
    lengths, page, D = [40 * 16 + (b % 3) * 16 - b % 5 for b in range(B)], 16, 64
    kb, table, q = serving_batch(lengths, H, Hkv, D, page, torch.bfloat16, 50)
    for b in range(B):
        at = table[b, :38].long()
        kb[at[5:38]] = kb[at[5]].clone()                  # 33 equal pages
        kb[at[b % 5], b % 2, b % Hkv, b % D] = float("nan")
        if b % 7 == 0:
            kb[at[3:30], 0] = float("nan")
    check_pages(lengths, H, Hkv, page, kb, table, q, (1, 2, 7, 36, 39, 60))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 150])
def test_select_pages_where_more_pages_are_near_than_are_held(B):
    """1500 pages whose bounds differ in one column's last bit: fp32 sums cannot tell them apart."""
    page, D, n_pages = 8, 64, 1500
    g = torch.Generator().manual_seed(51)
    kb = (torch.randn(1, 1, 1, D, generator=g).bfloat16() * 8).expand(n_pages, 2, 1, D).contiguous()
    for p in range(n_pages):
        x = kb[p, 1, 0, (p * 7) % D].float()
        kb[p, 1, 0, (p * 7) % D] = (x + x.abs() * torch.finfo(torch.bfloat16).eps).bfloat16()
    q = torch.randn(B, 2, D, generator=g).bfloat16() * 1e-3
    q[..., 0] = 30
    lengths = [n_pages * page - b for b in range(B)]      # the table is shared: the same pages for every sequence
    table = torch.randperm(n_pages, generator=g).int()[None].expand(B, n_pages).contiguous()
    check_pages(lengths, 2, 1, page, kb, table, q, (5, 40) if B > 1 else (1, 5, 40, 1200))
