"""Extremes of the paged calls' arguments."""
import ctypes as C

import pytest
import torch

import ma_transformer_b200 as mt
from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import paged_attention as paged
from test_paged_attention import _decode, _struct


@pytest.mark.parametrize("left", [2 ** 63 - 1, 2 ** 63 - 16, 2 ** 62])
@pytest.mark.parametrize("B, width", [(1, 40), (2, 1 << 16), (300, 512)])
def test_a_window_wider_than_any_sequence_plans_for_the_whole_cache(left, B, width):
    s, _ = _struct()
    size = lambda taps: nat.lib.mat_paged_decode_workspace_bytes(C.byref(s), B, 4, width, taps, 0)  # noqa: E731
    assert size(left) == size(-1) == size(width * 16)


@pytest.mark.parametrize("n_sel", [2 ** 27, 2 ** 59, 2 ** 60, 2 ** 63 - 1])
def test_a_list_of_more_pages_than_32_bits_of_tokens_is_refused(n_sel):
    s, base = _struct()
    assert nat.lib.mat_paged_decode_workspace_bytes(C.byref(s), 2, 4, 3, -1, n_sel) == 0
    assert _decode(s, base, pages=base, n_sel=n_sel) == 1 and b"list of pages" in nat.lib.mat_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_more_sequences_than_a_block_holds_in_place(dtype):
    """1500 sequences of 0 to 3 new tokens (their ranges are searched in memory), queries turned in place."""
    B, page, Hkv, H, D = 1500, 8, 1, 2, 64
    g = torch.Generator().manual_seed(61)
    new = torch.randint(0, 4, (B,), generator=g)
    start = torch.randint(0, 14, (B,), generator=g)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)])
    N = int(cu[-1])
    q, k, v = (torch.randn(N + 5, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv))
    table = torch.randperm(3 * B, generator=g).view(B, 3)
    cache = mt.PagedKVCache(3 * B, page, Hkv, D, dtype, key_bounds=True)
    before = [t.clone() for t in (cache.k, cache.v)]
    i32 = lambda t: t.to(torch.int32).cuda()  # noqa: E731
    dq = q.cuda()
    freq = mt.rotary_frequencies(D)
    got = paged.append(cache, k.cuda(), v.cuda(), i32(table), i32(start), cu_seqlens=i32(cu), query=dq, query_out=dq, inv_freq=freq)
    assert got is dq and nat.device_status() == 0 and torch.equal(dq[N:].cpu(), q[N:])
    seq = torch.repeat_interleave(torch.arange(B), new)
    pos = start[seq] + torch.arange(N) - cu[seq]
    t = pos.double()[:, None, None] * freq.cpu()
    turn = lambda x: torch.cat([x[..., :32] * t.cos() - x[..., 32:] * t.sin(), x[..., 32:] * t.cos() + x[..., :32] * t.sin()], -1)  # noqa: E731
    at, slot = table[seq, pos // page].cuda(), (pos % page).cuda()
    for a, x in ((dq[:N], q[:N]), (cache.k[at, slot], k[:N])):
        want = turn(x.double())
        size = x.double().abs().amax(-1, keepdim=True) * 2
        assert ((a.cpu().double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 10 * 2.0 ** -24 * size).all()
    assert torch.equal(cache.v[at, slot].cpu(), v[:N])
    written = torch.zeros(3 * B, page, dtype=torch.bool, device="cuda")
    written[at, slot] = True
    for a, x in zip((cache.k, cache.v), before):
        assert torch.equal(a[~written], x[~written])


@pytest.mark.gpu
@pytest.mark.parametrize("B", [3, 160])
def test_a_page_outside_the_cache_is_the_last_choice_and_reported(B):
    n_pages, page, D = 30, 16, 64
    g = torch.Generator().manual_seed(62)
    kb = torch.randn(n_pages, 2, 1, D, generator=g).sort(1).values.bfloat16()
    k = torch.zeros(n_pages, page, 1, D, dtype=torch.bfloat16, device="cuda")
    cache = mt.PagedKVCache.from_tensors(k, k, key_bounds=kb.cuda())
    table = torch.stack([torch.randperm(n_pages, generator=g) for _ in range(B)]).int()
    table[:, 7], table[:, 12] = 1 << 20, -1
    n = torch.full((B,), n_pages * page, dtype=torch.int32, device="cuda")
    q = torch.randn(B, 2, D, generator=g).bfloat16().cuda()
    pages = paged.select_pages(q, cache, table.cuda(), n, 20).cpu()
    assert nat.device_status() == 2 and not ((pages == 7) | (pages == 12)).any()
    pages = paged.select_pages(q, cache, table.cuda(), n, 29).cpu()
    assert nat.device_status() == 2
    assert (pages == torch.tensor([p for p in range(30) if p != 12])).all()      # the lower of the two


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_past_32_bits_of_elements(dtype):
    """The last pages of a cache of more than 2^32 elements hold what the pages of a small one do."""
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 40 GiB")
    page, D, N, H = 16, 64, 200, 4
    big = mt.PagedKVCache(2 ** 22 + 16, page, 1, D, dtype, key_bounds=True)
    small = mt.PagedKVCache(16, page, 1, D, dtype, key_bounds=True)
    g = torch.Generator().manual_seed(63)
    q, k, v = (torch.randn(N, h, D, generator=g).to(dtype).cuda() for h in (H, 1, 1))
    order = torch.randperm(16, generator=g)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    freq, got = mt.rotary_frequencies(D), []
    for cache, base in ((big, 2 ** 22), (small, 0)):
        table = (order + base).int().cuda()
        turned = paged.append(cache, k, v, table, i32(0), cu_seqlens=i32(0, N), query=q, inv_freq=freq)
        last = turned[-1:].contiguous()
        pages = paged.select_pages(last, cache, table, i32(N), 4)
        got.append((turned, pages, paged.decode(last, cache, table, i32(N)), paged.decode(last, cache, table, i32(N), pages=pages),
                    paged.decode(last, cache, table, i32(N), spec=mt.PatternSpec.causal_window(20, 3)), cache.k[base:], cache.v[base:], cache.key_bounds[base:]))
    assert nat.device_status() == 0 and all(torch.equal(a, b) for a, b in zip(*got))
    assert not big.k[:2 ** 22].any() and not big.v[:2 ** 22].any()
