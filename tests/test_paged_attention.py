"""The paged cache: appending with rotation, attention of one new token, page selection; against plain 64-bit code.

Tolerances count roundings.  u is half a step of the element type (finfo.eps / 2).  An output row o = sum p v is rounded
once (u |o|); the weights may be rounded to the element type before the product (u A, A = sum p |v|; fp32 keeps them);
fp32 arithmetic adds c A with c from the error of a score, 2 D 2^-24 sum |q k| scale, doubled for the exponential's
reference, plus 2^-19 for the exponential itself and the sums."""
import ctypes as C
import math

import pytest
import torch

import ma_transformer_b200 as mt
from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import paged_attention as paged
from ma_transformer_b200.patterns import PatternSpec

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- inputs and plain code ---------------------------------------------------------------------------------

def make_cache(lengths, page, Hkv, D, dtype, seed=0, extra_width=0, heads_first=False, bounds=False):
    """A cache whose unused slots, unused pages and unused table entries hold what must not be read."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lengths]
    n_pages = sum(used) + 2
    shape = (n_pages, Hkv, page, D) if heads_first else (n_pages, page, Hkv, D)
    k, v = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
    if heads_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    kb = torch.full((n_pages, 2, Hkv, D), float("nan"), dtype=dtype) if bounds else None
    table = torch.full((len(lengths), max(max(used), 1) + extra_width), -7, dtype=torch.int32)
    table[:, 1::2] = 1 << 30
    ids = torch.randperm(n_pages, generator=g).tolist()
    logical = []
    for b, n in enumerate(lengths):
        lk, lv = (torch.randn(n, Hkv, D, generator=g).to(dtype) for _ in range(2))
        for w in range(used[b]):
            p = ids.pop()
            table[b, w] = p
            part = lk[w * page:(w + 1) * page]
            k[p, :len(part)] = part
            v[p, :len(part)] = lv[w * page:(w + 1) * page]
            if bounds:
                kb[p, 0], kb[p, 1] = part.float().amin(0).to(dtype), part.float().amax(0).to(dtype)
        logical.append((lk, lv))
    return k, v, kb, table, logical


def attend(q, k, v, scale):
    """q [H, D]; k, v [n, Hkv, D] of what is seen: the output in 64 bits and A = sum p |v|, E = largest sum |q k| scale."""
    H, D = q.shape
    if k.shape[0] == 0:
        z = torch.zeros(H, D, dtype=torch.float64)
        return z, z, 0.0
    G = H // k.shape[1]
    kk, vv = (t.double().repeat_interleave(G, 1) for t in (k, v))
    s = torch.einsum("hd,nhd->hn", q.double(), kk) * scale
    p = torch.softmax(s, -1)
    E = float((torch.einsum("hd,nhd->hn", q.double().abs(), kk.abs()) * scale).max())
    return torch.einsum("hn,nhd->hd", p, vv), torch.einsum("hn,nhd->hd", p, vv.abs()), E


def allowance(o, A, E, D, dtype):
    u = half_step(dtype)
    c = 2 * 2 * D * 2.0 ** -24 * E + 2.0 ** -19
    return u * o.abs() + ((0 if dtype == torch.float32 else u) + c) * A + 1e-30


def page_scores(q, kb, table, n, page, h, G):
    used = table[:-(-n // page)].long()
    lo, hi = kb[used, 0, h].double(), kb[used, 1, h].double()
    qg = q[h * G:(h + 1) * G].double()
    return (qg.clamp(min=0).sum(0) * hi + qg.clamp(max=0).sum(0) * lo).sum(-1)


def best(score, own, topk):
    order = sorted(range(len(score)), key=lambda i: (i != own, -float(score[i]), i))[:topk]
    return sorted(order) + [-1] * (topk - len(order))


# ---- refusals (no GPU needed) ------------------------------------------------------------------------------

def _struct(**kw):
    s = nat.MatPagedCache()
    buf = (C.c_char * 64)()
    base = (C.addressof(buf) + 15) // 16 * 16
    s._keep = buf
    s.k = s.v = base
    s.n_pages, s.page_size, s.H_kv, s.D, s.dtype = 4, 16, 2, 64, nat.MAT_BF16
    s.k_page_stride = s.v_page_stride = 16 * 128
    s.k_token_stride = s.v_token_stride = 128
    s.k_head_stride = s.v_head_stride = 64
    for name, x in kw.items():
        setattr(s, name, x)
    return s, base


def _decode(s, base, **kw):
    a = dict(q=base, q_stride=256, o=base, B=2, H=4, table=base, width=3, stride=3, lengths=base, left=-1, dilation=1, pages=None,
             n_sel=0, scale=0.0, ws=None, ws_bytes=0)
    a.update(kw)
    return nat.lib.mat_paged_decode(C.byref(s), *a.values(), None)


def _append(s, base, **kw):
    a = dict(kn=base, vn=base, kts=128, vts=128, N=2, cu=None, start=base, table=base, width=3, stride=3, B=2, q=None, qo=None, H=0,
             qts=0, f=None, rot=0, inter=0)
    a.update(kw)
    return nat.lib.mat_paged_append(C.byref(s), *a.values(), None)


def _select(s, base, **kw):
    a = dict(q=base, q_stride=256, B=2, H=4, table=base, width=3, stride=3, lengths=base, topk=2, pages=base, ws=None, ws_bytes=0)
    a.update(kw)
    return nat.lib.mat_paged_select(C.byref(s), *a.values(), None)


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(dtype=7), dict(n_pages=0), dict(n_pages=1 << 31), dict(page_size=0), dict(page_size=4),
    dict(page_size=48), dict(page_size=2048), dict(H_kv=0), dict(H_kv=1 << 20), dict(D=0), dict(D=12), dict(D=264),
    dict(k_token_stride=-128), dict(v_head_stride=3), dict(key_bounds=8)])
def test_a_malformed_cache_is_refused(change):
    s, base = _struct(**change)
    for call in (_decode, _append, _select):
        assert call(s, base) in (1, 2)
    assert nat.lib.mat_last_error()
    assert nat.lib.mat_paged_decode_workspace_bytes(C.byref(s), 2, 4, 3, -1, 0) == 0


@pytest.mark.parametrize("change, code", [
    (dict(q=None), 1), (dict(o=None), 1), (dict(lengths=None), 1), (dict(table=None), 1), (dict(B=0), 1), (dict(B=70000), 1),
    (dict(H=3), 1), (dict(H=0), 1), (dict(width=0), 1), (dict(stride=2), 1), (dict(left=4, dilation=0), 1), (dict(n_sel=-1), 1),
    (dict(left=4, n_sel=2, pages=1 << 12), 1), (dict(pages=1 << 12), 1), (dict(q_stride=12), 1), (dict(q_stride=-8), 1),
    (dict(width=1 << 16, stride=1 << 16), 4), (dict(width=1 << 16, stride=1 << 16, ws=256, ws_bytes=1024), 4)])
def test_decode_refusals(change, code):
    s, base = _struct()
    assert _decode(s, base, **change) == code and nat.lib.mat_last_error()


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(N=3), dict(N=1 << 31, cu=16), dict(kn=None), dict(vn=None), dict(start=None), dict(table=None), dict(B=0, N=0),
    dict(q=16), dict(q=16, qo=16, H=3), dict(q=16, qo=16, H=1 << 17, qts=256), dict(rot=3, f=16), dict(rot=66, f=16), dict(rot=2), dict(rot=-2), dict(kts=4), dict(vts=-8),
    dict(q=16, qo=16, H=4, qts=4), dict(kn=8), dict(q=24, qo=16, H=4, qts=256)])
def test_append_refusals(change):
    s, base = _struct()
    assert _append(s, base, **change) in (1, 2) and nat.lib.mat_last_error()


def test_append_of_no_tokens_is_nothing_to_do():
    s, base = _struct()
    assert _append(s, base, N=0, cu=base) == 0


@pytest.mark.parametrize("change, code", [(dict(topk=0), 2), (dict(topk=1 << 20), 2), (dict(pages=None), 1), (dict(q=None), 1), (dict(H=5), 1),
                                          (dict(lengths=None), 1), (dict(), 4)])
def test_select_refusals(change, code):
    s, base = _struct()
    s.key_bounds = base
    assert _select(s, base, **change) == code
    s.key_bounds = None
    assert _select(s, base) == 1 and b"key_bounds" in nat.lib.mat_last_error()


def test_python_surface_refuses_host_tensors_and_bad_widths():
    z = torch.zeros(4, 16, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        mt.PagedKVCache.from_tensors(z, z)
    with pytest.raises(RuntimeError, match="even"):
        mt.rotary_frequencies(7, device="cpu")
    f = mt.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and f[0] == 1 and abs(float(f[1]) - 0.1) < 1e-15


# ---- decode -------------------------------------------------------------------------------------------------

DECODE = [
    # lengths, H, Hkv, D, page, dtype
    ([1], 1, 1, 64, 16, torch.bfloat16),
    ([0, 1, 2, 15, 16, 17, 33], 4, 4, 64, 16, torch.bfloat16),
    ([777], 8, 8, 64, 16, torch.float16),
    ([5, 64, 65, 300, 0, 1000], 8, 2, 128, 64, torch.bfloat16),
    ([129, 1], 16, 1, 64, 32, torch.float16),
    ([200, 31], 40, 2, 80, 8, torch.bfloat16),
    ([90, 250], 10, 2, 96, 128, torch.float32),
    ([3000, 7], 4, 4, 64, 64, torch.float32),
    ([1500], 6, 3, 256, 64, torch.bfloat16),
    ([1025], 3, 1, 256, 1024, torch.float32),
    ([40, 41], 2, 2, 8, 8, torch.bfloat16),
    ([70], 5, 1, 24, 16, torch.float32),
    ([66, 1], 64, 1, 128, 16, torch.bfloat16),
    ([8191, 4097, 1], 32, 8, 128, 64, torch.bfloat16),
    ([20000], 2, 1, 64, 64, torch.float16),
    ([300, 17, 0, 5000], 16, 2, 64, 16, torch.float32),
    ([700, 33], 24, 2, 128, 32, torch.float32),
    ([90], 9, 1, 8, 8, torch.float32),
    ([400, 1200], 8, 1, 32, 8, torch.bfloat16),
    ([9000, 100], 4, 4, 128, 64, torch.bfloat16),
    ([2500] * 40, 8, 8, 64, 64, torch.float16),
]


def run_decode(case, spec=None, seed=0, heads_first=False, extra_width=1, scale=None, strided=False):
    lengths, H, Hkv, D, page, dtype = case
    k, v, _, table, logical = make_cache(lengths, page, Hkv, D, dtype, seed, extra_width, heads_first)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lengths), H, D, generator=g).to(dtype)
    if heads_first:
        dk, dv = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v))
    else:
        dk, dv = k.cuda(), v.cuda()
    cache = mt.PagedKVCache.from_tensors(dk, dv)
    dq = torch.cat([q, q], -1).cuda().view(len(lengths), 2 * H, D)[:, :H] if strided else q.cuda()
    if strided:
        dq.copy_(q)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = paged.decode(dq, cache, table.cuda(), n, spec=spec, scale=scale)
    assert nat.device_status() == 0
    out = out.cpu().double()
    sc = scale or 1 / math.sqrt(D)
    for b, m in enumerate(lengths):
        lk, lv = logical[b]
        if spec is not None and m:
            pos = [m - 1 - t * spec.dilation for t in range(spec.left + 1) if m - 1 - t * spec.dilation >= 0][::-1]
            lk, lv = lk[pos], lv[pos]
        o, A, E = attend(q[b], lk, lv, sc)
        bad = (out[b] - o).abs() > allowance(o, A, E, D, dtype)
        assert not bad.any(), f"sequence {b} of {m} tokens: off by {float((out[b] - o).abs().max())}"
        if m == 0:
            assert (out[b] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(case):
    run_decode(case)


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [PatternSpec.causal_window(1), PatternSpec.causal_window(64, 2), PatternSpec.causal_window(200),
                                  PatternSpec.sliding_window(7), PatternSpec.causal_window(5000, 3)], ids=str)
@pytest.mark.parametrize("case", [DECODE[1], DECODE[3], DECODE[7], DECODE[15], DECODE[18]], ids=str)
def test_decode_of_a_window(case, spec):
    run_decode(case, spec=spec)


@pytest.mark.gpu
def test_decode_with_other_strides_widths_and_scale():
    run_decode(DECODE[3], heads_first=True, strided=True, scale=0.3)
    run_decode(DECODE[7], heads_first=True)
    for case in (DECODE[3], DECODE[15]):              # a table for far longer sequences than there are
        run_decode(case, extra_width=20000)
        run_decode(case, extra_width=2000)
    run_decode(([5] * 700, 2, 1, 64, 8, torch.bfloat16))


@pytest.mark.gpu
def test_a_windowed_decode_needs_only_the_pages_it_reads():
    """Pages before the window may be given back: their entries hold anything."""
    lengths, H, Hkv, D, page, dtype = case = ([1000], 4, 4, 64, 16, torch.bfloat16)
    k, v, _, table, logical = make_cache(lengths, page, Hkv, D, dtype)
    table[0, :(1000 - 64) // page] = -1
    q = torch.randn(1, H, D).to(dtype)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = paged.decode(q.cuda(), cache, table.cuda(), n, spec=PatternSpec.causal_window(64)).cpu().double()
    assert nat.device_status() == 0
    o, A, E = attend(q[0], logical[0][0][-64:], logical[0][1][-64:], 1 / 8)
    assert ((out[0] - o).abs() <= allowance(o, A, E, D, dtype)).all()


@pytest.mark.gpu
def test_decode_is_the_same_every_time_and_on_another_stream_and_in_a_graph():
    lengths, H, Hkv, D, page, dtype = case = ([5000, 3, 900], 8, 2, 128, 32, torch.bfloat16)
    k, v, _, table, _ = make_cache(lengths, page, Hkv, D, dtype)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    q, t = torch.randn(3, H, D).to(dtype).cuda(), table.cuda()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = paged.decode(q, cache, t, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged.decode(q, cache, t, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other) and torch.equal(want, paged.decode(q, cache, t, n))
    out1, out2 = torch.empty_like(q), torch.empty_like(q)
    graphs = []
    for out in (out1, out2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.decode(q, cache, t, n, out=out)
        graphs.append(graph)
    n.copy_(torch.tensor([17, 1, 0]))               # replays read the lengths of the time
    short = paged.decode(q, cache, t, n)
    n.copy_(torch.tensor(lengths))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        graphs[0].replay()
    with torch.cuda.stream(b):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(out1, want) and torch.equal(out2, want)
    n.copy_(torch.tensor([17, 1, 0]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(out1, short)


@pytest.mark.gpu
def test_pages_outside_the_cache_count_as_absent_and_are_reported():
    lengths, H, Hkv, D, page, dtype = ([100], 4, 2, 64, 16, torch.float32)
    k, v, _, table, logical = make_cache(lengths, page, Hkv, D, dtype)
    table[0, 2] = 1000000
    table[0, 4] = -3
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    q = torch.randn(1, H, D)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = paged.decode(q.cuda(), cache, table.cuda(), n).cpu().double()
    assert nat.device_status() == 2 and nat.device_status() == 0
    keep = [i for i in range(100) if i // 16 not in (2, 4)]
    o, A, E = attend(q[0], logical[0][0][keep], logical[0][1][keep], 1 / 8)
    assert ((out[0] - o).abs() <= allowance(o, A, E, D, dtype)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spec, first", [(None, 0), (PatternSpec.causal_window(50), 249 - 49), (PatternSpec.causal_window(40, 2), 249 - 78),
                                         (PatternSpec.causal_window(3), 249 - 2)])
def test_a_length_past_the_table_reads_what_the_table_holds(dtype, spec, first):
    """A sequence of 250 tokens whose table stops after 208, and the largest length there is."""
    k, v, _, table, logical = make_cache([208], 16, 2, 64, dtype)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    q = torch.randn(1, 4, 64).to(dtype)
    n = torch.tensor([250], dtype=torch.int32, device="cuda")
    step = spec.dilation if spec else 1
    pos = [p for p in range(first, 208) if (p - first) % step == 0]
    out = paged.decode(q.cuda(), cache, table.cuda(), n, spec=spec).cpu().double()
    assert nat.device_status() == 2
    o, A, E = attend(q[0], logical[0][0][pos], logical[0][1][pos], 1 / 8)
    assert ((out[0] - o).abs() <= allowance(o, A, E, 64, dtype)).all()
    n.fill_(2 ** 31 - 1)
    out = paged.decode(q.cuda(), cache, table.cuda(), n, spec=spec)
    assert nat.device_status() == 2 and (spec is None or not out.any())


@pytest.mark.gpu
def test_decode_with_rows_of_pages():
    lengths, H, Hkv, D, page, dtype = ([300, 33, 0, 1], 6, 3, 64, 16, torch.float16)
    k, v, _, table, logical = make_cache(lengths, page, Hkv, D, dtype)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    q = torch.randn(4, H, D).to(dtype)
    pages = torch.full((4, Hkv, 5), -1, dtype=torch.int32)
    pages[0, 0] = torch.tensor([0, 3, 7, 12, 18])
    pages[0, 1, :2] = torch.tensor([2, 18])
    pages[0, 2, :3] = torch.tensor([-1, 5, 4000])     # entries past the length are skipped
    pages[1, 0, 0], pages[1, 1, 0], pages[1, 1, 1] = 2, 0, 1
    pages[2, 0, 0] = 0                                # an idle sequence stays zero
    pages[3, :, 0] = 0
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = paged.decode(q.cuda(), cache, table.cuda(), n, pages=pages.cuda()).cpu().double()
    assert nat.device_status() == 0
    for b, m in enumerate(lengths):
        for h in range(Hkv):
            pos = [p * page + s for p in pages[b, h].tolist() if p >= 0 for s in range(page) if p * page + s < m]
            o, A, E = attend(q[b, 2 * h:2 * h + 2], logical[b][0][pos][:, h:h + 1], logical[b][1][pos][:, h:h + 1], 1 / 8)
            assert ((out[b, 2 * h:2 * h + 2] - o).abs() <= allowance(o, A, E, D, dtype)).all()


# ---- selection ----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("lengths, H, Hkv, D, page, dtype, topk", [
    ([1, 0, 16, 17, 500], 4, 4, 64, 16, torch.bfloat16, 4),
    ([2000, 37], 8, 2, 128, 16, torch.float16, 1),
    ([3000, 1], 10, 2, 80, 8, torch.float32, 100),
    ([20000, 9000], 4, 1, 64, 8, torch.bfloat16, 64),
    ([300], 2, 2, 256, 64, torch.bfloat16, 9),
    ([12000], 2, 1, 8, 8, torch.float32, 1499)])
def test_select_pages(lengths, H, Hkv, D, page, dtype, topk):
    k, v, kb, table, _ = make_cache(lengths, page, Hkv, D, dtype, bounds=True)
    q = torch.randn(len(lengths), H, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda(), key_bounds=kb.cuda())
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pages = paged.select_pages(q.cuda(), cache, table.cuda(), n, topk).cpu()
    assert nat.device_status() == 0
    for b, m in enumerate(lengths):
        for h in range(Hkv):
            s = page_scores(q[b], kb, table[b], m, page, h, H // Hkv) if m else []
            assert pages[b, h].tolist() == best(s, (m - 1) // page, topk), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("n_pages", [9, 40, 300, 700, 1500])
def test_selection_of_equal_scores_takes_the_lower_page(n_pages):
    page, Hkv, D = 8, 1, 64
    k, v, kb, table, _ = make_cache([n_pages * page], page, Hkv, D, torch.bfloat16, bounds=True)
    kb[table[0, :n_pages].long()] = kb[table[0, 0].long()].clone()
    some = [n_pages // 2, n_pages // 3]
    kb[table[0, some].long()] += 1
    kb[table[0, 1].long()] = float("nan")              # not a number: last
    q = torch.ones(1, 2, D, dtype=torch.bfloat16)
    cache = mt.PagedKVCache.from_tensors(k.cuda(), v.cuda(), key_bounds=kb.cuda())
    n = torch.tensor([n_pages * page], dtype=torch.int32, device="cuda")
    for topk in (1, 2, 4, 6, n_pages - 1, n_pages, n_pages + 3):
        got = paged.select_pages(q.cuda(), cache, table.cuda(), n, topk).cpu()[0, 0].tolist()
        rank = sorted(range(n_pages), key=lambda i: (i != n_pages - 1, i not in some, i == 1, i))[:topk]
        assert got == sorted(rank) + [-1] * (topk - len(rank)), topk


# ---- append -------------------------------------------------------------------------------------------------

def turned(x, pos, freq, interleaved):
    """x [n, heads, D] in 64 bits, rotated at integer positions."""
    x = x.double().clone()
    r = 2 * len(freq)
    t = pos.double()[:, None] * freq
    c, s = t.cos()[:, None], t.sin()[:, None]
    i = torch.arange(r // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


APPEND = [
    # start, new, H, Hkv, D, rot, page, dtype, interleaved
    ([0], [1], 1, 1, 64, 64, 16, torch.bfloat16, False),
    ([5, 0, 15, 16, 1000003], [1, 1, 1, 1, 1], 8, 2, 128, 128, 16, torch.bfloat16, False),
    ([7, 0, 100], [40, 1, 0], 4, 4, 64, 32, 16, torch.float16, True),
    ([0, 3, 63, 64], [200, 0, 2, 130], 6, 2, 80, 80, 64, torch.float32, False),
    ([11], [500], 5, 1, 256, 64, 128, torch.bfloat16, True),
    ([3, 9], [20, 30], 2, 2, 24, 6, 8, torch.float32, False),       # a rotation that no 16-byte vector fits
    ([3, 9], [20, 30], 2, 1, 72, 20, 8, torch.bfloat16, False),
    ([1, 2], [9, 70], 2, 1, 256, 254, 1024, torch.float16, False),
    ([2 ** 31 - 40], [9], 2, 1, 64, 64, 1024, torch.float32, False),
    ([4, 5], [33, 1], 4, 2, 64, 0, 32, torch.bfloat16, False),      # no rotation
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("variant", ["packed", "strided"])
def test_append(case, variant):
    start, new, H, Hkv, D, rot, page, dtype, inter = case
    B, N = len(start), sum(new)
    g = torch.Generator().manual_seed(5)
    pad = 3 if variant == "strided" else 0             # rows behind the last sequence
    q, k, v = (torch.randn(N + pad, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv))
    first, last = [s // page for s in start], [(s + max(n, 1) - 1) // page for s, n in zip(start, new)]
    width = max(last) + 1
    n_pages = sum(b - a + 1 for a, b in zip(first, last)) + 1
    ids = torch.randperm(n_pages, generator=g).tolist()
    kp = torch.randn(n_pages, page, Hkv, D, generator=g).to(dtype)
    vp = torch.randn(n_pages, page, Hkv, D, generator=g).to(dtype)
    kb = torch.full((n_pages, 2, Hkv, D), 77.0, dtype=dtype)
    off = min(first)                                    # tables of far positions: only the tail is stored, as a view would
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    rows = {}
    for b in range(B):
        for w in range(first[b], last[b] + 1):
            rows[b, w] = ids.pop()
            table[b, w] = rows[b, w]
    freq = mt.rotary_frequencies(rot, device="cpu") if rot else None
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
    if variant == "strided":                            # slices of a fused projection; heads-first storage
        fused = torch.cat([q, k, v], 1).cuda()
        dq, dk, dv = fused[:, :H], fused[:, H:H + Hkv], fused[:, H + Hkv:]
        ck, cv = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (kp, vp))
    else:
        dq, dk, dv, ck, cv = q.cuda(), k.cuda(), v.cuda(), kp.cuda(), vp.cuda()
    cache = mt.PagedKVCache.from_tensors(ck, cv, key_bounds=kb.cuda())
    qo = torch.full((N + pad, H, D), 9.0, dtype=dtype, device="cuda")
    one_each = variant == "packed" and all(n == 1 for n in new)
    got = paged.append(cache, dk, dv, table, torch.tensor(start, dtype=torch.int32, device="cuda"),
                       cu_seqlens=None if one_each else cu.cuda(), query=dq, inv_freq=freq.cuda() if rot else None, interleaved=inter,
                       query_out=qo)
    assert got is qo and nat.device_status() == 0
    u = half_step(dtype)
    f = freq if rot else torch.zeros(0, dtype=torch.float64)
    # a rounding of the result, and of the fp32 cosine, sine and products (5 roundings of 2^-24 on each of two terms)
    close = lambda x, want, size: bool(((x.double() - want).abs() <= u * want.abs() + 10 * 2.0 ** -24 * size).all())  # noqa: E731
    kept_k, kept_v = kp.clone(), vp.clone()
    for b in range(B):
        r = slice(int(cu[b]), int(cu[b + 1]))
        pos = torch.arange(start[b], start[b] + new[b])
        size_q, size_k = (x[r].double().abs().amax(-1, keepdim=True) * 2 if new[b] else 0 for x in (q, k))
        assert close(qo[r].cpu(), turned(q[r], pos, f, inter), size_q)
        where = torch.tensor([rows[b, int(p) // page] for p in pos], dtype=torch.long)
        assert close(ck[where.cuda(), (pos % page).cuda()].cpu(), turned(k[r], pos, f, inter), size_k)
        kept_k[where, pos % page] = ck[where.cuda(), (pos % page).cuda()].cpu()
        kept_v[where, pos % page] = v[r]
    assert torch.equal(ck.cpu(), kept_k) and torch.equal(cv.cpu(), kept_v)     # and nothing else was written
    assert (qo[N:] == 9).all()
    for b in range(B):
        for w in range(first[b], last[b] + 1):
            if not new[b]:
                assert (cache.key_bounds[rows[b, w]] == 77).all()
                continue
            end = min(page, start[b] + new[b] - w * page)
            filled = kept_k[rows[b, w], :end].float()
            assert torch.equal(cache.key_bounds[rows[b, w], 0].cpu().float(), filled.amin(0))
            assert torch.equal(cache.key_bounds[rows[b, w], 1].cpu().float(), filled.amax(0))


@pytest.mark.gpu
def test_append_piece_by_piece_and_after_a_rollback_leaves_the_same_cache():
    Hkv, D, page, N = 2, 64, 16, 75
    k, v = torch.randn(N, Hkv, D).bfloat16().cuda(), torch.randn(N, Hkv, D).bfloat16().cuda()
    f = mt.rotary_frequencies(D)
    table = torch.randperm(8).to(torch.int32).cuda()[None]
    at = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    caches = [mt.PagedKVCache(8, page, Hkv, D, torch.bfloat16, key_bounds=True) for _ in range(2)]
    paged.append(caches[0], k, v, table, at(0), cu_seqlens=torch.tensor([0, N], dtype=torch.int32, device="cuda"), inv_freq=f)
    for i in range(N):
        if i == 50:                                     # drafted tokens that were rejected
            for j in range(i, i + 9):
                paged.append(caches[1], 30 * k[i:i + 1], v[i:i + 1], table, at(j), inv_freq=f)
        paged.append(caches[1], k[i:i + 1], v[i:i + 1], table, at(i), inv_freq=f)
    used = table[0, :5].long()
    assert torch.equal(caches[0].key_bounds[used], caches[1].key_bounds[used])
    assert torch.equal(caches[0].k[used].flatten(0, 1)[:N], caches[1].k[used].flatten(0, 1)[:N])
    assert torch.equal(caches[0].v[used].flatten(0, 1)[:N], caches[1].v[used].flatten(0, 1)[:N])


@pytest.mark.gpu
def test_append_outside_the_cache_is_skipped_and_reported():
    cache = mt.PagedKVCache(4, 8, 1, 64, torch.float32, key_bounds=True)
    x = torch.randn(4, 1, 64).cuda()
    table = torch.tensor([[0, 9], [-1, 1], [2, 3], [3, 3]], dtype=torch.int32).cuda()
    start = torch.tensor([8, 3, 16, -5], dtype=torch.int32).cuda()
    q = paged.append(cache, x, x, table, start, query=x)
    assert nat.device_status() == 2 and not cache.k.any() and not cache.v.any() and not cache.key_bounds.any()
    assert torch.equal(q[:3], x[:3])                    # the queries do not need the pages


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    cache = mt.PagedKVCache(4, 16, 2, 64, torch.bfloat16)
    t, n = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q, kv = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    paged.decode(q, cache, t, n)
    for bad in (lambda: paged.decode(q.float(), cache, t, n), lambda: paged.decode(q[:, :3], cache, t, n), lambda: paged.decode(q.cpu(), cache, t, n),
                lambda: paged.decode(q, cache, t.long(), n), lambda: paged.decode(q, cache, t, n[:0]), lambda: paged.decode(q, cache, t, n.cpu()),
                lambda: paged.decode(q, cache, t, n, spec=PatternSpec.longformer(1, 1, [0])),
                lambda: paged.decode(q, cache, t, n, spec=PatternSpec.causal_window(4), pages=torch.zeros(1, 2, 1, dtype=torch.int32, device="cuda")),
                lambda: paged.decode(q, cache, t, n, pages=torch.zeros(1, 4, 1, dtype=torch.int32, device="cuda")),
                lambda: paged.select_pages(q, cache, t, n, 1), lambda: paged.select_pages(q, cache, t, n, 0),
                lambda: paged.append(cache, kv, kv[:, :1], t, n), lambda: paged.append(cache, kv[:0], kv[:0], t, n),
                lambda: paged.append(cache, kv, kv, t, n, inv_freq=torch.ones(4, device="cuda")),
                lambda: paged.append(cache, kv, kv, t, n, query=q, query_out=q[:, :2]),
                lambda: paged.append(cache, kv, kv, t, n, cu_seqlens=n),
                lambda: mt.PagedKVCache(4, 12, 2, 64), lambda: mt.PagedKVCache(4, 16, 2, 60),
                lambda: mt.PagedKVCache.from_tensors(cache.k, cache.v, key_bounds=cache.k)):
        with pytest.raises(RuntimeError):
            bad()
    assert nat.device_status() == 0
