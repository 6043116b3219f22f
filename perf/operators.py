"""Measured cases of the serving and block-selection operators.

Four paths, as a user's program calls them:

``append``    new keys and values rotated by position and written into a paged cache (with the pages' key bounds)
``decode``    attention of one new token per sequence over the paged cache
``selected``  pages chosen for each new token by a cheap score, then attention over the chosen pages
``train``     blocks chosen for each query of a sequence, attention over them, and its gradients

``own`` picks between the plain form in elementary torch operations and the package's operators.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of 64 conversations, at far positions; older pages have been given back
        dict(name="append-step", op="append", B=64, N=64, H=32, Hkv=8, D=128, rot=128, page=64, dtype="bf16",
             interleaved=False, far=1000000),
        # prompts of seven users packed without padding, half of each head rotated
        dict(name="append-prompts", op="append", B=7, N=32768, H=12, Hkv=4, D=64, rot=32, page=16, dtype="fp16",
             interleaved=True, far=500),
        # a single short conversation: latency
        dict(name="decode-one", op="decode", B=1, longest=777, H=8, Hkv=8, D=64, page=16, dtype="bf16", taps=0, dilation=1),
        # a serving batch of mixed lengths
        dict(name="decode-batch", op="decode", B=64, longest=8192, H=32, Hkv=8, D=128, page=64, dtype="bf16", taps=0,
             dilation=1),
        # few long documents
        dict(name="decode-long", op="decode", B=4, longest=131072, H=32, Hkv=8, D=128, page=64, dtype="bf16", taps=0,
             dilation=1),
        # the order-book model's dilated causal window, tick by tick, in fp32
        dict(name="decode-window", op="decode", B=16, longest=8192, H=4, Hkv=4, D=64, page=64, dtype="fp32", taps=64,
             dilation=2),
        # a batch that reads 32 pages of each long conversation
        dict(name="selected-batch", op="selected", B=32, longest=32768, H=32, Hkv=8, D=128, page=64, dtype="bf16", topk=32),
        # one very long document, a key head for every query head
        dict(name="selected-long", op="selected", B=1, longest=1000000, H=8, Hkv=8, D=64, page=64, dtype="fp16", topk=64),
        # a small fp32 model with a sequence that ends inside a block
        dict(name="train-fp32", op="train", B=2, S=1000, H=4, Hkv=4, D=32, block=32, topk=4, causal=True, dtype="fp32"),
        # the eight heads of 64 columns of the window benchmark
        dict(name="train-heads", op="train", B=1, S=8192, H=8, Hkv=8, D=64, block=64, topk=16, causal=True, dtype="bf16"),
        # key heads shared by four query heads
        dict(name="train-shared", op="train", B=2, S=4096, H=16, Hkv=4, D=128, block=64, topk=8, causal=True, dtype="bf16"),
        # an encoder's two-sided selection
        dict(name="train-encoder", op="train", B=2, S=2000, H=12, Hkv=12, D=64, block=32, topk=8, causal=False, dtype="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "selected", "train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "train":
        Hkv = rng.choice([1, 2, 4, 6])
        H = Hkv * rng.choice([1, 1, 2, 4])
        block = rng.choice([16, 32, 64, 128])
        S = _log_uniform(rng, 200, 4096)
        return dict(op=op, B=rng.choice([1, 1, 2]) if H <= 8 else 1, S=S, H=H, Hkv=Hkv, D=rng.choice([32, 64, 80, 128]),
                    block=block, topk=rng.randint(1, max(2, min(24, 1024 // block))), causal=rng.random() < 0.7, dtype=dtype)
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 2, 4, 5, 8])
    D = rng.choice([64, 80, 96, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        B = _log_uniform(rng, 1, 64)
        step = rng.random() < 0.5
        N = B if step else max(B, _log_uniform(rng, 100, 16384))
        return dict(op=op, B=B, N=N, H=H, Hkv=Hkv, D=D, rot=rng.choice([D, D // 2]), page=page, dtype=dtype,
                    interleaved=rng.random() < 0.5, far=_log_uniform(rng, 10, 1000000))
    width = Hkv * D * (4 if dtype == "fp32" else 2)
    B = _log_uniform(rng, 1, 128)
    most = max(64, min(200000, 400000 * 2048 // (B * max(width, 2048))))
    longest = _log_uniform(rng, 20, most)
    if op == "decode":
        window = rng.random() < 0.3
        return dict(op=op, B=B, longest=longest, H=H, Hkv=Hkv, D=D, page=page, dtype=dtype,
                    taps=_log_uniform(rng, 1, 1024) if window else 0, dilation=rng.choice([1, 2, 3]) if window else 1)
    return dict(op=op, B=B, longest=longest, H=H, Hkv=Hkv, D=D, page=page, dtype=dtype, topk=_log_uniform(rng, 1, 64))


# ---- inputs -----------------------------------------------------------------------------------------------

def _lengths(case):
    """Cached tokens of each sequence (the new one among them): from one token up to the longest, an idle slot in
    batches of eight and more.  The seed permutes them."""
    r = random.Random("%d %d" % (case["B"], case["longest"]))
    n = [case["longest"]] + [_log_uniform(r, max(1, case["longest"] // 16), case["longest"]) for _ in range(case["B"] - 1)]
    if len(n) >= 8:
        n[1], n[2] = 1, 0
    return n


def _prompt_lengths(case):
    """New tokens of each sequence of an append, at least one each."""
    B, N = case["B"], case["N"]
    r = random.Random("%d %d" % (B, N))
    cuts = sorted(r.sample(range(1, N), B - 1)) if B > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [N])]


def _page_bounds(k_pages):
    """Smallest and largest key of every page, column by column: [pages, 2, Hkv, D]."""
    return torch.stack([k_pages.amin(1), k_pages.amax(1)], dim=1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    dt = DTYPES[case["dtype"]]
    op, B, H, Hkv, D = case["op"], case["B"], case["H"], case["Hkv"], case["D"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if op == "train":
        S, block = case["S"], case["block"]
        nb = -(-S // block)
        centre = torch.randn(B, nb, 1, Hkv, D, generator=g, device="cuda") * 0.7   # the keys of a block resemble each other
        k = (torch.randn(B, nb, block, Hkv, D, generator=g, device="cuda") + centre).reshape(B, nb * block, Hkv, D)
        return dict(q=normal(B, S, H, D), k=k[:, :S].to(dt).contiguous(), v=normal(B, S, Hkv, D), dout=normal(B, S, H, D))

    page = case["page"]
    if op == "append":
        new = _prompt_lengths(case)
        host.shuffle(new)
        start = [host.randrange(case["far"]) for _ in new]
        first = [s // page for s in start]
        last = [(s + n - 1) // page for s, n in zip(start, new)]
        n_pages = sum(n // page + 2 for n in new)          # enough wherever the sequences start
        ids = list(range(n_pages))
        host.shuffle(ids)
        table = torch.full((B, max(last) + 1), -1, dtype=torch.int32)   # pages before the first touched one were given back
        at = 0
        for b in range(B):
            n = last[b] - first[b] + 1
            table[b, first[b]:last[b] + 1] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        k_pages, v_pages = normal(n_pages, page, Hkv, D), normal(n_pages, page, Hkv, D)
        # what the cache holds before: the first touched page of a sequence up to its start
        bounds = _page_bounds(k_pages)
        for b in range(B):
            used = start[b] % page
            if used:
                p = int(table[b, first[b]])
                bounds[p] = _page_bounds(k_pages[p:p + 1, :used])[0]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        rot = case["rot"]
        inv_freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        return dict(q=normal(case["N"], H, D), k=normal(case["N"], Hkv, D), v=normal(case["N"], Hkv, D), k_pages=k_pages,
                    v_pages=v_pages, bounds=bounds, table=table.cuda(), start=ints(start), cu=ints(cu), inv_freq=inv_freq)

    lengths = _lengths(case)
    host.shuffle(lengths)
    width = -(-case["longest"] // page)
    used = [-(-n // page) for n in lengths]
    n_pages = max(1, sum(used))
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    k_pages, v_pages = normal(n_pages, page, Hkv, D), normal(n_pages, page, Hkv, D)
    s = dict(q=normal(B, H, D), k_pages=k_pages, v_pages=v_pages, table=table, lengths=ints(lengths))
    if op == "selected":
        k_pages += torch.randn(n_pages, 1, Hkv, D, generator=g, device="cuda").to(dt)
        s["bounds"] = _page_bounds(k_pages)
        for b, n in enumerate(lengths):
            if n % page:
                p = int(table[b, n // page])
                s["bounds"][p] = _page_bounds(k_pages[p:p + 1, :n % page])[0]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] != "train":
        from ma_transformer_b200.paged_attention import PagedKVCache
        s["cache"] = PagedKVCache.from_tensors(s["k_pages"], s["v_pages"], key_bounds=s.get("bounds"))
    if own and case["op"] == "decode" and case["taps"]:
        from ma_transformer_b200 import PatternSpec
        s["spec"] = PatternSpec.causal_window(case["taps"], case["dilation"])
    return s


# ---- plain forms ------------------------------------------------------------------------------------------

def _rotated(x, cos, sin, rot, interleaved):
    """The first ``rot`` columns of [N, heads, D] turned by the token's angles (fp32), rounded once."""
    f = x.float()
    part = f[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rot // 2], part[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, f[..., rot:]], -1).to(x.dtype)


def _plain_append(s):
    c = s["case"]
    page, rot = c["page"], c["rot"]
    n = torch.arange(c["N"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), n, right=True)
    pos = s["start"].long()[seq] + n - s["cu"].long()[seq]
    angle = pos.double()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotated(s["q"], cos, sin, rot, c["interleaved"])
    k = _rotated(s["k"], cos, sin, rot, c["interleaved"])
    at, slot = s["table"].long()[seq, pos // page], pos % page
    s["k_pages"][at, slot] = k
    s["v_pages"][at, slot] = s["v"]
    fresh = torch.zeros(s["bounds"].shape[0], dtype=torch.int32, device="cuda")
    fresh.scatter_reduce_(0, at, (slot == 0).int(), "amax")
    fresh = (fresh > 0)[:, None, None]
    lo = torch.where(fresh, math.inf, s["bounds"][:, 0].float()).index_reduce_(0, at, k.float(), "amin")
    hi = torch.where(fresh, -math.inf, s["bounds"][:, 1].float()).index_reduce_(0, at, k.float(), "amax")
    s["bounds"].copy_(torch.stack([lo, hi], 1))
    return {"query": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "bounds": s["bounds"]}


def _plain_attend(q, k, v, seen):
    """q [B, Hkv, G, D] over k, v [B, Hkv, n, D] in fp32 where ``seen`` [B, 1 or Hkv, n]; a row that sees nothing is zero."""
    score = torch.einsum("bhgd,bhnd->bhgn", q.float(), k.float()) / math.sqrt(q.shape[-1])
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bhgn,bhnd->bhgd", weight, v.float())
    return torch.where(total > 0, out / total, 0.0)


def _plain_decode(s):
    c = s["case"]
    page, taps, dil = c["page"], c["taps"], c["dilation"]
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    length = s["lengths"].long()[:, None]
    if taps:
        pos = length - 1 - torch.arange(taps, device="cuda") * dil
        seen = pos >= 0
        pos = pos.clamp(min=0)
        at = s["table"].long().gather(1, pos // page).clamp(min=0)
        k, v = s["k_pages"][at, pos % page], s["v_pages"][at, pos % page]
    else:
        at = s["table"].long().clamp(min=0)
        k, v = s["k_pages"][at].flatten(1, 2), s["v_pages"][at].flatten(1, 2)
        seen = torch.arange(k.shape[1], device="cuda") < length
    out = _plain_attend(s["q"].view(B, Hkv, H // Hkv, D), k.transpose(1, 2), v.transpose(1, 2), seen[:, None])
    return {"out": out.reshape(B, H, D).to(s["q"].dtype)}


def _best(score, visible, always, topk):
    """The ``topk`` best entries of the last axis, ``always`` among them, equal scores by the lower index; ascending,
    -1 behind the last."""
    score = torch.where(always, math.inf, torch.where(visible, score, -math.inf))
    n = score.shape[-1]
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    index = torch.where(order.values[..., :topk] > -math.inf, order.indices[..., :topk], n).sort(-1).values
    index = torch.nn.functional.pad(index, (0, max(0, topk - n)), value=n)
    return torch.where(index < n, index, -1).int()


def _plain_selected(s):
    c = s["case"]
    page, topk = c["page"], c["topk"]
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    q = s["q"].view(B, Hkv, H // Hkv, D)
    table = s["table"].long().clamp(min=0)
    bounds = s["bounds"][table].double()                       # [B, W, 2, Hkv, D]
    up, down = q.double().clamp(min=0).sum(2), q.double().clamp(max=0).sum(2)
    score = torch.einsum("bhd,bwhd->bhw", up, bounds[:, :, 1]) + torch.einsum("bhd,bwhd->bhw", down, bounds[:, :, 0])
    length = s["lengths"].long()[:, None, None]
    w = torch.arange(table.shape[1], device="cuda")
    pages = _best(score, w * page < length, (w == (length - 1) // page) & (length > 0), topk)
    chosen = pages.long().clamp(min=0)
    at = table[:, None].expand(-1, Hkv, -1).gather(2, chosen)[..., None]
    slot, head = torch.arange(page, device="cuda"), torch.arange(Hkv, device="cuda")[:, None, None]
    k, v = s["k_pages"][at, slot, head].flatten(2, 3), s["v_pages"][at, slot, head].flatten(2, 3)
    seen = ((pages >= 0)[..., None] & (chosen[..., None] * page + slot < length[..., None])).flatten(2, 3)
    out = _plain_attend(q, k, v, seen)
    return {"pages": pages, "out": out.reshape(B, H, D).to(s["q"].dtype)}


def _plain_train(s):
    c = s["case"]
    B, S, H, Hkv, D, block, topk = c["B"], c["S"], c["H"], c["Hkv"], c["D"], c["block"], c["topk"]
    nb, group, dt = -(-S // block), H // Hkv, s["q"].dtype
    k64 = s["k"].double()
    fill = k64[:, -1:].expand(-1, nb * block - S, -1, -1)     # repeats of the last key leave its block's bounds as they are
    kb = torch.cat([k64, fill], 1).view(B, nb, block, Hkv, D)
    q64 = s["q"].double().view(B, S, Hkv, group, D)
    score = torch.einsum("bshd,bnhd->bshn", q64.clamp(min=0).sum(3), kb.amax(2)) + torch.einsum(
        "bshd,bnhd->bshn", q64.clamp(max=0).sum(3), kb.amin(2))
    mine = (torch.arange(S, device="cuda") // block)[:, None, None]
    n = torch.arange(nb, device="cuda")
    blocks = _best(score, (n <= mine) if c["causal"] else (n >= 0).expand(S, 1, nb), n == mine, topk)     # [B, S, Hkv, topk]
    picked = torch.zeros(B, S, Hkv, nb + 1, dtype=torch.bool, device="cuda")
    picked.scatter_(3, torch.where(blocks >= 0, blocks, nb).long(), True)
    i = torch.arange(S, device="cuda")
    seen = picked[..., :nb].repeat_interleave(block, -1)[..., :S].permute(0, 2, 1, 3)                  # [B, Hkv, S, S]
    if c["causal"]:
        seen = seen & (i[None, :] <= i[:, None])
    q, k, v, dout = (s[x].float() for x in ("q", "k", "v", "dout"))
    q, dout = (x.view(B, S, Hkv, group, D).permute(0, 2, 3, 1, 4) for x in (q, dout))                  # [B, Hkv, G, S, D]
    k, v = k.transpose(1, 2), v.transpose(1, 2)                                                        # [B, Hkv, S, D]
    scale = 1 / math.sqrt(D)
    weight = torch.einsum("bhgid,bhjd->bhgij", q, k).mul_(scale).masked_fill_(~seen[:, :, None], -math.inf)
    top = weight.amax(-1, keepdim=True)
    weight = weight.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    weight = weight.div_(total)
    out = torch.einsum("bhgij,bhjd->bhgid", weight, v)
    dv = torch.einsum("bhgij,bhgid->bhjd", weight, dout)
    delta = (dout * out).sum(-1, keepdim=True)
    ds = torch.einsum("bhgid,bhjd->bhgij", dout, v).sub_(delta).mul_(weight).mul_(scale)
    dq = torch.einsum("bhgij,bhjd->bhgid", ds, k)
    dk = torch.einsum("bhgij,bhgid->bhjd", ds, q)
    rows = lambda x: x.permute(0, 3, 1, 2, 4).reshape(B, S, H, D).to(dt)  # noqa: E731
    return {"blocks": blocks, "out": rows(out), "lse": lse.permute(0, 3, 1, 2).reshape(B, S, H), "dq": rows(dq),
            "dk": dk.transpose(1, 2).to(dt), "dv": dv.transpose(1, 2).to(dt)}


# ---- the package's operators ------------------------------------------------------------------------------

def _own_run(s):
    c = s["case"]
    if c["op"] == "train":
        from ma_transformer_b200 import selected_attention as sel
        blocks = sel.select_blocks(s["q"], s["k"], c["block"], c["topk"], causal=c["causal"])
        out, lse = sel.forward_selected(s["q"], s["k"], s["v"], blocks, c["block"], causal=c["causal"])
        dq, dk, dv = sel.backward_selected(s["q"], s["k"], s["v"], out, lse, s["dout"], blocks, c["block"],
                                           causal=c["causal"])
        return {"blocks": blocks, "out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    from ma_transformer_b200 import paged_attention as paged
    if c["op"] == "append":
        q = paged.append(s["cache"], s["k"], s["v"], s["table"], s["start"], cu_seqlens=s["cu"], query=s["q"],
                         inv_freq=s["inv_freq"], interleaved=c["interleaved"])
        return {"query": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "bounds": s["bounds"]}
    if c["op"] == "decode":
        return {"out": paged.decode(s["q"], s["cache"], s["table"], s["lengths"], spec=s.get("spec"))}
    pages = paged.select_pages(s["q"], s["cache"], s["table"], s["lengths"], c["topk"])
    return {"pages": pages, "out": paged.decode(s["q"], s["cache"], s["table"], s["lengths"], pages=pages)}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "selected": _plain_selected, "train": _plain_train}


def run(state):
    return _own_run(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------

def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    H, Hkv, D, B = c["H"], c["Hkv"], c["D"], c["B"]
    if c["op"] == "append":
        rows = c["N"] * (2 * H + 4 * Hkv) * D * size                       # q, k, v read and written
        pages = max(B, c["N"] // c["page"])
        return {"bytes": rows + 4 * pages * Hkv * D * size, "flops": 3 * c["N"] * (H + Hkv) * c["rot"]}
    if c["op"] == "train":
        S, block, topk, nb = c["S"], c["block"], c["topk"], -(-c["S"] // c["block"])
        pairs = 0
        for n in range(nb):
            rows = min(block, S - n * block)
            if c["causal"]:
                pairs += rows * (min(topk, n + 1) - 1) * block + rows * (rows + 1) // 2
            else:
                pairs += rows * min(min(topk, nb) * block, S)
        scores = S * nb // (2 if c["causal"] else 1) * Hkv * 4 * D
        return {"bytes": B * S * ((4 * H + 4 * Hkv) * D * size + 4 * H + 4 * Hkv * topk),
                "flops": B * (14 * pairs * H * D + scores)}
    lengths, page = _lengths(c), c.get("page")
    rows = 2 * B * H * D * size
    if c["op"] == "decode":
        seen = sum(min(n, -(-n // c["dilation"]), c["taps"]) if c["taps"] else n for n in lengths)
        return {"bytes": rows + 2 * seen * Hkv * D * size, "flops": 4 * seen * H * D}
    held = [-(-n // page) for n in lengths]
    seen = sum(min(n, c["topk"] * page) for n in lengths)
    scored = sum(held)
    return {"bytes": rows + 2 * (seen + scored) * Hkv * D * size + 4 * B * Hkv * c["topk"],
            "flops": 4 * seen * H * D + 4 * scored * Hkv * D}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------

def _exact_softmax(score):
    """Rows of weights of a [rows, n] score with -inf where nothing is seen, and the log of their sums."""
    lse = torch.logsumexp(score, -1, keepdim=True)
    return torch.exp(score - lse), lse


def _exact_choice(score, own_entry, topk):
    """Truth values of the chosen entries of one row set [rows, n]: counts how many beat each entry."""
    n = score.shape[-1]
    score = score.clone()
    if own_entry is not None:
        score[torch.arange(score.shape[0], device=score.device), own_entry] = math.inf
    order = torch.argsort(score, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order)
    rank.scatter_(-1, order, torch.arange(n, device=score.device).expand_as(order).contiguous())
    return (rank < topk) & (score > -math.inf)


def _exact_append(c, s):
    rot, page = c["rot"], c["page"]
    cu, start, table = s["cu"].tolist(), s["start"].tolist(), s["table"].cpu()
    pos = torch.cat([torch.arange(a, a + cu[b + 1] - cu[b]) for b, a in enumerate(start)]).cuda()
    phase = torch.polar(torch.ones_like(s["inv_freq"])[None] * torch.ones_like(pos)[:, None],
                        pos[:, None].double() * s["inv_freq"][None])[:, None]

    def turn(x):
        x = x.double().clone()
        i = torch.arange(rot // 2, device="cuda")
        first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
        z = torch.complex(x[..., first], x[..., second]) * phase
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q, k, v = turn(s["q"]), turn(s["k"]), s["v"].double()
    kp, vp, bounds = s["k_pages"].double(), s["v_pages"].double(), s["bounds"].double()
    ids, ends = [], []
    for b, a in enumerate(start):
        p = pos[cu[b]:cu[b + 1]]
        at = table[b].cuda().long()[p // page]
        kp[at, p % page], vp[at, p % page] = k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]
        end = a + cu[b + 1] - cu[b]
        for w in range(a // page, (end - 1) // page + 1):
            ids.append(int(table[b, w]))
            ends.append(min(page, end - w * page))
    ids, ends = torch.tensor(ids).cuda(), torch.tensor(ends).cuda()
    outside = (torch.arange(page, device="cuda") >= ends[:, None])[:, :, None, None]
    bounds[ids, 0] = kp[ids].masked_fill(outside, math.inf).amin(1)
    bounds[ids, 1] = kp[ids].masked_fill(outside, -math.inf).amax(1)
    return {"query": q, "k_pages": kp, "v_pages": vp, "bounds": bounds}


def _exact_serve(c, s):
    B, H, Hkv, D, page = c["B"], c["H"], c["Hkv"], c["D"], c["page"]
    group = H // Hkv
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        held = s["table"][b, :-(-n // page)].long()
        q = s["q"][b].double()
        for h in range(Hkv):
            mine = q[h * group:(h + 1) * group]
            j = torch.arange(n, device="cuda")
            if c["op"] == "selected":
                lo, hi = s["bounds"][held, 0, h].double(), s["bounds"][held, 1, h].double()
                score = sum(torch.maximum(r * lo, r * hi).sum(-1) for r in mine)[None]
                kept = _exact_choice(score, torch.tensor([(n - 1) // page], device="cuda"), c["topk"])[0]
                j = j[kept[j // page]]
            elif c["taps"]:
                back = n - 1 - j
                j = j[(back % c["dilation"] == 0) & (back // c["dilation"] < c["taps"])]
            k, v = (s[x][held[j // page], j % page, h].double() for x in ("k_pages", "v_pages"))
            weight, _ = _exact_softmax(mine @ k.T / math.sqrt(D))
            out[b, h * group:(h + 1) * group] = weight @ v
    return {"pages": None, "out": out} if c["op"] == "selected" else {"out": out}


def _exact_train(c, s):
    B, S, H, Hkv, D, block = c["B"], c["S"], c["H"], c["Hkv"], c["D"], c["block"]
    group, nb = H // Hkv, -(-S // block)
    zeros = lambda heads: torch.zeros(B, S, heads, D, dtype=torch.float64, device="cuda")  # noqa: E731
    out, dq, dk, dv, lse = zeros(H), zeros(H), zeros(Hkv), zeros(Hkv), torch.zeros(B, S, H, dtype=torch.float64, device="cuda")
    i = torch.arange(S, device="cuda")
    for b in range(B):
        for h in range(Hkv):
            k, v = s["k"][b, :, h].double(), s["v"][b, :, h].double()
            lo = torch.stack([x.amin(0) for x in k.split(block)])
            hi = torch.stack([x.amax(0) for x in k.split(block)])
            heads = range(h * group, (h + 1) * group)
            score = torch.zeros(S, nb, dtype=torch.float64, device="cuda")
            for a in heads:
                q = s["q"][b, :, a].double()
                score += torch.relu(q) @ hi.T - torch.relu(-q) @ lo.T
            if c["causal"]:
                score[torch.arange(nb, device="cuda") > (i // block)[:, None]] = -math.inf
            hidden = ~_exact_choice(score, i // block, c["topk"])[:, i // block]
            if c["causal"]:
                hidden |= i[None] > i[:, None]
            for a in heads:
                q, do = s["q"][b, :, a].double(), s["dout"][b, :, a].double()
                p, l = _exact_softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf))
                o = p @ v
                ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(D)
                out[b, :, a], lse[b, :, a], dq[b, :, a] = o, l[:, 0], ds @ k
                dk[b, :, h] += ds.T @ q
                dv[b, :, h] += p.T @ do
    return {"blocks": None, "out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_train(case, s) if case["op"] == "train" else _exact_serve(case, s)
