"""Serving and training steps of the cache and selection operators captured into CUDA graphs, replayed on new data, from two
threads, and beside another graph."""
import threading

import pytest
import torch

import ma_transformer_b200 as mt
from ma_transformer_b200 import _native as nat
from ma_transformer_b200 import paged_attention as paged

pytestmark = pytest.mark.gpu


class Served:
    """One token for each of B sequences: append with rotation, selection, attention over the pages and over everything."""

    def __init__(self, B, H, Hkv, D, page, width, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        self.shape, self.dtype, self.g = (B, H, Hkv, D), dtype, g
        self.cache = mt.PagedKVCache(B * width, page, Hkv, D, dtype, key_bounds=True)
        self.table = torch.randperm(B * width, generator=g).view(B, width).int().cuda()
        self.freq = mt.rotary_frequencies(D)
        self.start = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.q, self.k, self.v = (torch.empty(B, h, D, dtype=dtype, device="cuda") for h in (H, Hkv, Hkv))

    def new_tokens(self, at):
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=self.g).to(self.dtype))
        self.start.copy_(torch.arange(self.start.shape[0]) % 3 + at)

    def step(self):
        lengths = self.start + 1
        q = paged.append(self.cache, self.k, self.v, self.table, self.start, query=self.q, inv_freq=self.freq)
        pages = paged.select_pages(q, self.cache, self.table, lengths, 3)
        return [q, pages, paged.decode(q, self.cache, self.table, lengths, pages=pages), paged.decode(q, self.cache, self.table, lengths)]


@pytest.mark.parametrize("B, dtype", [(2, torch.bfloat16), (40, torch.float16), (2, torch.float32)])
def test_a_captured_serving_step_replays_on_new_tokens(B, dtype):
    eager, captured = (Served(B, 8, 4, 64, 16, 8, dtype, 71) for _ in range(2))
    eager.new_tokens(0), captured.new_tokens(0)
    eager.step()
    captured.step()                                       # loads the kernels; appends the same tokens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step()
    for at in range(0, 60):
        eager.new_tokens(at), captured.new_tokens(at)
        want = eager.step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), at
    for a, b in ((eager.cache.k, captured.cache.k), (eager.cache.v, captured.cache.v), (eager.cache.key_bounds, captured.cache.key_bounds)):
        assert torch.equal(a, b)
    assert nat.device_status() == 0


def test_two_threads_serve_on_streams_of_their_own():
    both = [Served(3, 8, 4, 64, 16, 8, torch.bfloat16, 72 + i) for i in range(2)]
    alone = [Served(3, 8, 4, 64, 16, 8, torch.bfloat16, 72 + i) for i in range(2)]
    got, want = [[], []], [[], []]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for at in range(40):
                both[i].new_tokens(at)
                got[i].append(both[i].step())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        for at in range(40):
            alone[i].new_tokens(at)
            want[i].append(alone[i].step())
        for at, (a, b) in enumerate(zip(got[i], want[i])):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), (i, at)


@pytest.mark.parametrize("dtype, S, D, block", [(torch.bfloat16, 300, 64, 64), (torch.float16, 300, 80, 16), (torch.float32, 300, 64, 32)])
def test_a_captured_training_step_replays_on_new_inputs(dtype, S, D, block):
    g = torch.Generator().manual_seed(73)
    fresh = lambda: [torch.randn(1, S, h, D, generator=g).to(dtype).cuda() for h in (4, 2, 2, 4)]  # noqa: E731
    leaves = [t.requires_grad_(True) for t in fresh()[:3]]
    dout = fresh()[3]

    def step(x, grad):
        out = mt.selected_block_attention(*x, block, 4)
        return [out.detach(), *torch.autograd.grad(out, x, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaves, dout)
    for _ in range(3):
        new = fresh()
        with torch.no_grad():
            for a, b in zip((*leaves, dout), new):
                a.copy_(b)
        graph.replay()
        want = step([t.clone().requires_grad_(True) for t in new[:3]], new[3])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
