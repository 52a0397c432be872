"""Append, attention with weights and eviction captured together, the row counts staying on the device."""
import numpy as np
import pytest
import torch

from gufo_npu_b200.backend import Context
from gufo_npu_b200.cache8 import CudaCache8
from tests.test_gpu_cache8 import draw, ints

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
KV, HEADS, HD, CAPACITY, BUDGET = 2, 8, 96, 160, 100


class Layer:
    """A layer's step under a budget: the counts that the eviction leaves are those that the next step starts at."""

    def __init__(self, ctx, form, into):
        self.ctx = ctx
        self.cache = CudaCache8(ctx, 3, KV, HD, CAPACITY, format=form, weights=True)
        self.into = CudaCache8(ctx, 4, KV, HD, BUDGET // 16 * 16 + 16, format=form, weights=True) if into else None
        self.tokens = [4, 1, 7]
        n = sum(self.tokens)
        self.k, self.v = draw(1, n, KV, HD).to(DEV), draw(2, n, KV, HD).to(DEV)
        self.q, self.out = draw(3, n, HEADS, HD).to(DEV), torch.empty(n, HEADS, HD, device=DEV)
        self.held, self.total, self.left = ints(97, 40, 0), ints(0, 0, 0), ints(0, 0, 0)
        self.kept = torch.zeros(3, KV, BUDGET, dtype=torch.int32, device=DEV)
        self.counts = ints(*self.tokens)
        self.batch, self.all = self.cache.batch(self.held, self.tokens), self.cache.batch(self.total)
        self.scratch = self.cache.scratch(HEADS, n, accumulate=True)
        first, rows = draw(4, 97 + 40, KV, HD).to(DEV), self.cache.batch(ints(0, 0), [97, 40])
        torch.cuda.synchronize()
        self.cache.append_device(rows, first, first)
        ctx.synchronize()

    def step(self):
        """On torch's current stream, which is the context's."""
        self.cache.append_device(self.batch, self.k, self.v)
        self.cache.attend_device(self.batch, self.q, self.out, self.scratch, accumulate=True)
        torch.add(self.held, self.counts, out=self.total)
        self.cache.evict_device(self.all, BUDGET, self.kept, first=2, last=9, held=self.left, into=self.into,
                                into_slots=[3, 0, 1] if self.into else None)
        if not self.into:
            self.held.copy_(self.left)

    def state(self):
        cache, slots = (self.into, [3, 0, 1]) if self.into else (self.cache, None)
        rows = torch.empty(2, 3 * 96, KV, HD, device=DEV)
        cache.rows_device(cache.batch(ints(0, 0, 0), [96] * 3, slots), rows[0], rows[1])
        self.ctx.synchronize()
        some = self.left.tolist()
        rows = rows.view(2, 3, 96, KV, HD)
        whole = [rows[:, i, :n] for i, n in enumerate(some)] + [cache.weights[slots[i] if slots else i, :, :n] for i, n in enumerate(some)]
        return [x.cpu().numpy() for x in whole + [self.out, self.kept, self.left]]


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_captured_steps_under_a_budget(form, into):
    """Replays give what single calls give, to the bit, and two streams' replays do not meet."""
    layers = []
    for _ in range(3):
        s = torch.cuda.Stream()
        layers.append((Layer(Context(0, s.cuda_stream), form, into), s))
    (plain, s0), replayed = layers[0], layers[1:]
    torch.cuda.synchronize()
    graphs = []
    for layer, s in replayed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            layer.step()
        graphs.append(graph)
    for _ in range(6):
        with torch.cuda.stream(s0):
            plain.step()
        for graph, (_, s) in zip(graphs, replayed):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = plain.state()
        assert plain.left.tolist()[0] == BUDGET
        for layer, _ in replayed:
            for a, b in zip(layer.state(), want):
                np.testing.assert_array_equal(a, b)
        torch.cuda.synchronize()
    del graphs
    for layer, _ in layers:
        layer.ctx.close()
