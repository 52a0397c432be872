"""Attention calls over the 8-bit cache with very many query rows: what is taken, and what is refused as a whole."""
import ctypes as C

import numpy as np
import pytest
import torch

from gufo_npu_b200._capi import GufoCudaError
from gufo_npu_b200.backend import Context
from gufo_npu_b200.cache8 import CudaCache8
from tests import cache8_reference as R
from tests.test_gpu_cache8 import Pair, ints

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HD = 16
TOO_LARGE = 7


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def queries(seed, rows, heads):
    return torch.randn(rows, heads, HD, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)) * 1.5


@pytest.mark.parametrize("heads, tokens, capacity", [(4096, 520, 528), (2048, 1030, 1040)])
def test_many_query_heads_of_one_kv_head(ctx, heads, tokens, capacity):
    """Two million query rows of a sequence: a block a group of rows, and shared out."""
    p = Pair(ctx, 1, 1, HD, capacity, "e4m3", weights=False)
    p.fill([tokens])
    q = queries(3, tokens, heads)
    out = torch.full_like(q, float("nan"))
    scratch = p.gpu.scratch(heads, tokens)
    batch = p.gpu.batch(ints(0), [tokens])
    torch.cuda.synchronize()
    p.gpu.attend_device(batch, q, out, scratch)
    ctx.synchronize()
    assert bool(torch.isfinite(out).all())
    some = [0, 1, 7, heads // 2, heads - 1]
    for t in (0, 1, 15, 16, 300, tokens - 2, tokens - 1):
        want, _, size, mass = p.ref.attend(0, t + 1, q[t, some].cpu().numpy(), HD ** -0.5)
        assert np.all(np.abs(out[t, some].cpu().numpy() - want) <= R.attend_bound(size, mass, t + 1, HD)), t


def test_sequences_that_are_too_many_together(ctx):
    """Seventeen sequences of a long cache whose query rows are more than a launch takes, each of them fewer."""
    n, heads, capacity, rows = 17, 65536, 1 << 20, 40
    cache = CudaCache8(ctx, n, 1, HD, capacity)
    p = Pair(ctx, n, 1, HD, 48, "e4m3", weights=False)
    k, v = (torch.randn(n * rows, 1, HD, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    p.append([0] * n, [rows] * n, k, v)
    kd, vd, q = k.to(DEV), v.to(DEV), queries(3, n, heads)
    out = torch.full_like(q, float("nan"))
    scratch = cache.scratch(heads, n)
    start, at = ints(*[0] * n), ints(*[rows - 1] * n)
    torch.cuda.synchronize()
    cache.append_device(cache.batch(start, [rows] * n), kd, vd)
    cache.attend_device(cache.batch(at), q, out, scratch)
    ctx.synchronize()
    some = [0, 31, 32, heads - 1]
    for i in range(n):
        want, _, size, mass = p.ref.attend(i, rows, q[i, some].cpu().numpy(), HD ** -0.5)
        assert np.all(np.abs(out[i, some].cpu().numpy() - want) <= R.attend_bound(size, mass, rows, HD)), i
    cache.close()


def test_a_sequence_that_is_too_large_refuses_the_whole_call(ctx):
    """The last of 129 sequences has more query rows than a launch takes: nothing runs, not the first 128 either."""
    n, heads, capacity, last = 129, 8000, 1 << 20, 132
    cache = CudaCache8(ctx, n, 1, HD, capacity)
    tokens = [1] * (n - 1) + [last]
    q = torch.zeros(sum(tokens), heads, HD, device=DEV)
    out = torch.full_like(q, 7.0)
    scratch = cache.scratch(heads, sum(tokens))
    batch = cache.batch(torch.zeros(n, dtype=torch.int32, device=DEV), tokens)
    torch.cuda.synchronize()
    before = ctx.launch_count()
    with pytest.raises(GufoCudaError) as e:
        cache.attend_device(batch, q, out, scratch)
    assert e.value.status == TOO_LARGE
    ctx.synchronize()
    assert ctx.launch_count() == before and bool((out == 7.0).all())
    # 131 tokens are the most of a sequence (2^31 / (capacity / 16 + 17) groups of 32 rows): scratch for more is for nobody.
    size = C.c_size_t()
    for count, status in ((131 * n, 0), (131 * n + 1, TOO_LARGE)):
        assert ctx.lib.gufo_cuda_cache8_attend_scratch(ctx.handle, cache.handle, heads, count, 0, C.byref(size)) == status
    cache.close()
