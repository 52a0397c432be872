"""NaN in e4m3 cache rows: which outputs become NaN, for every way a call is cut up, and evictions of such rows."""
import numpy as np
import pytest
import torch

from gufo_npu_b200.backend import Context
from tests import cache8_reference as R
from tests.test_gpu_cache8 import Pair, attend, check_evict, draw, evict

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAN = float("nan")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def check(p, tokens, q, out, visible):
    """NaN where the definition has NaN, and nowhere else; the other values within the bound."""
    at = 0
    for slot, n in enumerate(tokens):
        for _ in range(n):
            want, _, size, mass = p.ref.attend(slot, visible[at], q[at].cpu().numpy(), p.head_dim ** -0.5)
            bound = R.attend_bound(size, mass, visible[at], p.head_dim)
            assert np.array_equal(np.isnan(out[at]), np.isnan(want)), (slot, at)
            there = ~np.isnan(want)
            assert np.all(np.abs(out[at] - want)[there] <= bound[there]), (slot, at)
            at += 1


@pytest.mark.parametrize("capacity", [320, 1040, 4112])     # a block a unit, a cluster, shared out
@pytest.mark.parametrize("group, most", [(1, 3), (4, 4), (8, 5)])     # up to 3, 16 and 40 query rows
@pytest.mark.parametrize("head_dim", [16, 64, 80, 112, 144, 192, 208, 256])
def test_only_queries_that_see_a_nan_get_it(ctx, head_dim, group, most, capacity):
    """Single values that are NaN, in the first and the last piece of a head and between, of rows in the middle of blocks and
    behind what any query sees; a key that is NaN; other heads and sequences have none."""
    kv, rows = 2, 300
    p = Pair(ctx, 2, kv, head_dim, capacity, "e4m3", weights=False)
    k, v = draw(1, 2 * rows, kv, head_dim), draw(2, 2 * rows, kv, head_dim)
    for row, dim in ((5, head_dim // 2), (200, 3), (200, head_dim - 2), (203, head_dim - 1), (207, 0), (259, head_dim // 3), (265, 1), (290, 2)):
        v[row, 0, dim] = NAN
    k[rows + 100, 1, 4] = NAN
    p.append([0, 0], [rows, rows], k, v)
    tokens = [most, 3]
    q = draw(5, most + 3, kv * group, head_dim).to(DEV) * 1.5
    seen = [4, 201, 203, 260, 264][5 - most:] + [100, 101, 300]
    check(p, tokens, q, attend(p, [0, 0], tokens, q, visible=seen), seen)
    seen = [200, 5, 207, 300, 208][:most] + [0, 300, 99]
    check(p, tokens, q, attend(p, [0, 0], tokens, q, visible=seen), seen)
    # What is hidden is as it was: the NaN stay in the cache.
    p.same(0, rows)
    p.same(1, rows)


@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("head_dim", [32, 80, 256])
def test_evict_of_rows_with_nan(ctx, other, head_dim):
    """Rows with NaN gathered beside rows of larger and smaller scales: NaN they stay, and count for nothing in the scale."""
    p = Pair(ctx, 1, 2, head_dim, 112, "e4m3")
    x = draw(1, 110, 2, head_dim)
    x[16:32] *= 2.0 ** 20
    x[48:64] *= 2.0 ** -20
    x[5, 0, 7] = x[20, 0, head_dim - 1] = x[21, 1, 0] = x[55, 0, 9] = x[100, 1, 3] = NAN
    x[80:96] = NAN                         # a block of nothing else
    p.append([0], [110], x, -x)
    w = torch.zeros(1, 2, 112)
    w[0, 0, [5, 6, 20, 50, 55, 56, 85, 101]] = 1.0
    w[0, 1, [0, 17, 21, 60, 84, 85, 100, 109]] = 1.0
    p.gpu.weights.copy_(w)
    torch.cuda.synchronize()
    p.ref.weights[:] = w.numpy()
    into = Pair(ctx, 1, 2, head_dim, 64, "e4m3") if other else None
    check_evict(p, [110], 50, 2, 5, evict(p, [110], 50, 2, 5, into=into), into=into)
    if not other:
        check_evict(p, [50], 9, 0, 1, evict(p, [50], 9, 0, 1))
