"""Draft rows that are not kept: what they leave in the 8-bit cache, and what they do not."""
import numpy as np
import pytest
import torch

from gufo_npu_b200.backend import Context
from tests.test_gpu_cache8 import Pair, attend, check_attend, draw

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HD, KV = 48, 2


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def rows(seed, n, size=1.0):
    return draw(seed, n, KV, HD) * size, draw(seed + 100, n, KV, HD) * size


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("held, draft, accepted", [(37, 4, 1), (37, 4, 0), (30, 8, 1), (30, 8, 4), (47, 3, 1), (33, 30, 2)])
def test_dropped_rows_leave_their_scale_in_their_block(ctx, form, held, draft, accepted):
    """Large draft rows, of which the first few are kept, and smaller rows behind those: to the bit what a cache holds whose scales
    only grow (the reference's), until the block's rows are appended again from its first one on."""
    p, plain = (Pair(ctx, 1, KV, HD, 96, form) for _ in range(2))
    old, large, after = rows(1, held), rows(2, draft, 1000.0), rows(3, 5, 0.5)
    p.append([0], [held], *old)
    p.append([held], [draft], *large)
    kept = held + accepted
    p.append([kept], [5], *after)
    p.same(0, kept + 5)
    # Without the draft: the same, but for the blocks in which dropped rows joined kept ones.
    every = [torch.cat([a, b[:accepted], c]) for a, b, c in zip(old, large, after)]
    plain.append([0], [held], *old)
    for n, at, part in ((accepted, held, [b[:accepted] for b in large]), (5, kept, after)):
        plain.append([at], [n], *part)
    plain.same(0, kept + 5)
    begun = held // 16 * 16                     # ahead of the block in which the draft began
    np.testing.assert_array_equal(p.read(0, 0, kept + 5)[:, :, :begun], plain.read(0, 0, kept + 5)[:, :, :begun])
    # From the block's first row on once more: nothing of the draft is left.
    again = Pair(ctx, 1, KV, HD, 96, form)
    again.append([0], [kept + 5], *every)
    p.append([begun], [kept + 5 - begun], *[x[begun:] for x in every])
    np.testing.assert_array_equal(p.read(0, 0, kept + 5), again.read(0, 0, kept + 5))


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_draft_that_begins_a_block_leaves_nothing(ctx, form):
    p, plain = (Pair(ctx, 1, KV, HD, 96, form) for _ in range(2))
    old, large, after = rows(1, 32), rows(2, 20, 1000.0), rows(3, 7, 0.01)
    for q in (p, plain):
        q.append([0], [32], *old)
    p.append([32], [20], *large)
    for q in (p, plain):
        q.append([32], [7], *after)
    np.testing.assert_array_equal(p.read(0, 0, 39), plain.read(0, 0, 39))


def test_weights_of_a_dropped_draft(ctx):
    """What a draft's queries added to the rows ahead of it stays; its own rows' weights go with the rows that take their place."""
    p = Pair(ctx, 1, KV, HD, 64, "e4m3")
    p.append([0], [30], *rows(1, 30))
    p.append([30], [4], *rows(2, 4))
    q = draw(5, 4, 4, HD).to(DEV)
    given = check_attend(p, [30], [4], q, attend(p, [30], [4], q, accumulate=True))[0]
    # (a weight is off by its score's error, some 1e-5 here, as in test_attend_adds_up_weights: of 4 tokens' 2 heads)
    np.testing.assert_allclose(p.gpu.weights.cpu().numpy()[0], given, rtol=2.0 ** -23, atol=3e-5)
    before = p.gpu.weights.clone()
    p.append([31], [2], *rows(3, 2))
    after = p.gpu.weights.cpu().numpy()[0]
    assert not after[:, 31:33].any()
    np.testing.assert_array_equal(np.delete(after, [31, 32], 1), np.delete(before.cpu().numpy()[0], [31, 32], 1))
