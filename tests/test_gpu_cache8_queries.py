"""Attention over int8 keys whose channels differ widely, with queries that are inverse to them."""
import numpy as np
import pytest
import torch

from gufo_npu_b200.backend import Context
from tests import cache8_reference as R
from tests.test_gpu_cache8 import Pair, attend

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("capacity", [512, 2064])      # a block or a cluster a unit, shared out
@pytest.mark.parametrize("heads, head_dim, tokens", [(4, 64, 1), (4, 80, 2), (8, 128, 1), (4, 192, 4), (16, 256, 2), (4, 256, 1)])
@pytest.mark.parametrize("part, ratio", [(1, 1), (32, 100), (2, 1000)])
def test_small_query_values_meet_large_key_channels(ctx, part, ratio, heads, head_dim, tokens, capacity):
    """One channel in `part` is `ratio` times the others in the keys, and as much smaller in the queries: what the small values
    add to a score is as much as the large ones do, and keeps its bits."""
    rows = 500
    g = torch.Generator().manual_seed(head_dim + ratio)
    channels = torch.ones(head_dim)
    channels[torch.randperm(head_dim, generator=g)[:max(head_dim // part, 1)]] = ratio
    k, v = torch.randn(rows, 1, head_dim, generator=g) * channels, torch.randn(rows, 1, head_dim, generator=g)
    q = torch.randn(tokens, heads, head_dim, generator=g) * 1.5 / channels
    p = Pair(ctx, 1, 1, head_dim, capacity, "int8")
    p.append([0], [rows], k, v)
    out = attend(p, [rows - tokens], [tokens], q.to(DEV))
    keys, values = (p.ref.values(side, 0, 0, rows) for side in range(2))
    for t in range(tokens):
        seen = rows - tokens + t + 1
        for h in range(heads):
            x = q[t, h].double().numpy()
            s = keys[:seen] @ x * head_dim ** -0.5
            w = np.exp(s - s.max())
            w /= w.sum()
            # Queries: whole numbers, the largest 2^29 or more, each half of one off; sums of those are exact. Scores:
            # three roundings of what the digits add up to, two products, and two roundings in the scale. Then as in
            # attend_bound: the score's error twice, 2^-20 for the weights, additions, and 2^-40 of every value.
            score = 2.0 ** -30 * np.abs(x).max() * np.abs(keys[:seen]).sum(1).max() * head_dim ** -0.5 + 8 * 2.0 ** -24 * np.abs(s).max()
            bound = (2 * score + 2.0 ** -20 + (seen / 16 + 64) * 2.0 ** -24) * (w @ np.abs(values[:seen])) \
                + 2.0 ** -40 * np.abs(values[:seen]).sum(0)
            err = np.abs(out[t, h] - w @ values[:seen])
            assert np.all(err <= bound), (t, h, float((err / bound).max()))
