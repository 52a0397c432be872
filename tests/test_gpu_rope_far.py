"""Rotary positions far from the first ones, against sines and cosines of angles in 60 decimal digits."""
import decimal
import math

import numpy as np
import pytest
import torch

from gufo_npu_b200.backend import Context

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
POSITIONS = [1, 1000003, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 - 98765, -2 ** 31]
TWO_PI = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


@pytest.mark.parametrize("rope_dim, theta, factor", [(512, 10000000, 1), (128, 10000, 1), (256, 500000, 8), (64, 1000000, 0.25)])
def test_angles_of_far_positions(rope_dim, theta, factor):
    ctx = Context(0)
    pairs = rope_dim // 2
    x = torch.zeros(len(POSITIONS), 1, rope_dim, device=DEV)
    x[:, :, :pairs] = 1.0           # (1, 0): what comes out is the cosine and the sine
    y = torch.empty_like(x)
    at = torch.tensor(POSITIONS, dtype=torch.int32, device=DEV)
    rope = ctx.rope_create(rope_dim, theta=theta, scaling="linear", factor=factor)
    torch.cuda.synchronize()
    ctx.rope_device(rope, ctx.rope_parts([(x, y, None)]), at)
    ctx.synchronize()
    got = y.cpu().numpy().astype(np.float64)
    with decimal.localcontext() as c:
        c.prec = 60
        turns = [[float(p * decimal.Decimal(theta) ** (decimal.Decimal(-i) / pairs) / decimal.Decimal(factor) / TWO_PI % 1)
                  for i in range(pairs)] for p in POSITIONS]
    angle = 2 * math.pi * np.array(turns)
    # A step of sincospif's results (2^-24: below 1), its argument's half step at a quarter of a half turn (2^-27 half turns),
    # and the angle: half of 2^-64 of a turn and two roundings of 64 bits of a frequency of at most 2/3 of a turn here, times
    # the position.
    bound = 2.0 ** -24 + math.pi * 2.0 ** -27 + 2 * math.pi * 2.0 ** 31 * (2.0 ** -65 + 2 * 2.0 ** -64 * 2 / 3)
    worst = max(float(np.abs(got[:, 0, :pairs] - np.cos(angle)).max()), float(np.abs(got[:, 0, pairs:] - np.sin(angle)).max()))
    assert worst <= bound, (worst, bound)
    ctx.rope_free(rope)
    ctx.close()
