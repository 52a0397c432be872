"""Rotary positions on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

from gufo_npu_b200._capi import GufoCudaError
from gufo_npu_b200.backend import Context
from tests import cache8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def draw(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def turned(ctx, rope, parts, positions, eps=0.0):
    torch.cuda.synchronize()
    ctx.rope_device(rope, ctx.rope_parts(parts, rms_eps=eps), positions)
    ctx.synchronize()


def check(x, got, positions, freq, layout, magnitude=1.0, norm=None, eps=0.0):
    """A sine or cosine of sincospif is off by a step or so of 1 (2^-22), its argument by half a step of an eighth of
    a turn, the products and the sum by half a step each; the magnitude's and a norm's factors (an 8-value sum a lane, a
    root, a quotient, two products) by half a step an operation: 32 halves of a step in all."""
    want, size = R.rope(x.cpu().numpy(), positions.tolist(), freq, layout, magnitude, None if norm is None else norm.cpu().numpy(), eps)
    assert np.all(np.abs(got.cpu().numpy() - want) <= 32 * 2.0 ** -24 * size + 1e-37)


POSITIONS = [0, 1, -5, 17, 32767, 1000003, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rope_dim, head_dim, heads", [
    (2, 2, 3), (16, 16, 1), (10, 14, 5), (64, 256, 8), (80, 80, 6), (64, 64, 33), (104, 112, 5), (128, 512, 2), (512, 512, 3),
    (254, 256, 1), (72, 96, 20)])
def test_matches_the_definition(ctx, layout, norm, rope_dim, head_dim, heads):
    x = draw(rope_dim + heads, len(POSITIONS), heads, head_dim) * 3
    at = torch.tensor(POSITIONS, dtype=torch.int32, device=DEV)
    w = draw(1, head_dim) if norm else None
    y = torch.full_like(x, float("nan"))
    rope = ctx.rope_create(rope_dim, theta=1e7, layout=layout)
    turned(ctx, rope, [(x, y, w)], at, 1e-6)
    # (far positions: the reference multiplies in 64 bits, so the angles of its largest, 2^31, are 2^-22 off at most)
    want, size = R.rope(x.cpu().numpy(), POSITIONS, R.frequencies(rope_dim, 1e7), layout, 1.0, None if w is None else w.cpu().numpy(), 1e-6)
    assert np.all(np.abs(y.cpu().numpy() - want) <= (32 * 2.0 ** -24 + 2.0 ** -22) * size)
    ctx.rope_free(rope)


@pytest.mark.parametrize("scaling, more", [("linear", {"factor": 4.0}), ("by_parts", {"factor": 8.0, "original": 32768.0})])
def test_scalings(ctx, scaling, more):
    kw = {"original_positions" if k == "original" else k: v for k, v in more.items()}
    rope = ctx.rope_create(64, theta=1e7, scaling=scaling, magnitude=1.25, **kw)
    x, at = draw(3, 50, 2, 96), torch.arange(0, 50 * 5000, 5000, dtype=torch.int32, device=DEV)
    y = torch.empty_like(x)
    turned(ctx, rope, [(x, y, None)], at)
    check(x, y, at, R.frequencies(64, 1e7, scaling, **more), "halves", 1.25)
    assert torch.equal(x[:, :, 64:], y[:, :, 64:])
    ctx.rope_free(rope)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_rows_of_an_input_product(ctx, offset, tokens):
    """Queries and keys where the attention layer's product leaves them (each head's query and gate, keys, values), in
    one call, the queries in place; at an odd address too. What lies between them stays."""
    heads, kv, hd, width = 8, 2, 128, 2 * 8 * 128 + 2 * 2 * 128
    flat = draw(tokens + offset, tokens * width + 1)
    before = flat.clone()
    rows = flat[offset:offset + tokens * width].view(tokens, width)
    q = rows[:, :2 * heads * hd].view(tokens, heads, 2, hd)[:, :, 0]
    k = rows[:, 2 * heads * hd:2 * heads * hd + kv * hd].view(tokens, kv, hd)
    out = torch.empty(tokens, kv, hd, device=DEV)
    wq, wk = draw(5, hd), draw(6, hd)
    at = torch.arange(tokens, dtype=torch.int32, device=DEV) + 100000
    old = q.clone()
    rope = ctx.rope_create(32, theta=1e6, layout="pairs")
    turned(ctx, rope, [(q, q, wq), (k, out, wk)], at, 1e-6)
    check(old, q, at, R.frequencies(32, 1e6), "pairs", norm=wq, eps=1e-6)
    check(k, out, at, R.frequencies(32, 1e6), "pairs", norm=wk, eps=1e-6)
    was = before[offset:offset + tokens * width].view(tokens, width)
    assert torch.equal(rows[:, 2 * heads * hd:], was[:, 2 * heads * hd:])
    assert torch.equal(rows[:, :2 * heads * hd].view(tokens, heads, 2, hd)[:, :, 1], was[:, :2 * heads * hd].view(tokens, heads, 2, hd)[:, :, 1])
    ctx.rope_free(rope)


def test_parts_of_different_widths(ctx):
    """Four parts of different heads and widths, a row of one of them empty of numbers."""
    parts, kept = [], []
    at = torch.tensor([5, 6, 70000], dtype=torch.int32, device=DEV)
    for i, (heads, hd) in enumerate([(3, 64), (1, 34), (17, 256), (2, 500)]):
        x = draw(20 + i, 3, heads, hd)
        y = torch.empty_like(x)
        parts.append((x, y, draw(30 + i, hd) if i % 2 else None))
    parts[0][0][1, 2] = float("nan")
    parts[2][0][0, 0, 40] = float("inf")       # passed on, and nobody else's
    rope = ctx.rope_create(34, theta=1e4)
    turned(ctx, rope, parts, at, 1e-5)
    freq = R.frequencies(34, 1e4)
    for i, (x, y, w) in enumerate(parts):
        if i == 0:
            assert torch.isnan(y[1, 2]).all() and int(torch.isnan(y).sum()) == 64
            x, y = x[::2], y[::2]
            check(x, y, at[::2], freq, "halves")
        elif i == 2:
            assert y[0, 0, 40] == float("inf") and int(torch.isfinite(y).logical_not().sum()) == 1
            check(x[1:], y[1:], at[1:], freq, "halves")
        else:
            check(x, y, at, freq, "halves", norm=w, eps=1e-5)
    ctx.rope_free(rope)


def test_captured_call_follows_positions(ctx):
    x, y = draw(9, 4, 2, 64), torch.empty(4, 2, 64, device=DEV)
    at = torch.zeros(4, dtype=torch.int32, device=DEV)
    s = torch.cuda.Stream()
    c = Context(0, s.cuda_stream)
    rope = c.rope_create(64, theta=1e4)
    parts = c.rope_parts([(x, y, None)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.rope_device(rope, parts, at)
    for first in (7, 90000):
        at.copy_(torch.arange(first, first + 4))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(x, y, at, R.frequencies(64, 1e4), "halves")
    del graph
    c.close()


def test_refusals(ctx):
    x = draw(1, 2, 3, 64)
    at = torch.zeros(2, dtype=torch.int32, device=DEV)
    rope = ctx.rope_create(32)
    before = ctx.launch_count()

    def refused(status, rope, parts, positions=at, edit=None):
        arr = ctx.rope_parts(parts)
        if edit:
            edit(arr[0])
        with pytest.raises(GufoCudaError) as e:
            ctx.rope_device(rope, arr, positions)
        assert e.value.status == status
    refused(1, 12345, [(x, x, None)])
    refused(1, rope, [(x, x, None)] * 5)
    refused(2, rope, [(x[:, :, :30], x[:, :, :30], None)])
    refused(2, rope, [(x[:, :, :33], x[:, :, :33], None)])
    refused(2, rope, [(draw(1, 2, 1, 514), draw(1, 2, 1, 514), None)])
    for field, value in (("in_", None), ("out", None), ("out_head_stride", 5)):
        refused(1, rope, [(x, x, None)], edit=lambda p: setattr(p, field, value))
    refused(2, rope, [(x, x, None)], edit=lambda p: setattr(p, "heads", 0))
    for parts in ([(x.double(), x, None)], [(x, x.cpu(), None)], [(x[0], x[0], None)], [(x, x[:, :2], None)],
                  [(x[:, :, ::2], x[:, :, ::2], None)], [(x, x, draw(1, 63))]):
        with pytest.raises(ValueError):
            ctx.rope_parts(parts)
    for positions in (at.long(), at.cpu(), torch.zeros(3, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError):
            ctx.rope_device(rope, ctx.rope_parts([(x, x, None)]), positions)
    with pytest.raises(GufoCudaError):
        ctx.rope_create(7)
    # No tokens: nothing to do.
    ctx.rope_device(rope, ctx.rope_parts([(x[:0], x[:0], None)]), at[:0])
    assert ctx.launch_count() == before
    ctx.rope_free(rope)
    with pytest.raises(GufoCudaError):
        ctx.rope_free(rope)
