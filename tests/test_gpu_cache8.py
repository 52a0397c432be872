"""The 8-bit key / value cache on the GPU: append, rows, attention and eviction against their
definitions in 64 bits (tests/cache8_reference.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

from gufo_npu_b200._capi import GufoCudaError
from gufo_npu_b200.backend import Context
from gufo_npu_b200.cache8 import CudaCache8
from tests import cache8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def draw(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(shape[-1], generator=g))


class Pair:
    """A cache on the GPU and the reference of it."""

    def __init__(self, ctx, slots, kv_heads, head_dim, capacity, form, weights=True):
        self.ctx, self.form = ctx, form
        self.gpu = CudaCache8(ctx, slots, kv_heads, head_dim, capacity, format=form, weights=weights)
        self.ref = R.Cache(slots, kv_heads, head_dim, capacity, form)
        self.slots, self.kv_heads, self.head_dim, self.capacity = slots, kv_heads, head_dim, capacity

    def append(self, positions, tokens, keys, values, slots=None):
        """keys, values: [sum of tokens, kv_heads, head_dim] on the CPU."""
        k, v = keys.to(DEV), values.to(DEV)
        torch.cuda.synchronize()
        self.gpu.append_device(self.gpu.batch(ints(*positions), tokens, slots), k, v)
        self.ctx.synchronize()
        at = 0
        for i, (p, n) in enumerate(zip(positions, tokens)):
            if n:
                self.ref.append(i if slots is None else slots[i], p, (keys[at:at + n].numpy(), values[at:at + n].numpy()))
            at += n

    def fill(self, lengths, seed=1):
        n = sum(lengths)
        self.append([0] * len(lengths), lengths, draw(seed, n, self.kv_heads, self.head_dim), draw(seed + 1, n, self.kv_heads, self.head_dim))

    def read(self, slot, first, rows):
        """Keys and values of rows of a slot: [2, kv_heads, rows, head_dim] (the GPU's)."""
        out = torch.full((2, rows, self.kv_heads, self.head_dim), float("nan"), device=DEV)
        torch.cuda.synchronize()
        self.gpu.rows_device(self.gpu.batch(ints(first), [rows], [slot]), out[0], out[1])
        self.ctx.synchronize()
        return out.permute(0, 2, 1, 3).cpu().numpy()

    def same(self, slot, rows):
        """Whether the first rows of a slot are the reference's, to the bit."""
        got = self.read(slot, 0, rows)
        for side in range(2):
            for h in range(self.kv_heads):
                want = self.ref.values(side, slot, h, rows)
                np.testing.assert_array_equal(got[side, h], want, err_msg=f"side {side}, slot {slot}, head {h}")


# ---- append and rows --------------------------------------------------------------------


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("head_dim, kv_heads", [(16, 3), (80, 2), (128, 1), (192, 1), (256, 2)])
def test_append_matches_the_definition(ctx, form, head_dim, kv_heads):
    """Ragged appends one behind another, in slots of any order: blocks that begin, fill up, span several; scales that grow."""
    p = Pair(ctx, 5, kv_heads, head_dim, 96, form)
    held = [0] * 5
    for call, (slots, tokens) in enumerate([([0, 1, 2, 3, 4], [1, 15, 16, 17, 0]), ([3, 0, 4], [1, 30, 40]),
                                            ([1, 2], [1, 33]), ([0, 1, 2, 3, 4], [2, 2, 2, 2, 2])]):
        n = sum(tokens)
        # Each call's rows are larger than the last one's, some much.
        k = draw(10 * call, n, kv_heads, head_dim) * 2.0 ** (1.5 * call)
        v = draw(10 * call + 1, n, kv_heads, head_dim) * 2.0 ** (4 * (call % 2))
        p.append([held[s] for s in slots], tokens, k, v, slots)
        for s, t in zip(slots, tokens):
            held[s] += t
        for s in range(5):
            if held[s]:
                p.same(s, held[s])


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_append_of_extreme_values(ctx, form):
    """Nothing but zeros, the smallest numbers, the largest, infinities, NaN; largest codes and ties."""
    hd = 32
    most = R.MOST[form]
    rows = torch.zeros(8 * 16, 1, hd)
    rows[16:32] = 1e-45 * torch.arange(1, hd + 1)
    rows[32:48] = torch.linspace(-3.4e38, 3.4e38, hd)
    rows[48, 0, 3], rows[49, 0, 4], rows[50, 0, 5] = float("inf"), float("-inf"), 1.0
    rows[64:80] = torch.randn(16, 1, hd, generator=torch.Generator().manual_seed(1))
    rows[66, 0, 7] = float("nan")
    rows[80:96] = torch.linspace(-most, most, hd)            # exactly the largest code: the scale is 1
    rows[96:112] = torch.linspace(-most * 1.001, most * 1.001, hd)
    rows[112:128] = torch.arange(hd) * 0.5 - 8               # halves: ties of int8
    rows[127, 0, 0] = most
    p = Pair(ctx, 1, 1, hd, 128, form)
    p.append([0], [128], rows, -rows)
    p.same(0, 128)
    got = p.read(0, 0, 128)
    assert np.isnan(got).sum() == (2 * int(torch.isnan(rows).sum()) if form == "e4m3" else 0)
    # Row by row, larger than before each time: the codes there are rounded again.
    q = Pair(ctx, 1, 1, hd, 16, form)
    for r in range(16):
        x = draw(r, 1, 1, hd) * 1.9 ** r
        q.append([r], [1], x, x * 2.0 ** (-10 * (r % 2)))
        q.same(0, r + 1)


@pytest.mark.parametrize("position, tokens", [(60, 10), (64, 5), (70, 3), (-3, 10), (-20, 5), (2 ** 31 - 1, 4), (-2 ** 31, 4), (2 ** 31 - 30, 64)])
def test_append_outside_is_left_out(ctx, position, tokens):
    p = Pair(ctx, 3, 2, 64, 64, "e4m3")
    p.fill([64, 64, 64])
    before = [p.read(s, 0, 64) for s in range(3)]
    k, v = draw(5, tokens, 2, 64) * 0.01, draw(6, tokens, 2, 64) * 0.01
    p.append([position], [tokens], k, v, [1])
    for s in (0, 2):
        np.testing.assert_array_equal(p.read(s, 0, 64), before[s])
    p.same(1, 64)
    if position >= 64 or position + tokens <= 0:
        np.testing.assert_array_equal(p.read(1, 0, 64), before[1])


def test_append_takes_rows_as_they_lie(ctx):
    """Keys and values inside rows of an input product, at odd addresses, and a head's stride of its own."""
    flat = draw(3, 1, 20 * (7 * 48 + 1) + 1).to(DEV).view(-1)
    rows = flat[1:1 + 20 * (7 * 48 + 1)].view(20, 7 * 48 + 1)
    k = rows[:, :4 * 48].view(20, 2, 2, 48)[:, :, 1]
    v = rows[:, 4 * 48:6 * 48].view(20, 2, 48)
    p = Pair(ctx, 1, 2, 48, 32, "int8")
    torch.cuda.synchronize()
    p.gpu.append_device(p.gpu.batch(ints(3), [20]), k, v)
    p.ctx.synchronize()
    p.ref.append(0, 3, (k.cpu().numpy(), v.cpu().numpy()))
    got = p.read(0, 3, 20)
    for side in range(2):
        for h in range(2):
            np.testing.assert_array_equal(got[side, h], p.ref.values(side, 0, h, 23)[3:])


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("head_dim, kv_heads", [(16, 8), (48, 5), (112, 3), (64, 32), (128, 16)])
def test_rows_of_many_heads(ctx, form, head_dim, kv_heads):
    """Ragged appends and reads of many heads: whole blocks written together, rows read from inside a block."""
    p = Pair(ctx, 3, kv_heads, head_dim, 96, form)
    tokens = [90, 37, 16]
    n = sum(tokens)
    p.append([5, 0, 40], tokens, draw(1, n, kv_heads, head_dim), draw(2, n, kv_heads, head_dim), [1, 2, 0])
    first, count, slots = [3, 20, 41], [60, 17, 14], [1, 2, 0]
    total = sum(count)
    out = torch.full((2, total, kv_heads, head_dim), float("nan"), device=DEV)
    torch.cuda.synchronize()
    p.gpu.rows_device(p.gpu.batch(ints(*first), count, slots), out[0], out[1])
    ctx.synchronize()
    got, at = out.cpu().numpy(), 0
    for f, c, s in zip(first, count, slots):
        for side in range(2):
            for h in range(kv_heads):
                np.testing.assert_array_equal(got[side, at:at + c, h], p.ref.values(side, s, h, f + c)[f:])
        at += c


def test_rows_outside_are_zeros(ctx):
    p = Pair(ctx, 2, 1, 16, 32, "e4m3")
    p.fill([32, 32])
    got = np.concatenate([p.read(1, -4, 32), p.read(1, 28, 8)], 2)     # (a call takes `capacity` rows at most)
    assert not got[:, :, :4].any() and not got[:, :, 36:].any()
    np.testing.assert_array_equal(got[:, :, 4:36], p.read(1, 0, 32))
    one = torch.full((3, 1, 16), 7.0, device=DEV)
    torch.cuda.synchronize()
    batch = p.gpu.batch(ints(2), [3])
    ctx._check(ctx.lib.gufo_cuda_cache8_rows_device(ctx.handle, p.gpu.handle, C.byref(batch.args), None, C.c_void_p(one.data_ptr())))
    ctx.synchronize()
    np.testing.assert_array_equal(one.cpu().numpy().transpose(1, 0, 2), p.read(0, 2, 3)[1])


def test_many_sequences(ctx):
    """More sequences than one launch takes: appends, attention and eviction of each are its own."""
    n, kv, hd = 300, 1, 64
    p = Pair(ctx, n, kv, hd, 32, "e4m3")
    order = [(i * 77) % n for i in range(n)]
    tokens = [(i * 5) % 21 for i in range(n)]
    total = sum(tokens)
    p.append([0] * n, tokens, draw(1, total, kv, hd), draw(2, total, kv, hd), order)
    for i in range(0, n, 13):
        if tokens[i]:
            p.same(order[i], tokens[i])
    q = draw(3, n, 2, hd).to(DEV)
    out = torch.full((n, 2, hd), float("nan"), device=DEV)
    scratch = p.gpu.scratch(2, n, accumulate=True)
    seen = ints(*tokens)
    torch.cuda.synchronize()
    p.gpu.attend_device(p.gpu.batch(seen, slots=order), q, out, scratch, visible=seen, accumulate=True)
    ctx.synchronize()
    for i in range(n):
        want, weights, size, mass = p.ref.attend(order[i], tokens[i], q[i].cpu().numpy(), hd ** -0.5)
        assert np.all(np.abs(out[i].cpu().numpy() - want) <= R.attend_bound(size, mass, tokens[i], hd)), i
        p.ref.weights[order[i], 0, :tokens[i]] += weights.sum(0).astype(np.float32)
    got = p.gpu.weights.cpu().numpy()
    np.testing.assert_allclose(got, p.ref.weights, rtol=1e-4, atol=1e-6)
    p.ref.weights[:] = got      # the very weights that the eviction goes by
    kept = torch.full((n, kv, 6), -7, dtype=torch.int32, device=DEV)
    held = torch.full((n,), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    p.gpu.evict_device(p.gpu.batch(seen, slots=order), 6, kept, first=1, last=2, held=held)
    ctx.synchronize()
    for i in range(n):
        stay = p.ref.evict(order[i], tokens[i], 6, 1, 2)[0]
        assert kept[i, 0].tolist() == stay + [-1] * (6 - len(stay)) and int(held[i]) == len(stay)
        if stay:
            p.same(order[i], len(stay))


# ---- attention --------------------------------------------------------------------------


def attend(p, positions, tokens, q, gate=None, visible=None, slots=None, accumulate=False, scale=0.0, scratch=None):
    """The GPU's outputs for query rows on the device."""
    out = torch.full(tuple(q.shape), float("nan"), device=DEV)
    scratch = scratch or p.gpu.scratch(q.shape[1], q.shape[0], accumulate)
    torch.cuda.synchronize()
    p.gpu.attend_device(p.gpu.batch(ints(*positions), tokens, slots), q, out, scratch, gate=gate,
                        visible=None if visible is None else ints(*visible), accumulate=accumulate, scale=scale)
    p.ctx.synchronize()
    return out.cpu().numpy()


def check_attend(p, positions, tokens, q, out, gate=None, visible=None, slots=None, scale=None):
    """Outputs against the reference; returns the weights that each row was given, [slot][kv_heads, seen]."""
    hd = p.head_dim
    scale = hd ** -0.5 if scale is None else scale
    x = q.cpu().numpy()
    at, given = 0, {}
    for i, (position, n) in enumerate(zip(positions, tokens)):
        slot = i if slots is None else slots[i]
        for t in range(n):
            seen = min(max(position + t + 1 if visible is None else visible[at], 0), p.capacity)
            want, weights, size, mass = p.ref.attend(slot, seen, x[at], scale)
            bound = R.attend_bound(size, mass, seen, hd)
            if gate is not None:
                g = 1.0 / (1.0 + np.exp(-gate[at].cpu().numpy().astype(np.float64)))
                want, bound = want * g, (bound + 8 * 2.0 ** -24 * mass[:, 0]) * g      # expf, a sum, a quotient, a product
            err = np.abs(out[at] - want)
            assert np.all(err <= bound), (i, t, seen, float((err - bound).max()))
            if seen:
                w = weights.reshape(p.kv_heads, -1, seen).sum(1)
                given.setdefault(slot, np.zeros((p.kv_heads, p.capacity)))[:, :seen] += w
            at += 1
    return given


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("heads, kv_heads, head_dim", [
    (1, 1, 16), (4, 4, 64), (12, 1, 64), (6, 2, 80), (2, 1, 128), (32, 8, 128), (9, 3, 192), (8, 2, 256), (16, 1, 256), (40, 2, 48)])
def test_attend_matches_the_definition(ctx, form, heads, kv_heads, head_dim):
    """Sequences of one row to some hundred, one to eight query tokens, gated, queries beside their gates."""
    lengths = [1, 15, 16, 17, 127, 129, 300]
    tokens = [1, 2, 3, 1, 4, 8, 1]
    p = Pair(ctx, 7, kv_heads, head_dim, 320, form)
    p.fill(lengths)
    rows = sum(tokens)
    both = (draw(5, rows, heads, 2 * head_dim) * 1.5).to(DEV).view(rows, heads, 2, head_dim)
    q, gate = both[:, :, 0], both[:, :, 1]
    positions = [n - t for n, t in zip(lengths, tokens)]       # the last tokens of what is there
    out = attend(p, positions, tokens, q, gate)
    check_attend(p, positions, tokens, q, out, gate)
    # Without gates, and at an odd address.
    flat = torch.empty(rows * heads * head_dim + 1, device=DEV)
    odd = flat[1:].view(rows, heads, head_dim)
    odd.copy_(q)
    check_attend(p, positions, tokens, odd, attend(p, positions, tokens, odd, scale=0.3), scale=0.3)


@pytest.mark.parametrize("form, heads, kv_heads, head_dim, length, tokens", [
    ("e4m3", 8, 2, 256, 5000, 1), ("int8", 4, 1, 128, 20011, 1), ("e4m3", 4, 1, 64, 9000, 9), ("int8", 2, 2, 96, 3333, 40)])
def test_attend_over_long_contexts(ctx, form, heads, kv_heads, head_dim, length, tokens):
    """One sequence over many splits, and many query tokens in groups."""
    p = Pair(ctx, 1, kv_heads, head_dim, (length + 15) // 16 * 16, form)
    p.fill([length])
    q = (draw(5, tokens, heads, head_dim) * 1.5).to(DEV)
    scratch = p.gpu.scratch(heads, tokens)
    out = attend(p, [length - tokens], [tokens], q, scratch=scratch)
    check_attend(p, [length - tokens], [tokens], q, out)
    # The same again, to the bit: sums are taken in one order, and the scratch is as it was.
    for _ in range(3):
        np.testing.assert_array_equal(attend(p, [length - tokens], [tokens], q, scratch=scratch), out)


@pytest.mark.parametrize("capacity", [1040, 2064])
@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("heads, kv_heads, head_dim, most", [
    (4, 4, 64, 1), (4, 2, 48, 8), (12, 1, 64, 8), (32, 8, 128, 1), (8, 2, 112, 4), (6, 1, 128, 8), (8, 2, 256, 1), (8, 2, 256, 4),
    (9, 3, 192, 8), (40, 2, 256, 2)])
def test_attend_shares_ragged_sequences_out(ctx, form, heads, kv_heads, head_dim, most, capacity):
    """Sequences of one row to a thousand, whose tiles many blocks, or a cluster's, take parts of: every group of query rows,
    ragged."""
    lengths = [9, 15, 1033, 700, 64, 65, 1, 400, 1040]
    tokens = [min(n, most) for n in (1, 2, 8, 3, 4, 8, 1, 5, 2)]
    p = Pair(ctx, 9, kv_heads, head_dim, capacity, form)
    p.fill(lengths)
    rows = sum(tokens)
    q, gate = (draw(5, rows, heads, head_dim) * 1.5).to(DEV), draw(6, rows, heads, head_dim).to(DEV)
    slots = [(4 * i) % 9 for i in range(9)]
    positions = [lengths[s] - t if lengths[s] >= t else 0 for s, t in zip(slots, tokens)]
    out = attend(p, positions, tokens, q, gate, slots=slots)
    check_attend(p, positions, tokens, q, out, gate, slots=slots)
    # The tokens in any order, some that see nothing, and their weights.
    seen = [(331 * i * i) % 1041 if i % 4 else 0 for i in range(rows)]
    p.gpu.weights.zero_()
    out = attend(p, positions, tokens, q, slots=slots, visible=seen, accumulate=True)
    given = check_attend(p, positions, tokens, q, out, slots=slots, visible=seen)
    got = p.gpu.weights.cpu().numpy()
    for slot in range(9):
        # (as in test_attend_adds_up_weights, for each of up to 8 tokens' 20 heads)
        np.testing.assert_allclose(got[slot], given.get(slot, np.zeros((kv_heads, capacity))), rtol=2.0 ** -23, atol=3e-5 * 8)


@pytest.mark.parametrize("capacity", [400, 1040])
@pytest.mark.parametrize("form, sequences, heads, kv_heads, head_dim, most", [
    ("int8", 130, 10, 5, 64, 3), ("e4m3", 70, 56, 14, 128, 4), ("e4m3", 33, 32, 16, 256, 3)])
def test_attend_with_more_units_than_blocks(ctx, form, sequences, heads, kv_heads, head_dim, most, capacity):
    """Blocks that go through several sequences' heads, and share the last of them with the next block; or a block for each."""
    p = Pair(ctx, sequences, kv_heads, head_dim, capacity, form, weights=False)
    lengths = [most + (i * 149) % (capacity + 1 - most) for i in range(sequences)]
    # One content for all slots (the reference holds one): a sequence is told by its length and its queries.
    one = R.Cache(1, kv_heads, head_dim, capacity, form)
    k, v = draw(1, capacity, kv_heads, head_dim), draw(2, capacity, kv_heads, head_dim)
    one.append(0, 0, (k.numpy(), v.numpy()))
    kd, vd = k.to(DEV), v.to(DEV)
    torch.cuda.synchronize()
    for slot in range(sequences):
        p.gpu.append_device(p.gpu.batch(ints(0), [capacity], [slot]), kd, vd)
    p.ctx.synchronize()
    p.ref = one
    tokens = [1 + i % most for i in range(sequences)]
    rows = sum(tokens)
    q = (draw(5, rows, heads, head_dim) * 1.5).to(DEV)
    positions = [n - t for n, t in zip(lengths, tokens)]
    out = attend(p, positions, tokens, q)
    check_attend(p, positions, tokens, q, out, slots=[0] * sequences)


def test_scratch_is_anybodys(ctx):
    """One scratch, full of NaN, for calls of different shapes one behind another."""
    p = Pair(ctx, 4, 2, 128, 1024, "e4m3")
    p.fill([1000, 30, 500, 1024])
    q = draw(5, 16, 8, 128).to(DEV)
    scratch = p.gpu.scratch(8, 16, accumulate=True)
    nan = np.full(scratch.bytes // 4, np.nan, dtype=np.float32)
    for tokens in ([1, 1, 1, 1], [4, 4, 4, 4], [0, 0, 0, 1], [1, 8, 2, 0]):
        ctx.upload(scratch.ptr, nan)
        n = sum(tokens)
        for accumulate in (False, True, False):
            positions = [a - b for a, b in zip((1000, 30, 500, 1024), tokens)]
            out = attend(p, positions, tokens, q[:n], accumulate=accumulate, scratch=scratch)
            check_attend(p, positions, tokens, q[:n], out)


def test_attend_with_peaked_and_flat_scores(ctx):
    """Weights of 1 beside weights of 2^-60, and rows that all weigh the same."""
    p = Pair(ctx, 2, 1, 64, 4096, "e4m3")
    p.fill([4000, 4000])
    q = torch.cat([draw(5, 1, 4, 64) * 40, draw(6, 1, 4, 64) * 1e-6]).to(DEV)
    out = attend(p, [3999, 3999], [1, 1], q)
    check_attend(p, [3999, 3999], [1, 1], q, out)
    # Queries of any size: their largest value is what the halves are scaled by.
    for size in (1e-30, 1e30):
        tiny = q * size
        check_attend(p, [3999, 3999], [1, 1], tiny, attend(p, [3999, 3999], [1, 1], tiny, scale=0.125 / size), scale=0.125 / size)


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("largest", [2.0 ** -130, 2.0 ** -100, 1.99, 1.9922, 1.99225, 1.9999, 2.0 ** 123.5, 2.0 ** 124.5, 2.0 ** 127, 3.4e38])
def test_attend_with_queries_of_any_size(ctx, form, largest):
    """Largest values on both sides of where the queries' scaling changes, to the ends of fp32; the scale makes up for it."""
    p = Pair(ctx, 1, 1, 64, 512, form)
    k, v = draw(1, 400, 1, 64) * 2.0 ** -60, draw(2, 400, 1, 64)
    p.append([0], [400], k, v)
    q = draw(5, 2, 4, 64)
    q = (q.double() / q.abs().amax(-1, keepdim=True) * largest).float().to(DEV)
    scale = float(np.float32(min(2.0 ** 62 / largest, 2.0 ** 126)))
    out = attend(p, [398], [2], q, scale=scale)
    check_attend(p, [398], [2], q, out, scale=scale)


def test_attend_hides_what_is_not_seen(ctx):
    """Rows behind the ones a token sees hold NaN, and change nothing; tokens that see nothing get zeros."""
    p = Pair(ctx, 3, 2, 64, 64, "e4m3")
    p.fill([37, 37, 37])
    q = draw(5, 6, 4, 64).to(DEV)
    gate = draw(6, 6, 4, 64).to(DEV)
    gate[1] = float("nan")       # of a token that sees nothing
    visible = [37, 0, 16, 5, -3, 1]
    tokens = [2, 1, 3]
    clean = attend(p, [0, 0, 0], tokens, q, gate, visible)
    check_attend(p, [0, 0, 0], [0, 1, 3], q[2:], clean[2:], gate[2:], visible[2:])
    assert not clean[1].any() and not clean[4].any()
    p.ref = R.Cache(3, 2, 64, 64, "e4m3")      # (behind row 37 only)
    bad = torch.full((27, 2, 64), float("nan"))
    torch.cuda.synchronize()
    k = bad.repeat(3, 1, 1).to(DEV)
    p.gpu.append_device(p.gpu.batch(ints(37, 37, 37), [27] * 3), k, k)
    ctx.synchronize()
    np.testing.assert_array_equal(attend(p, [0, 0, 0], tokens, q, gate, visible), clean)
    # A NaN that is seen is seen: of its KV head's queries, where the row is among those seen.
    seen = attend(p, [0, 0, 0], tokens, q, None, [38, 0, 16, 5, 0, 64])
    assert np.isnan(seen[0]).all() and np.isnan(seen[5]).all() and np.isfinite(seen[1:5]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attend_of_rows_that_are_not_finite(ctx, bad):
    """A query row that is not finite makes NaN of its own outputs and of nobody else's."""
    p = Pair(ctx, 1, 1, 128, 256, "int8")
    p.fill([200])
    q = draw(5, 3, 2, 128).to(DEV)
    clean = attend(p, [197], [3], q)
    q[1, 1, 77] = bad
    out = attend(p, [197], [3], q)
    assert np.isnan(out[1, 1]).all()
    out[1, 1] = clean[1, 1]
    np.testing.assert_array_equal(out, clean)


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_attend_adds_up_weights(ctx, form):
    lengths, tokens, slots = [5, 1000, 40, 333], [1, 3, 2, 1], [2, 0, 3, 1]
    p = Pair(ctx, 5, 2, 64, 1024, form)
    n = sum(lengths)
    p.append([0] * 4, lengths, draw(1, n, 2, 64), draw(2, n, 2, 64), slots)
    start = torch.rand(5, 2, 1024, generator=torch.Generator().manual_seed(3))
    torch.cuda.synchronize()
    p.gpu.weights.copy_(start)
    q = draw(5, sum(tokens), 6, 64).to(DEV) * 2
    positions = [a - b for a, b in zip(lengths, tokens)]
    out = attend(p, positions, tokens, q, slots=slots, accumulate=True)
    given = check_attend(p, positions, tokens, q, out, slots=slots)
    got = p.gpu.weights.cpu().numpy()
    for slot in range(5):
        added = given.get(slot, np.zeros((2, 1024)))
        # A weight is off by its score's error (1e-5 here) as a part of itself, the sum by half a step.
        np.testing.assert_allclose(got[slot], start[slot].numpy() + added, rtol=2.0 ** -23, atol=0.0 if slot == 4 else 3e-5)
    assert np.array_equal(got[4], start[4].numpy())
    np.testing.assert_array_equal(attend(p, positions, tokens, q, slots=slots), out)     # the weights come on top


def test_attend_far_into_a_large_cache(ctx):
    """Offsets beyond 32 bits: the last slot of a cache of gigabytes, all its rows seen, few of them written."""
    capacity, kv, hd, slots = 1 << 21, 2, 256, 3
    cache = CudaCache8(ctx, slots, kv, hd, capacity, format="int8")
    p = Pair(ctx, 1, kv, hd, 64, "int8")
    k, v = draw(1, 40, kv, hd), draw(2, 40, kv, hd)
    p.append([8], [40], k, v)                # the same places in their blocks
    at = capacity - 56
    q = draw(5, 1, 4, hd) * 3
    kd, vd, qd = k.to(DEV), v.to(DEV), q.to(DEV)
    out = torch.empty(1, 4, hd, device=DEV)
    back = torch.empty(2, 40, kv, hd, device=DEV)
    scratch = cache.scratch(4, 1)
    torch.cuda.synchronize()
    cache.append_device(cache.batch(ints(at), [40], [2]), kd, vd)
    cache.rows_device(cache.batch(ints(at), [40], [2]), back[0], back[1])
    cache.attend_device(cache.batch(ints(at + 39), slots=[2]), qd, out, scratch)
    ctx.synchronize()
    for h in range(kv):
        want = [p.ref.values(side, 0, h, 48)[8:] for side in range(2)]
        np.testing.assert_array_equal(back[0, :, h].cpu().numpy(), want[0])
        np.testing.assert_array_equal(back[1, :, h].cpu().numpy(), want[1])
        for i in (2 * h, 2 * h + 1):
            s = want[0] @ q[0, i].double().numpy() / 16
            top = max(s.max(), 0.0)
            p_ = np.exp(s - top)
            total = p_.sum() + (at * np.exp(-top))       # zeros score zero
            o = p_ @ want[1] / total
            size = (np.abs(want[0]) @ np.abs(q[0, i].double().numpy())).max() / 16
            mass = np.stack([p_ @ np.abs(want[1]) / total, np.abs(want[1]).sum(0)])
            bound = R.attend_bound(np.array(size), mass, 40, hd)
            # (and the sum of two million weights, in the lanes' fp32 sums of some hundred)
            assert np.all(np.abs(out[0, i].cpu().numpy() - o) <= bound + 2.0 ** -16 * np.abs(o))
    cache.close()


def test_calls_on_two_streams_and_in_graphs(ctx):
    """Two contexts' calls in flight together, each with scratch of its own; a captured chain that follows the
    positions it finds."""
    kv, hd, heads, capacity = 2, 128, 8, 4096
    streams = [torch.cuda.Stream() for _ in range(2)]
    parts = []
    for i, s in enumerate(streams):
        c = Context(0, s.cuda_stream)
        p = Pair(c, 2, kv, hd, capacity, "e4m3")
        p.fill([3000, 1200], seed=10 * i)
        q = draw(7 + i, 2, heads, hd).to(DEV)
        k, v = draw(8 + i, 2, kv, hd).to(DEV), draw(9 + i, 2, kv, hd).to(DEV)
        out = torch.empty(2, heads, hd, device=DEV)
        at = ints(3000, 1200)
        parts.append((c, p, q, k, v, out, at, p.gpu.batch(at), p.gpu.scratch(heads, 2, accumulate=True)))
    torch.cuda.synchronize()

    def step(part):
        c, p, q, k, v, out, at, batch, scratch = part
        p.gpu.append_device(batch, k, v)
        p.gpu.attend_device(batch, q, out, scratch, accumulate=True)
    graphs = []
    for part, s in zip(parts, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(part)
        graphs.append(graph)
    for lengths in ((3000, 1200), (3001, 1201), (17, 4095)):
        for part, s in zip(parts, streams):
            part[6].copy_(ints(*lengths))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for c, p, q, k, v, out, at, batch, scratch in parts:
            for i in range(2):
                p.ref.append(i, lengths[i], (k[i:i + 1].cpu().numpy(), v[i:i + 1].cpu().numpy()))
            check_attend(p, lengths, [1, 1], q, out.cpu().numpy())
    del graphs
    for part in parts:
        part[0].close()


@pytest.mark.parametrize("capacity", [320, 1024])
def test_captured_calls_of_short_caches(capacity):
    """A block, or a cluster of blocks, a sequence and head, captured once: lengths from none to all of the cache, and weights."""
    stream = torch.cuda.Stream()
    c = Context(0, stream.cuda_stream)
    p = Pair(c, 2, 2, 80, capacity, "e4m3")
    p.fill([capacity, capacity])
    q, gate = draw(7, 3, 6, 80).to(DEV), draw(8, 3, 6, 80).to(DEV)
    out = torch.empty(3, 6, 80, device=DEV)
    at = ints(5, 5)
    batch, scratch = p.gpu.batch(at, [1, 2]), p.gpu.scratch(6, 3, accumulate=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        p.gpu.attend_device(batch, q, out, scratch, gate=gate, accumulate=True)
    for positions in ((5, 17), (-1, 62), (capacity - 1, -3), (capacity - 2, capacity), (63, 0), (0, capacity // 2)):
        at.copy_(ints(*positions))
        p.gpu.weights.zero_()
        torch.cuda.synchronize()
        first = None
        for _ in range(3):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            first = out.clone() if first is None else first
            assert torch.equal(first, out)
        given = check_attend(p, positions, [1, 2], q, out.cpu().numpy(), gate)
        got = p.gpu.weights.cpu().numpy()
        for slot in range(2):
            np.testing.assert_allclose(got[slot], 3 * given.get(slot, np.zeros((2, capacity))), rtol=2.0 ** -22, atol=3e-5 * 6)
    del graph
    c.close()


def test_a_new_cache_is_used_on_another_stream():
    """A cache made on a stream that is busy, and written on another: nothing clears it afterwards."""
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    c = Context(0, busy.cuda_stream)
    with torch.cuda.stream(busy):
        x = torch.ones(4096, 4096, device=DEV)
        for _ in range(50):
            x = x @ x * 2.0 ** -12
    p = Pair(c, 1, 1, 16, 32, "e4m3")
    c.set_stream(other.cuda_stream)
    k = draw(1, 20, 1, 16)
    kd = k.to(DEV)
    other.wait_stream(torch.cuda.current_stream())
    p.gpu.append_device(p.gpu.batch(ints(0), [20]), kd, kd)
    torch.cuda.synchronize()
    p.ref.append(0, 0, (k.numpy(), k.numpy()))
    p.same(0, 20)
    c.close()


# ---- eviction ---------------------------------------------------------------------------


def evict(p, rows, budget, first, last, slots=None, into=None, into_slots=None, held=True):
    n = len(rows)
    kept = torch.full((n, p.kv_heads, budget), -7, dtype=torch.int32, device=DEV)
    count = torch.full((n,), -7, dtype=torch.int32, device=DEV) if held else None
    torch.cuda.synchronize()
    p.gpu.evict_device(p.gpu.batch(ints(*rows), slots=slots), budget, kept, first=first, last=last, held=count,
                       into=into.gpu if into else None, into_slots=into_slots)
    p.ctx.synchronize()
    return kept.cpu().numpy(), None if count is None else count.cpu().numpy()


def set_weights(p, seed, ties=False):
    w = torch.exp(2 * torch.randn(p.slots, p.kv_heads, p.capacity, generator=torch.Generator().manual_seed(seed)))
    if ties:
        w = torch.round(w.clamp(max=3.0))
    p.gpu.weights.copy_(w)
    torch.cuda.synchronize()
    p.ref.weights[:] = w.numpy()
    return w


def check_evict(p, rows, budget, first, last, got, slots=None, into=None, into_slots=None):
    kept, held = got
    to = into or p
    for i, n in enumerate(rows):
        slot = i if slots is None else slots[i]
        there = slot if into_slots is None else into_slots[i]
        stay = p.ref.evict(slot, n, budget, first, last, into.ref if into else None, there)
        for h in range(p.kv_heads):
            assert kept[i, h].tolist() == stay[h] + [-1] * (budget - len(stay[h])), (i, h)
        assert held is None or held[i] == min(n, budget)
        if min(n, budget):
            to.same(there, min(n, budget))
        np.testing.assert_array_equal(to.gpu.weights.cpu().numpy()[there, :, :min(n, budget)], to.ref.weights[there, :, :min(n, budget)])


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("head_dim, rows, budget, first, last, ties", [
    (64, [100, 50, 33, 49], 48, 4, 8, False), (128, [500, 0, 1, 499], 200, 0, 0, True), (80, [300, 300, 17, 3], 299, 1, 1, False),
    (256, [64, 63, 16, 15], 1, 0, 0, False), (16, [700, 650, 300, 699], 97, 60, 60, True), (48, [200, 100, 60, 50], 50, 80, 3, True),
    (64, [400, 5, 90, 400], 60, 20, 40, False)])
def test_evict_matches_the_definition(ctx, form, other, head_dim, rows, budget, first, last, ties):
    """Sequences longer and shorter than the budget, ends that do not fit it, ties; in place and into other slots of another cache."""
    p = Pair(ctx, 4, 2, head_dim, 704, form)
    p.fill(rows)
    set_weights(p, budget, ties)
    if other:
        into = Pair(ctx, 6, 2, head_dim, (budget + 15) // 16 * 16 + 16, form)
        into.fill([7] * 6, seed=50)
        before = [p.read(s, 0, 704) for s in range(4)], p.gpu.weights.clone()
        got = evict(p, rows, budget, first, last, into=into, into_slots=[5, 0, 2, 3])
        check_evict(p, rows, budget, first, last, got, into=into, into_slots=[5, 0, 2, 3])
        for s in range(4):
            np.testing.assert_array_equal(p.read(s, 0, 704), before[0][s])
        assert torch.equal(p.gpu.weights, before[1])
        for s in (1, 4):
            into.same(s, 7)
    else:
        got = evict(p, rows, budget, first, last)
        check_evict(p, rows, budget, first, last, got)


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_evict_in_place_over_many_blocks(ctx, form):
    """Several rounds of a cluster's blocks, one head of a slot among others."""
    p = Pair(ctx, 3, 1, 32, 6016, form)
    p.fill([6000, 16, 6000])
    w = set_weights(p, 1)
    w[0, 0, :3000] += 100.0      # the first half stays as it is, and is not touched
    p.gpu.weights.copy_(w)
    torch.cuda.synchronize()
    p.ref.weights[:] = w.numpy()
    got = evict(p, [6000, 6000], 4500, 3, 50, slots=[2, 0])
    check_evict(p, [6000, 6000], 4500, 3, 50, got, slots=[2, 0])
    p.same(1, 16)


@pytest.mark.parametrize("other", [False, True])
def test_evict_of_many_rows(ctx, other):
    """More rows than a thread holds weights of at a time, with and without ties."""
    rows, budget = [20000, 4097, 16385], 6001
    p = Pair(ctx, 3, 1, 16, 20000, "int8")
    p.fill(rows)
    for ties in (False, True):
        set_weights(p, 5, ties)
        into = Pair(ctx, 3, 1, 16, 6016, "int8") if other else None
        check_evict(p, rows, budget, 4, 100, evict(p, rows, budget, 4, 100, into=into, into_slots=[2, 1, 0] if other else None),
                    into=into, into_slots=[2, 1, 0] if other else None)
        rows = rows if other else [min(n, budget) for n in rows]
        budget -= 3000


def test_evict_goes_by_any_weight(ctx):
    """Negative weights, zeros of both signs, infinities, NaN last; the positions left alone."""
    p = Pair(ctx, 1, 1, 16, 64, "e4m3")
    p.fill([64])
    w = torch.zeros(1, 1, 64)
    w[0, 0, ::2] = -0.0
    w[0, 0, 5], w[0, 0, 9], w[0, 0, 11], w[0, 0, 20], w[0, 0, 30] = float("inf"), -1.0, float("nan"), 1e-45, float("-inf")
    w[0, 0, 40] = -float("nan")
    p.gpu.weights.copy_(w)
    torch.cuda.synchronize()
    p.ref.weights[:] = w.numpy()
    for budget in (61, 60, 59, 40, 2, 1):
        into = Pair(ctx, 1, 1, 16, 64, "e4m3")
        got = evict(p, [64], budget, 0, 0, into=into, held=False)
        check_evict(p, [64], budget, 0, 0, got, into=into)


def test_evict_tightens_scales(ctx):
    """Blocks take the scale of what they hold: a large row that leaves gives its neighbours no bits back, but the rows that come
    after it to the block are held as finely as alone."""
    p = Pair(ctx, 1, 1, 16, 48, "int8")
    x = draw(1, 40, 1, 16)
    x[20] *= 1000.0
    p.append([0], [40], x, x)
    w = torch.ones(1, 1, 48)
    w[0, 0, 20] = 0.0
    p.gpu.weights.copy_(w)
    torch.cuda.synchronize()
    p.ref.weights[:] = w.numpy()
    check_evict(p, [40], 39, 0, 0, evict(p, [40], 39, 0, 0))
    y = draw(2, 1, 1, 16) * 0.5
    p.append([39], [1], y, y)
    p.same(0, 40)


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("other", [False, True])
def test_evict_of_zeros_from_under_a_large_scale(ctx, form, other):
    """Zeros that shared a scale with large rows, by themselves and beside the smallest numbers: zeros they stay."""
    p = Pair(ctx, 1, 1, 32, 96, form)
    x = torch.zeros(96, 1, 32)
    x[0:16:2] = draw(1, 8, 1, 32) * 2.0 ** 100        # rows 1, 3, ...: zeros under their scale
    x[16:32] = draw(2, 16, 1, 32)
    x[16:32:4] = 0.0
    x[32:48] = 1e-40 * torch.arange(32)
    x[64:80] = draw(3, 16, 1, 32) * 2.0 ** -100
    x[80:96] = float("inf")
    x[81:96:3] = 0.0
    p.append([0], [96], x, -x)
    for rows in (list(range(1, 16, 2)) + [16, 20, 24, 28] + list(range(32, 37)), list(range(1, 16, 2)) + list(range(64, 74)),
                 [81, 84, 87], [16, 81]):
        w = torch.zeros(1, 1, 96)
        w[0, 0, rows] = 1.0
        q = Pair(ctx, 1, 1, 32, 96, form)
        q.append([0], [96], x, -x)
        q.gpu.weights.copy_(w)
        torch.cuda.synchronize()
        q.ref.weights[:] = w.numpy()
        into = Pair(ctx, 1, 1, 32, 96, form) if other else None
        check_evict(q, [96], len(rows), 0, 0, evict(q, [96], len(rows), 0, 0, into=into), into=into)


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("other", [False, True])
def test_evict_tightens_the_last_block(ctx, form, other):
    """The last block keeps its first rows in their places and loses a large one: what comes after it is held as finely as beside
    those rows alone, in place as in another cache."""
    p = Pair(ctx, 1, 1, 16, 48, form)
    x = draw(1, 40, 1, 16)
    x[38] *= 1000.0
    p.append([0], [40], x, x)
    p.gpu.weights.copy_(torch.arange(48, 0, -1).float().view(1, 1, 48))
    torch.cuda.synchronize()
    p.ref.weights[:] = p.gpu.weights.cpu().numpy()
    into = Pair(ctx, 1, 1, 16, 48, form) if other else None
    check_evict(p, [40], 37, 0, 0, evict(p, [40], 37, 0, 0, into=into), into=into)
    y = draw(2, 4, 1, 16)
    (into or p).append([37], [4], y, y)
    (into or p).same(0, 41)


# ---- as they are used together ----------------------------------------------------------


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_decoding_under_a_budget(ctx, form):
    """Steps of an attention layer of three sequences: rotary positions, append, attention with weights, and an eviction when
    a sequence has outgrown its budget; positions go on, the rows do not."""
    heads, kv, hd, budget, room = 4, 2, 64, 40, 16
    p = Pair(ctx, 3, kv, hd, 64, form)
    rope = ctx.rope_create(32, theta=1e6, scaling="by_parts", factor=4.0, original_positions=1024)
    freq = R.frequencies(32, 1e6, "by_parts", 4.0, 1024.0)
    magnitude = float(np.float32(0.1 * np.log(4.0) + 1.0))
    q_norm, k_norm = draw(70, hd).to(DEV), draw(71, hd).to(DEV)
    held, place = [3, 0, 11], [1000, 0, 5]
    p.fill(held)
    p.gpu.weights.zero_()
    torch.cuda.synchronize()
    scratch = p.gpu.scratch(heads, 9, accumulate=True)
    for step in range(30):
        tokens = [1 + (step + i) % 3 for i in range(3)]
        n = sum(tokens)
        x = draw(100 + step, n, 1, 2 * heads * hd + 2 * kv * hd).view(n, -1).to(DEV)
        q = x[:, :2 * heads * hd].view(n, heads, 2, hd)
        k = x[:, 2 * heads * hd:(2 * heads + kv) * hd].view(n, kv, hd)
        v = x[:, (2 * heads + kv) * hd:].view(n, kv, hd)
        turned_q, turned_k = torch.empty(n, heads, hd, device=DEV), torch.empty(n, kv, hd, device=DEV)
        out = torch.empty(n, heads, hd, device=DEV)
        at = ints(*[place[i] + t for i in range(3) for t in range(tokens[i])])
        batch = p.gpu.batch(ints(*held), tokens)
        torch.cuda.synchronize()
        ctx.rope_device(rope, ctx.rope_parts([(q[:, :, 0], turned_q, q_norm), (k, turned_k, k_norm)], rms_eps=1e-6), at)
        p.gpu.append_device(batch, turned_k, v)
        p.gpu.attend_device(batch, turned_q, out, scratch, gate=q[:, :, 1], accumulate=True)
        ctx.synchronize()
        for got, rows, w in ((turned_q, q[:, :, 0], q_norm), (turned_k, k, k_norm)):
            want, size = R.rope(rows.cpu().numpy(), at.tolist(), freq, "halves", magnitude, w.cpu().numpy(), 1e-6)
            assert np.all(np.abs(got.cpu().numpy() - want) <= 32 * 2.0 ** -24 * size)
        first = 0
        for i, t in enumerate(tokens):
            p.ref.append(i, held[i], (turned_k[first:first + t].cpu().numpy(), v[first:first + t].cpu().numpy()))
            first += t
        given = check_attend(p, held, tokens, turned_q, out.cpu().numpy(), q[:, :, 1])
        got = p.gpu.weights.cpu().numpy()
        for i in range(3):
            total = held[i] + tokens[i]
            np.testing.assert_allclose(got[i, :, :total], p.ref.weights[i, :, :total] + given[i][:, :total], rtol=1e-4, atol=1e-5)
            p.ref.weights[i, :, :total] = got[i, :, :total]
            held[i] += tokens[i]
            place[i] += tokens[i]
        if max(held) > budget + room:
            check_evict(p, held, budget, 2, 10, evict(p, held, budget, 2, 10))
            held = [min(h, budget) for h in held]
    assert place[0] > 1050 and max(held) <= budget + room
    ctx.rope_free(rope)


# ---- what is refused, and lifetimes -----------------------------------------------------


def test_refusals(ctx):
    p = Pair(ctx, 3, 2, 64, 64, "e4m3")
    plain = CudaCache8(ctx, 3, 2, 64, 64)
    gpu = p.gpu
    k = torch.zeros(2, 2, 64, device=DEV)
    out = torch.zeros(2, 4, 64, device=DEV)
    kept = torch.zeros(2, 2, 8, dtype=torch.int32, device=DEV)
    at = ints(0, 0)
    scratch = gpu.scratch(4, 2)
    before = ctx.launch_count()

    def refused(status, call, *args, **kw):
        with pytest.raises(GufoCudaError) as e:
            call(*args, **kw)
        assert e.value.status == status, e.value
    for slots in ([0, 3], [0, -1], [1, 1]):
        refused(1, gpu.append_device, gpu.batch(at, slots=slots), k, k)
        refused(1, gpu.rows_device, gpu.batch(at, slots=slots), k, k)
        refused(1, gpu.attend_device, gpu.batch(at, slots=slots), out, out, scratch)
        refused(1, gpu.evict_device, gpu.batch(at, slots=slots), 8, kept)
    four = gpu.batch(ints(0, 0, 0, 0))
    refused(1, gpu.append_device, four, k.repeat(2, 1, 1), k.repeat(2, 1, 1))
    refused(1, gpu.append_device, gpu.batch(at, tokens=[-1, 3]), k, k)
    long = torch.zeros(65, 2, 64, device=DEV)
    refused(1, gpu.append_device, gpu.batch(at, tokens=[65, 0]), long, long)
    # The library's own checks behind the tensors' ones.
    b = gpu.batch(at)
    lib, h = ctx.lib, ctx.handle
    ptr = C.c_void_p(k.data_ptr())
    assert lib.gufo_cuda_cache8_append_device(h, gpu.handle, None, ptr, 128, 64, ptr, 128, 64) == 1
    assert lib.gufo_cuda_cache8_append_device(h, gpu.handle, C.byref(b.args), None, 128, 64, ptr, 128, 64) == 1
    assert lib.gufo_cuda_cache8_append_device(h, 999999, C.byref(b.args), ptr, 128, 64, ptr, 128, 64) == 1
    assert lib.gufo_cuda_cache8_rows_device(h, gpu.handle, C.byref(b.args), C.c_void_p(k.data_ptr() + 4), None) == 1
    none = type(b.args)(2, None, None, None)
    assert lib.gufo_cuda_cache8_append_device(h, gpu.handle, C.byref(none), ptr, 128, 64, ptr, 128, 64) == 1
    # Attention.
    small = gpu.scratch(4, 2)
    small.bytes -= 1
    refused(1, gpu.attend_device, b, out, out, small)
    small.bytes += 1
    refused(1, gpu.attend_device, b, out, out, scratch, accumulate=True)     # scratch for calls without
    refused(1, plain.attend_device, plain.batch(at), out, out, plain.scratch(4, 2, accumulate=True), accumulate=True)
    three = torch.zeros(2, 3, 64, device=DEV)
    refused(2, gpu.attend_device, b, three, three, scratch)
    # Eviction.
    refused(1, plain.evict_device, plain.batch(at), 8, kept)
    refused(2, gpu.evict_device, b, 65, torch.zeros(2, 2, 65, dtype=torch.int32, device=DEV))
    refused(2, gpu.evict_device, b, 8, kept, first=-1)
    refused(2, gpu.evict_device, b, 8, kept, last=-1)
    refused(1, gpu.evict_device, b, 8, kept, held=at)
    refused(1, gpu.evict_device, b, 8, kept, into=gpu)
    refused(1, gpu.evict_device, b, 8, kept, into_slots=[0, 1])
    refused(1, gpu.evict_device, b, 8, kept, into=plain, into_slots=[1, 1])
    for other in (CudaCache8(ctx, 3, 2, 64, 64, format="int8"), CudaCache8(ctx, 3, 1, 64, 64), CudaCache8(ctx, 3, 2, 80, 64)):
        refused(2, gpu.evict_device, b, 8, kept, into=other)
    refused(2, gpu.evict_device, b, 32, torch.zeros(2, 2, 32, dtype=torch.int32, device=DEV), into=CudaCache8(ctx, 3, 2, 64, 16))
    assert lib.gufo_cuda_cache8_evict_device(h, gpu.handle, C.byref(b.args), 8, 0, 0, None, None, 0, None) == 1
    # Shapes and types of the tensors.
    for bad in (k.half(), k.cpu(), k[:1], k[:, :1], k[:, :, :32], k.transpose(1, 2)):
        with pytest.raises(ValueError):
            gpu.append_device(b, bad, k)
        with pytest.raises(ValueError):
            gpu.rows_device(b, k, bad)
    with pytest.raises(ValueError):
        gpu.rows_device(b, k, torch.zeros(2, 2, 128, device=DEV)[:, :, :64])
    for kw in ({"gate": out[:1]}, {"visible": ints(1)}, {"visible": at.long()}):
        with pytest.raises(ValueError):
            gpu.attend_device(b, out, out, scratch, **kw)
    with pytest.raises(ValueError):
        gpu.evict_device(b, 8, kept[:, :1])
    with pytest.raises(ValueError):
        gpu.evict_device(b, 8, kept, held=ints(0))
    with pytest.raises(ValueError):
        gpu.batch(at, tokens=[1])
    # Batches and scratch of another device (as they would be: there may be one device only).
    elsewhere = gpu.batch(at)
    elsewhere.device = 1
    foreign = type("Scratch", (), {"ctx": type("Context", (), {"device": 1}), "ptr": scratch.ptr, "bytes": scratch.bytes})
    for call, *args in ((gpu.append_device, elsewhere, k, k), (gpu.rows_device, elsewhere, k, k),
                        (gpu.attend_device, elsewhere, out, out, scratch), (gpu.attend_device, b, out, out, foreign),
                        (gpu.evict_device, elsewhere, 8, kept)):
        with pytest.raises(ValueError):
            call(*args)
    for args in ((0, 1, 64, 64), (4097, 1, 64, 64), (1, 0, 64, 64), (1, 1, 8, 64), (1, 1, 72, 64), (1, 1, 272, 64), (1, 1, 64, 0),
                 (1, 1, 64, 24), (1, 1, 64, 1 << 29)):
        with pytest.raises(GufoCudaError) as e:
            CudaCache8(ctx, *args)
        assert e.value.status == 2
    with pytest.raises(GufoCudaError) as e:
        CudaCache8(ctx, 4096, 1024, 256, 1 << 20)
    assert e.value.status == 5
    # Batches without rows: nothing to do.
    empty = gpu.batch(at, tokens=[0, 0])
    gpu.append_device(empty, k[:0], k[:0])
    gpu.rows_device(empty, k[:0], k[:0])
    gpu.attend_device(empty, out[:0], out[:0], scratch)
    nobody = gpu.batch(at[:0])
    gpu.evict_device(nobody, 8, kept[:0])
    assert ctx.launch_count() == before


def test_weights_outlive_the_cache_object():
    """A tensor over the accumulated weights keeps their memory; a closed cache answers no more."""
    c = Context(0)
    cache = CudaCache8(c, 2, 1, 16, 32, weights=True)
    w = cache.weights
    c.synchronize()
    w.fill_(3.0)
    del cache
    again = CudaCache8(c, 2, 1, 16, 32, weights=True)
    c.synchronize()
    assert float(w.sum()) == 3.0 * 64 and float(again.weights.sum()) == 0.0
    del w
    torch.cuda.synchronize()
    again.close()
    with pytest.raises(GufoCudaError):
        again.append_device(again.batch(ints(0)), torch.zeros(1, 1, 16, device=DEV), torch.zeros(1, 1, 16, device=DEV))
    c.close()
