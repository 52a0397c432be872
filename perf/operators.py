"""Operators around a key / value cache that is held in 8 bits, as cases that can be timed.

`kind` picks the operator:

  rope      Context.rope_device: RMSNorm of each head and rotary positions, queries and keys in one call
  append    CudaCache8.append_device: rows of keys and values into the cache (and rows_device: the blocks that
            this touched, read back as the fp32 values they stand for)
  attend    CudaCache8.attend_device: a few query tokens of each sequence over its cached rows; with `weights`,
            what each row was given is added up beside it
  evict     CudaCache8.evict_device: of each sequence and KV head the rows of least weight leave the cache. `step`
            rows > 0: in place, behind an append of that many rows, as a decode loop runs it; 0: from a prompt's
            cache into the sequence's own smaller one

The cache: blocks of 16 rows of a head share a scale, a power of two, the smallest with which the block's largest
magnitude is a code (e4m3: 448, int8: 127) or less. Rows that join a block may make its scale grow; the rows there
are rounded to it again. Where `own` is false everything is computed here in plain torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
BLOCK = 16


def listed():
    return [
        # A decode step of 32 sequences far into their contexts: rotary part of 64, frequencies stretched by parts.
        {"name": "rope_decode", "kind": "rope", "tokens": 32, "heads": 16, "kv_heads": 4, "head_dim": 256, "rope_dim": 64,
         "layout": "halves", "scaling": "by_parts", "farthest": 1000000, "norm": True},
        # A prompt of one sequence, interleaved pairs over the whole head, positions scaled linearly.
        {"name": "rope_prompt", "kind": "rope", "tokens": 8000, "heads": 8, "kv_heads": 2, "head_dim": 256, "rope_dim": 256,
         "layout": "pairs", "scaling": "linear", "farthest": 32000, "norm": False},
        # The ragged verify batch's new rows: 32 sequences, one to four draft tokens each.
        {"name": "append_verify", "kind": "append", "sequences": 32, "kv_heads": 4, "head_dim": 256, "positions": 2000,
         "tokens": 4, "format": "e4m3"},
        # A prompt's rows behind an odd number that is there.
        {"name": "append_prompt", "kind": "append", "sequences": 1, "kv_heads": 2, "head_dim": 256, "positions": 37,
         "tokens": 16001, "format": "int8"},
        # The smallest: a short conversation of one sequence.
        {"name": "attend_one", "kind": "attend", "sequences": 1, "heads": 8, "kv_heads": 2, "head_dim": 256, "positions": 500,
         "tokens": 1, "format": "e4m3", "gate": True, "weights": False},
        # The verify batch over its contexts: 32 sequences of up to 4096 rows, one to four query tokens.
        {"name": "attend_verify", "kind": "attend", "sequences": 32, "heads": 16, "kv_heads": 4, "head_dim": 256,
         "positions": 4096, "tokens": 4, "format": "e4m3", "gate": True, "weights": False},
        # One sequence with a very long context.
        {"name": "attend_long", "kind": "attend", "sequences": 1, "heads": 16, "kv_heads": 4, "head_dim": 256,
         "positions": 131000, "tokens": 1, "format": "int8", "gate": True, "weights": False},
        # Heads that share no keys: many short sequences, the first of a single row.
        {"name": "attend_short", "kind": "attend", "sequences": 64, "heads": 4, "kv_heads": 4, "head_dim": 64, "positions": 333,
         "tokens": 1, "format": "int8", "gate": False, "weights": False},
        # Decoding under a budget: the weight of every row is kept.
        {"name": "attend_weights", "kind": "attend", "sequences": 16, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "positions": 4096, "tokens": 1, "format": "e4m3", "gate": False, "weights": True},
        # Sixteen steps past the budget: the least wanted rows of eight sequences leave.
        {"name": "evict_step", "kind": "evict", "sequences": 8, "kv_heads": 8, "head_dim": 128, "positions": 2048,
         "step": 16, "budget": 2048, "first": 4, "last": 64, "format": "e4m3"},
        # Prompts of 16384 rows brought down to 2048.
        {"name": "evict_prompt", "kind": "evict", "sequences": 4, "kv_heads": 4, "head_dim": 256, "positions": 16384,
         "step": 0, "budget": 2048, "first": 4, "last": 256, "format": "e4m3"},
        # One short prompt, int8, odd numbers.
        {"name": "evict_small", "kind": "evict", "sequences": 1, "kv_heads": 2, "head_dim": 256, "positions": 777,
         "step": 0, "budget": 255, "first": 3, "last": 31, "format": "int8"},
    ]


def _log(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


HEADS = [(2, 1, 128), (8, 2, 256), (16, 4, 256), (4, 4, 64), (32, 8, 128), (6, 2, 80), (12, 1, 64), (20, 4, 96), (9, 3, 192),
         (5, 5, 112)]


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "evict", "evict"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    form = rng.choice(["e4m3", "int8"])
    if kind == "rope":
        return {"kind": kind, "tokens": _log(rng, 1, min(8000, 30000000 // ((heads + kv_heads) * head_dim))), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "rope_dim": 2 * rng.randint(8, head_dim // 2), "layout": rng.choice(["halves", "pairs"]),
                "scaling": rng.choice(["none", "linear", "by_parts"]), "farthest": _log(rng, 1000, 1000000),
                "norm": rng.random() < 0.5}
    row = kv_heads * head_dim
    if kind == "append":
        sequences = _log(rng, 1, 64)
        most = 8000000 // (sequences * row)
        return {"kind": kind, "sequences": sequences, "kv_heads": kv_heads, "head_dim": head_dim, "positions": _log(rng, 1, 3000),
                "tokens": _log(rng, 1, max(8, most)), "format": form}
    if kind == "attend":
        sequences = _log(rng, 1, 64)
        most = min(131000, 120000000 // (sequences * row))
        weights = rng.random() < 0.3
        tokens = rng.choice([1, 1, 2, 3, 4, 8])
        most = min(most, 650000000 // (sequences * heads * head_dim * tokens))
        return {"kind": kind, "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "positions": _log(rng, 1, most), "tokens": tokens, "format": form, "gate": rng.random() < 0.5, "weights": weights}
    sequences = _log(rng, 1, 16)
    positions = _log(rng, 300, min(20000, 20000000 // (sequences * row)))
    budget = rng.randint(200, positions)
    step = rng.choice([0, 1, 16, 40])
    return {"kind": kind, "sequences": sequences, "kv_heads": kv_heads, "head_dim": head_dim,
            "positions": budget if step else positions, "step": step, "budget": budget, "first": rng.randint(0, 20),
            "last": rng.randint(40, 100), "format": form}


# ---- inputs ----------------------------------------------------------------------------


class State:
    """What a case's program keeps between passes."""


def _normal(gen, *shape):
    return torch.randn(*shape, device=DEVICE, generator=gen)


def _channels(gen, width):
    """Some channels of real keys are many times larger than the rest."""
    return torch.exp(0.5 * _normal(gen, width))


def _counts(case):
    """Query or new tokens of each sequence: a verify batch brings one to `tokens` of them."""
    n, most = case["sequences"], case["tokens"]
    return [most if n == 1 else 1 + i % most for i in range(n)] if most <= 8 else [most - (i * 7) % (most // 2) for i in range(n)]


def _held(case):
    """Rows that each sequence has in its cache ahead of the call."""
    n, most = case["sequences"], case["positions"]
    if n == 1 or case["kind"] == "evict":
        return [most] * n
    return [most * i // (n - 1) for i in range(n)] if case["kind"] == "attend" else [max(0, most - 13 * i) for i in range(n)]


def _inputs(case, seed):
    """The case's inputs, the same for every way to compute it."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    d = {}
    if case["kind"] == "rope":
        heads, kv, hd, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
        # Rows of an attention layer's input product: each head's query and gate, then keys and values.
        d["in"] = _normal(gen, tokens, 2 * heads * hd + 2 * kv * hd) * torch.exp(0.5 * _normal(gen, 1, 2 * heads * hd + 2 * kv * hd))
        d["q_norm"], d["k_norm"] = 1.0 + 0.1 * _normal(gen, hd), 1.0 + 0.1 * _normal(gen, hd)
        if tokens > 64:   # a prompt: one position after another
            d["at"] = (torch.arange(tokens, device=DEVICE) + max(0, case["farthest"] - tokens)).int()
        else:
            d["at"] = torch.randint(0, case["farthest"], (tokens,), device=DEVICE, generator=gen).int()
        return d
    n, kv, hd = case["sequences"], case["kv_heads"], case["head_dim"]
    held = _held(case)
    d["positions"] = torch.tensor(held, dtype=torch.int32, device=DEVICE)
    scale = _channels(gen, kv * hd).view(kv, hd)
    d["old_k"], d["old_v"] = _normal(gen, sum(held), kv, hd) * scale, _normal(gen, sum(held), kv, hd)
    if case["kind"] == "append":
        rows = sum(_counts(case))
        # A later row may be larger than all that its block holds.
        d["k"], d["v"] = _normal(gen, rows, kv, hd) * scale * 1.5, _normal(gen, rows, kv, hd) * 1.5
    elif case["kind"] == "attend":
        counts = _counts(case)
        d["new_k"], d["new_v"] = _normal(gen, sum(counts), kv, hd) * scale, _normal(gen, sum(counts), kv, hd)
        d["q"] = _normal(gen, sum(counts), case["heads"], 2 if case["gate"] else 1, hd)   # query, gate
        d["q"][:, :, 0] *= 1.5 / scale.repeat_interleave(case["heads"] // kv, 0)
        if case["weights"]:
            d["weights"] = torch.rand(n, kv, _capacity(case), device=DEVICE, generator=gen)
    else:
        # Sums of softmax weights: a few rows hold most of them, many have next to none, some the same.
        w = torch.exp(2.0 * _normal(gen, n, kv, _capacity(case)))
        d["weights"] = torch.where(w < 0.2, torch.zeros_like(w), w)
        if case["step"]:
            d["k"], d["v"] = _normal(gen, n * case["step"], kv, hd) * scale * 1.5, _normal(gen, n * case["step"], kv, hd)
    return d


def _capacity(case):
    most = case["positions"] + (case["step"] if case["kind"] == "evict" else case["tokens"])
    return (most + BLOCK - 1) // BLOCK * BLOCK


def prepare(case, seed):
    s = State()
    s.case = case
    s.d = _inputs(case, seed)
    (_prepare_own if own else _prepare_plain)(s)
    torch.cuda.synchronize()
    return s


def _prepare_own(s):
    from gufo_npu_b200.backend import Context
    from gufo_npu_b200.cache8 import CudaCache8
    case, d = s.case, s.d
    torch.cuda.synchronize()
    s.ctx = Context(0)
    if case["kind"] == "rope":
        tokens, hd = case["tokens"], case["head_dim"]
        s.rope = s.ctx.rope_create(case["rope_dim"], theta=1e7, layout=case["layout"], **_scaling(case))
        s.q, s.k = (torch.empty(tokens, case[h], hd, device=DEVICE) for h in ("heads", "kv_heads"))
        q, k = _rope_rows(case, d["in"])
        norms = (d["q_norm"], d["k_norm"]) if case["norm"] else (None, None)
        s.parts = s.ctx.rope_parts([(q, s.q, norms[0]), (k, s.k, norms[1])], rms_eps=1e-6)
        return
    n, kv, hd = case["sequences"], case["kv_heads"], case["head_dim"]
    held = _held(case)
    s.cache = CudaCache8(s.ctx, n, kv, hd, _capacity(case), format=case["format"], weights="weights" in d)
    s.zero = torch.zeros(n, dtype=torch.int32, device=DEVICE)
    torch.cuda.synchronize()
    s.cache.append_device(s.cache.batch(s.zero, tokens=held), d["old_k"], d["old_v"])
    if case["kind"] == "append":
        s.batch = s.cache.batch(d["positions"], tokens=_counts(case))
        first, rows = _touched(case)
        s.first = torch.tensor(first, dtype=torch.int32, device=DEVICE)
        s.read = s.cache.batch(s.first, tokens=rows)
        s.out = torch.empty(2, sum(rows), kv, hd, device=DEVICE)
    elif case["kind"] == "attend":
        s.batch = s.cache.batch(d["positions"], tokens=_counts(case))
        s.cache.append_device(s.batch, d["new_k"], d["new_v"])
        s.out = torch.empty(sum(_counts(case)), case["heads"], hd, device=DEVICE)
        s.scratch = s.cache.scratch(case["heads"], sum(_counts(case)), accumulate=case["weights"])
    else:
        s.rows = min(case["budget"], case["positions"] + case["step"])
        s.kept = torch.empty(n, kv, case["budget"], dtype=torch.int32, device=DEVICE)
        s.out = torch.empty(2, n * s.rows, kv, hd, device=DEVICE)
        s.into = None
        if case["step"]:
            s.batch = s.cache.batch(d["positions"], tokens=[case["step"]] * n)
        else:
            s.into = CudaCache8(s.ctx, n, kv, hd, (s.rows + BLOCK - 1) // BLOCK * BLOCK, format=case["format"], weights=True)
        s.total = d["positions"] + case["step"]
        s.all = s.cache.batch(s.total)
        s.read = (s.into or s.cache).batch(s.zero, tokens=[s.rows] * n)
    s.ctx.synchronize()
    if "weights" in d:
        s.cache.weights.copy_(d["weights"])


def _prepare_plain(s):
    case, d = s.case, s.d
    if case["kind"] == "rope":
        s.inv_freq, s.magnitude = _frequencies(case)
        return
    n, kv, hd = case["sequences"], case["kv_heads"], case["head_dim"]
    cap = _capacity(case)
    held = _held(case)
    kind = torch.float8_e4m3fn if case["format"] == "e4m3" else torch.int8
    s.codes = [torch.zeros(n, kv, cap, hd, device=DEVICE).to(kind) for _ in "kv"]
    s.scales = [torch.zeros(n, kv, cap // BLOCK, device=DEVICE) for _ in "kv"]
    zero = torch.zeros(n, dtype=torch.int32, device=DEVICE)
    _append(s, zero, held, (d["old_k"], d["old_v"]))
    if case["kind"] == "attend":
        _append(s, d["positions"], _counts(case), (d["new_k"], d["new_v"]))
    if "weights" in d:
        s.weights = d["weights"].clone()


def _scaling(case):
    """Arguments of rope_create for contexts longer than the first 32768 positions."""
    return {"none": {}, "linear": {"scaling": "linear", "factor": 4.0},
            "by_parts": {"scaling": "by_parts", "factor": 8.0, "original_positions": 32768, "fast_turns": 32.0,
                         "slow_turns": 1.0, "magnitude": 1.2079}}[case["scaling"]]


def _rope_rows(case, rows):
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    q = rows[:, :2 * heads * hd].view(-1, heads, 2, hd)[:, :, 0]
    return q, rows[:, 2 * heads * hd:2 * heads * hd + kv * hd].view(-1, kv, hd)


def _touched(case):
    """The first row of the first block that an append reaches, and the rows from there on, of each sequence."""
    held = _held(case)
    first = [p // BLOCK * BLOCK for p in held]
    return first, [p + c - f for p, c, f in zip(held, _counts(case), first)]


# ---- one pass --------------------------------------------------------------------------


def run(state):
    return globals()[("_own_" if own else "_plain_") + state.case["kind"]](state)


def _own_rope(s):
    s.ctx.rope_device(s.rope, s.parts, s.d["at"])
    return [s.q, s.k]


def _own_append(s):
    s.cache.append_device(s.batch, s.d["k"], s.d["v"])
    s.cache.rows_device(s.read, s.out[0], s.out[1])
    return s.out


def _own_attend(s):
    q = s.d["q"]
    s.cache.attend_device(s.batch, q[:, :, 0], s.out, gate=q[:, :, 1] if s.case["gate"] else None, scratch=s.scratch,
                          accumulate=s.case["weights"])
    return {"out": s.out, "weights": s.cache.weights} if s.case["weights"] else {"out": s.out}


def _own_evict(s):
    case = s.case
    if case["step"]:
        s.cache.append_device(s.batch, s.d["k"], s.d["v"])
    s.cache.evict_device(s.all, case["budget"], s.kept, first=case["first"], last=case["last"], into=s.into)
    cache = s.into or s.cache
    cache.rows_device(s.read, s.out[0], s.out[1])
    return {"kept": s.kept, "rows": s.out, "weights": cache.weights[:, :, :s.rows]}


# ---- the plain forms -------------------------------------------------------------------


def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor of the rotated values."""
    more = _scaling(case)
    pairs = case["rope_dim"] // 2
    freq = 1e7 ** (-torch.arange(pairs, device=DEVICE, dtype=torch.float64) / pairs)
    if case["scaling"] == "linear":
        freq = freq / more["factor"]
    elif case["scaling"] == "by_parts":
        # Pairs that turn more than `fast_turns` times over the original positions stay, those that turn less than
        # `slow_turns` times are stretched, the ones between are mixed, evenly over the pair's number.
        def pair_of(turns):
            return pairs * math.log(more["original_positions"] / (turns * 2.0 * math.pi)) / math.log(1e7)
        low, high = max(math.floor(pair_of(more["fast_turns"])), 0), min(math.ceil(pair_of(more["slow_turns"])), pairs - 1)
        ramp = ((torch.arange(pairs, device=DEVICE, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / more["factor"] * ramp
    return freq, more.get("magnitude", 1.0)


def _rotate(x, cos, sin, rope_dim, layout):
    turned, rest = x[..., :rope_dim], x[..., rope_dim:]
    if layout == "halves":
        a, b = turned[..., :rope_dim // 2], turned[..., rope_dim // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    case, d = s.case, s.d
    angle = d["at"].double()[:, None] * s.inv_freq
    cos, sin = ((f(angle) * s.magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    out = []
    for x, w in zip(_rope_rows(case, d["in"]), (d["q_norm"], d["k_norm"])):
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        out.append(_rotate(x, cos, sin, case["rope_dim"], case["layout"]))
    return out


def _power(e):
    """2^e in fp32 for whole numbers from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _scale_of(top, kind):
    """The smallest power of two (2^-126 or more) with which `top` is at most the largest code."""
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8) if kind == torch.float8_e4m3fn else torch.where(m <= 127 / 128, e - 7, e - 6)
    return _power(torch.where(top > 0, e, torch.full_like(e, -126)).clamp(min=-126))


def _encode(x, kind):
    return x.clamp(-448.0, 448.0).to(kind) if kind == torch.float8_e4m3fn else torch.round(x).clamp(-127.0, 127.0).to(kind)


def _append(s, positions, counts, rows):
    """Rows of every sequence behind its `positions`, a block's codes rounded to its new scale."""
    n, kv, cap, hd = s.codes[0].shape
    blocks = min(cap // BLOCK, (max(counts) + BLOCK - 1) // BLOCK + 1)
    count = torch.tensor(counts, device=DEVICE)
    start = positions.long() // BLOCK
    first = torch.minimum(start, torch.full_like(start, cap // BLOCK - blocks))
    seq = torch.repeat_interleave(torch.arange(n, device=DEVICE), count)
    nth = torch.arange(sum(counts), device=DEVICE) - torch.repeat_interleave(count.cumsum(0) - count, count)
    row = positions.long()[seq] + nth - first[seq] * BLOCK
    at = (first[:, None] + torch.arange(blocks, device=DEVICE))            # [n, blocks]
    place = torch.arange(blocks * BLOCK, device=DEVICE).view(1, 1, blocks, BLOCK, 1) + (first * BLOCK).view(n, 1, 1, 1, 1)
    old = place < positions.view(n, 1, 1, 1, 1)
    new = ~old & (place < (positions + count).view(n, 1, 1, 1, 1))
    who = torch.arange(n, device=DEVICE)[:, None]
    for i in range(2):
        x = torch.zeros(n, blocks * BLOCK, kv, hd, device=DEVICE)
        x[seq, row] = rows[i]
        x = x.view(n, blocks, BLOCK, kv, hd).permute(0, 3, 1, 2, 4)       # [n, kv, blocks, 16, hd]
        codes = s.codes[i].view(n, kv, cap // BLOCK, BLOCK, hd)
        here = codes.view(torch.int8).permute(0, 2, 1, 3, 4)[who, at].permute(0, 2, 1, 3, 4).contiguous().view(codes.dtype)
        was = s.scales[i].permute(0, 2, 1)[who, at].permute(0, 2, 1)[..., None, None]
        top = x.abs().amax((-2, -1), keepdim=True)
        scale = torch.where(new.any(-2, keepdim=True), _scale_of(top, codes.dtype), was)
        scale = torch.where(old.any(-2, keepdim=True), torch.maximum(scale, was), scale)
        again = _encode(here.float() * (was / scale).nan_to_num(), codes.dtype)
        done = torch.where(new, _encode(x / scale, codes.dtype).view(torch.int8),
                           torch.where(old, again.view(torch.int8), here.view(torch.int8)))
        codes.view(torch.int8).permute(0, 2, 1, 3, 4)[who, at] = done.permute(0, 2, 1, 3, 4)
        s.scales[i].permute(0, 2, 1)[who, at] = scale[..., 0, 0].permute(0, 2, 1)


def _values(s, i, rows):
    """What the first `rows` rows of every head stand for: [n, kv, rows, hd]."""
    n, kv, cap, hd = s.codes[i].shape
    blocks = (rows + BLOCK - 1) // BLOCK
    x = s.codes[i][:, :, :blocks * BLOCK].float().view(n, kv, blocks, BLOCK, hd) * s.scales[i][:, :, :blocks, None, None]
    return x.view(n, kv, blocks * BLOCK, hd)[:, :, :rows]


def _plain_append(s):
    case, d = s.case, s.d
    _append(s, d["positions"], _counts(case), (d["k"], d["v"]))
    first, rows = _touched(case)
    n = case["sequences"]
    count = torch.tensor(rows, device=DEVICE)
    seq = torch.repeat_interleave(torch.arange(n, device=DEVICE), count)
    row = torch.arange(sum(rows), device=DEVICE) - torch.repeat_interleave(count.cumsum(0) - count, count)
    row = row + torch.tensor(first, device=DEVICE)[seq]
    out = []
    for i in range(2):
        codes = s.codes[i].view(torch.int8).permute(0, 2, 1, 3)[seq, row].view(s.codes[i].dtype).float()
        out.append(codes * s.scales[i].permute(0, 2, 1)[seq, row // BLOCK][..., None])
    return torch.stack(out)


def _padded(case):
    """Where each query token stands in [sequences, most tokens], as flat numbers."""
    counts = _counts(case)
    most = max(counts)
    return most, torch.tensor([i * most + t for i, c in enumerate(counts) for t in range(c)], device=DEVICE)


def _plain_attend(s):
    case, d = s.case, s.d
    n, kv, hd, heads = case["sequences"], case["kv_heads"], case["head_dim"], case["heads"]
    group = heads // kv
    most, at = _padded(case)
    rows = case["positions"] + case["tokens"]
    q = torch.zeros(n * most, heads, hd, device=DEVICE)
    q[at] = d["q"][:, :, 0]
    q = q.view(n, most, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, hd)
    k, v = _values(s, 0, rows), _values(s, 1, rows)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(hd)
    seen = d["positions"].view(n, 1) + 1 + torch.arange(most, device=DEVICE)           # token t sees the rows up to its own
    hidden = torch.arange(rows, device=DEVICE).view(1, 1, 1, rows) >= seen.repeat_interleave(group, 1).view(n, 1, -1, 1)
    score = score.masked_fill(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).view(n, kv, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n * most, heads, hd)[at]
    if case["gate"]:
        out = out / (1.0 + torch.exp(-d["q"][:, :, 1]))
    if not case["weights"]:
        return {"out": out}
    there = torch.zeros(n * most, device=DEVICE)
    there[at] = 1.0
    p = p * there.view(n, 1, most, 1).expand(n, 1, most, group).reshape(n, 1, -1, 1)
    s.weights[:, :, :rows] += p.sum(-2)
    return {"out": out, "weights": s.weights}


def _chosen(weights, rows, budget, first, last):
    """The rows that stay, ascending: `first` and `last` ones, and of the others those of most weight (ties: the
    lowest row): [n, kv, budget]; -1 behind them where there are fewer."""
    n, kv = weights.shape[:2]
    if rows <= budget:
        kept = torch.arange(budget, device=DEVICE)
        return torch.where(kept < rows, kept, -1).int().expand(n, kv, budget).contiguous()
    # The oldest rows come first where the two do not fit together.
    first = min(first, budget)
    last = min(last, budget - first)
    more = budget - first - last
    order = torch.sort(weights[:, :, first:rows - last], dim=-1, descending=True, stable=True)[1][:, :, :more] + first
    ends = [torch.arange(first, device=DEVICE), torch.arange(rows - last, rows, device=DEVICE)]
    ends = [e.expand(n, kv, e.numel()) for e in ends]
    return torch.cat([ends[0], order, ends[1]], -1).sort(-1).values.int()


def _plain_evict(s):
    case, d = s.case, s.d
    n, kv, hd = case["sequences"], case["kv_heads"], case["head_dim"]
    total = case["positions"] + case["step"]
    if case["step"]:
        _append(s, d["positions"], [case["step"]] * n, (d["k"], d["v"]))
        s.weights[:, :, case["positions"]:total] = 0.0
    kept = _chosen(s.weights, total, case["budget"], case["first"], case["last"])
    rows = min(total, case["budget"])
    blocks = (rows + BLOCK - 1) // BLOCK
    at = kept[:, :, :rows].long()
    weights = s.weights.gather(-1, at)
    out = []
    for i in range(2):
        kind = s.codes[i].dtype
        x = _values(s, i, total).gather(2, at[..., None].expand(n, kv, rows, hd))
        x = torch.cat([x, torch.zeros(n, kv, blocks * BLOCK - rows, hd, device=DEVICE)], 2).view(n, kv, blocks, BLOCK, hd)
        scale = _scale_of(x.abs().amax((-2, -1)), kind)
        codes = _encode(x / scale[..., None, None], kind).view(n, kv, blocks * BLOCK, hd)
        out.append((codes.float().view(n, kv, blocks, BLOCK, hd) * scale[..., None, None]).view(n, kv, -1, hd)[:, :, :rows])
        if case["step"]:
            s.codes[i].view(torch.int8)[:, :, :rows] = codes.view(torch.int8)[:, :, :rows]
            s.scales[i][:, :, :blocks] = scale
    if case["step"]:
        s.weights[:, :, :rows] = weights
    return {"kept": kept, "rows": torch.stack(out).permute(0, 1, 3, 2, 4).reshape(2, n * rows, kv, hd),
            "weights": weights}


# ---- what a pass cannot do without, and the same from the definitions in 64 bits --------


def work(case):
    kv, hd, kind = case["kv_heads"], case["head_dim"], case["kind"]
    if kind == "rope":
        rows = case["tokens"] * (case["heads"] + kv)
        return {"bytes": 4 * (2 * rows * hd + case["tokens"] + 2 * hd), "flops": rows * (6 * case["rope_dim"] // 2 + 4 * hd * case["norm"])}
    n = case["sequences"]
    row = 2 * kv * hd          # bytes of a row's codes, keys and values
    if kind == "append":
        new, touched = sum(_counts(case)), sum(_touched(case)[1])
        # New rows in; the rows beside them in their blocks in; all of them as codes out, and as values.
        return {"bytes": new * row * 4 + (touched - new) * row + touched * row * 5, "flops": 2 * touched * row}
    if kind == "attend":
        counts, held = _counts(case), _held(case)
        rows = sum(h + c for h, c in zip(held, counts))
        seen = sum(sum(h + 1 + t for t in range(c)) for h, c in zip(held, counts))
        wide = sum(counts) * case["heads"] * hd
        return {"bytes": rows * (row + 8 * kv // BLOCK + 8 * kv * case["weights"]) + 4 * wide * (3 if case["gate"] else 2),
                "flops": 4 * seen * case["heads"] * hd}
    total = case["positions"] + case["step"]
    rows = min(case["budget"], total)
    # The weights in; the rows that stay in, as codes out, and as values; their numbers and weights out.
    return {"bytes": n * (4 * kv * total + rows * row * 6 + 8 * kv * rows + 4 * case["step"] * row), "flops": n * rows * row}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, d)
    n, kv, hd = case["sequences"], case["kv_heads"], case["head_dim"]
    held, e4m3 = _held(case), case["format"] == "e4m3"

    def split(rows, counts):
        """[rows, kv, hd] in fp32 as a list of each sequence's [kv, rows, hd] in 64 bits."""
        return [x.double().permute(1, 0, 2) for x in rows.split(counts)]
    old = [split(d[name], held) for name in ("old_k", "old_v")]
    kept = [[_rounded(x, e4m3, None, 0)[0] for x in side] for side in old]
    if case["kind"] == "append":
        counts = _counts(case)
        new = [split(d[name], counts) for name in ("k", "v")]
        first, _ = _touched(case)
        out = []
        for side in range(2):
            rows = []
            for i in range(n):
                x = _joined(kept[side][i], old[side][i], new[side][i], e4m3)
                rows.append(x[:, first[i]:].permute(1, 0, 2))
            out.append(torch.cat(rows))
        return torch.stack(out)
    if case["kind"] == "attend":
        return _exact_attend(case, d, kept, old, split)
    return _exact_evict(case, d, kept, old, split)


def _exact_rope(case, d):
    more, rope = _scaling(case), case["rope_dim"]
    theta = []
    for i in range(rope // 2):
        f = 1e7 ** (-2.0 * i / rope)
        if case["scaling"] == "linear":
            f /= more["factor"]
        elif case["scaling"] == "by_parts":
            ends = [rope * math.log(more["original_positions"] / (2 * math.pi * more[t])) / (2 * math.log(1e7))
                    for t in ("fast_turns", "slow_turns")]
            low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rope // 2 - 1)
            slow = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
            f = f * (1.0 - slow) + slow * f / more["factor"]
        theta.append(f)
    angle = d["at"].double()[:, None, None] * torch.tensor(theta, dtype=torch.float64, device=DEVICE)
    turn = torch.polar(torch.full_like(angle, more.get("magnitude", 1.0)), angle)      # complex: [tokens, 1, pairs]
    out = []
    for x, w in zip(_rope_rows(case, d["in"]), (d["q_norm"], d["k_norm"])):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
        y = x.clone()
        halves = case["layout"] == "halves"
        a, b = (slice(0, rope // 2), slice(rope // 2, rope)) if halves else (slice(0, rope, 2), slice(1, rope, 2))
        z = torch.complex(x[..., a], x[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    return out


def _nearest(x, e4m3):
    """Multiples of a code's step nearest to x, halves to even: e4m3 has 3 fraction bits down to 2^-6."""
    if not e4m3:
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    # (log2 of a value just under a power of two may round up to it.)
    step = torch.where(x.abs().clamp(min=2.0 ** -6) < 8 * step, step / 2, step)
    return torch.round(x / step) * step


def _rounded(x, e4m3, least, held):
    """x: [kv, rows, hd] in 64 bits, a block's rows rounded to codes of its scale; `least`: the first block's scale is
    no smaller, as `held` rows ahead of x are in it already. Returns the values and each row's scale."""
    kv, rows, hd = x.shape
    pad = -(held + rows) % BLOCK
    z = torch.cat([x.new_zeros(kv, held, hd), x, x.new_zeros(kv, pad, hd)], 1).view(kv, -1, BLOCK, hd)
    top = z.abs().amax((2, 3), keepdim=True)
    most = 448.0 if e4m3 else 127.0
    scale = torch.exp2(torch.ceil(torch.log2(top / most)).clamp(min=-126.0))
    scale = torch.where(top > most * scale, scale * 2, torch.where(top <= most * scale / 2, scale / 2, scale)).clamp(min=2.0 ** -126)
    if least is not None and held:
        scale[:, :1] = torch.maximum(scale[:, :1], least.view(kv, 1, 1, 1))
    y = (_nearest(z / scale, e4m3) * scale).view(kv, -1, hd)[:, held:held + rows]
    return y, scale.view(kv, -1).repeat_interleave(BLOCK, 1)[:, held:held + rows]


def _joined(kept, old, new, e4m3):
    """The cache of one sequence and side behind an append: `kept` holds the values of `old`."""
    held = kept.shape[1] % BLOCK
    whole = kept.shape[1] - held
    if not held:
        return torch.cat([kept, _rounded(new, e4m3, None, 0)[0]], 1)
    was = _rounded(old[:, whole:], e4m3, None, 0)[1][:, 0]
    values, scale = _rounded(new, e4m3, was, held)
    now = scale[:, :1, None]
    return torch.cat([kept[:, :whole], _nearest(kept[:, whole:] / now, e4m3) * now, values], 1)


def _exact_attend(case, d, kept, old, split):
    kv, hd, heads, counts = case["kv_heads"], case["head_dim"], case["heads"], _counts(case)
    e4m3 = case["format"] == "e4m3"
    new = [split(d[name], counts) for name in ("new_k", "new_v")]
    queries = d["q"].double().split(counts)
    outs = []
    weights = d["weights"].double() if case["weights"] else None
    for i, (held, count) in enumerate(zip(_held(case), counts)):
        k, v = (_joined(kept[side][i], old[side][i], new[side][i], e4m3) for side in range(2))
        for t in range(count):
            see = held + 1 + t
            q = queries[i][t, :, 0].view(kv, heads // kv, hd)
            p = torch.softmax(torch.einsum("kgd,knd->kgn", q, k[:, :see]) / math.sqrt(hd), -1)
            o = torch.einsum("kgn,knd->kgd", p, v[:, :see]).reshape(heads, hd)
            outs.append(o * torch.sigmoid(queries[i][t, :, 1]) if case["gate"] else o)
            if weights is not None:
                weights[i, :, :see] += p.sum(1)
    out = {"out": torch.stack(outs)}
    if weights is not None:
        out["weights"] = weights
    return out


def _exact_evict(case, d, kept, old, split):
    n, kv, total = case["sequences"], case["kv_heads"], case["positions"] + case["step"]
    e4m3, budget = case["format"] == "e4m3", case["budget"]
    rows = min(total, budget)
    weights = d["weights"].double().cpu().numpy().copy()
    new = [split(d[name], [case["step"]] * n) for name in ("k", "v")] if case["step"] else None
    weights[:, :, case["positions"]:total] = 0.0
    choice = np.full((n, kv, budget), -1, dtype=np.int32)
    for i in range(n):
        for h in range(kv):
            stay = np.arange(total)
            if total > budget:
                first = min(case["first"], budget)
                last = min(case["last"], budget - first)
                inner = np.arange(first, total - last)
                by = np.lexsort((inner, -weights[i, h, inner]))[:budget - first - last]
                stay = np.sort(np.concatenate([np.arange(first), inner[by], np.arange(total - last, total)]))
            choice[i, h, :rows] = stay
    at = torch.from_numpy(choice[:, :, :rows].astype(np.int64)).to(DEVICE)
    sides = []
    for side in range(2):
        values = []
        for i in range(n):
            x = kept[side][i]
            if case["step"]:
                x = _joined(x, old[side][i], new[side][i], e4m3)
            x = torch.stack([x[h, at[i, h]] for h in range(kv)])
            values.append(_rounded(x, e4m3, None, 0)[0].permute(1, 0, 2))
        sides.append(torch.cat(values))
    chosen = torch.from_numpy(np.take_along_axis(weights, choice[:, :, :rows].astype(np.int64), -1)).to(DEVICE)
    return {"kept": torch.from_numpy(choice).to(DEVICE), "rows": torch.stack(sides), "weights": chosen}
