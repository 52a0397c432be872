"""The key / value cache in 8 bits: `CudaCache8` over the C ABI's gufo_cuda_cache8 entries.

One cache holds the keys and values of one attention layer for a number of sequences. A call
takes a batch of them (`batch`: made once, used for every layer and step); the number of rows a
sequence holds is a device tensor of the caller's, one for all layers, as it is for the fp16
cache of gufo_cuda_attention_device. Everything here only enqueues on the context's stream.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

from . import _capi
from .backend import Context, _DeviceArray, check_ints


class Batch:
    """Sequences of a call: slots and tokens as the library takes them, and the positions they start at."""

    def __init__(self, device: int, positions, tokens: Optional[Sequence[int]], slots: Optional[Sequence[int]]):
        check_ints("cache8", device, positions)
        self.device = device
        n = positions.numel()
        for name, values in (("tokens", tokens), ("slots", slots)):
            if values is not None and len(values) != n:
                raise ValueError(f"cache8: {n} positions and {len(values)} {name}")
        self.sequences = n
        self.positions = positions
        self.rows = n if tokens is None else sum(tokens)
        self._tokens = None if tokens is None else (C.c_int * n)(*tokens)
        self._slots = None if slots is None else (C.c_int * n)(*slots)
        self.args = _capi.Cache8Batch(n, C.cast(self._slots, C.c_void_p) if slots is not None else None,
                                      C.cast(self._tokens, C.c_void_p) if tokens is not None else None,
                                      positions.data_ptr())


class Scratch:
    """Scratch of attention calls that run one after another: one for each stream or captured graph that
    may be in flight beside others."""

    def __init__(self, ctx: Context, nbytes: int):
        self.ctx, self.bytes, self.ptr = ctx, nbytes, 0
        self.ptr = ctx.malloc(nbytes)

    def close(self) -> None:
        if self.ptr and self.ctx.handle:
            self.ctx.free(self.ptr)
        self.ptr = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _Owner:
    """The library's cache: freed when neither its CudaCache8 nor a tensor over its memory is left."""

    def __init__(self, ctx: Context, config: "_capi.Cache8Config"):
        self.ctx, self.handle = ctx, 0
        out = C.c_int64()
        ctx._check(ctx.lib.gufo_cuda_cache8_create(ctx.handle, C.byref(config), C.byref(out)))
        self.handle = int(out.value)

    def close(self) -> None:
        if self.handle and self.ctx.handle:
            self.ctx.lib.gufo_cuda_cache8_free(self.ctx.handle, self.handle)
        self.handle = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class CudaCache8:
    """Keys and values of one attention layer, a byte a value (gufo_cuda_cache8)."""

    def __init__(self, ctx: Context, sequences: int, kv_heads: int, head_dim: int, capacity: int, format: str = "e4m3",
                 weights: bool = False):
        if format not in _capi.CACHE8_FORMATS:
            raise ValueError(f"cache8: formats are {sorted(_capi.CACHE8_FORMATS)}")
        self.ctx = ctx
        self.sequences, self.kv_heads, self.head_dim, self.capacity = sequences, kv_heads, head_dim, capacity
        self.format = format
        config = _capi.Cache8Config(sequences, kv_heads, head_dim, capacity, _capi.CACHE8_FORMATS[format], int(weights))
        self._owner = _Owner(ctx, config)
        self.handle = self._owner.handle
        self._weights = None
        if weights:
            import torch
            ptr = C.c_void_p()
            ctx._check(ctx.lib.gufo_cuda_cache8_weights(ctx.handle, self.handle, C.byref(ptr)))
            memory = _DeviceArray(int(ptr.value), sequences * kv_heads * capacity)
            memory.owner = self._owner      # (the tensor keeps `memory`)
            flat = torch.as_tensor(memory, device=torch.device("cuda", ctx.device))
            self._weights = flat.view(sequences, kv_heads, capacity)

    def close(self) -> None:
        """Frees the cache at once; tensors over its weights must not be used after."""
        self._owner.close()
        self.handle = 0
        self._weights = None

    @property
    def weights(self):
        """The accumulated weights [sequences, kv_heads, capacity], the cache's own memory; None without."""
        return self._weights

    def batch(self, positions, tokens: Optional[Sequence[int]] = None, slots: Optional[Sequence[int]] = None) -> Batch:
        """Sequences of a call: `positions` (int32, device) rows held ahead of it, `tokens` rows each (one
        without), in `slots` (0, 1, ... without)."""
        return Batch(self.ctx.device, positions, tokens, slots)

    def _ctx_of(self, batch: Batch) -> Context:
        if batch.device != self.ctx.device:
            raise ValueError("cache8: the batch is another device's")
        return self.ctx

    def scratch(self, heads: int, tokens: int, accumulate: bool = False) -> Scratch:
        """Scratch of attend_device calls with up to `tokens` query tokens in all."""
        nbytes = C.c_size_t()
        self.ctx._check(self.ctx.lib.gufo_cuda_cache8_attend_scratch(self.ctx.handle, self.handle, heads, tokens,
                                                                     int(accumulate), C.byref(nbytes)))
        return Scratch(self.ctx, nbytes.value)

    def append_device(self, batch: Batch, keys, values) -> None:
        """Writes the batch's rows, [rows, kv_heads, head_dim] each, at their positions."""
        ctx = self._ctx_of(batch)
        ctx._check(_capi.native.cache8_append(ctx._address, ctx.device, self.handle, batch.args, batch.rows, self.kv_heads,
                                              self.head_dim, keys, values))

    def rows_device(self, batch: Batch, keys, values) -> None:
        """What the rows of an append with this batch stand for, into contiguous [rows, kv_heads, head_dim]."""
        ctx = self._ctx_of(batch)
        ctx._check(_capi.native.cache8_rows(ctx._address, ctx.device, self.handle, batch.args, batch.rows, self.kv_heads,
                                            self.head_dim, keys, values))

    def attend_device(self, batch: Batch, queries, out, scratch: Scratch, gate=None, scale: float = 0.0, visible=None,
                      accumulate: bool = False) -> None:
        """out = softmax(queries K^T scale) V [* sigmoid(gate)] for [rows, heads, head_dim] query rows. Token t of
        a sequence sees the rows up to position + t, or the first visible[...] (int32, a value per row of
        queries). `accumulate` adds what each cached row was given to `weights`."""
        ctx = self._ctx_of(batch)
        if scratch.ctx.device != ctx.device:
            raise ValueError("cache8: the scratch is another device's")
        ctx._check(_capi.native.cache8_attend(ctx._address, ctx.device, self.handle, batch.args, batch.rows, self.head_dim,
                                              queries, out, gate, visible, scale, accumulate, scratch.ptr, scratch.bytes))

    def evict_device(self, batch: Batch, budget: int, kept, first: int = 0, last: int = 0, held=None,
                     into: Optional["CudaCache8"] = None, into_slots: Optional[Sequence[int]] = None) -> None:
        """Brings the batch's sequences (their `positions` rows) down to `budget` rows: the first `first`, the
        last `last`, and the rest by weight; in place, or into another cache's slots. `kept` (int32
        [sequences, kv_heads, budget]) gets the rows that stayed, `held` (int32 [sequences]) how many."""
        if tuple(kept.shape) != (batch.sequences, self.kv_heads, budget):
            raise ValueError(f"cache8: kept is [{batch.sequences}, {self.kv_heads}, {budget}], not {list(kept.shape)}")
        slots = None
        if into_slots is not None:
            if len(into_slots) != batch.sequences:
                raise ValueError(f"cache8: {batch.sequences} sequences and {len(into_slots)} slots")
            slots = (C.c_int * batch.sequences)(*into_slots)
        if into is not None and into.ctx is not self.ctx:
            raise ValueError("cache8: both caches belong to one context")
        if into is not None and not into.handle:      # (0 is the library's word for an eviction in place)
            raise ValueError("cache8: into is closed")
        ctx = self._ctx_of(batch)
        ctx._check(_capi.native.cache8_evict(ctx._address, ctx.device, self.handle, batch.args, batch.sequences, self.kv_heads,
                                             budget, first, last, kept, held, into.handle if into is not None else 0, slots))
