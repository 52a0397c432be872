// The key / value cache in 8 bits: its two formats, its blocks, the sequences of a call.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace gufo {

constexpr int kCacheBlock = GUFO_CUDA_CACHE8_BLOCK;   // rows that share a scale
constexpr int kCacheMaxSequences = 4096;
constexpr int kCacheMaxDim = 256;
constexpr int kBatchSequences = 128;   // of one launch: they are 2.6 KB of its arguments

// A sequence of a call.
struct BatchEntry {
  int index;    // in the call: of its position
  int slot;
  int tokens;
  int row;      // of the call's packed rows: its first
};
struct BatchArgs {
  BatchEntry of[kBatchSequences];
  int first_item[kBatchSequences + 1];   // work items ahead of a sequence's own (what an item is depends on the kernel)
  int sequences;
  const int* positions;
};
static_assert(sizeof(BatchArgs) <= 2600, "leaves room beside it in 4 KB of arguments");

// What a kernel sees of a cache. A block of 16 rows of a head is their codes, then their scale and
// 12 bytes of nothing: one contiguous copy. The codes stand by pairs of pieces (32 values), the 16
// rows' bytes of a pair together: a row's part of a pair is a sector, which is what a row that is
// gathered or written by itself costs (pieces alone: half of what is fetched is of another row; 8192
// rows scattered over 64 MB 24 us, not 16). The order of the rows within a pair lets the
// attention's lanes read their fragments from different places of shared memory: for keys eight
// lanes read four pieces of two rows, for values two pieces of every second row.
struct CacheView {
  uint8_t* sides[2];
  float* weights;
  int kv_heads, head_dim, capacity;
};
inline CacheView ViewOf(const Cache8& c) {
  return {{c.sides[0], c.sides[1]}, c.weights, c.c.kv_heads, c.c.head_dim, c.c.capacity};
}
__host__ __device__ inline int CodeBytes(int head_dim) { return (head_dim + 31) / 32 * 32 * kCacheBlock; }
__host__ __device__ inline int BlockBytes(int head_dim) { return CodeBytes(head_dim) + 16; }
// The first block of a head of a slot, and of a side's block its scale.
__device__ __forceinline__ uint8_t* BlocksOf(const CacheView& c, int side, size_t of_head) {
  return c.sides[side] + of_head * (c.capacity / kCacheBlock) * BlockBytes(c.head_dim);
}
__device__ __forceinline__ float* ScaleOf(uint8_t* block, int head_dim) {
  return reinterpret_cast<float*>(block + CodeBytes(head_dim));
}
__device__ __forceinline__ const float* ScaleOf(const uint8_t* block, int head_dim) {
  return reinterpret_cast<const float*>(block + CodeBytes(head_dim));
}
// Where a piece of a row stands in its block.
__device__ __forceinline__ int PieceAt(int side, int row, int piece) {
  const int pair = piece >> 1;
  const int at = side == 0 ? row ^ (2 * (pair & 1)) : row ^ (row >> 2 & 1);
  return pair * 512 + at * 32 + (piece & 1) * 16;
}

// Calls launch(args) for every run of at most kBatchSequences sequences with work and `limit` items;
// items(tokens) says how many items a sequence has, at most `limit`. Checks the batch (CheckBatch) has passed.
template <typename Items, typename Launch>
int ForEachRun(const gufo_cuda_cache8_batch& b, Items items, Launch launch, int limit = INT32_MAX) {
  BatchArgs a;
  a.positions = b.positions;
  int row = 0;
  for (int i = 0; i < b.sequences;) {
    a.sequences = 0;
    int at = 0;
    for (; i < b.sequences && a.sequences < kBatchSequences; ++i) {
      const int tokens = b.tokens != nullptr ? b.tokens[i] : 1;
      const int n = items(tokens);
      if (n > limit - at) {
        break;
      }
      if (n > 0) {
        a.of[a.sequences] = {i, b.slots != nullptr ? b.slots[i] : i, tokens, row};
        a.first_item[a.sequences++] = at;
        at += n;
      }
      row += tokens;
    }
    for (int s = a.sequences; s <= kBatchSequences; ++s) {
      a.first_item[s] = at;
    }
    if (at > 0) {
      if (const int rc = launch(a, at); rc != GUFO_CUDA_OK) {
        return rc;
      }
    }
  }
  return GUFO_CUDA_OK;
}

// The cache of a handle; ctx->mu is held.
int FindCache(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const char* what, const Cache8** out);
// Whether a batch's sequences, slots and (where `counted`) tokens are ones of the cache; the rows of all.
int CheckBatch(const Cache8& cache, const gufo_cuda_cache8_batch* b, const char* what, bool counted, int64_t* rows);

// The sequence of an item: the last one whose items start at or ahead of it.
__device__ __forceinline__ int SequenceOf(const BatchArgs& b, int item) {
  int low = 0, high = b.sequences - 1;
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (b.first_item[mid] <= item) {
      low = mid;
    } else {
      high = mid - 1;
    }
  }
  return low;
}

__device__ __forceinline__ int PositionOf(const CacheView& c, const BatchArgs& b, const BatchEntry& e) {
  return min(max(b.positions[e.index], 0), c.capacity);
}

// ---- formats ---------------------------------------------------------------
//
// Encode takes four values and the block's scale inverted (a power of two; the products are at most the
// largest code, or NaN) and rounds to the nearest code, ties to even: half a step, 2^-4 of the value for
// e4m3 (2^-10 below its smallest normal value), 0.5 for int8. Decode is exact in fp16.

struct E4m3 {
  static constexpr bool kHasNan = true;    // codes 0x7F and 0xFF
  static constexpr bool kWhole = false;    // codes are not whole numbers
  // The power of two of the smallest scale that holds a magnitude with these fp32 bits: 448 = 1.75 * 2^8.
  __device__ static int ScaleExponent(uint32_t bits) {
    return static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7);
  }
  __device__ static uint32_t Encode(float4 v, float inverse) {
    uint16_t low, high;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(v.y * inverse), "f"(v.x * inverse));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(v.w * inverse), "f"(v.z * inverse));
    return low | static_cast<uint32_t>(high) << 16;
  }
  // Bytes 0, 1 and bytes 2, 3 of a word as pairs of fp16.
  __device__ static void Decode(uint32_t word, uint32_t& first, uint32_t& second) {
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
        : "=r"(first), "=r"(second) : "r"(word));
  }
};

struct Int8 {
  static constexpr bool kHasNan = false;
  static constexpr bool kWhole = true;
  // 127 = 1.984375 * 2^6.
  __device__ static int ScaleExponent(uint32_t bits) {
    return static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x7E0000u ? 6 : 5);
  }
  // Beside 1.5 * 2^23 a value is rounded to a whole number in the low bits of the sum (a conversion runs at
  // a quarter of the rate). NaN, whose bits are anything, is 0.
  __device__ static uint32_t Encode(float4 v, float inverse) {
    const auto bits = [&](float x) { return __float_as_uint(fmaf(x == x ? x : 0.f, inverse, 12582912.0f)); };
    return __byte_perm(__byte_perm(bits(v.x), bits(v.y), 0x0040), __byte_perm(bits(v.z), bits(v.w), 0x0040), 0x5410);
  }
  // fp16 1024 + n has n in its low bits: bytes moved up by 128 beside 0x64, less 1152.
  __device__ static void Decode(uint32_t word, uint32_t& first, uint32_t& second) {
    const uint32_t up = word ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(up, 0x64646464u, 0x4140), b = __byte_perm(up, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    first = *reinterpret_cast<const uint32_t*>(&x);
    second = *reinterpret_cast<const uint32_t*>(&y);
  }
};

// 2^e for e from -126 to 127.
__device__ __forceinline__ float PowerOfTwo(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// The scale's exponent for a block whose largest magnitude is `top` (finite).
template <typename Format>
__device__ __forceinline__ int ScaleExponentOf(float top) {
  return max(Format::ScaleExponent(__float_as_uint(top)), -126);
}
__device__ __forceinline__ int ExponentOf(float scale) {   // of a power of two
  return static_cast<int>(__float_as_uint(scale) >> 23) - 127;
}
// Four codes as values.
template <typename Format>
__device__ __forceinline__ float4 DecodeFour(uint32_t word) {
  uint32_t a, b;
  Format::Decode(word, a, b);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return make_float4(x.x, x.y, y.x, y.y);
}

}  // namespace gufo
