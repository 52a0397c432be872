// The key / value cache in 8 bits: its memory, the append, and its rows as fp32.
//
// The append. What a block of 16 rows of a head becomes depends on all its new rows, through
// their largest magnitude, and on the scale of the rows that it holds already: four warps take
// a block's keys and four its values, four rows each, and meet once in shared memory. The
// rows that were there are read and rounded again only where the scale grew. Bound by the 4
// bytes a value that come in (16001 rows of 2 heads of 256, cold: 20 us, 4.1 TB/s in and out);
// decode steps (a row or a few a sequence: 6.5 us cold, 4 behind another kernel) by latency alone.
#include "cache8.cuh"

#include <new>

namespace gufo {
namespace {

constexpr int kAppendThreads = 256;
constexpr float kLargest = 0x1p127f;
constexpr uint32_t kLargestBits = 0x7F000000u;

struct AppendArgs {
  CacheView cache;
  const float* rows[2];
  int64_t token_stride[2], head_stride[2];
  int whole;      // rows may be read four values at a time
};

// Grid: (blocks that the batch may touch, KV heads).
template <typename Format>
__global__ void __launch_bounds__(kAppendThreads)
AppendKernel(const __grid_constant__ AppendArgs a, const __grid_constant__ BatchArgs batch) {
  __shared__ uint32_t tops[2][4];
  __shared__ __align__(16) uint8_t image[2][kCacheBlock * kCacheMaxDim];
  GridLaunchDependents();
  GridDependencyWait();
  const BatchEntry& e = batch.of[SequenceOf(batch, blockIdx.x)];
  const CacheView& c = a.cache;
  const int held = batch.positions[e.index];
  const int start = min(max(held, 0), c.capacity);
  const int end = static_cast<int>(min(static_cast<int64_t>(held) + e.tokens, static_cast<int64_t>(c.capacity)));
  const int nth = blockIdx.x - batch.first_item[&e - batch.of];
  const int block = start / kCacheBlock + nth;
  const int row0 = block * kCacheBlock;
  if (row0 >= end) {
    return;
  }
  const int head = blockIdx.y;
  const int side = threadIdx.x / 128, warp = threadIdx.x / 32 & 3, lane = threadIdx.x & 31;
  const size_t of_head = static_cast<size_t>(e.slot) * c.kv_heads + head;
  const int fours = c.head_dim / 4;
  constexpr int kTimes = kCacheMaxDim / 128;

  // This warp's new rows: r = row0 + 4 warp + i where start <= r < end.
  float4 x[4][kTimes];
  uint32_t bits = 0;     // of the largest magnitude: as whole numbers they order alike, NaN above all
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + 4 * warp + i;
    const float* from = a.rows[side] + (static_cast<int64_t>(e.row) + (r - held)) * a.token_stride[side] + head * a.head_stride[side];
#pragma unroll
    for (int n = 0; n < kTimes; ++n) {
      const int f = lane + 32 * n;
      x[i][n] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= start && r < end && f < fours) {
        if (a.whole) {
          x[i][n] = __ldcs(reinterpret_cast<const float4*>(from) + f);
        } else {
          x[i][n] = make_float4(__ldcs(from + 4 * f), __ldcs(from + 4 * f + 1), __ldcs(from + 4 * f + 2), __ldcs(from + 4 * f + 3));
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int n = 0; n < kTimes; ++n) {
      const auto magnitude = [](float v) { return __float_as_uint(v) & 0x7FFFFFFFu; };
      bits = max(bits, max(max(magnitude(x[i][n].x), magnitude(x[i][n].y)), max(magnitude(x[i][n].z), magnitude(x[i][n].w))));
    }
  }
  const bool joins = row0 < start;   // rows that stay are in the block
  uint8_t* codes = BlocksOf(c, side, of_head) + static_cast<size_t>(block) * BlockBytes(c.head_dim);
  float* scale_at = ScaleOf(codes, c.head_dim);
  const float was = joins ? *scale_at : 0.f;
  const auto most_of_side = [&](uint32_t mine) {
    mine = __reduce_max_sync(0xFFFFFFFFu, mine);
    if (lane == 0) {
      tops[side][warp] = mine;
    }
    __syncthreads();
    return max(max(tops[side][0], tops[side][1]), max(tops[side][2], tops[side][3]));
  };
  bits = most_of_side(bits);
  if (__syncthreads_or(bits >= kLargestBits)) {
    // Magnitudes from there on saturate: what a code stands for is finite. NaN stays, and counts for nothing.
    uint32_t finite = 0;
    const auto hold = [&](float& v) {
      if (v == v) {
        v = fminf(fmaxf(v, -kLargest), kLargest);
        finite = max(finite, __float_as_uint(v) & 0x7FFFFFFFu);
      }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < kTimes; ++n) {
        hold(x[i][n].x), hold(x[i][n].y), hold(x[i][n].z), hold(x[i][n].w);
      }
    }
    bits = most_of_side(finite);
  }
  int exponent = ScaleExponentOf<Format>(__uint_as_float(bits));
  if (joins) {
    exponent = max(exponent, ExponentOf(was));
  }
  const float inverse = PowerOfTwo(-exponent);   // (exponent is -126 .. 121)
  if (row0 >= start && row0 + kCacheBlock <= end) {
    // A whole block: put together in shared memory and written sixteen bytes a thread. (The half
    // that a last single piece leaves of its pair holds zeros.)
    if (c.head_dim % 32 != 0 && lane < 16 && warp == 0) {
      *reinterpret_cast<uint4*>(image[side] + PieceAt(side, lane, c.head_dim / 16)) = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < kTimes; ++n) {
        const int f = lane + 32 * n;
        if (f < fours) {
          *(reinterpret_cast<uint32_t*>(image[side] + PieceAt(side, 4 * warp + i, f / 4)) + f % 4) = Format::Encode(x[i][n], inverse);
        }
      }
    }
    __syncthreads();
    for (int at = threadIdx.x % 128 * 16; at < CodeBytes(c.head_dim); at += 128 * 16) {
      *reinterpret_cast<uint4*>(codes + at) = *reinterpret_cast<const uint4*>(image[side] + at);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row0 + 4 * warp + i;
#pragma unroll
      for (int n = 0; n < kTimes; ++n) {
        const int f = lane + 32 * n;
        if (f >= fours) {
          continue;
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(codes + PieceAt(side, 4 * warp + i, f / 4)) + f % 4;
        if (r >= start && r < end) {
          *to = Format::Encode(x[i][n], inverse);
        } else if (r < start && exponent > ExponentOf(was)) {
          // (was * inverse is 0 where the scales are more than 2^149 apart, as the codes are then.)
          *to = Format::Encode(DecodeFour<Format>(*to), was * inverse);
        }
      }
    }
  }
  if (warp == 0 && lane == 0) {
    *scale_at = PowerOfTwo(exponent);
  }
  if (side == 0 && warp == 0 && lane < kCacheBlock && c.weights != nullptr && row0 + lane >= start && row0 + lane < end) {
    c.weights[of_head * c.capacity + row0 + lane] = 0.f;
  }
}

struct RowsArgs {
  CacheView cache;
  float* out[2];
  int each;       // heads a block of threads
};
constexpr int kRowsThreads = 256;

// Grid: (blocks that the batch touches, KV heads / each, 2). A block's rows are read a word of four codes a
// lane, rows beside one another from the same sectors, and go out sixteen bytes a lane: bound by those
// (16001 rows of 2 heads of 256, cold: 20 us, 4.0 TB/s in and out).
template <typename Format>
__global__ void __launch_bounds__(kRowsThreads)
RowsKernel(const __grid_constant__ RowsArgs a, const __grid_constant__ BatchArgs batch) {
  GridLaunchDependents();
  GridDependencyWait();
  const int side = blockIdx.z;
  float* out = a.out[side];
  if (out == nullptr) {
    return;
  }
  const BatchEntry& e = batch.of[SequenceOf(batch, blockIdx.x)];
  const CacheView& c = a.cache;
  const int64_t position = batch.positions[e.index];
  const int nth = blockIdx.x - batch.first_item[&e - batch.of];
  // The first row of the block, counted from the slot's first (a block may lie outside).
  const int64_t row0 = ((position >> 4) + nth) * kCacheBlock;
  const int fours = c.head_dim / 4;
  int shift = 2;      // 2^shift lanes a row
  while (1 << shift < fours) {
    ++shift;
  }
  const int f = threadIdx.x & ((1 << shift) - 1);
  const bool inside = row0 >= 0 && row0 < c.capacity;
  const int64_t token0 = row0 - position;     // of the block's first row
  const int64_t stride = static_cast<int64_t>(c.kv_heads) * fours;
  const int head0 = blockIdx.y * a.each;
  const int all = min(a.each, c.kv_heads - head0) * kCacheBlock;    // rows of the heads, one head's after another's
  const size_t first_head = static_cast<size_t>(e.slot) * c.kv_heads + head0;
  const size_t of_head = static_cast<size_t>(c.capacity / kCacheBlock) * BlockBytes(c.head_dim);
  const uint8_t* block = c.sides[side] + first_head * of_head + static_cast<size_t>(inside ? row0 / kCacheBlock : 0) * BlockBytes(c.head_dim);
  float4* to = reinterpret_cast<float4*>(out + ((e.row + token0) * c.kv_heads + head0) * c.head_dim) + f;
  constexpr int kEach = 4;
  const int step = kRowsThreads >> shift;
  for (int n0 = threadIdx.x >> shift; n0 < all; n0 += kEach * step) {
    uint32_t word[kEach];
    float scale[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int n = n0 + i * step, r = n % kCacheBlock;
      word[i] = 0;
      scale[i] = 0.f;
      if (inside && n < all && f < fours) {
        const uint8_t* from = block + (n / kCacheBlock) * of_head;
        word[i] = *(reinterpret_cast<const uint32_t*>(from + PieceAt(side, r, f / 4)) + f % 4);
        scale[i] = *ScaleOf(from, c.head_dim);
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int n = n0 + i * step, r = n % kCacheBlock;
      if (n < all && f < fours && token0 + r >= 0 && token0 + r < e.tokens) {
        float4 v = DecodeFour<Format>(word[i]);
        v.x *= scale[i], v.y *= scale[i], v.z *= scale[i], v.w *= scale[i];
        __stcs(to + r * stride + (n / kCacheBlock) * fours, v);
      }
    }
  }
}

// Blocks that `tokens` rows touch at most.
int BlocksOfRows(int tokens) { return tokens > 0 ? (tokens - 1 + kCacheBlock - 1) / kCacheBlock + 1 : 0; }

int CheckConfig(const gufo_cuda_cache8_config& c) {
  if (c.format != GUFO_CUDA_CACHE8_E4M3 && c.format != GUFO_CUDA_CACHE8_INT8) {
    return Fail(GUFO_CUDA_UNSUPPORTED_TYPE, "cache8: formats are e4m3 and int8");
  }
  if (c.sequences < 1 || c.sequences > kCacheMaxSequences || c.kv_heads < 1 || c.kv_heads > 1024) {
    return Fail(GUFO_CUDA_SHAPE, "cache8: 1 to 4096 sequences of 1 to 1024 KV heads");
  }
  if (c.head_dim < 16 || c.head_dim > kCacheMaxDim || c.head_dim % 16 != 0) {
    return Fail(GUFO_CUDA_SHAPE, "cache8: head_dim is a multiple of 16, 16 to 256");
  }
  if (c.capacity < kCacheBlock || c.capacity % kCacheBlock != 0 || c.capacity > (1 << 28)) {
    return Fail(GUFO_CUDA_SHAPE, "cache8: the capacity is a multiple of 16 rows, 2^28 at most");
  }
  return GUFO_CUDA_OK;
}

}  // namespace

int CheckBatch(const Cache8& cache, const gufo_cuda_cache8_batch* b, const char* what, bool counted, int64_t* rows) {
  const auto fail = [&](const char* why) { return Fail(GUFO_CUDA_BAD_ARGUMENT, std::string(what) + ": " + why); };
  if (b == nullptr) {
    return fail("null pointer");
  }
  if (b->sequences < 0 || b->sequences > cache.c.sequences) {
    return fail("more sequences than the cache has");
  }
  if (b->positions == nullptr && b->sequences > 0) {
    return fail("null pointer");
  }
  uint64_t seen[kCacheMaxSequences / 64] = {};
  int64_t total = 0;
  for (int i = 0; i < b->sequences; ++i) {
    const int slot = b->slots != nullptr ? b->slots[i] : i;
    if (slot < 0 || slot >= cache.c.sequences) {
      return fail("no such slot");
    }
    if (seen[slot / 64] >> (slot % 64) & 1) {
      return fail("a slot comes twice");
    }
    seen[slot / 64] |= 1ull << (slot % 64);
    const int tokens = counted && b->tokens != nullptr ? b->tokens[i] : 1;
    if (tokens < 0 || tokens > cache.c.capacity) {
      return fail("a sequence has 0 to `capacity` tokens");
    }
    total += tokens;
  }
  if (total > (1 << 30)) {
    return Fail(GUFO_CUDA_TOO_LARGE, std::string(what) + ": too many rows for one call");
  }
  *rows = total;
  return GUFO_CUDA_OK;
}

int FindCache(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const char* what, const Cache8** out) {
  const auto it = ctx->caches.find(handle);
  if (it == ctx->caches.end()) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, std::string(what) + ": unknown cache handle");
  }
  *out = &it->second;
  return GUFO_CUDA_OK;
}

}  // namespace gufo

using gufo::Fail;

extern "C" {

int gufo_cuda_cache8_create(gufo_cuda_ctx* ctx, const gufo_cuda_cache8_config* config, gufo_cuda_cache8* out) {
  if (ctx == nullptr || config == nullptr || out == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_create: null pointer");
  }
  if (const int rc = gufo::CheckConfig(*config); rc != GUFO_CUDA_OK) {
    return rc;
  }
  gufo::Cache8 cache;
  cache.c = *config;
  const size_t heads = static_cast<size_t>(config->sequences) * config->kv_heads;
  const auto whole = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
  const size_t rows = heads * static_cast<size_t>(config->capacity);   // at most 2^50
  const size_t side = whole(rows / gufo::kCacheBlock * gufo::BlockBytes(config->head_dim));
  const size_t weights = config->weights != 0 ? whole(rows * 4) : 0;
  std::lock_guard<std::mutex> lock(ctx->mu);
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  uint8_t* data = nullptr;
  const size_t bytes = 2 * side + weights;
  GUFO_CUDA_TRY(cudaMalloc(reinterpret_cast<void**>(&data), bytes));
  cudaError_t e = cudaMemsetAsync(data, 0, bytes, ctx->stream);
  if (e == cudaSuccess) {
    e = cudaStreamSynchronize(ctx->stream);   // (the next call may be on another stream)
  }
  if (e != cudaSuccess) {
    cudaFree(data);
    return gufo::CudaFail(e, "cache8_create");
  }
  cache.sides[0] = data;
  cache.sides[1] = data + side;
  cache.weights = weights != 0 ? reinterpret_cast<float*>(data + 2 * side) : nullptr;
  const int64_t id = ctx->next_id++;
  try {
    ctx->caches.emplace(id, cache);
  } catch (const std::bad_alloc&) {
    cudaFree(data);
    return Fail(GUFO_CUDA_OUT_OF_MEMORY, "cache8_create: host allocation failed");
  }
  *out = id;
  return GUFO_CUDA_OK;
}

int gufo_cuda_cache8_free(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle) {
  if (ctx == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_free: ctx is null");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const auto it = ctx->caches.find(handle);
  if (it == ctx->caches.end()) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_free: unknown cache handle");
  }
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  GUFO_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
  GUFO_CUDA_TRY(cudaFree(it->second.sides[0]));
  ctx->caches.erase(it);
  return GUFO_CUDA_OK;
}

int gufo_cuda_cache8_weights(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, float** weights) {
  if (ctx == nullptr || weights == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_weights: null pointer");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  if (const int rc = gufo::FindCache(ctx, handle, "cache8_weights", &cache); rc != GUFO_CUDA_OK) {
    return rc;
  }
  *weights = cache->weights;
  return GUFO_CUDA_OK;
}

int gufo_cuda_cache8_append_device(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const gufo_cuda_cache8_batch* batch,
                                   const float* keys, int64_t key_token_stride, int64_t key_head_stride,
                                   const float* values, int64_t value_token_stride, int64_t value_head_stride) {
  if (ctx == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_append: ctx is null");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  int64_t rows = 0;
  int rc = gufo::FindCache(ctx, handle, "cache8_append", &cache);
  if (rc == GUFO_CUDA_OK) {
    rc = gufo::CheckBatch(*cache, batch, "cache8_append", true, &rows);
  }
  if (rc != GUFO_CUDA_OK || rows == 0) {
    return rc;
  }
  if (keys == nullptr || values == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_append: null pointer");
  }
  gufo::AppendArgs a{gufo::ViewOf(*cache), {keys, values}, {key_token_stride, value_token_stride},
                     {key_head_stride, value_head_stride}, 0};
  a.whole = ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15) == 0 &&
            ((key_token_stride | key_head_stride | value_token_stride | value_head_stride) & 3) == 0;
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  const auto kernel = cache->c.format == GUFO_CUDA_CACHE8_E4M3 ? gufo::AppendKernel<gufo::E4m3> : gufo::AppendKernel<gufo::Int8>;
  return gufo::ForEachRun(
      *batch, gufo::BlocksOfRows,
      [&](const gufo::BatchArgs& b, int blocks) -> int {
        GUFO_CUDA_TRY(gufo::LaunchOverlapped(kernel, dim3(blocks, cache->c.kv_heads), dim3(gufo::kAppendThreads), 0, ctx->stream,
                                             1, a, b));
        ctx->launches.fetch_add(1);
        return GUFO_CUDA_OK;
      });
}

int gufo_cuda_cache8_rows_device(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const gufo_cuda_cache8_batch* batch, float* keys,
                                 float* values) {
  if (ctx == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_rows: ctx is null");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  int64_t rows = 0;
  int rc = gufo::FindCache(ctx, handle, "cache8_rows", &cache);
  if (rc == GUFO_CUDA_OK) {
    rc = gufo::CheckBatch(*cache, batch, "cache8_rows", true, &rows);
  }
  if (rc != GUFO_CUDA_OK || rows == 0 || (keys == nullptr && values == nullptr)) {
    return rc;
  }
  if (((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15) != 0) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_rows: rows go to 16-byte boundaries");
  }
  gufo::RowsArgs a{gufo::ViewOf(*cache), {keys, values}, 1};
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  const auto kernel = cache->c.format == GUFO_CUDA_CACHE8_E4M3 ? gufo::RowsKernel<gufo::E4m3> : gufo::RowsKernel<gufo::Int8>;
  return gufo::ForEachRun(
      *batch, gufo::BlocksOfRows,
      [&](const gufo::BatchArgs& b, int blocks) -> int {
        // Heads a block of threads: 1024 values of a row where that leaves the device full, as what a block costs
        // by itself is as much as four groups of values a thread (2048 rows of 8 heads of 128, 8 sequences: 54 us
        // with a head a block).
        const int wide = 1024 / cache->c.head_dim < cache->c.kv_heads ? 1024 / cache->c.head_dim : cache->c.kv_heads;
        a.each = static_cast<int64_t>(blocks) * cache->c.kv_heads * 2 / wide >= 4 * ctx->sm_count ? wide : 1;
        GUFO_CUDA_TRY(gufo::LaunchOverlapped(kernel, dim3(blocks, (cache->c.kv_heads + a.each - 1) / a.each, 2),
                                             dim3(gufo::kRowsThreads), 0, ctx->stream, 1, a, b));
        ctx->launches.fetch_add(1);
        return GUFO_CUDA_OK;
      });
}

}  // extern "C"
