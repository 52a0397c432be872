// Eviction from the 8-bit cache by accumulated attention weight, in two launches.
//
// Which rows stay. A block of threads per sequence and KV head finds the weight of the last row
// that stays by radix selection over the weights' 32 bits (histograms of 11, 11 and 10 of them,
// whole numbers, so that nothing depends on the order of the atomics), then walks the rows once
// in their order, writes down the ones that stay and moves their weights. Bound by latency: four
// walks over 4 bytes a row, which are in L2 behind the first, and a scan of the block a walk
// of 4096 rows.
//
// Moving them. A warp makes one block of 16 rows: it gathers them, takes their largest
// magnitude, and rounds what had another scale. In place, the rows a block receives come from
// its own place or behind it, so blocks written in order overwrite nothing that is still wanted:
// a cluster of thread blocks does the next 64 blocks of a head at a time, all read before any
// is written. Blocks whose rows stay where they are are not touched. Into another cache there
// is no order to keep, and every block is a warp of its own.
#include <cooperative_groups.h>

#include "cache8.cuh"

namespace gufo {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kMoveCluster = 8;

struct EvictArgs {
  CacheView cache, into;
  int into_slots[kBatchSequences];
  int budget, first, last;
  int* kept;
  int* held;
};

// Weights in the order of these: NaN below everything, both zeros the same.
__device__ __forceinline__ uint32_t KeyOf(float w) {
  const uint32_t bits = __float_as_uint(w + 0.f);
  return w != w ? 0u : (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

// Exclusive sum over the block in thread order, and the sum of all. `spare`: 33 words.
__device__ __forceinline__ unsigned long long BlockScan(unsigned long long v, unsigned long long* spare, unsigned long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned long long sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long below = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    sum += lane >= o ? below : 0;
  }
  __syncthreads();   // what the last call left has been read
  if (lane == 31) {
    spare[warp] = sum;
  }
  __syncthreads();
  unsigned long long w = spare[lane];   // kSelectThreads / 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long below = __shfl_up_sync(0xFFFFFFFFu, w, o);
    w += lane >= o ? below : 0;
  }
  *total = __shfl_sync(0xFFFFFFFFu, w, 31);
  const unsigned long long ahead = __shfl_sync(0xFFFFFFFFu, w, warp == 0 ? 0 : warp - 1);
  return sum - v + (warp == 0 ? 0 : ahead);
}

// Grid: (KV heads, sequences).
__global__ void __launch_bounds__(kSelectThreads)
SelectKernel(const __grid_constant__ EvictArgs a, const __grid_constant__ BatchArgs batch) {
  __shared__ unsigned bins[kBins];
  __shared__ unsigned long long spare[32];
  __shared__ unsigned found[2];   // the bin, and how many more are wanted from it
  GridLaunchDependents();
  GridDependencyWait();
  const BatchEntry& e = batch.of[blockIdx.y];
  const CacheView& c = a.cache;
  const int head = blockIdx.x;
  const int rows = PositionOf(c, batch, e);
  const int budget = a.budget;
  int* kept = a.kept + (static_cast<size_t>(e.index) * c.kv_heads + head) * budget;
  const float* from = c.weights + (static_cast<size_t>(e.slot) * c.kv_heads + head) * c.capacity;
  float* to = a.into.weights == nullptr
                  ? nullptr
                  : a.into.weights + (static_cast<size_t>(a.into_slots[blockIdx.y]) * c.kv_heads + head) * a.into.capacity;
  if (head == 0 && threadIdx.x == 0 && a.held != nullptr) {
    a.held[e.index] = min(rows, budget);
  }
  if (rows <= budget) {
    for (int i = threadIdx.x; i < budget; i += kSelectThreads) {
      kept[i] = i < rows ? i : -1;
      if (i < rows && to != nullptr && to != from) {
        to[i] = from[i];
      }
    }
    return;
  }
  const int first = min(a.first, budget);
  const int last = min(a.last, budget - first);
  const int low = first, high = rows - last;        // the rows that compete
  int wanted = budget - first - last;               // of them; fewer than there are

  // The key of the last row that stays: its bits from the top, 11, 11 and 10.
  uint32_t key = 0, mask = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3 && wanted > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int width = pass == 2 ? 1024 : 2048;
    for (int i = threadIdx.x; i < kBins; i += kSelectThreads) {
      bins[i] = 0;
    }
    __syncthreads();
    for (int base = 0; base < rows; base += 4 * kSelectThreads) {
      const int i = base + 4 * threadIdx.x;
      const float4 w = i < rows ? *reinterpret_cast<const float4*>(from + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float f[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = KeyOf(f[j]);
        const bool counts = i + j >= low && i + j < high && (k & mask) == key;
        // Many rows have the same weight, none: lanes with the same bin add up first.
        const unsigned bin = counts ? (k >> shift) & (width - 1) : kBins;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, bin);
        if (counts && (threadIdx.x & 31) == __ffs(same) - 1) {
          atomicAdd(&bins[bin], __popc(same));
        }
      }
    }
    __syncthreads();
    const unsigned top = bins[kBins - 1 - 2 * threadIdx.x], next = bins[kBins - 2 - 2 * threadIdx.x];
    unsigned long long total;
    const unsigned ahead = static_cast<unsigned>(BlockScan(top + next, spare, &total));
    const unsigned want = static_cast<unsigned>(wanted);
    if (ahead < want && want <= ahead + top) {
      found[0] = kBins - 1 - 2 * threadIdx.x;
      found[1] = want - ahead;
    } else if (ahead + top < want && want <= ahead + top + next) {
      found[0] = kBins - 2 - 2 * threadIdx.x;
      found[1] = want - ahead - top;
    }
    __syncthreads();
    key |= found[0] << shift;
    mask |= static_cast<uint32_t>(width - 1) << shift;
    wanted = static_cast<int>(found[1]);
    __syncthreads();
  }

  // The rows above the key stay, the ends, and the first `wanted` rows with that very key.
  unsigned long long before = 0;   // rows that stay anyway | rows with the key << 32
#pragma unroll 1
  for (int base = 0; base < rows; base += 4 * kSelectThreads) {
    const int i = base + 4 * threadIdx.x;
    const float4 w = i < rows ? *reinterpret_cast<const float4*>(from + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float f[4] = {w.x, w.y, w.z, w.w};
    bool stays[4], ties[4];
    unsigned long long mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = KeyOf(f[j]);
      const bool competes = i + j >= low && i + j < high && mask != 0;
      stays[j] = i + j < rows && (i + j < low || i + j >= high || (competes && k > key));
      ties[j] = competes && k == key;
      mine += (stays[j] ? 1ull : 0ull) + (ties[j] ? 1ull << 32 : 0ull);
    }
    unsigned long long total;
    unsigned long long at = before + BlockScan(mine, spare, &total);   // (a barrier: the weights have been read)
    before += total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned equal = static_cast<unsigned>(at >> 32);
      const unsigned place = static_cast<unsigned>(at) + min(equal, static_cast<unsigned>(wanted));
      if (stays[j] || (ties[j] && equal < static_cast<unsigned>(wanted))) {
        kept[place] = i + j;
        if (to != nullptr) {
          to[place] = f[j];
        }
      }
      at += (stays[j] ? 1ull : 0ull) + (ties[j] ? 1ull << 32 : 0ull);
    }
  }
}

// Grid: (groups of kMoveWarps blocks, 2 * KV heads, sequences); in place the first is a cluster.
template <typename Format, bool kInPlace>
__global__ void __launch_bounds__(kMoveThreads, 3)
MoveKernel(const __grid_constant__ EvictArgs a, const __grid_constant__ BatchArgs batch) {
  constexpr int kTimes = kCacheBlock * kCacheMaxDim / 16 / 32;   // 16-byte pieces of a block, a lane's
  GridLaunchDependents();
  GridDependencyWait();
  const BatchEntry& e = batch.of[blockIdx.z];
  const CacheView& c = a.cache;
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int* kept = a.kept + (static_cast<size_t>(e.index) * c.kv_heads + head) * a.budget;
  const size_t source = static_cast<size_t>(e.slot) * c.kv_heads + head;
  const size_t target = static_cast<size_t>(a.into_slots[blockIdx.z]) * c.kv_heads + head;
  const uint8_t* from = BlocksOf(c, side, source);
  uint8_t* to = BlocksOf(a.into, side, target);
  const int bytes = BlockBytes(c.head_dim);
  const int pieces = c.head_dim / 16;   // of a row
  const int blocks = (a.budget + kCacheBlock - 1) / kCacheBlock;
  for (int first = blockIdx.x * kMoveWarps; first - static_cast<int>(blockIdx.x * kMoveWarps) < blocks;
       first += gridDim.x * kMoveWarps) {   // (in place every block of the cluster goes round as often)
    const int block = first + warp;
    const int row = block * kCacheBlock + lane;
    const int mine = block < blocks && lane < kCacheBlock && row < a.budget ? kept[row] : -1;
    const bool moves = __any_sync(0xFFFFFFFFu, mine >= 0 && (!kInPlace || mine != row));
    const float was = moves && mine >= 0 ? *ScaleOf(from + static_cast<size_t>(mine / kCacheBlock) * bytes, c.head_dim) : 0.f;
    uint4 word[kTimes];
    float top = 0.f;
    if (moves) {
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        // (Sixteen lanes gather a piece of all rows: what they write is together.)
        const int r = lane & 15, piece = (lane >> 4) + 2 * i;
        const int row_of = __shfl_sync(0xFFFFFFFFu, mine, r);
        word[i] = make_uint4(0, 0, 0, 0);
        if (piece < pieces && row_of >= 0) {
          word[i] = __ldcg(reinterpret_cast<const uint4*>(from + static_cast<size_t>(row_of / kCacheBlock) * bytes +
                                                          PieceAt(side, row_of % kCacheBlock, piece)));
        }
      }
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        const float scale = __shfl_sync(0xFFFFFFFFu, was, lane & 15);
        __half2 most = __float2half2_rn(0.f);
        const uint32_t w[4] = {word[i].x, word[i].y, word[i].z, word[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t x, y;
          Format::Decode(w[j], x, y);
          most = __hmax2(most, __hmax2(__habs2(*reinterpret_cast<const __half2*>(&x)), __habs2(*reinterpret_cast<const __half2*>(&y))));
        }
        const float m = fmaxf(__low2float(most), __high2float(most));   // (maxima pass NaN by)
        top = fmaxf(top, m * scale);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      }
    }
    if constexpr (kInPlace) {
      cooperative_groups::this_cluster().sync();   // every block of the round has been read
    }
    if (moves) {
      const int exponent = ScaleExponentOf<Format>(top);
      const float now = PowerOfTwo(exponent), inverse = PowerOfTwo(-exponent);
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        const int r = lane & 15, piece = (lane >> 4) + 2 * i;
        const float scale = __shfl_sync(0xFFFFFFFFu, was, r);
        const int there = __shfl_sync(0xFFFFFFFFu, mine, r);
        if (piece >= pieces || there < 0) {
          continue;
        }
        uint4 out = word[i];
        if (scale != now) {
          const float by = scale * inverse;
          const auto again = [&](uint32_t w) {
            const float4 v = DecodeFour<Format>(w);
            return Format::Encode(v.x * by, v.y * by, v.z * by, v.w * by);
          };
          out = make_uint4(again(out.x), again(out.y), again(out.z), again(out.w));
        }
        *reinterpret_cast<uint4*>(to + static_cast<size_t>(block) * bytes + PieceAt(side, r, piece)) = out;
      }
      if (lane == 0) {
        *ScaleOf(to + static_cast<size_t>(block) * bytes, c.head_dim) = now;
      }
    }
  }
}

template <typename Format>
int LaunchMove(gufo_cuda_ctx* ctx, const EvictArgs& a, const BatchArgs& b, bool in_place) {
  const int groups = ((a.budget + kCacheBlock - 1) / kCacheBlock + kMoveWarps - 1) / kMoveWarps;
  const int x = in_place ? kMoveCluster : groups;
  const auto kernel = in_place ? MoveKernel<Format, true> : MoveKernel<Format, false>;
  GUFO_CUDA_TRY(LaunchOverlapped(kernel, dim3(x, 2 * a.cache.kv_heads, b.sequences), dim3(kMoveThreads), 0, ctx->stream,
                                 in_place ? kMoveCluster : 1, a, b));
  ctx->launches.fetch_add(1);
  return GUFO_CUDA_OK;
}

}  // namespace
}  // namespace gufo

using gufo::Fail;

extern "C" int gufo_cuda_cache8_evict_device(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const gufo_cuda_cache8_batch* batch,
                                             int budget, int first, int last, int* kept, int* held, gufo_cuda_cache8 into_handle,
                                             const int* into_slots) {
  if (ctx == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: ctx is null");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  int64_t sequences = 0;
  int rc = gufo::FindCache(ctx, handle, "cache8_evict", &cache);
  if (rc == GUFO_CUDA_OK) {
    rc = gufo::CheckBatch(*cache, batch, "cache8_evict", false, &sequences);
  }
  if (rc != GUFO_CUDA_OK) {
    return rc;
  }
  if (cache->weights == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: the cache keeps no weights");
  }
  if (budget < 1 || budget > cache->c.capacity || first < 0 || last < 0) {
    return Fail(GUFO_CUDA_SHAPE, "cache8_evict: a budget of 1 to `capacity` rows, and no negative first or last");
  }
  if (into_handle == 0 && into_slots != nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: into_slots without into");
  }
  const bool in_place = into_handle == 0;
  const gufo::Cache8* into = cache;
  if (!in_place) {
    rc = gufo::FindCache(ctx, into_handle, "cache8_evict", &into);
    if (rc != GUFO_CUDA_OK) {
      return rc;
    }
    if (into == cache) {
      return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: into is another cache (0: in place)");
    }
    if (into->c.kv_heads != cache->c.kv_heads || into->c.head_dim != cache->c.head_dim || into->c.format != cache->c.format ||
        into->c.capacity < budget) {
      return Fail(GUFO_CUDA_SHAPE, "cache8_evict: into has the same heads and format, and room for the budget");
    }
    gufo_cuda_cache8_batch there = *batch;
    there.slots = into_slots != nullptr ? into_slots : batch->slots;
    rc = gufo::CheckBatch(*into, &there, "cache8_evict", false, &sequences);
    if (rc != GUFO_CUDA_OK) {
      return rc;
    }
  }
  if (batch->sequences == 0) {
    return GUFO_CUDA_OK;
  }
  if (kept == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: null pointer");
  }
  if (held != nullptr && held == batch->positions) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_evict: held and positions are different arrays");
  }
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  gufo_cuda_cache8_batch each = *batch;
  each.tokens = nullptr;
  return gufo::ForEachRun(
      each, [](int) { return 1; },
      [&](const gufo::BatchArgs& b, int) -> int {
        gufo::EvictArgs a{gufo::ViewOf(*cache), gufo::ViewOf(*into), {}, budget, first, last, kept, held};
        for (int i = 0; i < b.sequences; ++i) {
          a.into_slots[i] = in_place || into_slots == nullptr ? b.of[i].slot : into_slots[b.of[i].index];
        }
        GUFO_CUDA_TRY(gufo::LaunchOverlapped(gufo::SelectKernel, dim3(cache->c.kv_heads, b.sequences), dim3(gufo::kSelectThreads),
                                             0, ctx->stream, 1, a, b));
        ctx->launches.fetch_add(1);
        return cache->c.format == GUFO_CUDA_CACHE8_E4M3 ? gufo::LaunchMove<gufo::E4m3>(ctx, a, b, in_place)
                                                        : gufo::LaunchMove<gufo::Int8>(ctx, a, b, in_place);
      });
}
