// Eviction from the 8-bit cache by accumulated attention weight, in two launches.
//
// Which rows stay. A block of threads per sequence and KV head finds the weight of the last row
// that stays by radix selection over the weights' 32 bits (histograms of 11, 11 and 10 of them,
// whole numbers, so that nothing depends on the order of the atomics), then goes through the rows
// in their order, writes down the ones that stay and moves their weights. Bound by latency: up
// to 16384 rows are read once and stay in registers, and behind the first histogram only the
// rows of one bin are looked at (64 heads of 2064 rows 11 us cold, 16 heads of 16384 rows 20).
//
// Moving them. A warp makes one block of 16 rows: it gathers them, takes their largest
// magnitude, and rounds what had another scale. In place, the rows a block receives come from
// its own place or behind it, so blocks written in order overwrite nothing that is still wanted:
// a cluster of thread blocks does the next 64 blocks of a head at a time, all read before any
// is written (2048 rows of 64 heads of 128: 18 us cold, two rounds). Blocks that stay as they are
// are not touched. Into another cache there is no order to keep, and every block is a warp of its own (2048 of 16384 rows, 16 heads of 256:
// 16 us cold).
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

// Grid: (KV heads, sequences). Threads take four rows beside one another of each of C chunks of
// 4096; up to 4096 * C rows stay in their registers from the first look to the last.
template <int C>
__global__ void __launch_bounds__(kSelectThreads)
SelectKernel(const __grid_constant__ EvictArgs a, const __grid_constant__ BatchArgs batch) {
  __shared__ unsigned bins[kBins];
  __shared__ uint32_t listed[kBins];       // keys that share the first bits of the one that is looked for
  __shared__ unsigned of_warp[C][32];
  __shared__ unsigned found[3];            // the bin, how many more are wanted from it, how many it holds
  __shared__ unsigned list_count;
  constexpr int kChunk = 4 * kSelectThreads, kSpan = C * kChunk;
  GridLaunchDependents();
  GridDependencyWait();
  const BatchEntry& e = batch.of[blockIdx.y];
  const CacheView& c = a.cache;
  const int head = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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

  float4 w[C];
  const bool one_span = rows <= kSpan;
  const auto load = [&](int base) {
#pragma unroll
    for (int n = 0; n < C; ++n) {
      const int i = base + n * kChunk + 4 * threadIdx.x;
      w[n] = i < rows ? *reinterpret_cast<const float4*>(from + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  const auto key_of = [&](int n, int j) { return KeyOf(j == 0 ? w[n].x : j == 1 ? w[n].y : j == 2 ? w[n].z : w[n].w); };
  // Adds a key's bits to the bins. Many rows have the same weight, none: their lanes add up first.
  const auto count = [&](uint32_t k, int shift, unsigned bits, bool counts) {
    const bool none = counts && k == KeyOf(0.f);
    const unsigned all = __ballot_sync(0xFFFFFFFFu, none);
    if (none ? lane == __ffs(all) - 1 : counts) {
      atomicAdd(&bins[k >> shift & bits], none ? __popc(all) : 1u);
    }
  };
  load(0);
  if (threadIdx.x == 0) {
    list_count = 0;
  }
  // The key of the last row that stays: its bits from the top, 11, 11 and 10. Behind the first
  // look the keys that share its bits are listed, where they are few enough, and the rest is
  // left alone.
  uint32_t key = 0, mask = 0;
  bool list = false;
#pragma unroll 1
  for (int pass = 0; pass < 3 && wanted > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const unsigned bits = pass == 2 ? 1023 : 2047;
    for (int i = threadIdx.x; i < kBins; i += kSelectThreads) {
      bins[i] = 0;
    }
    __syncthreads();
    if (list) {
      const unsigned n = list_count;
      for (unsigned i = threadIdx.x; i < (n + 31) / 32 * 32; i += kSelectThreads) {
        const uint32_t k = i < n ? listed[i] : 0;
        count(k, shift, bits, i < n && (k & mask) == key);
      }
    } else {
      for (int base = 0; base < rows; base += kSpan) {
        if (!one_span && (pass > 0 || base > 0)) {
          load(base);
        }
#pragma unroll
        for (int n = 0; n < C; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = base + n * kChunk + 4 * threadIdx.x + j;
            const uint32_t k = key_of(n, j);
            count(k, shift, bits, i >= low && i < high && (k & mask) == key);
          }
        }
      }
    }
    __syncthreads();
    // The bin with the last wanted one, from the top: thread t has bins 2047 - 2 t and 2046 - 2 t.
    const unsigned top = bins[kBins - 1 - 2 * threadIdx.x], next = bins[kBins - 2 - 2 * threadIdx.x];
    unsigned sum = top + next;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned below = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      sum += lane >= o ? below : 0;
    }
    if (lane == 31) {
      of_warp[0][warp] = sum;
    }
    __syncthreads();
    unsigned ahead = of_warp[0][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned below = __shfl_up_sync(0xFFFFFFFFu, ahead, o);
      ahead += lane >= o ? below : 0;
    }
    ahead = __shfl_sync(0xFFFFFFFFu, ahead, warp == 0 ? 0 : warp - 1);
    ahead = (warp == 0 ? 0 : ahead) + sum - top - next;
    const unsigned want = static_cast<unsigned>(wanted);
    if (ahead < want && want <= ahead + top) {
      found[0] = kBins - 1 - 2 * threadIdx.x, found[1] = want - ahead, found[2] = top;
    } else if (ahead + top < want && want <= ahead + top + next) {
      found[0] = kBins - 2 - 2 * threadIdx.x, found[1] = want - ahead - top, found[2] = next;
    }
    __syncthreads();
    key |= found[0] << shift;
    mask |= bits << shift;
    wanted = static_cast<int>(found[1]);
    if (found[1] == found[2]) {
      break;      // all of the bin stay, whatever their other bits
    }
    if (!list && one_span && pass < 2 && found[2] <= kBins) {
      list = true;
#pragma unroll
      for (int n = 0; n < C; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = n * kChunk + 4 * threadIdx.x + j;
          const uint32_t k = key_of(n, j);
          if (i >= low && i < high && (k & mask) == key) {
            listed[atomicAdd(&list_count, 1u)] = k;
          }
        }
      }
    }
    __syncthreads();
  }

  // The rows above the key stay, the ends, and the first `wanted` rows with the key's bits. Rows that
  // stay anyway and rows with the key are counted together, 16 bits each (a chunk has 4096).
  unsigned before = 0, ties_before = 0;
#pragma unroll 1
  for (int base = 0; base < rows; base += kSpan) {
    if (!one_span) {
      load(base);
    }
    unsigned marks[C], sums[C];      // a thread's rows: stays 1 << j, ties 16 << j; counts up to this thread
#pragma unroll
    for (int n = 0; n < C; ++n) {
      marks[n] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = base + n * kChunk + 4 * threadIdx.x + j;
        const uint32_t k = key_of(n, j);
        const bool competes = i >= low && i < high && mask != 0;
        marks[n] |= i < rows && (i < low || i >= high || (competes && (k & mask) > key)) ? 1u << j : 0u;
        marks[n] |= competes && (k & mask) == key ? 16u << j : 0u;
      }
      sums[n] = __popc(marks[n] & 15u) | __popc(marks[n] & 0xF0u) << 16;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned below = __shfl_up_sync(0xFFFFFFFFu, sums[n], o);
        sums[n] += lane >= o ? below : 0;
      }
      if (lane == 31) {
        of_warp[n][warp] = sums[n];
      }
    }
    __syncthreads();     // (the weights have been read, too)
#pragma unroll
    for (int n = 0; n < C; ++n) {
      unsigned ahead = of_warp[n][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned below = __shfl_up_sync(0xFFFFFFFFu, ahead, o);
        ahead += lane >= o ? below : 0;
      }
      const unsigned chunk = __shfl_sync(0xFFFFFFFFu, ahead, 31);
      ahead = __shfl_sync(0xFFFFFFFFu, ahead, warp == 0 ? 0 : warp - 1);
      const unsigned up_to = (warp == 0 ? 0 : ahead) + sums[n];
      unsigned stays = before + (up_to & 0xFFFFu) - __popc(marks[n] & 15u);
      unsigned ties = ties_before + (up_to >> 16) - __popc(marks[n] & 0xF0u);
      const float f[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool stay = marks[n] >> j & 1u, tie = marks[n] >> (4 + j) & 1u;
        if (stay || (tie && ties < static_cast<unsigned>(wanted))) {
          const unsigned place = stays + min(ties, static_cast<unsigned>(wanted));
          kept[place] = base + n * kChunk + 4 * threadIdx.x + j;
          if (to != nullptr) {
            to[place] = f[j];
          }
        }
        stays += stay;
        ties += tie;
      }
      before += chunk & 0xFFFFu;
      ties_before += chunk >> 16;
    }
    __syncthreads();     // before the counts' next use
  }
}

// Grid: (groups of kMoveWarps blocks, 2 * KV heads, sequences); in place the first is a cluster.
template <typename Format, bool kInPlace>
__global__ void __launch_bounds__(kMoveThreads, kInPlace ? 3 : 2)
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
  // In place the last block may keep its first rows where they are, and lose others.
  const bool loses = kInPlace && a.budget % kCacheBlock != 0 && batch.positions[e.index] > a.budget;
  for (int first = blockIdx.x * kMoveWarps; first - static_cast<int>(blockIdx.x * kMoveWarps) < blocks;
       first += gridDim.x * kMoveWarps) {   // (in place every block of the cluster goes round as often)
    const int block = first + warp;
    const int row = block * kCacheBlock + lane;
    const int mine = block < blocks && lane < kCacheBlock && row < a.budget ? kept[row] : -1;
    const bool moves = __any_sync(0xFFFFFFFFu, mine >= 0 && (!kInPlace || mine != row)) || (loses && block == blocks - 1);
    const float was = moves && mine >= 0 ? *ScaleOf(from + static_cast<size_t>(mine / kCacheBlock) * bytes, c.head_dim) : 0.f;
    uint4 word[kTimes];
    float top = 0.f;
    if (moves) {
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        // (Two lanes a row's part of a pair of pieces, the rows of a pair together.)
        const int r = lane >> 1, piece = (lane & 1) + 2 * i;
        const int row_of = __shfl_sync(0xFFFFFFFFu, mine, r);
        word[i] = make_uint4(0, 0, 0, 0);
        if (piece < pieces && row_of >= 0) {
          word[i] = __ldcg(reinterpret_cast<const uint4*>(from + static_cast<size_t>(row_of / kCacheBlock) * bytes +
                                                          PieceAt(side, row_of % kCacheBlock, piece)));
        }
      }
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        const float scale = __shfl_sync(0xFFFFFFFFu, was, lane >> 1);
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
        const int r = lane >> 1, piece = (lane & 1) + 2 * i;
        const float scale = __shfl_sync(0xFFFFFFFFu, was, r);
        const int there = __shfl_sync(0xFFFFFFFFu, mine, r);
        if (piece >= pieces || there < 0) {
          continue;
        }
        uint4 out = word[i];
        if (scale != now) {
          const float by = fminf(scale * inverse, 0x1p127f);   // (beyond: of zeros beside much smaller rows, or alone)
          const auto again = [&](uint32_t w) {
            return Format::Encode(DecodeFour<Format>(w), by);
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
        const auto select = cache->c.capacity <= 4 * gufo::kSelectThreads ? gufo::SelectKernel<1> : gufo::SelectKernel<4>;
        GUFO_CUDA_TRY(gufo::LaunchOverlapped(select, dim3(cache->c.kv_heads, b.sequences), dim3(gufo::kSelectThreads),
                                             0, ctx->stream, 1, a, b));
        ctx->launches.fetch_add(1);
        return cache->c.format == GUFO_CUDA_CACHE8_E4M3 ? gufo::LaunchMove<gufo::E4m3>(ctx, a, b, in_place)
                                                        : gufo::LaunchMove<gufo::Int8>(ctx, a, b, in_place);
      });
}
