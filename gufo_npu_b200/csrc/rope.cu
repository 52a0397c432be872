// Rotary positions for rows of any number of tokens: RMSNorm of a head where asked, then
//   (a, b) -> (a cos - b sin, a sin + b cos)
// for each pair of the head's first rope_dim values, the angle being position times the
// pair's frequency.
//
// The angle. In turns: the frequency is kept as a 64-bit fraction of a turn per position,
// the product with the position wraps around at whole turns by itself, and what is lost is the
// fraction's own rounding times the position: 2^-33 of a turn at the farthest one, 2^-44 at a
// million (fp32 angles are 0.06 off there). The nearest quarter is split off as whole numbers, so
// what sincospif sees is an eighth of a turn at most with 24 significant bits (2^-28 of a turn off),
// near the zeros of both functions too.
//
// What bounds it. The copy: 4 bytes in, 4 out per value (8000 tokens of 10 heads of 256 32 us, 5.2
// TB/s; a decode step 3 us, a launch). A sine and cosine per pair would
// cost as much again at 1 KB rows, so a group of lanes computes them once for its token and
// keeps them for several heads. A row is spread over the fewest lanes (a power of two) that
// hold it four pairs each, so that rows of 64 to 256 values leave no lane idle.
#include <cmath>
#include <new>

#include "common.cuh"

namespace gufo {
namespace {

constexpr int kMaxRopeDim = 512;
constexpr int kRopeThreads = 256;

struct RopePart {
  gufo_cuda_rope_rows rows;
  int first;     // of the token's items: where this part's start
};

struct RopeArgs {
  RopePart parts[GUFO_CUDA_ROPE_PARTS];
  int nparts;
  const unsigned long long* turns;   // [rope_dim / 2]: 2^-64 turns per position
  const int* positions;
  int tokens;
  int rope_dim;
  float magnitude;
  int items;      // a token's: groups of up to `each` heads
  int each;
  int lanes;      // of a row: a power of two
};

// Cosine and sine of `position` times the frequency.
__device__ __forceinline__ void Turn(unsigned long long per, int position, float magnitude, float* cs, float* sn) {
  const unsigned long long at = per * static_cast<unsigned long long>(static_cast<long long>(position));
  const unsigned quarter = static_cast<unsigned>((at + (1ull << 61)) >> 62);
  const long long rest = static_cast<long long>(at - (static_cast<unsigned long long>(quarter) << 62));
  float s, c;
  sincospif(static_cast<float>(rest) * 0x1p-63f, &s, &c);
  const float x = (quarter & 1u) != 0 ? s : c;
  const float y = (quarter & 1u) != 0 ? c : s;
  *cs = (quarter == 1u || quarter == 2u ? -x : x) * magnitude;
  *sn = (quarter >= 2u ? -y : y) * magnitude;
}

// V pairs a lane at a time, up to N times, U heads.
template <int V, int N, int U>
__global__ void __launch_bounds__(kRopeThreads)
RopeKernel(const __grid_constant__ RopeArgs a, bool interleaved) {
  GridLaunchDependents();
  const int lane = threadIdx.x & (a.lanes - 1);
  const int group = (blockIdx.x * kRopeThreads + threadIdx.x) / a.lanes;   // lanes of one item
  const int token = group / a.items, item = group - token * a.items;
  GridDependencyWait();
  const bool there = token < a.tokens;   // (whole warps stay for the shuffles)
  int p = 0;
  while (p + 1 < a.nparts && item >= a.parts[p + 1].first) {
    ++p;
  }
  const gufo_cuda_rope_rows& r = a.parts[p].rows;
  const int head0 = (item - a.parts[p].first) * a.each;
  const int heads = there ? min(a.each, r.heads - head0) : 0;
  const int half = a.rope_dim / 2, pairs = r.head_dim / 2;
  const int position = there ? a.positions[token] : 0;
  const bool norm = r.norm_weight != nullptr;
  // Where a pair's values stand: halves apart in the turning part of that layout, else side by side.
  const bool apart = !interleaved;
  float cs[N][V], sn[N][V], wa[N][V], wb[N][V];
  auto at = [&](int n) { return (n * a.lanes + lane) * V; };
  auto index = [&](int pair, int v, bool second) {
    return apart && pair < half ? pair + v + (second ? half : 0) : 2 * (pair + v) + (second ? 1 : 0);
  };
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int pair = at(n);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      cs[n][v] = 1.f, sn[n][v] = 0.f, wa[n][v] = 1.f, wb[n][v] = 1.f;
      if (heads > 0 && pair < pairs) {
        if (pair < half) {
          Turn(a.turns[pair + v], position, a.magnitude, &cs[n][v], &sn[n][v]);
        }
        if (norm) {
          wa[n][v] = r.norm_weight[index(pair, v, false)];
          wb[n][v] = r.norm_weight[index(pair, v, true)];
        }
      }
    }
  }
  const float* in = r.in + token * r.in_token_stride + head0 * r.in_head_stride;
  float* out = r.out + token * r.out_token_stride + head0 * r.out_head_stride;
  // Several heads' rows are on their way at once. (Every lane of a warp goes round as often as the
  // longest group of it, for the shuffles.)
  const int rounds = __reduce_max_sync(0xFFFFFFFFu, heads);
  for (int h0 = 0; h0 < rounds; h0 += U) {
    float x[U][N][V], y[U][N][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* row = in + (h0 + u) * r.in_head_stride;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int pair = at(n);
        const bool mine = h0 + u < heads && pair < pairs;
        if constexpr (V == 4) {
          float4 first = make_float4(0.f, 0.f, 0.f, 0.f), second = first;
          const bool split = apart && pair < half;
          if (mine) {
            const float* from = row + (split ? pair : 2 * pair);
            first = __ldcs(reinterpret_cast<const float4*>(from));
            second = __ldcs(reinterpret_cast<const float4*>(from + (split ? half : 4)));
          }
          const float f[8] = {first.x, first.y, first.z, first.w, second.x, second.y, second.z, second.w};
#pragma unroll
          for (int v = 0; v < V; ++v) {
            x[u][n][v] = split ? f[v] : f[2 * v];
            y[u][n][v] = split ? f[4 + v] : f[2 * v + 1];
          }
        } else {
          x[u][n][0] = mine ? __ldcs(row + index(pair, 0, false)) : 0.f;
          y[u][n][0] = mine ? __ldcs(row + index(pair, 0, true)) : 0.f;
        }
      }
    }
    float inv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      inv[u] = 1.f;
    }
    if (__any_sync(0xFFFFFFFFu, norm)) {
      float sq[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sq[u] = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            sq[u] = fmaf(x[u][n][v], x[u][n][v], sq[u]);
            sq[u] = fmaf(y[u][n][v], y[u][n][v], sq[u]);
          }
        }
      }
      for (int o = a.lanes / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          sq[u] += __shfl_xor_sync(0xFFFFFFFFu, sq[u], o);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        inv[u] = norm ? 1.0f / sqrtf(sq[u] / static_cast<float>(r.head_dim) + r.rms_eps) : 1.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float* row = out + (h0 + u) * r.out_head_stride;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int pair = at(n);
        if (h0 + u >= heads || pair >= pairs) {
          continue;
        }
        const bool turns = pair < half;   // the others are passed on as they are, NaN and infinities too
        float f[V], g[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float p = x[u][n][v] * inv[u] * wa[n][v], w = y[u][n][v] * inv[u] * wb[n][v];
          f[v] = turns ? fmaf(p, cs[n][v], -(w * sn[n][v])) : p;
          g[v] = turns ? fmaf(p, sn[n][v], w * cs[n][v]) : w;
        }
        if constexpr (V == 4) {
          const bool split = apart && turns;
          float* to = row + (split ? pair : 2 * pair);
          const float4 first = split ? make_float4(f[0], f[1], f[2], f[3]) : make_float4(f[0], g[0], f[1], g[1]);
          const float4 second = split ? make_float4(g[0], g[1], g[2], g[3]) : make_float4(f[2], g[2], f[3], g[3]);
          *reinterpret_cast<float4*>(to) = first;
          *reinterpret_cast<float4*>(to + (split ? half : 4)) = second;
        } else {
          row[index(pair, 0, false)] = f[0];
          row[index(pair, 0, true)] = g[0];
        }
      }
    }
  }
}

int CheckRope(const gufo_cuda_rope_params* p) {
  if (p == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: null pointer");
  }
  if (p->rope_dim < 2 || p->rope_dim > kMaxRopeDim || p->rope_dim % 2 != 0) {
    return Fail(GUFO_CUDA_SHAPE, "rope: rope_dim is even, 2 to 512");
  }
  if (p->layout != GUFO_CUDA_ROPE_HALVES && p->layout != GUFO_CUDA_ROPE_PAIRS) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: unknown layout");
  }
  if (!(p->theta > 1.0) || !std::isfinite(p->theta)) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: theta is above 1");
  }
  const bool by_parts = p->scaling == GUFO_CUDA_ROPE_BY_PARTS;
  if (p->scaling != GUFO_CUDA_ROPE_UNSCALED && p->scaling != GUFO_CUDA_ROPE_LINEAR && !by_parts) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: unknown scaling");
  }
  if (p->scaling != GUFO_CUDA_ROPE_UNSCALED && (!(p->factor > 0.0) || !std::isfinite(p->factor) || !std::isfinite(1.0 / p->factor))) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: the scaling's factor is above 0");
  }
  if (by_parts && (!(p->original_positions > 0.0) || !std::isfinite(p->original_positions) || !(p->slow_turns > 0.0) ||
                   !(p->fast_turns > p->slow_turns) || !std::isfinite(p->fast_turns))) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: by parts takes original_positions > 0 and fast_turns > slow_turns > 0");
  }
  if (!std::isfinite(static_cast<float>(p->magnitude))) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: the magnitude is finite");
  }
  return GUFO_CUDA_OK;
}

// Angles per position, in more than a double's bits: positions multiply what they are off by.
void Frequencies(const gufo_cuda_rope_params& p, long double* frequencies, double* magnitude) {
  const int pairs = p.rope_dim / 2;
  const bool by_parts = p.scaling == GUFO_CUDA_ROPE_BY_PARTS;
  // The pair that turns `turns` times over the original positions.
  const auto pair_of = [&](double turns) {
    return pairs * std::log(p.original_positions / (turns * 2.0 * M_PI)) / std::log(p.theta);
  };
  double low = 0.0, high = 0.0;
  if (by_parts) {
    // (The ramp may end behind the last pair, and keeps its slope there: held to 2 pairs - 1.)
    low = std::fmin(std::fmax(std::floor(pair_of(p.fast_turns)), 0.0), p.rope_dim - 1.0);
    high = std::fmin(std::fmax(std::ceil(pair_of(p.slow_turns)), 0.0), p.rope_dim - 1.0);
  }
  for (int i = 0; i < pairs; ++i) {
    long double f = std::pow(static_cast<long double>(p.theta), -static_cast<long double>(i) / pairs);
    if (p.scaling == GUFO_CUDA_ROPE_LINEAR) {
      f /= p.factor;
    } else if (by_parts) {
      const long double slow = std::fmin(std::fmax((i - low) / std::fmax(static_cast<long double>(high - low), 1e-3L), 0.0L), 1.0L);
      f = f * (1.0L - slow) + f / p.factor * slow;
    }
    frequencies[i] = f;
  }
  *magnitude = p.magnitude != 0.0 ? p.magnitude : by_parts && p.factor > 1.0 ? 0.1 * std::log(p.factor) + 1.0 : 1.0;
}

template <int V, int N, int U>
cudaError_t LaunchOf(gufo_cuda_ctx* ctx, const RopeArgs& a, bool interleaved) {
  const int64_t threads = static_cast<int64_t>(a.tokens) * a.items * a.lanes;
  return LaunchOverlapped(RopeKernel<V, N, U>, dim3(static_cast<unsigned>((threads + kRopeThreads - 1) / kRopeThreads)),
                          dim3(kRopeThreads), 0, ctx->stream, 1, a, interleaved);
}

// A prompt's rows: several heads on their way at once (8000 tokens of 10 heads 35.6 -> 32 us); a decode step's,
// with a head a group of lanes: one (32 tokens of 20 heads 3.1 us, 4.4 with four).
template <int V, int N>
cudaError_t Launch(gufo_cuda_ctx* ctx, const RopeArgs& a, bool interleaved) {
  return a.each > 1 ? LaunchOf<V, N, (N * V <= 4 ? 4 : 2)>(ctx, a, interleaved) : LaunchOf<V, N, 1>(ctx, a, interleaved);
}

}  // namespace
}  // namespace gufo

using gufo::Fail;

extern "C" {

int gufo_cuda_rope_frequencies(const gufo_cuda_rope_params* params, double* frequencies, double* magnitude) {
  if (const int rc = gufo::CheckRope(params); rc != GUFO_CUDA_OK) {
    return rc;
  }
  if (frequencies == nullptr || magnitude == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: null pointer");
  }
  long double exact[gufo::kMaxRopeDim / 2];
  gufo::Frequencies(*params, exact, magnitude);
  for (int i = 0; i < params->rope_dim / 2; ++i) {
    frequencies[i] = static_cast<double>(exact[i]);
  }
  return GUFO_CUDA_OK;
}

int gufo_cuda_rope_create(gufo_cuda_ctx* ctx, const gufo_cuda_rope_params* params, gufo_cuda_rope* out) {
  if (ctx == nullptr || out == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope_create: null pointer");
  }
  if (const int rc = gufo::CheckRope(params); rc != GUFO_CUDA_OK) {
    return rc;
  }
  long double frequencies[gufo::kMaxRopeDim / 2];
  double magnitude = 1.0;
  gufo::Frequencies(*params, frequencies, &magnitude);
  unsigned long long turns[gufo::kMaxRopeDim / 2];
  const int pairs = params->rope_dim / 2;
  for (int i = 0; i < pairs; ++i) {
    // Positions are whole numbers: whole turns per position count for nothing.
    const long double t = frequencies[i] / (2.0L * 3.14159265358979323846264338327950288L);
    turns[i] = static_cast<unsigned long long>(std::rint((t - std::floor(t)) * 0x1p64L));   // (whole from a half on: below 2^64)
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  gufo::Rope rope;
  rope.rope_dim = params->rope_dim;
  rope.interleaved = params->layout == GUFO_CUDA_ROPE_PAIRS;
  rope.magnitude = static_cast<float>(magnitude);
  GUFO_CUDA_TRY(cudaMalloc(reinterpret_cast<void**>(&rope.turns), pairs * sizeof(turns[0])));
  cudaError_t e = cudaMemcpyAsync(rope.turns, turns, pairs * sizeof(turns[0]), cudaMemcpyHostToDevice, ctx->stream);
  if (e == cudaSuccess) {
    e = cudaStreamSynchronize(ctx->stream);
  }
  if (e != cudaSuccess) {
    cudaFree(rope.turns);
    return gufo::CudaFail(e, "rope_create");
  }
  const int64_t id = ctx->next_id++;
  try {
    ctx->ropes.emplace(id, rope);
  } catch (const std::bad_alloc&) {
    cudaFree(rope.turns);
    return Fail(GUFO_CUDA_OUT_OF_MEMORY, "rope_create: host allocation failed");
  }
  *out = id;
  return GUFO_CUDA_OK;
}

int gufo_cuda_rope_free(gufo_cuda_ctx* ctx, gufo_cuda_rope rope) {
  if (ctx == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope_free: ctx is null");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const auto it = ctx->ropes.find(rope);
  if (it == ctx->ropes.end()) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope_free: unknown handle");
  }
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  GUFO_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
  cudaFree(it->second.turns);
  ctx->ropes.erase(it);
  return GUFO_CUDA_OK;
}

int gufo_cuda_rope_device(gufo_cuda_ctx* ctx, gufo_cuda_rope handle, const gufo_cuda_rope_rows* parts, int nparts,
                          const int* positions, int tokens) {
  if (ctx == nullptr || parts == nullptr || (positions == nullptr && tokens > 0)) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: null pointer");
  }
  if (nparts < 1 || nparts > GUFO_CUDA_ROPE_PARTS || tokens < 0) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: 1 to 4 parts and no negative number of tokens");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const auto it = ctx->ropes.find(handle);
  if (it == ctx->ropes.end()) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: unknown handle");
  }
  const gufo::Rope& rope = it->second;
  gufo::RopeArgs a{};
  int widest = 0, most = 0, rows = 0;
  bool fours = rope.rope_dim % 8 == 0;   // four pairs at a time, on 16-byte boundaries
  for (int i = 0; i < nparts; ++i) {
    const gufo_cuda_rope_rows& r = parts[i];
    if (tokens > 0 && (r.in == nullptr || r.out == nullptr)) {
      return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: null pointer in a part");
    }
    if (r.heads < 1 || r.heads > 65536 || r.head_dim < rope.rope_dim || r.head_dim > gufo::kMaxRopeDim || r.head_dim % 2 != 0) {
      return Fail(GUFO_CUDA_SHAPE, "rope: 1 to 65536 heads of rope_dim to 512 values, an even number");
    }
    if (r.in == r.out && (r.in_token_stride != r.out_token_stride || r.in_head_stride != r.out_head_stride)) {
      return Fail(GUFO_CUDA_BAD_ARGUMENT, "rope: rows that are turned in place keep their strides");
    }
    a.parts[i].rows = r;
    widest = widest > r.head_dim ? widest : r.head_dim;
    most = most > r.heads ? most : r.heads;
    rows += r.heads;
    fours = fours && r.head_dim % 8 == 0 &&
            ((reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out)) & 15) == 0 &&
            ((r.in_token_stride | r.in_head_stride | r.out_token_stride | r.out_head_stride) & 3) == 0;
  }
  if (tokens == 0) {
    return GUFO_CUDA_OK;
  }
  const int per = fours ? 4 : 1;
  a.lanes = 1;
  while (a.lanes < 32 && a.lanes * per * 2 < widest) {
    a.lanes *= 2;
  }
  // Heads that share a token's sines: up to eight, as many as leave the device 16 warps an SM. (8000
  // tokens of 10 heads: 49 us with a head a group of lanes, 32 with eight.)
  const int64_t room = static_cast<int64_t>(ctx->sm_count) * 16 * (32 / a.lanes);
  const int64_t want = static_cast<int64_t>(tokens) * rows / room;
  a.each = want < 1 ? 1 : want > most ? most : static_cast<int>(want);
  a.each = a.each > 8 ? 8 : a.each;
  for (int i = 0; i < nparts; ++i) {
    a.parts[i].first = a.items;
    a.items += (parts[i].heads + a.each - 1) / a.each;
  }
  if (static_cast<int64_t>(tokens) * a.items * a.lanes > static_cast<int64_t>(INT32_MAX) - gufo::kRopeThreads) {
    return Fail(GUFO_CUDA_TOO_LARGE, "rope: too many rows for one call");
  }
  a.nparts = nparts;
  a.turns = rope.turns;
  a.positions = positions;
  a.tokens = tokens;
  a.rope_dim = rope.rope_dim;
  a.magnitude = rope.magnitude;
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  const int times = (widest / 2 + a.lanes * per - 1) / (a.lanes * per);
  cudaError_t e;
  if (fours) {
    e = times <= 1 ? gufo::Launch<4, 1>(ctx, a, rope.interleaved) : gufo::Launch<4, 2>(ctx, a, rope.interleaved);
  } else {
    e = times <= 2 ? gufo::Launch<1, 2>(ctx, a, rope.interleaved)
        : times <= 4 ? gufo::Launch<1, 4>(ctx, a, rope.interleaved)
                     : gufo::Launch<1, 8>(ctx, a, rope.interleaved);
  }
  GUFO_CUDA_TRY(e);
  ctx->launches.fetch_add(1);
  return GUFO_CUDA_OK;
}

}  // extern "C"
