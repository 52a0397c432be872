// Attention of a few query tokens of each sequence over the 8-bit cache.
//
// What bounds it. The cache is read once, two bytes a row and dimension of a KV head: far into
// the contexts that is all the time there is, if loads are never waited for and the arithmetic
// stays hidden under them: one int8 sequence of 131000 rows of 4 heads of 256 65 us, 4.1 TB/s, of
// which the loop alone takes 4.4; half of all cycles issue, and three warps a scheduler do not cover
// more of what instructions wait for one another. Short contexts are bound by latency (500 rows
// 7 us), ragged batches by both (verify batch of 32 sequences 64 us: 23, and 3.4
// TB/s behind them).
//
// The arithmetic. A group of one, two or four warps (64 dimensions each) goes through tiles of
// as many blocks of the cache (16 rows, one scale for the keys, one for the values), streamed
// through rings in shared memory (bulk copies). For each block one warp takes the scores, over all
// dimensions; its weights then go to the group's warps, each of which adds up its 64 dimensions
// of the group's blocks. So nothing is decoded twice, a warp's sums take 16 registers for eight
// query rows whatever the head's size, and the group meets once a tile.
// The cache rows are the A operand of mma.sync m16n8k16, eight query rows (tokens times the
// query heads of the KV head) the B operand:
//   S^T = K Q^T   [16 rows x 8 queries],     O^T = V^T P^T   [16 dimensions x 8 queries]
// Codes become fp16 exactly, in registers. The fp32 operands (queries; probabilities) go in as
// two fp16 halves, 22 bits of them, scaled by a power of two first so that small ones keep
// their bits (queries against int8 keys: as whole numbers of four digits); each sixteen products'
// sum is added up in fp32, as the tensor core cuts off what its adder does not hold. S^T comes out
// with a query's column in the lanes that O^T wants it in; P^T is turned into a B operand by
// movmatrix. A lane's dimensions are permuted (16 bytes
// of a key row, 8 of a value row are its own), which a sum over all of them does not see and
// the output undoes.
// A block's weights are taken against the maximum that the group knew, or the block's own where
// that is larger; only then, and with the first tiles, is anything rescaled.
//
// The split. A unit of work is (sequence, group of query rows, KV head) with all the tiles
// that the sequence is long. The device's resident blocks of threads share out the tiles of all
// units, in order, to one tile: each finds its stretch from the lengths that it reads, whatever
// they are, and goes through the units that it touches. What several blocks have a part of, a
// second kernel puts together, part by part in order: as a last block's work behind a counter
// it took 5 us more of the first one's time (fence, counter, two rounds through L2 by one block).
// Where the cache is short, a unit has a block or a cluster of blocks instead, which join in
// distributed shared memory.
//
// The weights of the rows (for eviction) need every query's final maximum and sum: the scores
// are written down as they come, 4 bytes against 2 * head_dim / group read for them, and a
// second kernel turns them into weights and adds those up, one thread a row, in order.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "cache8.cuh"
#include "decode_device.cuh"
#include "mma_common.cuh"

namespace gufo {
namespace {

constexpr int kMostUnitRows = 256;
constexpr int kRanks = 8;
constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kMostSms = 160;                 // whose blocks a call uses
constexpr int kMostBlocks = 4 * kMostSms;     // of threads: four an SM at most
constexpr float kProbScale = 32768.f;
constexpr float kLog2e = 1.4426950408889634f;

// A unit that several blocks have a part of: what the second kernel needs to know. One for every
// unit, or, where they are more than the blocks, for the last one that each block begins.
struct Cut {
  int first;       // block
  int parts;       // blocks with a part of it; 0: none is cut here
  int rows;        // query rows
  int token, head; // of its first row
  int first_flat;  // that row's place among the sequence's tokens' heads of this KV head
};

struct AttendArgs {
  CacheView cache;
  const float* queries;
  int64_t query_token_stride, query_head_stride;
  const float* gate;
  int64_t gate_token_stride, gate_head_stride;
  float* out;
  int64_t out_token_stride, out_head_stride;
  const int* visible;
  int heads, group;
  float scale;             // times log2 e
  int whole;               // rows of queries, gates and outputs may be taken four values at a time
  Cut* cuts;               // [units or blocks]
  int by_unit;
  int ranks;               // blocks of a unit that is not shared out: 1, or a cluster's kRanks
  float* sums;             // [blocks][2: the unit it goes on with, the one it begins][rows][head_dim]
  float* stats;            // [blocks][2][rows][2]
  float* scores;           // [query rows][capacity]; null: no weights
  float* finals;           // [query rows][2]: maximum, 1 / sum
};

// NS: segments of 64 dimensions (1, 2, 4), warps of a group; RT: groups of eight query rows.
// Small blocks of threads, several of which an SM holds: one's queries and join pass under
// another's tiles (one block of 16 warps an SM: the verify batch 90 us, not 75; one long sequence
// 60, not 64).
template <int NS, int RT>
struct Shape {
  static constexpr int kTile = NS * kCacheBlock;            // rows that a group takes at a time
  static constexpr int kGroups = kWarps / NS;
  // What a unit costs besides its tiles (queries, the join), in tiles: as much as so many rows of the
  // cache. (The verify batch, heads of 256: 68, 64 and 67 us with 64, 128 and 256 rows; heads of 128:
  // 50, 46, 48; 100 sequences, heads of 64: 77, 60, 52.)
  static constexpr int kUnitCost = (NS == 1 ? kMostUnitRows : 128) / kTile;
  static constexpr int kRowBytes = 64 * NS;
  static constexpr int kSlot = kCacheBlock * kRowBytes + 16;   // a block's keys or values, their scale
  static constexpr int kSlots = NS == 4 ? 3 : NS == 2 ? 5 : 8;
  static constexpr int kRing = kWarps * kSlots * kSlot;
  static constexpr int kJoin = kGroups * 8 * RT * kRowBytes * 4;
  // Of threads that an SM holds: as many as keep their sums in registers, but for 4 to 40 bytes that eleven of
  // the 72 kernels spill (e4m3, heads of 256, 16 query rows: 40). (32 sequences of some 2000
  // rows, heads of 128: 16 query rows 66 us with four, 48 with three; 32 query rows 129 with three,
  // 95 with two. Heads of 256, 16 query rows: 70 with three, 79 with two.)
  static constexpr int kBlocks = RT == 4 ? 2 : NS == 4 || RT == 2 ? 3 : 4;
  static constexpr int kShared = kRing > kJoin ? kRing : kJoin;
  static constexpr int kQuery = RT * NS * 4 * 32 * 16;      // B operands, in the lanes' order (two fp16 halves, or four digits)
  static constexpr int kWeights = NS == 1 ? 0 : 2 * kWarps * RT * 32 * 16;   // the same of two tiles' weights
  static constexpr int kBytes = kShared + kQuery + kWeights;
  static_assert(kBlocks * (kBytes + 1024 + 2880) <= 228 * 1024 || RT == 4, "kBlocks fit an SM with what else is in shared memory");
};

// Waits until a copy that this kernel asked for has landed; false, once, where it has not after
// about a second: what comes of it is made NaN then, and the warp waits for nothing any more and asks
// for nothing. Ahead of that it waits as long again for the copies into its own ring that are under way
// (slots `slot`, of this `phase`, up to the one that is filled next): they must not find the shared
// memory of the next block of threads.
template <int kSlots>
__device__ __noinline__ bool LandedLate(uint32_t bar, uint32_t parity, uint32_t own, int slot, int fill_slot) {
  const long long began = clock64();
  while (!MbarTryWait(bar, parity)) {
    if (clock64() - began > kLandLimit) {
      do {
        while (!MbarTryWait(own + 8 * slot, parity) && clock64() - began < 2 * kLandLimit) {
        }
        if (++slot == kSlots) {
          slot = 0;
          parity ^= 1;
        }
      } while (slot != fill_slot);
      return false;
    }
  }
  return true;
}

// The warps of a group meet.
template <int NS>
__device__ __forceinline__ void Meet(int group) {
  if constexpr (NS == 1) {
    __syncwarp();
  } else {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * NS) : "memory");
  }
}
// d = a b, sixteen products added by the instruction; d += a b. Volatile, so that a product stays
// ahead of the barrier behind which its operands' place in shared memory is given back: its
// issue is what waits for their loads.
__device__ __forceinline__ void MmaFirst(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void MmaMore(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d += a b in whole numbers, thirty-two products.
__device__ __forceinline__ void MmaWhole(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transpose(uint32_t v) {
  uint32_t t;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}
__device__ __forceinline__ uint32_t PackHalves(__half x, __half y) {
  return __half_as_ushort(x) | static_cast<uint32_t>(__half_as_ushort(y)) << 16;
}

// A unit: query rows [row0, row0 + rows) of a sequence, one KV head.
struct Task {
  BatchEntry e;
  int rows, row0;
  int position;
};

__device__ __forceinline__ int SeenBy(const AttendArgs& a, const BatchEntry& e, int position, int token) {
  const int64_t seen = a.visible != nullptr ? __ldcg(a.visible + e.row + token) : static_cast<int64_t>(position) + token + 1;
  return static_cast<int>(min(max(seen, static_cast<int64_t>(0)), static_cast<int64_t>(a.cache.capacity)));
}

// Tiles of each sequence in `tiles` (one at least: a row that sees nothing is an output too) and
// the cost of the units of all sequences ahead of it in `ahead` ([sequences + 1]). (The sum of
// all is an int: the caller has made sure.) Threads: 128 at least.
struct Shares {
  int tiles[kBatchSequences];
  int ahead[kBatchSequences + 1];
  int position[kBatchSequences];
};
__device__ __forceinline__ void ShareOut(const AttendArgs& a, const BatchArgs& batch, int tile_rows, int unit_cost, Shares& shares) {
  int* const tiles = shares.tiles;
  int* const ahead = shares.ahead;
  __shared__ int of_warp[kBatchSequences / 32];
  const int n = batch.sequences, i = threadIdx.x, warp = i >> 5, lane = i & 31;
  if (i < n) {
    shares.position[i] = __ldcg(batch.positions + batch.of[i].index);
  }
  if (a.visible == nullptr) {
    if (i < n) {
      tiles[i] = SeenBy(a, batch.of[i], shares.position[i], batch.of[i].tokens - 1);
    }
  } else {
    for (int s = warp; s < n; s += blockDim.x / 32) {
      int most = 0;
      for (int token = lane; token < batch.of[s].tokens; token += 32) {
        most = max(most, SeenBy(a, batch.of[s], 0, token));
      }
      most = __reduce_max_sync(0xFFFFFFFFu, most);
      if (lane == 0) {
        tiles[s] = most;
      }
    }
    __syncthreads();
  }
  int sum = 0;
  if (i < kBatchSequences) {
    int mine = 0;
    if (i < n) {
      const int of = max(1, (tiles[i] + tile_rows - 1) / tile_rows);
      tiles[i] = of;
      mine = (batch.first_item[i + 1] - batch.first_item[i]) * a.cache.kv_heads * (of + unit_cost);
    }
    sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      sum += lane >= o ? below : 0;
    }
    if (lane == 31) {
      of_warp[warp] = sum;
    }
  }
  __syncthreads();
  if (i < kBatchSequences) {
    for (int w = 0; w < warp; ++w) {
      sum += of_warp[w];
    }
    ahead[i + 1] = sum;
    if (i == 0) {
      ahead[0] = 0;
    }
  }
  __syncthreads();
}

// The blocks' stretches of the whole cost: one more for the first `more` of them. A unit's own
// cost comes ahead of its tiles: a block whose stretch ends within it has no part of the unit.
struct Stretches {
  int blocks, each, more;
  __device__ __forceinline__ Stretches(int all, int least, int most) : blocks(min(most, max(all / least, 1))) {
    each = all / blocks;
    more = all - each * blocks;
  }
  __device__ __forceinline__ int start_of(int block) const { return each * block + min(block, more); }
  __device__ __forceinline__ int owner_of(int at) const {     // the block whose stretch it is in
    const int split = (each + 1) * more;
    return at < split ? at / (each + 1) : more + (at - split) / each;
  }
};
// The unit that `at` of the whole cost is of.
struct Unit {
  int sequence, tiles;
  int start;      // of its tiles
  int chunk, kh;
  int number;     // of all units of the batch
  Unit() = default;
  __device__ __forceinline__ Unit(const BatchArgs& batch, const Shares& shares, int kv_heads, int unit_cost, int at) {
    const int sequences = batch.sequences;
    int low = 0, high = sequences - 1;
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (shares.ahead[mid] <= at) {
        low = mid;
      } else {
        high = mid - 1;
      }
    }
    sequence = low;
    tiles = shares.tiles[low];
    const int unit = (at - shares.ahead[low]) / (tiles + unit_cost);
    start = shares.ahead[low] + unit * (tiles + unit_cost) + unit_cost;
    chunk = unit / kv_heads;
    kh = unit - chunk * kv_heads;
    number = batch.first_item[low] * kv_heads + unit;
  }
};
__device__ __forceinline__ Task TaskOf(const AttendArgs& a, const BatchArgs& batch, int position, const Unit& unit, int rows) {
  Task task;
  task.e = batch.of[unit.sequence];
  task.row0 = unit.chunk * rows;
  task.rows = min(rows, task.e.tokens * a.group - task.row0);
  task.position = position;
  return task;
}
// Where a block's part of a unit starts, in rows: of the one that it goes on with, or begins.
__device__ __forceinline__ size_t PartOf(int block, bool begins, int rows) { return (static_cast<size_t>(block) * 2 + (begins ? 1 : 0)) * rows; }
// The call's query row of a task's row r: token and head.
struct QueryRow {
  int64_t token;
  int head;
  QueryRow() = default;
  __device__ __forceinline__ QueryRow(const AttendArgs& a, const Task& task, int kh, int r) {
    const int flat = task.row0 + r, t = flat / a.group;
    token = static_cast<int64_t>(task.e.row) + t;
    head = kh * a.group + flat - t * a.group;
  }
};
// Four dimensions of a row of the output, gated; a row that saw nothing is zero.
__device__ __forceinline__ void Finish(const AttendArgs& a, const QueryRow& q, int f, float4 v, float sum, bool sees) {
  float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.gate != nullptr) {
    const float* gate = a.gate + q.token * a.gate_token_stride + q.head * a.gate_head_stride + 4 * f;
    if (a.whole) {
      g = *reinterpret_cast<const float4*>(gate);
    } else {
      g = make_float4(gate[0], gate[1], gate[2], gate[3]);
    }
  }
  const float by = 1.f / sum;
  float4 o = make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
  if (a.gate != nullptr) {
    o.x *= SigmoidDev(g.x), o.y *= SigmoidDev(g.y), o.z *= SigmoidDev(g.z), o.w *= SigmoidDev(g.w);
  }
  if (!sees) {
    o = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float* out = a.out + q.token * a.out_token_stride + q.head * a.out_head_stride + 4 * f;
  if (a.whole) {
    *reinterpret_cast<float4*>(out) = o;
  } else {
    out[0] = o.x, out[1] = o.y, out[2] = o.z, out[3] = o.w;
  }
}
// What the weights need of a row.
__device__ __forceinline__ void Note(const AttendArgs& a, const QueryRow& q, float most, float sum) {
  if (a.finals != nullptr) {
    reinterpret_cast<float2*>(a.finals)[q.token * a.heads + q.head] = make_float2(most, 1.f / sum);
  }
}

// D: tiles are shared out, grid: resident blocks; otherwise grid: units times ranks. W: the scores are written
// down. (Apart, as what the loop has to fetch counts: with
// the stores behind a test in it a verify batch that writes none took 97 us, not 63.)
template <typename Format, int NS, int RT, bool W, bool D>
__global__ void __launch_bounds__(kThreads, (Shape<NS, RT>::kBlocks))
AttendKernel(const __grid_constant__ AttendArgs a, const __grid_constant__ BatchArgs batch) {
  using S = Shape<NS, RT>;
  constexpr int kTile = S::kTile;
  constexpr int kDigits = 4;                 // of queries as whole numbers
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ float row_factor[8 * RT];       // of a query row's scores; then their weights' sum
  __shared__ int row_seen[8 * RT];
  __shared__ float2 row_stats[D ? 1 : 8 * RT];       // a cluster's blocks': maximum and sum
  __shared__ float* row_scores[W ? 8 * RT : 1];      // where a query row's scores are written
  __shared__ __align__(8) float block_top[2][kWarps][8 * RT];    // what a block's weights are taken against
  __shared__ float group_top[S::kGroups][8 * RT], warp_total[kWarps][8 * RT];
  __shared__ std::conditional_t<D, Shares, int> shares;
  __shared__ __align__(16) uint4 nothing;        // a piece of zeros
  __shared__ __align__(8) uint64_t bars[kWarps][S::kSlots];
  if (threadIdx.x < kWarps * S::kSlots) {
    MbarInit(SharedAddress(&bars[0][0] + threadIdx.x), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    nothing = make_uint4(0, 0, 0, 0);
  }
  GridDependencyWait();
  GridLaunchDependents();
  const CacheView& c = a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / NS, member = warp % NS;
  const int g = lane >> 2, t = lane & 3;
  int begin = 0, end = 1, all = 1;
  if constexpr (D) {
    ShareOut(a, batch, kTile, S::kUnitCost, shares);
    all = shares.ahead[batch.sequences];
  }
  const Stretches stretches(all, S::kGroups, gridDim.x);   // a tile a group at least
  if constexpr (D) {
    if (threadIdx.x == 0 && !a.by_unit) {
      a.cuts[blockIdx.x].parts = 0;      // unless it begins a unit that others have parts of
    }
    if (blockIdx.x >= stretches.blocks) {
      return;
    }
    begin = stretches.start_of(blockIdx.x);
    end = stretches.start_of(blockIdx.x + 1);
  }

  const auto ring_of = [&](int w) { return raw + w * (S::kSlots * S::kSlot); };
  uint8_t* const ring = ring_of(warp);
  const int codes_bytes = CodeBytes(c.head_dim), block_bytes = BlockBytes(c.head_dim);
  const int pieces = c.head_dim / 16;
  // This lane's places in a block: keys of row g (g + 8: 256 further), piece t of a segment
  // (a segment: 1024 further); values of rows 2 t and 2 t + 1 (+ 8), eight dimensions of this
  // warp's segment (past the last piece any: nobody asks for them).
  const int key_place = PieceAt(0, g, t);
  const int value_piece = min(4 * member + (g >> 1), pieces - 1);
  const int value_place = PieceAt(1, 2 * t, value_piece) + 8 * (g & 1);
  // The ring's slots go round, through all units: the next to be filled, the next to be read.
  int fill_slot = 0, slot = 0, phase = 0;
  bool late = false;
  const auto wait_for = [&](int of_warp) {
    const uint32_t bar = SharedAddress(&bars[of_warp][slot]);
    if (!late && !MbarTryWait(bar, phase)) {
      late = !LandedLate<S::kSlots>(bar, phase, SharedAddress(&bars[warp][0]), slot, fill_slot);
    }
  };
  const auto next_slot = [&]() {
    if (++slot == S::kSlots) {
      slot = 0;
      phase ^= 1;
    }
  };
  uint4* const query = reinterpret_cast<uint4*>(raw + S::kShared);   // [rt][seg * 4 + j][lane]: high pair, pair, low pair, pair
  uint4* const shared_p = reinterpret_cast<uint4*>(raw + S::kShared + S::kQuery);   // [2][warp][rt][lane]

#pragma unroll 1
  for (int from = begin; from < end;) {
    Unit unit;
    Task task;
    int first_tile = 0, last_tile = INT_MAX;
    if constexpr (!D) {
      const int number = blockIdx.x / a.ranks, item = number / c.kv_heads;
      unit.sequence = SequenceOf(batch, item);
      unit.kh = number - item * c.kv_heads;
      unit.chunk = item - batch.first_item[unit.sequence];
      unit.tiles = last_tile;
      unit.start = unit.number = 0;
      from = end;
      task = TaskOf(a, batch, __ldcg(batch.positions + batch.of[unit.sequence].index), unit, 8 * RT);
    } else {
      unit = Unit(batch, shares, c.kv_heads, S::kUnitCost, from);
      first_tile = max(from - unit.start, 0);
      last_tile = min(end - unit.start, unit.tiles);
      from = unit.start + unit.tiles;
      if (last_tile <= first_tile) {
        continue;
      }
      task = TaskOf(a, batch, shares.position[unit.sequence], unit, 8 * RT);
    }
    const int kh = unit.kh;
    if (threadIdx.x < 8 * RT) {
      const int r = min(static_cast<int>(threadIdx.x), task.rows - 1);
      row_seen[threadIdx.x] = SeenBy(a, task.e, task.position, (task.row0 + r) / a.group);
      if constexpr (W) {
        const QueryRow q(a, task, kh, r);
        row_scores[threadIdx.x] = a.scores + (q.token * a.heads + q.head) * c.capacity;
      }
    }
    __syncthreads();
    int length = 0, least = INT_MAX;
#pragma unroll
    for (int r = 0; r < 8 * RT; ++r) {
      length = max(length, row_seen[r]);
      least = min(least, row_seen[r]);
    }
    // (These rows may see less than the sequence's last ones.)
    const int all_tiles = (length + kTile - 1) / kTile;
    const int rank = D || a.ranks == 1 ? 0 : blockIdx.x % kRanks;
    if (!D && a.ranks > 1) {
      first_tile = all_tiles * rank / kRanks;
      last_tile = all_tiles * (rank + 1) / kRanks;
    }
    const int end_tile = min(last_tile, all_tiles);
    const size_t of_head = static_cast<size_t>(task.e.slot) * c.kv_heads + kh;

    // ---- the ring: a warp copies its block of every tile, keys and values in turn (a block that
    // nobody sees is not copied)
    const uint8_t* const keys_from = BlocksOf(c, 0, of_head);
    const uint8_t* const values_from = BlocksOf(c, 1, of_head);
    int next_tile = first_tile + group;
    bool next_values = false;
    auto load = [&]() {
      if (next_tile < end_tile) {
        if (lane == 0 && !late) {
          const int block = next_tile * NS + member;
          const uint32_t bar = SharedAddress(&bars[warp][fill_slot]);
          if (block * kCacheBlock < length) {
            MbarArriveExpectTx(bar, block_bytes);
            BulkCopy(SharedAddress(ring + fill_slot * S::kSlot),
                     (next_values ? values_from : keys_from) + static_cast<size_t>(block) * block_bytes, block_bytes, bar);
          } else {
            MbarArrive(bar);
          }
        }
        next_tile += next_values ? S::kGroups : 0;
        next_values = !next_values;
        fill_slot = fill_slot + 1 == S::kSlots ? 0 : fill_slot + 1;
      }
    };
#pragma unroll
    for (int i = 0; i < S::kSlots - 1; ++i) {
      load();
    }

    // ---- the queries: every fourth row to a warp, in the order of the B operands
    constexpr int kTimes = (16 * NS + 31) / 32;
    constexpr int kEach = 8 * RT / kWarps;
    float4 rows_in[kEach][kTimes];
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const bool there = warp + kWarps * n < task.rows;
      const QueryRow q(a, task, kh, there ? warp + kWarps * n : 0);
      const float* row = a.queries + q.token * a.query_token_stride + q.head * a.query_head_stride;
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        const int f = lane + 32 * i;
        rows_in[n][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there && 4 * f < c.head_dim) {
          if (a.gate != nullptr && f % 8 == 0) {      // (wanted at the end: from L2 then)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a.gate + q.token * a.gate_token_stride + q.head * a.gate_head_stride + 4 * f));
          }
          if (a.whole) {
            rows_in[n][i] = *reinterpret_cast<const float4*>(row + 4 * f);
          } else {
            rows_in[n][i] = make_float4(row[4 * f], row[4 * f + 1], row[4 * f + 2], row[4 * f + 3]);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int r = warp + kWarps * n;
      const float4(&x)[kTimes] = rows_in[n];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        top = max(max(top, __float_as_uint(x[i].x) & 0x7FFFFFFFu), __float_as_uint(x[i].y) & 0x7FFFFFFFu);
        top = max(max(top, __float_as_uint(x[i].z) & 0x7FFFFFFFu), __float_as_uint(x[i].w) & 0x7FFFFFFFu);
      }
      top = __reduce_max_sync(0xFFFFFFFFu, top);
      if constexpr (Format::kWhole) {
        // Whole numbers as four signed bytes, base 256, the largest from 2^29 to 2^30: rounded to half of 2^-29 of
        // it. What is smaller keeps as many bits less, and may meet the keys' largest channels, so three bytes are
        // too few: queries inverse to keys of which 4 channels in 128 are a hundred times the others, 2e-6 off, this
        // way 2e-8 (fp32 operations 2.4e-7). A row that is not finite: any, its factor is NaN.
        const int e = min(max(static_cast<int>(top >> 23), 30), 254);
        const int by = 156 - e;
        const float up = PowerOfTwo(by);
#pragma unroll
        for (int i = 0; i < kTimes; ++i) {
          const int f = lane + 32 * i;     // dimensions 64 seg + 16 c + 4 j ..
          if (f < 16 * NS) {
            const int seg = f / 16, of = f % 16 / 4, j = f % 4;
            const int v[4] = {__float2int_rn(x[i].x * up), __float2int_rn(x[i].y * up), __float2int_rn(x[i].z * up),
                              __float2int_rn(x[i].w * up)};
            uint32_t digits[kDigits] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // Offset by 128 each, the bytes are the balanced digits.
              constexpr uint32_t kOffset = 0x80808080u;
              const uint32_t z = (static_cast<uint32_t>(v[k]) + kOffset) ^ kOffset;
#pragma unroll
              for (int l = 0; l < kDigits; ++l) {
                digits[l] |= (z >> (8 * l) & 0xFFu) << (8 * k);
              }
            }
            uint32_t* to = reinterpret_cast<uint32_t*>(query);     // [rt][seg][digit][lane][j]
#pragma unroll
            for (int l = 0; l < kDigits; ++l) {
              to[((((r / 8 * NS + seg) * kDigits + l) * 32) + r % 8 * 4 + of) * 4 + j] = digits[l];
            }
          }
        }
        if (lane == 0) {
          row_factor[r] = top < 0x7F800000u ? a.scale * PowerOfTwo(-by) : NAN;
        }
      } else {
        // The largest to 2^14 .. 2^15. (Products with codes of up to 448 and their sums stay in fp32's range.)
        const int e = min(max(static_cast<int>(top >> 23), 16), 254);
        const float up = PowerOfTwo(141 - e);
#pragma unroll
        for (int i = 0; i < kTimes; ++i) {
          const int f = lane + 32 * i;     // dimensions 64 seg + 16 c + 4 j ..
          if (f < 16 * NS) {
            const int seg = f / 16, of = f % 16 / 4, j = f % 4;
            const float v[4] = {x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up};
            __half high[4], low[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              high[k] = __float2half_rn(v[k]);
              low[k] = __float2half_rn(v[k] - __half2float(high[k]));
            }
            query[(r / 8 * 4 * NS + seg * 4 + j) * 32 + r % 8 * 4 + of] = make_uint4(
                PackHalves(high[0], high[1]), PackHalves(high[2], high[3]), PackHalves(low[0], low[1]), PackHalves(low[2], low[3]));
          }
        }
        if (lane == 0) {
          row_factor[r] = a.scale * PowerOfTwo(e - 141);
        }
      }
    }
    __syncthreads();

    // ---- the tiles
    float factor[RT][2];
    int seen[RT][2];
    float top[RT][2], total[RT][2];      // of query rows 8 rt + 2 t, + 1: the group's maximum, the sum of this lane's rows
    float acc[RT][4][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        factor[rt][i] = row_factor[8 * rt + 2 * t + i];
        seen[rt][i] = row_seen[8 * rt + 2 * t + i];
        top[rt][i] = -INFINITY;
        total[rt][i] = 0.f;
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        acc[rt][m][0] = acc[rt][m][1] = acc[rt][m][2] = acc[rt][m][3] = 0.f;
      }
    }
    // (All groups of eight rows, also where the sequence has fewer: a second loop for those is code that
    // the SM fetches in vain; a ragged batch of one to four tokens took 70 us with it and 64 without,
    // one to eight tokens 157 and 131.)
    int parity = 0;
#pragma unroll 1
    for (int tile = first_tile + group; tile < end_tile; tile += S::kGroups) {
      if ((tile * NS + member) * kCacheBlock < length) {
        wait_for(warp);
      }
      // Scores of this warp's block.
      const uint8_t* keys = ring + slot * S::kSlot;
      next_slot();
      float s[RT][4];
      const auto key_words = [&](int seg, int more) {
        const uint8_t* at = keys + key_place + 1024 * seg + more;
        return *reinterpret_cast<const uint4*>(4 * seg + t < pieces ? at : reinterpret_cast<const uint8_t*>(&nothing));
      };
      // (A block behind the last row that is seen was not copied, and weighs nothing.)
      const bool there = (tile * NS + member) * kCacheBlock < length;
      if (!there) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          s[rt][0] = s[rt][1] = s[rt][2] = s[rt][3] = 0.f;
        }
      } else if constexpr (Format::kWhole) {
        int d[RT][kDigits][4];      // by the queries' digits
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int l = 0; l < kDigits; ++l) {
            d[rt][l][0] = d[rt][l][1] = d[rt][l][2] = d[rt][l][3] = 0;
          }
        }
#pragma unroll
        for (int seg = 0; seg < NS; ++seg) {
          const uint4 k0 = key_words(seg, 0), k1 = key_words(seg, 256);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int l = 0; l < kDigits; ++l) {
              const uint4 q = query[((rt * NS + seg) * kDigits + l) * 32 + lane];
              MmaWhole(d[rt][l], k0.x, k1.x, k0.y, k1.y, q.x, q.y);
              MmaWhole(d[rt][l], k0.z, k1.z, k0.w, k1.w, q.z, q.w);
            }
          }
        }
        // (A digit's sum is at most 256 * 128 * 127, the highest's half of that: two of them fit an int.)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[rt][i] = fmaf(static_cast<float>(d[rt][3][i] * 256 + d[rt][2][i]), 65536.f,
                            static_cast<float>(d[rt][1][i] * 256 + d[rt][0][i]));
          }
        }
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          s[rt][0] = s[rt][1] = s[rt][2] = s[rt][3] = 0.f;
        }
#pragma unroll
        for (int seg = 0; seg < NS; ++seg) {
          const uint4 k0 = key_words(seg, 0), k1 = key_words(seg, 256);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          uint32_t k[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            Format::Decode(w0[j], k[j][0], k[j][2]);
            Format::Decode(w1[j], k[j][1], k[j][3]);
          }
          // Four products at a time, low halves first: an instruction's result is not waited for.
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            uint4 q[4];
            float d[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              q[j] = query[(rt * 4 * NS + seg * 4 + j) * 32 + lane];
              MmaFirst(d[j], k[j], q[j].z, q[j].w);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              MmaMore(d[j], k[j], q[j].x, q[j].y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[rt][i] += (d[0][i] + d[1][i]) + (d[2][i] + d[3][i]);
            }
          }
        }
      }
      const float key_scale = *reinterpret_cast<const float*>(keys + codes_bytes);
      const int r0 = (tile * NS + member) * kCacheBlock + g;
      const bool hides = (tile + 1) * kTile > least;     // some rows from some queries
      uint4 p[RT];             // high pair of rows 0-7, of 8-15; low pairs
      float sum[RT][2];        // of this lane's weights
      float own[RT][2];        // what they are taken against
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[rt][i] *= factor[rt][i & 1] * key_scale;
        }
        if constexpr (W) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 8 * rt + 2 * t + (i & 1), row = r0 + 8 * (i >> 1);
            if (r < task.rows && row < length) {
              __stcg(row_scores[r] + row, s[rt][i]);
            }
          }
        }
        if (hides) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[rt][i] = r0 + 8 * (i >> 1) < seen[rt][i & 1] ? s[rt][i] : -INFINITY;
          }
        }
        float m0 = fmaxf(fmaxf(s[rt][0], s[rt][2]), top[rt][0]), m1 = fmaxf(fmaxf(s[rt][1], s[rt][3]), top[rt][1]);
        if (__any_sync(0xFFFFFFFFu, m0 > top[rt][0] || m1 > top[rt][1])) {
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(0xFFFFFFFFu, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, o));
          }
        }
        own[rt][0] = m0, own[rt][1] = m1;
        if constexpr (NS > 1) {
          if (g == 0) {
            *reinterpret_cast<float2*>(&block_top[parity][warp][8 * rt + 2 * t]) = make_float2(m0, m1);
          }
        }
        const float t0 = m0 == -INFINITY ? 0.f : m0, t1 = m1 == -INFINITY ? 0.f : m1;
        const float e0 = exp2f(s[rt][0] - t0), e1 = exp2f(s[rt][1] - t1), e2 = exp2f(s[rt][2] - t0), e3 = exp2f(s[rt][3] - t1);
        sum[rt][0] = e0 + e2;
        sum[rt][1] = e1 + e3;
        const float x[4] = {e0 * kProbScale, e1 * kProbScale, e2 * kProbScale, e3 * kProbScale};
        __half high[4], low[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          high[i] = __float2half_rn(x[i]);
          low[i] = __float2half_rn(x[i] - __half2float(high[i]));
        }
        p[rt] = make_uint4(Transpose(PackHalves(high[0], high[1])), Transpose(PackHalves(high[2], high[3])),
                           Transpose(PackHalves(low[0], low[1])), Transpose(PackHalves(low[2], low[3])));
        if constexpr (NS > 1) {
          shared_p[((parity * kWarps + warp) * RT + rt) * 32 + lane] = p[rt];
        }
      }
      Meet<NS>(group);       // the weights are there; the last tile's values and this one's keys are done with
      load();
      load();
      // Where a block has raised the maximum: the sums to it.
      bool raised = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float n0 = own[rt][0], n1 = own[rt][1];
        if constexpr (NS > 1) {
#pragma unroll
          for (int b = 0; b < NS; ++b) {
            const float2 of = *reinterpret_cast<const float2*>(&block_top[parity][group * NS + b][8 * rt + 2 * t]);
            n0 = fmaxf(n0, of.x), n1 = fmaxf(n1, of.y);
          }
        }
        if (__any_sync(0xFFFFFFFFu, n0 > top[rt][0] || n1 > top[rt][1])) {
          raised = true;
          const float keep0 = n0 == top[rt][0] ? 1.f : exp2f(top[rt][0] - n0), keep1 = n1 == top[rt][1] ? 1.f : exp2f(top[rt][1] - n1);
          top[rt][0] = n0, top[rt][1] = n1;
          const float mine0 = own[rt][0] == n0 ? 1.f : exp2f(own[rt][0] - n0), mine1 = own[rt][1] == n1 ? 1.f : exp2f(own[rt][1] - n1);
          total[rt][0] = total[rt][0] * keep0 + sum[rt][0] * mine0;
          total[rt][1] = total[rt][1] * keep1 + sum[rt][1] * mine1;
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            acc[rt][m][0] *= keep0, acc[rt][m][1] *= keep1, acc[rt][m][2] *= keep0, acc[rt][m][3] *= keep1;
          }
        } else {
          total[rt][0] += sum[rt][0];
          total[rt][1] += sum[rt][1];
        }
      }
      // This warp's dimensions of the group's blocks.
#pragma unroll
      for (int b = 0; b < NS; ++b) {
        const int block = tile * NS + b;
        if (block * kCacheBlock >= length) {
          break;
        }
        wait_for(group * NS + b);
        uint8_t* values = ring_of(group * NS + b) + slot * S::kSlot;
        if constexpr (Format::kHasNan) {
          // A value that is NaN makes NaN of the sums of the queries that see its row, and of no
          // others, whose weight of 0 times NaN would: where some do not see all rows of a block, such
          // values are put into the sums by hand and taken out of the block.
          if ((block + 1) * kCacheBlock > least) {
            const auto marks = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; };   // of 0x7F, 0xFF
            // This warp's pieces: 64 words each.
            uint32_t* const words = reinterpret_cast<uint32_t*>(values) + 256 * member;
            const int count = 64 * min(4, (pieces + 1) / 2 * 2 - 4 * member);
            uint32_t found = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              found |= lane + 32 * i < count ? marks(words[lane + 32 * i]) : 0;
            }
            if (__any_sync(0xFFFFFFFFu, found != 0)) {
#pragma unroll
              for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const int dim = 8 * g + 2 * m + half;
                  int row = INT_MAX;      // the first with NaN
#pragma unroll 1
                  for (int r = kCacheBlock - 1; r >= 0; --r) {
                    const uint8_t code = values[PieceAt(1, r, value_piece) + dim % 16];
                    row = (code & 0x7F) == 0x7F ? block * kCacheBlock + r : row;
                  }
#pragma unroll
                  for (int rt = 0; rt < RT; ++rt) {
                    acc[rt][m][2 * half] = row < seen[rt][0] ? NAN : acc[rt][m][2 * half];
                    acc[rt][m][2 * half + 1] = row < seen[rt][1] ? NAN : acc[rt][m][2 * half + 1];
                  }
                }
              }
              __syncwarp();
#pragma unroll 1
              for (int i = lane; i < count; i += 32) {
                words[i] &= ~((marks(words[i]) >> 7) * 255u);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // ahead of the slot's next copy
              __syncwarp();
            }
          }
        }
        // (Read ahead of the values, which the products wait for: the slot is given back behind
        // those.)
        float by;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(by) : "r"(SharedAddress(values + codes_bytes)) : "memory");
        by *= 1.f / kProbScale;
        float each[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          each[rt][0] = each[rt][1] = by;
          if constexpr (NS > 1) {
            p[rt] = shared_p[((parity * kWarps + group * NS + b) * RT + rt) * 32 + lane];
            if (raised) {
              const float2 of = *reinterpret_cast<const float2*>(&block_top[parity][group * NS + b][8 * rt + 2 * t]);
              each[rt][0] *= of.x == top[rt][0] ? 1.f : exp2f(of.x - top[rt][0]);
              each[rt][1] *= of.y == top[rt][1] ? 1.f : exp2f(of.y - top[rt][1]);
            }
          }
        }
        uint2 v[4];     // this lane's eight dimensions of rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = *reinterpret_cast<const uint2*>(values + (value_place ^ (32 * (i & 1))) + 256 * (i >> 1));
        }
        uint32_t of[4][4];   // dimensions 2 m, 2 m + 1 of the eight: rows beside one another
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint32_t w0 = m < 2 ? v[0].x : v[0].y, w1 = m < 2 ? v[1].x : v[1].y;
          const uint32_t w2 = m < 2 ? v[2].x : v[2].y, w3 = m < 2 ? v[3].x : v[3].y;
          Format::Decode(__byte_perm(w0, w1, m & 1 ? 0x7362 : 0x5140), of[m][0], of[m][1]);
          Format::Decode(__byte_perm(w2, w3, m & 1 ? 0x7362 : 0x5140), of[m][2], of[m][3]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float d[4][4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            MmaFirst(d[m], of[m], p[rt].z, p[rt].w);
          }
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            MmaMore(d[m], of[m], p[rt].x, p[rt].y);
          }
#pragma unroll
          for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              acc[rt][m][i] = fmaf(d[m][i], each[rt][i & 1], acc[rt][m][i]);
            }
          }
        }
      }
      next_slot();
      parity ^= 1;
    }
    if (late) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        total[rt][0] = total[rt][1] = NAN;
      }
    }

    // ---- the groups' parts together
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = total[rt][i];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        }
        if (g == 0) {
          if (member == 0) {
            group_top[group][8 * rt + 2 * t + i] = top[rt][i];
          }
          warp_total[warp][8 * rt + 2 * t + i] = sum;
        }
      }
    }
    __syncthreads();     // the rings are free
    float* join = reinterpret_cast<float*>(raw);      // [group][row][64 NS]
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (8 * rt < task.rows) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float* out = join + (group * 8 * RT + 8 * rt + 2 * t + i) * S::kRowBytes + 64 * member + 8 * g;
          *reinterpret_cast<float4*>(out) = make_float4(acc[rt][0][i], acc[rt][0][i + 2], acc[rt][1][i], acc[rt][1][i + 2]);
          *reinterpret_cast<float4*>(out + 4) = make_float4(acc[rt][2][i], acc[rt][2][i + 2], acc[rt][3][i], acc[rt][3][i + 2]);
        }
      }
    }
    const bool alone = D ? first_tile == 0 && last_tile == unit.tiles : a.ranks == 1;
    const size_t part = PartOf(blockIdx.x, first_tile == 0, 8 * RT);
    if (threadIdx.x < 8 * RT) {
      // A row's maximum and sum, and the factors of the groups' parts.
      const int r = threadIdx.x;
      float most = -INFINITY;
#pragma unroll
      for (int of = 0; of < S::kGroups; ++of) {
        most = fmaxf(most, group_top[of][r]);
      }
      float sum = 0.f;
#pragma unroll
      for (int of = 0; of < S::kGroups; ++of) {
        const float by = group_top[of][r] == most ? 1.f : exp2f(group_top[of][r] - most);
#pragma unroll
        for (int w = 0; w < NS; ++w) {
          sum += warp_total[of * NS + w][r] * by;
        }
        group_top[of][r] = by;      // from now on the part's factor
      }
      row_factor[r] = sum;
      if constexpr (!D) {
        row_stats[r] = make_float2(most, sum);
      }
      if (r < task.rows) {
        if (alone) {
          Note(a, QueryRow(a, task, kh, r), most, sum);
        } else if (D) {
          // (A row that sees nothing is told by its sum, whatever its parts.)
          reinterpret_cast<float2*>(a.stats)[part + r] = make_float2(most, row_seen[r] > 0 ? sum : -1.f);
        }
      }
    }
    __syncthreads();
    const int fours = c.head_dim / 4;
#pragma unroll 4
    for (int at = threadIdx.x; at < task.rows * fours; at += kThreads) {
      const int r = at / fours, f = at - r * fours;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int of = 0; of < S::kGroups; ++of) {
        const float4 v = *reinterpret_cast<const float4*>(join + (of * 8 * RT + r) * S::kRowBytes + 4 * f);
        const float by = group_top[of][r];
        sum.x = fmaf(v.x, by, sum.x), sum.y = fmaf(v.y, by, sum.y), sum.z = fmaf(v.z, by, sum.z), sum.w = fmaf(v.w, by, sum.w);
      }
      if (alone) {
        Finish(a, QueryRow(a, task, kh, r), f, sum, row_factor[r], row_seen[r] > 0);
      } else if (!D) {
        *reinterpret_cast<float4*>(join + r * S::kRowBytes + 4 * f) = sum;
      } else {
        reinterpret_cast<float4*>(a.sums + (part + r) * c.head_dim)[f] = sum;
      }
    }
    if (!D && a.ranks > 1) {
      // The cluster's blocks put their parts together, each an eighth of the outputs.
      const auto cluster = cooperative_groups::this_cluster();
      cluster.sync();
      const auto parts_of = [&](int r, float (&by)[kRanks], float& most, float& total) {
        float2 stats[kRanks];
        most = -INFINITY;
#pragma unroll
        for (int i = 0; i < kRanks; ++i) {
          stats[i] = cluster.map_shared_rank(row_stats, i)[r];
          most = fmaxf(most, stats[i].x);
        }
        total = 0.f;
#pragma unroll
        for (int i = 0; i < kRanks; ++i) {
          by[i] = stats[i].x == most ? 1.f : exp2f(stats[i].x - most);
          total = fmaf(stats[i].y, by[i], total);
        }
      };
      for (int at = rank * kThreads + threadIdx.x; at < task.rows * fours; at += kRanks * kThreads) {
        const int r = at / fours, f = at - r * fours;
        float4 v[kRanks];
#pragma unroll
        for (int i = 0; i < kRanks; ++i) {
          v[i] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(join, i) + r * S::kRowBytes + 4 * f);
        }
        float by[kRanks], most, total;
        parts_of(r, by, most, total);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kRanks; ++i) {
          sum.x = fmaf(v[i].x, by[i], sum.x), sum.y = fmaf(v[i].y, by[i], sum.y);
          sum.z = fmaf(v[i].z, by[i], sum.z), sum.w = fmaf(v[i].w, by[i], sum.w);
        }
        const QueryRow q(a, task, kh, r);
        Finish(a, q, f, sum, total, row_seen[r] > 0);
        if (f == 0) {
          Note(a, q, most, total);
        }
      }
      cluster.sync();      // (the others have read this block's part)
    }
    if (D && first_tile == 0 && threadIdx.x == 0 && (a.by_unit || !alone)) {
      a.cuts[a.by_unit ? unit.number : static_cast<int>(blockIdx.x)] = {
          static_cast<int>(blockIdx.x), alone ? 0 : stretches.owner_of(unit.start + unit.tiles - 1) - static_cast<int>(blockIdx.x) + 1,
          task.rows, task.e.row, kh * a.group, task.row0};
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the rings are written by copies again
    __syncthreads();
  }
}

// The units that several blocks have parts of: grid (cuts, rows of a unit / R). R query rows a block:
// the parts' factors, then their sums; groups of a row's threads take a part of the parts each.
// (Two blocks an SM, not four: they come while the first kernel's last blocks run, and take shared
// memory and issue slots from what follows: the verify batch 84 us with four, 70 with two.)
constexpr int kJoinThreads = 256;
template <int R>
__global__ void __launch_bounds__(kJoinThreads, 2)
JoinKernel(const __grid_constant__ AttendArgs a, int rows) {
  constexpr int kRowThreads = kJoinThreads / R, kRowWarps = kRowThreads / 32;
  __shared__ float factor[R][kMostBlocks];
  __shared__ float of_warp[R][kRowWarps][2];
  __shared__ float4 partial[R][kRowThreads];
  GridLaunchDependents();
  const CacheView& c = a.cache;
  const int at_row = threadIdx.x / kRowThreads, thread = threadIdx.x % kRowThreads, warp = thread >> 5, lane = thread & 31;
  const int r = blockIdx.y * R + at_row;
  GridDependencyWait();
  const Cut cut = a.cuts[blockIdx.x];
  const int first_block = cut.first, count = cut.parts;
  if (count == 0 || static_cast<int>(blockIdx.y) * R >= cut.rows) {
    return;
  }
  const bool mine = r < cut.rows;      // (the others come along to the barriers)
  const auto part_at = [&](int i) { return PartOf(first_block + i, i == 0, rows) + r; };
  const int fours = c.head_dim / 4;
  const int takers = kRowThreads / fours;
  const int taker = thread / fours, f = thread - taker * fours;
  const int i_first = count * taker / takers, i_end = mine && taker < takers ? count * (taker + 1) / takers : 0;
  // The first sums are on their way while the statistics are looked at.
  constexpr int kAhead = R == 1 ? 16 : 8;
  float4 v[kAhead];
  const auto get = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      v[i] = i0 + i < i_end ? __ldcg(reinterpret_cast<const float4*>(a.sums + part_at(i0 + i) * c.head_dim) + f) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  get(i_first);
  constexpr int kStats = (kMostBlocks + kRowThreads - 1) / kRowThreads;
  float2 stats[kStats];
  float most = -INFINITY;
#pragma unroll
  for (int n = 0; n < kStats; ++n) {
    const int i = thread + n * kRowThreads;
    stats[n] = mine && i < count ? __ldcg(reinterpret_cast<const float2*>(a.stats) + part_at(i)) : make_float2(-INFINITY, 0.f);
    most = fmaxf(most, stats[n].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  }
  if (lane == 0) {
    of_warp[at_row][warp][0] = most;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    most = fmaxf(most, of_warp[at_row][w][0]);
  }
  float total = 0.f;
#pragma unroll
  for (int n = 0; n < kStats; ++n) {
    const int i = thread + n * kRowThreads;
    const float by = stats[n].x == most ? 1.f : exp2f(stats[n].x - most);
    if (i < count) {
      factor[at_row][i] = by;
    }
    total += stats[n].y * by;
  }
  total = WarpSum(total);
  if (lane == 0) {
    of_warp[at_row][warp][1] = total;
  }
  __syncthreads();
  total = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    total += of_warp[at_row][w][1];
  }
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = i_first; i0 < i_end; i0 += kAhead) {
    if (i0 > i_first) {
      get(i0);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float by = i0 + i < i_end ? factor[at_row][i0 + i] : 0.f;
      sum.x = fmaf(v[i].x, by, sum.x), sum.y = fmaf(v[i].y, by, sum.y), sum.z = fmaf(v[i].z, by, sum.z), sum.w = fmaf(v[i].w, by, sum.w);
    }
  }
  partial[at_row][thread] = sum;
  __syncthreads();
  if (!mine) {
    return;
  }
  QueryRow q;
  q.token = cut.token + (cut.first_flat + r) / a.group;
  q.head = cut.head + (cut.first_flat + r) % a.group;
  if (taker == 0) {
    for (int i = 1; i < takers; ++i) {
      const float4 w = partial[at_row][i * fours + f];
      sum.x += w.x, sum.y += w.y, sum.z += w.z, sum.w += w.w;
    }
    Finish(a, q, f, sum, total, !(total < 0.f));
  }
  if (thread == 0) {
    Note(a, q, most, total);
  }
}

// Weights of the rows: grid (groups of kWeightsThreads rows, KV heads, sequences). Bound by latency (16
// sequences of some 2000 rows, 8 KV heads of 4 query heads, 5 MB of scores: 7.4 us cold by itself).
constexpr int kWeightsThreads = 128;
__global__ void __launch_bounds__(kWeightsThreads)
WeightsKernel(const __grid_constant__ AttendArgs a, const __grid_constant__ BatchArgs batch) {
  GridLaunchDependents();
  GridDependencyWait();
  const CacheView& c = a.cache;
  const int kh = blockIdx.y;
  const BatchEntry& e = batch.of[blockIdx.z];
  const int position = batch.positions[e.index];
  int length = 0;
  for (int token = 0; token < e.tokens; ++token) {
    length = max(length, SeenBy(a, e, position, token));
  }
  const int row = blockIdx.x * kWeightsThreads + threadIdx.x;
  if (row >= length) {
    return;
  }
  float sum = 0.f;
  for (int token = 0; token < e.tokens; ++token) {
    if (row >= SeenBy(a, e, position, token)) {
      continue;
    }
    const int64_t first = (static_cast<int64_t>(e.row) + token) * a.heads + kh * a.group;
    for (int h = 0; h < a.group; ++h) {
      const float2 f = reinterpret_cast<const float2*>(a.finals)[first + h];
      sum += exp2f(__ldcs(a.scores + (first + h) * c.capacity + row) - f.x) * f.y;
    }
  }
  c.weights[(static_cast<size_t>(e.slot) * c.kv_heads + kh) * c.capacity + row] += sum;
}

// Scratch of the blocks of threads that a device holds at once, four an SM at most: two units'
// rows times dimensions, 8 rt * 64 ns with rt, ns <= 4 (two blocks an SM then; one half as large
// has three or four), and two statistics a row.
int Sms(const gufo_cuda_ctx* ctx) { return ctx->sm_count < kMostSms ? ctx->sm_count : kMostSms; }
constexpr size_t kPartialFloats = 2 * 2 * (32 * 256);     // of an SM
constexpr size_t kStatsFloats = 4 * 2 * (32 * 2);
// Items (groups of a sequence's query rows, each a unit for every KV head) that one launch takes: the
// cost of all its units is counted in an int (ShareOut; tiles of a block, and what a unit costs besides).
int MostItems(const gufo_cuda_cache8_config& c) {
  return static_cast<int>(INT32_MAX / (static_cast<int64_t>(c.kv_heads) * (c.capacity / kCacheBlock + 1 + kMostUnitRows / kCacheBlock)));
}
constexpr int kMostItemRows = 32;
size_t PartialBytes(int sms) { return static_cast<size_t>(sms) * ((kPartialFloats + kStatsFloats) * sizeof(float) + 4 * 32); }

template <typename Format, int NS, int RT, bool W, bool D>
int LaunchTiles(gufo_cuda_ctx* ctx, const AttendArgs& a, const BatchArgs& b, int grid) {
  using S = Shape<NS, RT>;
  static std::atomic<bool> configured[64];
  if (ctx->device >= 64 || !configured[ctx->device].load()) {
    GUFO_CUDA_TRY(cudaFuncSetAttribute(AttendKernel<Format, NS, RT, W, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    if (ctx->device < 64) {
      configured[ctx->device].store(true);
    }
  }
  GUFO_CUDA_TRY(LaunchOverlapped(AttendKernel<Format, NS, RT, W, D>, dim3(grid), dim3(kThreads), S::kBytes, ctx->stream,
                                 D ? 1 : a.ranks, a, b));
  ctx->launches.fetch_add(1);
  return GUFO_CUDA_OK;
}

template <typename Format, int NS, int RT, bool W>
int LaunchAttend(gufo_cuda_ctx* ctx, AttendArgs a, const BatchArgs& b, int64_t units, int rows) {
  using S = Shape<NS, RT>;
  const int blocks = Sms(ctx) * S::kBlocks;
  a.by_unit = units <= blocks;
  static_assert(S::kBlocks * 2 * 8 * RT * S::kRowBytes <= static_cast<int>(kPartialFloats) && S::kBlocks * 2 * 8 * RT * 2 <= static_cast<int>(kStatsFloats),
                "a block's parts fit the scratch");
  // Short caches: a block a unit, and nothing to be shared out or joined, where the longest unit takes no
  // longer than that: 384 rows (4 heads of 64 of 64 sequences of up to 333 rows: 9.0 us, 14.2 shared out; one
  // sequence of 500 rows, 2 heads of 256: 20.5, 10.9), more where there are units for two blocks in five at
  // least (64 sequences, 500 rows: 11.9, 15.2; 100 sequences, 1000 rows: 21.4, 22.9; 200 sequences, 2000 rows:
  // 66, 63; heads of 256, 128 sequences of 4, 500 rows: 27.9, 29.7; 1000 rows: 44.5, 40.9).
  const int short_capacity = units * 5 >= blocks * 2 ? (NS == 4 ? 512 : 1024) : 384;
  if (a.cache.capacity <= short_capacity) {
    a.ranks = 1;
    return LaunchTiles<Format, NS, RT, W, false>(ctx, a, b, static_cast<int>(units));
  }
  // Few units of some length: a cluster of blocks a unit, no second launch. (8 heads on 2 of 256, 500 rows: 7.0
  // us, 10.6 shared out; 1500: 10.9, 11.9; 1900: 12.8, 12.3. Heads of 128, 2000 rows: 10.3, 10.5; 3900: 15.7, 12.0.)
  if (a.cache.capacity <= (NS == 4 ? 1536 : 2048) && units * kRanks <= blocks) {
    a.ranks = kRanks;
    return LaunchTiles<Format, NS, RT, W, false>(ctx, a, b, static_cast<int>(units) * kRanks);
  }
  if (const int rc = LaunchTiles<Format, NS, RT, W, true>(ctx, a, b, blocks); rc != GUFO_CUDA_OK) {
    return rc;
  }
  const int cuts = a.by_unit ? static_cast<int>(units) : blocks;
  // Units of many parts: a block a row. (With three digits of int8 queries, one sequence of 131000 rows, 111
  // parts: 63 us, 86 with four rows a block; the verify batch of 8 sequences, 14 parts: 33, 38; of 32, 3: 73, 63.)
  if (std::min<int64_t>(blocks / units, a.cache.capacity / S::kTile) > 8) {
    GUFO_CUDA_TRY(LaunchOverlapped(JoinKernel<1>, dim3(cuts, rows), dim3(kJoinThreads), 0, ctx->stream, 1, a, 8 * RT));
  } else {
    GUFO_CUDA_TRY(LaunchOverlapped(JoinKernel<4>, dim3(cuts, (rows + 3) / 4), dim3(kJoinThreads), 0, ctx->stream, 1, a, 8 * RT));
  }
  ctx->launches.fetch_add(1);
  return GUFO_CUDA_OK;
}

template <typename Format, bool W>
int PickAttend(gufo_cuda_ctx* ctx, const AttendArgs& a, const BatchArgs& b, int64_t units, int rows, int ns, int rt) {
  switch (ns * 8 + rt) {
    case 8 + 1: return LaunchAttend<Format, 1, 1, W>(ctx, a, b, units, rows);
    case 8 + 2: return LaunchAttend<Format, 1, 2, W>(ctx, a, b, units, rows);
    case 8 + 4: return LaunchAttend<Format, 1, 4, W>(ctx, a, b, units, rows);
    case 16 + 1: return LaunchAttend<Format, 2, 1, W>(ctx, a, b, units, rows);
    case 16 + 2: return LaunchAttend<Format, 2, 2, W>(ctx, a, b, units, rows);
    case 16 + 4: return LaunchAttend<Format, 2, 4, W>(ctx, a, b, units, rows);
    case 32 + 1: return LaunchAttend<Format, 4, 1, W>(ctx, a, b, units, rows);
    case 32 + 2: return LaunchAttend<Format, 4, 2, W>(ctx, a, b, units, rows);
    default: return LaunchAttend<Format, 4, 4, W>(ctx, a, b, units, rows);
  }
}

}  // namespace
}  // namespace gufo

using gufo::Fail;

extern "C" {

int gufo_cuda_cache8_attend_scratch(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, int heads, int tokens, int accumulate,
                                    size_t* bytes) {
  if (ctx == nullptr || bytes == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_attend_scratch: null pointer");
  }
  if (heads < 1 || heads > 65536 || tokens < 0) {
    return Fail(GUFO_CUDA_SHAPE, "cache8_attend_scratch: 1 to 65536 heads, and no negative number of tokens");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  if (const int rc = gufo::FindCache(ctx, handle, "cache8_attend_scratch", &cache); rc != GUFO_CUDA_OK) {
    return rc;
  }
  const size_t rows = static_cast<size_t>(heads) * tokens;
  // (However the tokens are spread over the cache's sequences.)
  const int64_t group = heads > cache->c.kv_heads ? heads / cache->c.kv_heads : 1;
  const int64_t each = static_cast<int64_t>(gufo::MostItems(cache->c)) * gufo::kMostItemRows / group;
  if ((each < cache->c.capacity && tokens > each * cache->c.sequences) ||
      (accumulate != 0 && rows > (static_cast<size_t>(1) << 48) / cache->c.capacity)) {
    return Fail(GUFO_CUDA_TOO_LARGE, "cache8_attend_scratch: too many query rows for one call");
  }
  *bytes = gufo::PartialBytes(gufo::Sms(ctx)) + (accumulate != 0 ? rows * (2 + static_cast<size_t>(cache->c.capacity)) * 4 : 0);
  return GUFO_CUDA_OK;
}

int gufo_cuda_cache8_attend_device(gufo_cuda_ctx* ctx, gufo_cuda_cache8 handle, const gufo_cuda_cache8_batch* batch,
                                   const gufo_cuda_cache8_attend_args* p) {
  if (ctx == nullptr || p == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_attend: null pointer");
  }
  std::lock_guard<std::mutex> lock(ctx->mu);
  const gufo::Cache8* cache = nullptr;
  int64_t tokens = 0;
  int rc = gufo::FindCache(ctx, handle, "cache8_attend", &cache);
  if (rc == GUFO_CUDA_OK) {
    rc = gufo::CheckBatch(*cache, batch, "cache8_attend", true, &tokens);
  }
  if (rc != GUFO_CUDA_OK) {
    return rc;
  }
  const gufo_cuda_cache8_config& c = cache->c;
  if (p->heads < 1 || p->heads > 65536 || p->heads % c.kv_heads != 0) {
    return Fail(GUFO_CUDA_SHAPE, "cache8_attend: heads is a multiple of the cache's KV heads, 65536 at most");
  }
  if (p->accumulate != 0 && cache->weights == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_attend: the cache keeps no weights");
  }
  if (tokens == 0) {
    return GUFO_CUDA_OK;
  }
  if (p->queries == nullptr || p->out == nullptr || p->scratch == nullptr) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_attend: null pointer");
  }
  const size_t rows = static_cast<size_t>(p->heads) * tokens;
  const size_t own = gufo::PartialBytes(gufo::Sms(ctx));
  if (p->accumulate != 0 && rows > (static_cast<size_t>(1) << 48) / c.capacity) {
    return Fail(GUFO_CUDA_TOO_LARGE, "cache8_attend: too many query rows for one call");
  }
  const size_t want = own + (p->accumulate != 0 ? rows * (2 + static_cast<size_t>(c.capacity)) * 4 : 0);
  if (p->scratch_bytes < want || reinterpret_cast<uintptr_t>(p->scratch) % 16 != 0) {
    return Fail(GUFO_CUDA_BAD_ARGUMENT, "cache8_attend: " + std::to_string(want) + " bytes of scratch on a 16-byte boundary");
  }
  gufo::AttendArgs a{};
  a.cache = gufo::ViewOf(*cache);
  a.queries = p->queries;
  a.query_token_stride = p->query_token_stride;
  a.query_head_stride = p->query_head_stride;
  a.gate = p->gate;
  a.gate_token_stride = p->gate_token_stride;
  a.gate_head_stride = p->gate_head_stride;
  a.out = p->out;
  a.out_token_stride = p->out_token_stride;
  a.out_head_stride = p->out_head_stride;
  a.visible = p->visible;
  a.heads = p->heads;
  a.group = p->heads / c.kv_heads;
  a.scale = (p->scale != 0.f ? p->scale : 1.0f / sqrtf(static_cast<float>(c.head_dim))) * gufo::kLog2e;
  a.whole = ((reinterpret_cast<uintptr_t>(p->queries) | reinterpret_cast<uintptr_t>(p->gate) | reinterpret_cast<uintptr_t>(p->out)) & 15) == 0 &&
            ((p->query_token_stride | p->query_head_stride | p->gate_token_stride | p->gate_head_stride | p->out_token_stride |
              p->out_head_stride) & 3) == 0;
  uint8_t* scratch = static_cast<uint8_t*>(p->scratch);
  a.sums = reinterpret_cast<float*>(scratch);
  if (p->accumulate != 0) {
    a.finals = reinterpret_cast<float*>(scratch + own);
    a.scores = a.finals + 2 * rows;
  }
  // Query rows of an item: as few groups of eight as hold a sequence's, four at most.
  const int ns = c.head_dim <= 64 ? 1 : c.head_dim <= 128 ? 2 : 4;
  int most = 1;
  for (int i = 0; i < batch->sequences; ++i) {
    const int n = batch->tokens != nullptr ? batch->tokens[i] : 1;
    most = n > most ? n : most;
  }
  const int64_t rows_each = static_cast<int64_t>(most) * a.group;
  a.stats = a.sums + static_cast<size_t>(gufo::Sms(ctx)) * gufo::kPartialFloats;
  a.cuts = reinterpret_cast<gufo::Cut*>(a.stats + static_cast<size_t>(gufo::Sms(ctx)) * gufo::kStatsFloats);
  static_assert(sizeof(gufo::Cut) <= 32, "the scratch has 32 bytes a block for it");
  const int rt = rows_each <= 8 ? 1 : rows_each <= 16 ? 2 : 4;
  static_assert(8 * 4 == gufo::kMostItemRows, "of the largest rt");
  // (The longest sequence's: the others of a batch go to a launch of their own where they are too many together.)
  const int most_items = gufo::MostItems(c);
  if ((rows_each + 8 * rt - 1) / (8 * rt) > most_items) {
    return Fail(GUFO_CUDA_TOO_LARGE, "cache8_attend: too many query rows of one sequence");
  }
  GUFO_CUDA_TRY(cudaSetDevice(ctx->device));
  const int group = a.group;
  return gufo::ForEachRun(
      *batch, [&](int n) { return static_cast<int>((static_cast<int64_t>(n) * group + 8 * rt - 1) / (8 * rt)); },
      [&](const gufo::BatchArgs& b, int items) -> int {
        const int64_t units = static_cast<int64_t>(items) * c.kv_heads;
        const int rows = rows_each < 8 * rt ? static_cast<int>(rows_each) : 8 * rt;
        const bool e4m3 = c.format == GUFO_CUDA_CACHE8_E4M3;
        const int run = a.scores != nullptr ? (e4m3 ? gufo::PickAttend<gufo::E4m3, true>(ctx, a, b, units, rows, ns, rt)
                                                    : gufo::PickAttend<gufo::Int8, true>(ctx, a, b, units, rows, ns, rt))
                                            : (e4m3 ? gufo::PickAttend<gufo::E4m3, false>(ctx, a, b, units, rows, ns, rt)
                                                    : gufo::PickAttend<gufo::Int8, false>(ctx, a, b, units, rows, ns, rt));
        if (run != GUFO_CUDA_OK || a.scores == nullptr) {
          return run;
        }
        GUFO_CUDA_TRY(gufo::LaunchOverlapped(gufo::WeightsKernel,
                                             dim3((c.capacity + gufo::kWeightsThreads - 1) / gufo::kWeightsThreads, c.kv_heads,
                                                  b.sequences),
                                             dim3(gufo::kWeightsThreads), 0, ctx->stream, 1, a, b));
        ctx->launches.fetch_add(1);
        return GUFO_CUDA_OK;
      },
      most_items);
}

}  // extern "C"
