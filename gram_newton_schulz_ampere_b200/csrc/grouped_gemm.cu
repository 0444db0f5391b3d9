// Matrix products grouped by expert, with ragged groups of rows, on tcgen05.
//
//   rows product     out[r]  = left[r] . right[e]          for the rows r of expert e
//   reduced product  out[e]  = left[rows of e]^T . right[rows of e]
//
// Rows are sorted by expert: expert e owns the rows [end[e - 1], end[e]). The ends
// are read on the device, so routing needs no host synchronisation; they are
// clamped to [0, rows] and to ascending order, so no value of them leads out of
// the buffers. Rows past the last end belong to nobody and come out zero.
//
// Both are persistent, warp-specialised kernels of the same shape: warp 0 loads
// tiles with TMA into a ring of 128-byte-swizzled stages, lane 0 of warp 1 issues
// tcgen05.mma into one of two TMEM accumulators, warps 2..9 empty the other.
// PAIR: a cluster of two CTAs shares a 256-row MMA (cta_group::2).
//
// Rows product: the MMA's M side is the expert's matrix (128 or 256 of its output
// columns, the "features") and its N side is the expert's rows. N is a run-time
// field of the instruction, so a group of 40 rows costs a 48- or 64-wide MMA
// instead of a 128-row tile, and a group is cut into equal parts rather than full
// tiles and a remainder. The accumulator is the transpose of the output tile and
// is turned while it is staged. A tile may load rows of the next group; they only
// fill other columns of the accumulator, which are not stored.
//
// Reduced product: the rows are the contraction, so rows of other groups must not
// enter. A group's last 64 rows may reach into the next group: only the 16-row steps
// with rows of the group are multiplied, and the foreign rows of the last step are
// zeroed in shared memory (in both operands: a NaN times zero is a NaN) by a warp
// of its own between the loads and the MMA. A tile's contraction is not cut, so few
// tiles over many rows leave SMs idle (2 groups of 16384 rows, 64 x 64: 99 us for 8 MB).
//
// Few tiles with a long contraction: a cluster of up to 8 CTAs shares a tile, each
// with a part of the contraction, and adds up the fp32 partial sums out of the CTAs'
// shared memory in the order of the parts.
//
// Sums are fp32 in TMEM, rounded once at the store. Every wait is bounded.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"
#include "staging.cuh"

namespace gns {
namespace {

__device__ int g_grouped_status = 0;

constexpr int kMaxGroups = 1024;
constexpr int kBK = 64;   // contraction per stage: 128 bytes of a 16-bit type
constexpr int kBM = 128;  // rows of the MMA's M side per CTA
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr uint32_t kMBytes = kBM * kBK * 2;

struct Groups {
  const void* ends;
  int ends64;
  int count;
  int rows;
};

__device__ __forceinline__ int64_t group_end(const Groups& g, int e) {
  return g.ends64 ? static_cast<const int64_t*>(g.ends)[e] : static_cast<int64_t>(static_cast<const int32_t*>(g.ends)[e]);
}

// Row ranges of the 32 groups of a warp's lanes: ends clamped to [0, rows] and to the
// largest end before them (`carry`, updated for the next 32).
__device__ __forceinline__ void group_rows(int64_t value, int rows, int lane, int& carry, int& begin, int& end) {
  end = static_cast<int>(value < 0 ? 0 : (value > rows ? rows : value));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, end, o);
    if (lane >= o) end = max(end, other);
  }
  end = max(end, carry);
  begin = __shfl_up_sync(0xffffffffu, end, 1);
  if (lane == 0) begin = carry;
  carry = __shfl_sync(0xffffffffu, end, 31);
}

__device__ __forceinline__ int inclusive_sum(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += other;
  }
  return v;
}

// A group of `rows` rows is cut into `parts` parts of `size` rows (the last may be
// shorter): as few as the tile allows, equal up to the MMA's granularity.
struct Cut {
  int parts, size;
};

__device__ __forceinline__ Cut cut_group(int rows, int tile, int unit) {
  if (rows <= tile) return {rows > 0 ? 1 : 0, (rows + unit - 1) / unit * unit};
  const unsigned least = (rows + tile - 1) / tile;
  const int size = static_cast<int>((rows + least - 1) / least + unit - 1) / unit * unit;
  return {static_cast<int>(static_cast<unsigned>(rows + size - 1) / static_cast<unsigned>(size)), size};
}

// The groups as a CTA works through them, in shared memory: place i holds group
// order[i], whose tiles follow first_tile[i]. Where the tiles take more than one turn
// of the persistent grid, groups with costly tiles come first. The tiles are dealt to
// the CTAs in turn, so the sums of the shares then differ by less than one tile, and
// the tiles of the last, partial turn are the cheap ones. (In the groups' own order
// the busiest CTA pair of a ragged batch had about a quarter more than the mean.)
struct Table {
  int* first_row;   // [count + 1], by group
  int* first_tile;  // [count + 1], by place
  int* parts;       // [count], by group
  uint16_t* size;   // [count], by group: rows of a part
  uint16_t* order;  // [count], by place
  int* counts;      // [32]: scratch of the sort
  static constexpr uint32_t kBytes = 2 * (kMaxGroups + 1) * 4 + kMaxGroups * 8 + 32 * 4;

  __device__ __forceinline__ explicit Table(uint8_t* at)
      : first_row(reinterpret_cast<int*>(at)),
        first_tile(first_row + kMaxGroups + 1),
        parts(first_tile + kMaxGroups + 1),
        size(reinterpret_cast<uint16_t*>(parts + kMaxGroups)),
        order(size + kMaxGroups),
        counts(reinterpret_cast<int*>(order + kMaxGroups)) {}

  __device__ __forceinline__ int rows(int e) const { return first_row[e + 1] - first_row[e]; }
};

// One warp fills the table. cut(rows) gives a group's parts, each of `per_part` tiles,
// and their size; cost(rows, size) the cost of its tiles, in [0, 31].
template <class CutFn, class Cost>
__device__ __forceinline__ void fill_table(const Table& table, const Groups& groups, int lane, int workers,
                                           int per_part, CutFn cut, Cost cost) {
  constexpr int kAhead = 4;  // ends that a lane loads at once
  int carry = 0, before = 0;
  for (int base = 0; base < groups.count; base += 32 * kAhead) {
    int64_t value[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int e = base + 32 * q + lane;
      value[q] = e < groups.count ? group_end(groups, e) : 0;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int e = base + 32 * q + lane;
      if (e - lane >= groups.count) break;
      int begin, end;
      group_rows(value[q], groups.rows, lane, carry, begin, end);
      const Cut c = cut(end - begin);
      const int tiles = e < groups.count ? c.parts * per_part : 0;
      const int sum = inclusive_sum(tiles, lane);
      if (e < groups.count) {
        table.first_row[e] = begin;
        table.parts[e] = c.parts;
        table.size[e] = static_cast<uint16_t>(c.size);
        table.order[e] = static_cast<uint16_t>(e);
        table.first_tile[e] = before + sum - tiles;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  if (lane == 0) {
    table.first_row[groups.count] = carry;
    table.first_tile[groups.count] = before;
  }
  table.counts[lane] = 0;
  __syncwarp();
  if (before <= workers) return;
  // A counting sort: the groups of each cost are counted, then placed behind the
  // costlier ones.
  for (int base = 0; base < groups.count; base += 32) {
    const int e = base + lane;
    const int c = e < groups.count ? cost(table.rows(e), table.size[e]) : 32;
    const uint32_t same = __match_any_sync(0xffffffffu, c);
    if (c < 32 && lane == __ffs(same) - 1) table.counts[c] += __popc(same);
    __syncwarp();
  }
  const int with_cost = table.counts[lane];
  int place = with_cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_down_sync(0xffffffffu, place, o);
    if (lane + o < 32) place += other;
  }
  table.counts[lane] = place - with_cost;  // the costlier groups
  __syncwarp();
  for (int base = 0; base < groups.count; base += 32) {
    const int e = base + lane;
    const int c = e < groups.count ? cost(table.rows(e), table.size[e]) : 32;
    const uint32_t same = __match_any_sync(0xffffffffu, c);
    const int at = c < 32 ? table.counts[c] : 0;
    __syncwarp();
    if (c < 32) {
      table.order[at + __popc(same & ((1u << lane) - 1u))] = static_cast<uint16_t>(e);
      if (lane == __ffs(same) - 1) table.counts[c] = at + __popc(same);
    }
    __syncwarp();
  }
  before = 0;
  for (int base = 0; base < groups.count; base += 32) {
    const int i = base + lane;
    const int tiles = i < groups.count ? table.parts[table.order[i]] * per_part : 0;
    const int sum = inclusive_sum(tiles, lane);
    if (i < groups.count) table.first_tile[i] = before + sum - tiles;
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}

struct Output {
  void* d;
  int64_t ldd, bstride;
  int bf16;  // 16-bit outputs: 1 = bf16, 0 = fp16
  int vec;   // base, row and group strides are multiples of 16 bytes
  int linear;  // reduced product: rows and groups follow one another without gaps
};

// One whole 32 x 32 block of a staging slot to rows [r0, r0 + live) of the output.
template <bool OUT_F32>
__device__ __forceinline__ void store_rows(const uint8_t* slot, const Output& out, int64_t at, int live, int cols_left,
                                           int lane) {
  constexpr int kPieces = OUT_F32 ? 8 : 4;
  constexpr int kElems = OUT_F32 ? 4 : 8;
  constexpr int kRows = 32 / kPieces;
  constexpr int es = OUT_F32 ? 4 : 2;
  uint8_t* d = static_cast<uint8_t*>(out.d);
  if (out.vec && cols_left >= 32) {
    const int pc = lane % kPieces;
#pragma unroll
    for (int pass = 0; pass < 32 / kRows; ++pass) {
      const int r = pass * kRows + lane / kPieces;
      if (r < live)
        *reinterpret_cast<uint4*>(d + (at + r * out.ldd + pc * kElems) * es) =
            *reinterpret_cast<const uint4*>(slot + stage_off<OUT_F32>(static_cast<uint32_t>(r), 16u * pc));
    }
    return;
  }
  // Blocks on the right edge and outputs without aligned rows: lane = column.
  if (lane >= cols_left) return;
#pragma unroll 8
  for (int r = 0; r < live; ++r) {
    const int64_t i = at + r * out.ldd + lane;
    if (OUT_F32)
      static_cast<uint32_t*>(out.d)[i] = *reinterpret_cast<const uint32_t*>(slot + stage_off<true>(r, 4u * lane));
    else
      static_cast<uint16_t*>(out.d)[i] = *reinterpret_cast<const uint16_t*>(slot + stage_off<false>(r, 2u * lane));
  }
}

// Zeros in `bytes` bytes (an even number) from p on, by thread `id` of `threads`.
__device__ __forceinline__ void zero_fill(uint8_t* p, int64_t bytes, int id, int threads) {
  const int64_t head = min(bytes, static_cast<int64_t>((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u));
  const int64_t words = (bytes - head) / 16;
  for (int64_t i = 2 * id; i < head; i += 2 * threads) *reinterpret_cast<uint16_t*>(p + i) = 0;
  for (int64_t i = id; i < words; i += threads) *reinterpret_cast<uint4*>(p + head + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = head + 16 * words + 2 * id; i < bytes; i += 2 * threads) *reinterpret_cast<uint16_t*>(p + i) = 0;
}

// A lane's 32 accumulators rounded to the output type.
template <bool OUT_F32>
__device__ __forceinline__ void round_row(const float (&v)[32], int bf16, XRow<OUT_F32>& x) {
  if (OUT_F32) {
#pragma unroll
    for (int q = 0; q < 32; ++q) x.w[q % (OUT_F32 ? 32 : 16)] = __float_as_uint(v[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 32; q += 2) x.w[q >> 1] = pack_pair(v[q], v[q + 1], bf16);
  }
}

// ----------------------------------------------------------- barrier plumbing
// full / empty of each stage and of each accumulator; in a pair the full and the
// accumulator-empty barriers of CTA 0 serve both CTAs.
template <int S, bool PAIR>
struct Barriers {
  uint64_t* full;
  uint64_t* empty;
  uint64_t* tfull;
  uint64_t* tempty;
  uint64_t* tail;  // reduced product: a stage whose rows end inside it has landed in this CTA
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  static constexpr uint32_t kBytes = (3 * S + 4) * 8 + 8;

  __device__ __forceinline__ explicit Barriers(uint8_t* at) {
    full = reinterpret_cast<uint64_t*>(at);
    empty = full + S;
    tfull = full + 2 * S;
    tempty = full + 2 * S + 2;
    tail = full + 2 * S + 4;
    tmem_slot = reinterpret_cast<uint32_t*>(tail + S);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }

  __device__ __forceinline__ void init(uint32_t full_arrivals) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], full_arrivals);
      mbar_init(&empty[s], 1);
      mbar_init(&tail[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (PAIR ? 2 : 1) * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
};

template <bool CLUSTER>
__device__ __forceinline__ void meet() {
  if (CLUSTER)
    cluster_sync_all();
  else
    __syncthreads();
}

// Set-up common to both kernels: barriers, TMEM, and the wait for the stream's
// previous kernel. Returns the TMEM base.
template <int S, bool PAIR, bool CLUSTER = PAIR>
__device__ __forceinline__ uint32_t set_up(const Barriers<S, PAIR>& bar, int warp, uint32_t tmem_cols,
                                           uint32_t full_arrivals = 1) {
  if (threadIdx.x == 0) const_cast<Barriers<S, PAIR>&>(bar).init(full_arrivals);
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(bar.tmem_slot, tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(bar.tmem_slot, tmem_cols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  meet<CLUSTER>();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_predecessor();
  return *bar.tmem_slot;
}

// The producer's end: it waits until every stage it filled has been released. In a
// pair the releases of CTA 1's stages are arrivals that CTA 0's MMAs send when they
// complete; none may be on its way when the CTA leaves and its shared memory goes to
// another.
template <int S, bool PAIR>
__device__ __forceinline__ void drain(const Barriers<S, PAIR>& bar, int st, uint32_t ph, bool ok) {
  for (int i = 0; i < S && ok; ++i) {
    ok = mbar_wait_bounded(&bar.empty[st], ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusProducerTimeout);
    if (++st == S) {
      st = 0;
      ph ^= 1u;
    }
  }
}

// Teardown: all roles meet; after an abort, copies and MMAs in flight get time to
// land before TMEM and shared memory are released.
template <int S, bool PAIR, bool CLUSTER = PAIR>
__device__ __forceinline__ void tear_down(const Barriers<S, PAIR>& bar, int warp, uint32_t tmem_base,
                                          uint32_t tmem_cols) {
  tc_fence_before();
  meet<CLUSTER>();
  if (*bar.abort_flag) settle_for_ns(2000000ull);
  meet<CLUSTER>();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    if (PAIR)
      tmem_dealloc_pair(tmem_base, tmem_cols);
    else
      tmem_dealloc(tmem_base, tmem_cols);
  }
}

// ------------------------------------------------------------- rows product
struct RowsShape {
  int n, k_blocks, feature_tiles;
};

// Maps of the row operand with boxes of 32, 64, 96 and 128 rows: a part of any
// width comes with one copy a stage (several small boxes instead cost up to 8%).
struct RowMaps {
  CUtensorMap box[4];
};

// A tile's rows lie in one or two units of at most 256 columns of the accumulator,
// and the unit buffers are used in turn. TOK = 512: both units of a tile share the
// loads of the expert's columns.
//
// SPLIT: a tile belongs to a cluster of 2, 4 or 8 CTAs, each of which multiplies an
// equal share of the contraction (the join below).
template <int TOK, bool OUT_F32, bool PAIR, bool SPLIT>
struct RowsConfig {
  static_assert(!SPLIT || (TOK == 64 && !PAIR), "a split tile has one block of 32 x 32 accumulators a warp");
  static constexpr int kUnits = TOK > 256 ? 2 : 1;
  static constexpr int kUnitCols = TOK / kUnits;
  static constexpr int kFeatures = PAIR ? 2 * kBM : kBM;             // features of a tile
  static constexpr int kUnitRows = PAIR ? kUnitCols / 2 : kUnitCols;  // rows of a unit that one CTA loads, at most
  static constexpr int kGrain = PAIR ? 32 : 16;                       // granularity of N
  static constexpr uint32_t kUnitBytes = kUnitRows * kBK * 2;
  static constexpr uint32_t kStageBytes = kMBytes + kUnits * kUnitBytes;
  static constexpr int kStages = 6 * 32768 / kStageBytes - (OUT_F32 || SPLIT ? 1 : 0);
  static constexpr uint32_t kSlotBytes = 32 * (OUT_F32 || SPLIT ? 128 : 64);
  static constexpr uint32_t kJoinBytes = SPLIT ? 2 * kEpiWarps * 8 : 0;
  static constexpr uint32_t kTmemCols = 2 * kUnitCols;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes + Table::kBytes +
                                       Barriers<kStages, PAIR>::kBytes + kJoinBytes;
};

// A tile: `rows` rows from `row0` of group e, feature tile `f`.
struct RowsTile {
  int e, row0, rows, f;
};

__device__ __forceinline__ RowsTile rows_tile(const Table& table, int count, int t, int& place) {
  // Mostly the next tile is of the same place or the next one; else it is searched for.
  if (t >= table.first_tile[place + 1] && t >= table.first_tile[++place + 1]) {
    int hi = count - 1;
    while (place < hi) {
      const int mid = (place + hi + 1) >> 1;
      if (table.first_tile[mid] <= t)
        place = mid;
      else
        hi = mid - 1;
    }
  }
  RowsTile tile;
  tile.e = table.order[place];
  const int parts = table.parts[tile.e], size = table.size[tile.e];
  const int l = t - table.first_tile[place];
  tile.f = l / parts;  // a group's row parts are neighbours: they share the expert's columns in L2
  const int part = l - tile.f * parts;
  tile.row0 = table.first_row[tile.e] + part * size;
  tile.rows = min(size, table.first_row[tile.e + 1] - tile.row0);
  return tile;
}

// Rows of the tile's first unit: all of them if a unit holds them, else half (an
// MMA of a narrow remainder would wait for its other operand's shared memory reads).
template <class Cfg>
__device__ __forceinline__ int first_unit(const RowsTile& tile) {
  if (tile.rows <= Cfg::kUnitCols) return tile.rows;
  return ((tile.rows + 1) / 2 + Cfg::kGrain - 1) / Cfg::kGrain * Cfg::kGrain;
}

// N of the MMA for `rows` rows.
template <class Cfg>
__device__ __forceinline__ int mma_width(int rows) {
  return (rows + Cfg::kGrain - 1) / Cfg::kGrain * Cfg::kGrain;
}

// The join of a split tile, by one warp of each CTA of the cluster: the same 32 x 32
// block of all partial accumulators. The warp leaves its own in its slot (fp32, row =
// row of the output), tells the others, and adds up every size-th stretch of four rows
// from all slots, always in the order of the CTAs. `there` counts the CTAs whose
// partial is in place, `read` those that have read this CTA's.
struct Join {
  uint64_t* there;
  uint64_t* read;
  uint32_t phase, rank, size;

  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) const {
    return __all_sync(0xffffffffu,
                      mbar_wait_bounded<true>(bar, parity, abort_flag, &g_grouped_status, kStatusEpilogueTimeout));
  }

  // After every lane's accesses of the slots.
  __device__ __forceinline__ void tell(uint64_t* bar, int lane) const {
    __syncwarp();
    if (lane < static_cast<int>(size)) mbar_arrive_release_cluster(cluster_addr(bar, static_cast<uint32_t>(lane)));
  }

  // Sums are told as read before they are stored: a release waits for earlier stores.
  template <bool OUT_F32>
  __device__ __forceinline__ void add_up(const uint8_t* slot, const Output& out, int64_t at, int live, int cols_left,
                                         int lane) const {
    const int piece = lane % 8, first = 4 * static_cast<int>(rank) + lane / 8, step = 4 * static_cast<int>(size);
    float4 sum[4];  // a cluster has two CTAs at least
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      sum[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const int r = first + q * step;
      if (r >= live) continue;
      const uint32_t off = stage_off<true>(static_cast<uint32_t>(r), 16u * piece);
#pragma unroll 4
      for (uint32_t c = 0; c < size; ++c) {
        float4 p;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w)
                     : "r"(cluster_addr(slot, c) + off)
                     : "memory");
        sum[q] = make_float4(sum[q].x + p.x, sum[q].y + p.y, sum[q].z + p.z, sum[q].w + p.w);
      }
    }
    tell(read, lane);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = first + q * step;
      if (r >= live) continue;
      const int64_t i = at + r * out.ldd + 4 * piece;
      const int left = cols_left - 4 * piece;
      const float v[4] = {sum[q].x, sum[q].y, sum[q].z, sum[q].w};
      if (OUT_F32) {
        float* d = static_cast<float*>(out.d) + i;
        if (out.vec && left >= 4) {
          *reinterpret_cast<float4*>(d) = sum[q];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < left) d[k] = v[k];
        }
      } else {
        uint16_t* d = static_cast<uint16_t*>(out.d) + i;
        if (out.vec && left >= 4) {
          *reinterpret_cast<uint2*>(d) = make_uint2(pack_pair(v[0], v[1], out.bf16), pack_pair(v[2], v[3], out.bf16));
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < left) d[k] = float_to_half_bits(v[k], out.bf16);
        }
      }
    }
  }
};

template <bool F_MN, int TOK, bool OUT_F32, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_rows_kernel(const __grid_constant__ CUtensorMap map_right, const __grid_constant__ RowMaps map_rows,
                        const Groups groups, const RowsShape shape, const Output out, const int ab_bf16) {
  using Cfg = RowsConfig<TOK, OUT_F32, PAIR, SPLIT>;
  constexpr int S = Cfg::kStages;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int ctas = PAIR ? 2 : (SPLIT ? static_cast<int>(cluster_nctarank()) : 1);  // of a tile
  const int tile_begin = static_cast<int>(blockIdx.x) / ctas;
  const int tile_step = static_cast<int>(gridDim.x) / ctas;
  // This CTA's share of the contraction.
  const int share = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const int kb_begin = SPLIT ? share * shape.k_blocks / ctas : 0;
  const int kb_end = SPLIT ? (share + 1) * shape.k_blocks / ctas : shape.k_blocks;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_m = smem;
  uint8_t* smem_n = smem + S * kMBytes;
  uint8_t* smem_epi = smem + S * Cfg::kStageBytes;
  const Barriers<S, PAIR> bar(smem_epi + kEpiWarps * Cfg::kSlotBytes);
  uint64_t* join = reinterpret_cast<uint64_t*>(smem_epi + kEpiWarps * Cfg::kSlotBytes + Barriers<S, PAIR>::kBytes);
  const Table table(smem_epi + kEpiWarps * Cfg::kSlotBytes + Barriers<S, PAIR>::kBytes + Cfg::kJoinBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_right);
    for (int i = 0; i < Cfg::kUnitRows / 32; ++i) tma_prefetch_desc(&map_rows.box[i]);
    if (SPLIT)
      for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(&join[i], static_cast<uint32_t>(ctas));
  }
  const uint32_t tmem_base = set_up<S, PAIR, PAIR || SPLIT>(bar, warp, Cfg::kTmemCols);

  // A tile's cost is its rows.
  if (warp == 0)
    fill_table(
        table, groups, lane, tile_step, shape.feature_tiles, [](int rows) { return cut_group(rows, TOK, Cfg::kGrain); },
        [](int, int size) { return size * 31 / TOK; });
  __syncthreads();
  const int tiles = table.first_tile[groups.count];

  if (warp == 0) {
    if (lane == 0) {
      int st = 0, place = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = PAIR ? cluster_addr(&bar.full[0], 0) : 0u;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const RowsTile tile = rows_tile(table, groups.count, t, place);
        const int f0 = tile.f * Cfg::kFeatures + static_cast<int>(rank) * kBM;
        const int split = first_unit<Cfg>(tile);
        // This CTA's rows of each unit, and the smallest box that holds them.
        int row[2], box[2];
        uint32_t bytes = kMBytes;
#pragma unroll
        for (int u = 0; u < Cfg::kUnits; ++u) {
          const int width = mma_width<Cfg>(u == 0 ? split : tile.rows - split);
          const int mine = PAIR ? width / 2 : width;
          row[u] = tile.row0 + u * split + static_cast<int>(rank) * mine;
          box[u] = (mine + 31) / 32;
          bytes += static_cast<uint32_t>(box[u]) * 32u * kBK * 2u;
        }
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_wait_bounded(&bar.empty[st], ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusProducerTimeout)) {
            ok = false;
            break;
          }
          const int k0 = kb * kBK;
          uint8_t* sm = smem_m + st * kMBytes;
          uint8_t* sn = smem_n + st * Cfg::kUnits * Cfg::kUnitBytes;
          if (PAIR) {
            if (rank == 0) mbar_arrive_expect_tx(&bar.full[st], 2 * bytes);
            const uint32_t fb = full0 + static_cast<uint32_t>(st) * 8u;
            if (!F_MN) {
              tma_load_3d_pair(sm, &map_right, fb, k0, f0, tile.e);
            } else {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c) tma_load_3d_pair(sm + c * 8192, &map_right, fb, f0 + 64 * c, k0, tile.e);
            }
#pragma unroll
            for (int u = 0; u < Cfg::kUnits; ++u)
              if (box[u] > 0)
                tma_load_3d_pair(sn + u * Cfg::kUnitBytes, &map_rows.box[box[u] - 1], fb, k0, row[u], 0);
          } else {
            mbar_arrive_expect_tx(&bar.full[st], bytes);
            if (!F_MN) {
              tma_load_3d(sm, &map_right, &bar.full[st], k0, f0, tile.e);
            } else {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c) tma_load_3d(sm + c * 8192, &map_right, &bar.full[st], f0 + 64 * c, k0, tile.e);
            }
#pragma unroll
            for (int u = 0; u < Cfg::kUnits; ++u)
              if (box[u] > 0)
                tma_load_3d(sn + u * Cfg::kUnitBytes, &map_rows.box[box[u] - 1], &bar.full[st], k0, row[u], 0);
          }
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
      drain<S, PAIR>(bar, st, ph, ok);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint64_t desc_k = make_smem_desc_sw128(0, 16, 1024);
      const uint64_t desc_t = make_smem_desc_sw128(0, 8192, 1024);
      const uint32_t empty0 = PAIR ? cluster_addr(&bar.empty[0], 0) : 0u;
      const uint32_t empty1 = PAIR ? cluster_addr(&bar.empty[0], 1) : 0u;
      const uint32_t tfull0 = PAIR ? cluster_addr(&bar.tfull[0], 0) : 0u;
      const uint32_t tfull1 = PAIR ? cluster_addr(&bar.tfull[0], 1) : 0u;
      auto hand_over = [&](int b) {
        if (PAIR) {
          tc_commit_pair(tfull0 + static_cast<uint32_t>(b) * 8u);
          tc_commit_pair(tfull1 + static_cast<uint32_t>(b) * 8u);
        } else {
          tc_commit(&bar.tfull[b]);
        }
      };
      int st = 0, place = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const RowsTile tile = rows_tile(table, groups.count, t, place);
        const int split = first_unit<Cfg>(tile);
        int units = 0, buffer[2];
        uint32_t idesc[2];
#pragma unroll
        for (int u = 0; u < Cfg::kUnits; ++u) {
          const int width = mma_width<Cfg>(u == 0 ? split : tile.rows - split);
          if (width == 0 || !ok) continue;
          idesc[u] = make_idesc_f16(ab_bf16, F_MN ? 1 : 0, 0, Cfg::kFeatures, width);
          ok = mbar_wait_bounded(&bar.tempty[acc], acc_ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout);
          buffer[u] = acc;
          units = u + 1;
          acc ^= 1;
          if (acc == 0) acc_ph ^= 1u;
        }
        if (!ok) break;
        tc_fence_after();
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_wait_bounded(&bar.full[st], ph, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t m0 = (F_MN ? desc_t : desc_k) + ((smem_u32(smem_m + st * kMBytes) >> 4) & 0x3FFFu);
#pragma unroll
          for (int u = 0; u < Cfg::kUnits; ++u) {
            if (u > 0 && u >= units) continue;
            const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(buffer[u] * Cfg::kUnitCols);
            const uint64_t n0 =
                desc_k + ((smem_u32(smem_n + (st * Cfg::kUnits + u) * Cfg::kUnitBytes) >> 4) & 0x3FFFu);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk) {
              const uint32_t more = (kb > kb_begin || kk > 0) ? 1u : 0u;
              if (PAIR)
                tc_mma_f16_pair(d_tmem, m0 + kk * (F_MN ? 128u : 2u), n0 + kk * 2u, idesc[u], more);
              else
                tc_mma_f16(d_tmem, m0 + kk * (F_MN ? 128u : 2u), n0 + kk * 2u, idesc[u], more);
            }
            // The first unit of two is handed over as soon as its last products are issued.
            if (u + 1 < Cfg::kUnits && u + 1 < units && kb + 1 == kb_end) hand_over(buffer[u]);
          }
          if (PAIR) {
            tc_commit_pair(empty0 + static_cast<uint32_t>(st) * 8u);
            tc_commit_pair(empty1 + static_cast<uint32_t>(st) * 8u);
          } else {
            tc_commit(&bar.empty[st]);
          }
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
        // Last of the tile's commits, so that a CTA whose epilogue has seen it has seen
        // every earlier arrival on its barriers.
        if (ok) hand_over(buffer[units - 1]);
      }
    }
  } else {
    const int ew = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    const int half = ew >> 2;      // even (0) or odd (1) blocks of 32 rows
    uint8_t* slot = smem_epi + ew * Cfg::kSlotBytes;
    const uint32_t tempty0 = PAIR ? cluster_addr(&bar.tempty[0], 0) : 0u;
    int place = 0, acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    Join parts{join + ew, join + kEpiWarps + ew, 0u, static_cast<uint32_t>(share), static_cast<uint32_t>(ctas)};
    for (int t = tile_begin; t < tiles && ok; t += tile_step) {
      const RowsTile tile = rows_tile(table, groups.count, t, place);
      const int f0 = tile.f * Cfg::kFeatures + static_cast<int>(rank) * kBM + quarter * 32;
      const int split = first_unit<Cfg>(tile);
      for (int first = 0; first < tile.rows; first += split) {
        ok = mbar_wait_bounded(&bar.tfull[acc], acc_ph, bar.abort_flag, &g_grouped_status, kStatusEpilogueTimeout);
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        const uint32_t at =
            tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * Cfg::kUnitCols);
        const int rows = first == 0 ? split : tile.rows - split;
        const bool joins = SPLIT && 32 * half < rows && f0 < shape.n;  // the same in all CTAs of the cluster
        if (joins) {
          float v[32];
          __syncwarp();
          tmem_load_32cols(at + 32 * half, v);
          ok = parts.wait(parts.read, parts.phase ^ 1u, bar.abort_flag);  // of the tile before
          if (!ok) break;
          XRow<true> x;
          round_row<true>(v, out.bf16, x);
          stage_write_col<true>(slot, lane, x);
          parts.tell(parts.there, lane);
        }
#pragma unroll 1
        for (int c = 32 * half; c < rows && f0 < shape.n && !SPLIT; c += 64) {
          float v[32];
          __syncwarp();
          tmem_load_32cols(at + c, v);
          XRow<OUT_F32> x;
          round_row<OUT_F32>(v, out.bf16, x);
          // Lane = feature, value = row of the output: the block is turned in its slot.
          stage_write_col<OUT_F32>(slot, lane, x);
          __syncwarp();
          store_rows<OUT_F32>(slot, out, static_cast<int64_t>(tile.row0 + first + c) * out.ldd + f0, min(32, rows - c),
                              shape.n - f0, lane);
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR)
            mbar_arrive_cluster(tempty0 + static_cast<uint32_t>(acc) * 8u);
          else
            mbar_arrive(&bar.tempty[acc]);
        }
        if (joins) {
          ok = parts.wait(parts.there, parts.phase, bar.abort_flag);
          if (!ok) break;
          parts.template add_up<OUT_F32>(slot, out, static_cast<int64_t>(tile.row0 + 32 * half) * out.ldd + f0,
                                         min(32, rows - 32 * half), shape.n - f0, lane);
          parts.phase ^= 1u;
        }
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
    }
    // No CTA leaves while another reads its slots.
    if (SPLIT && ok) parts.wait(parts.read, parts.phase ^ 1u, bar.abort_flag);
    // Rows that no group owns.
    for (int r = table.first_row[groups.count] + static_cast<int>(blockIdx.x) * kEpiWarps + ew; r < groups.rows;
         r += static_cast<int>(gridDim.x) * kEpiWarps) {
      const int64_t base = static_cast<int64_t>(r) * out.ldd;
      for (int c = lane; c < shape.n; c += 32) {
        if (OUT_F32)
          static_cast<float*>(out.d)[base + c] = 0.0f;
        else
          static_cast<uint16_t*>(out.d)[base + c] = 0;
      }
    }
  }
  tear_down<S, PAIR, PAIR || SPLIT>(bar, warp, tmem_base, Cfg::kTmemCols);
}

// ---------------------------------------------------------- reduced product
struct ReduceShape {
  int m, n, tiles_m, tiles_n;
};

constexpr int kReduceN = 256;

template <bool OUT_F32, bool PAIR>
struct ReduceConfig {
  static constexpr int kStages = (PAIR ? 6 : 4) - (OUT_F32 ? 1 : 0);
  static constexpr int kTileM = PAIR ? 2 * kBM : kBM;
  static constexpr int kNRows = PAIR ? kReduceN / 2 : kReduceN;
  static constexpr uint32_t kNBytes = kNRows * kBK * 2;
  static constexpr uint32_t kStageBytes = kMBytes + kNBytes;
  static constexpr uint32_t kSlotBytes = 32 * (OUT_F32 ? 128 : 64);
  static constexpr uint32_t kTmemCols = 2 * kReduceN;
  static constexpr size_t kSmemBytes =
      1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes + Table::kBytes + Barriers<kStages, PAIR>::kBytes;
};

constexpr int kReduceThreads = kThreads + 32;  // and the warp that zeroes foreign rows

// The order of a tile's blocks of 64 rows. A last block with foreign rows needs the
// zeroing warp, about 800 clocks after it has landed. So it is loaded up to two
// blocks ahead of its turn: the ring holds (.., last, a, b), the MMAs take
// (.., a, b, last). (Taken in the ring's order, its wait was exposed in every
// tile: 275 against 249 us for 64 groups of 500 rows, 1024 x 4096.)
struct Blocks {
  int rows, count, ahead;

  __device__ __forceinline__ explicit Blocks(int rows_)
      : rows(rows_), count((rows_ + kBK - 1) / kBK), ahead(rows_ % 16 == 0 ? 0 : min(2, count - 1)) {}
  // Place in the tile's stretch of the ring of the last block.
  __device__ __forceinline__ int last_place() const { return count - 1 - ahead; }
  // The block that is loaded at ring place `at`.
  __device__ __forceinline__ int block_at(int at) const {
    return at < last_place() ? at : (at == last_place() ? count - 1 : at - 1);
  }
};

template <bool OUT_F32, bool PAIR>
__global__ void __launch_bounds__(kReduceThreads, 1)
    grouped_reduce_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_r,
                          const Groups groups, const ReduceShape shape, const Output out, const int ab_bf16) {
  using Cfg = ReduceConfig<OUT_F32, PAIR>;
  constexpr int S = Cfg::kStages;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int tile_begin = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int tile_step = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_m = smem;
  uint8_t* smem_n = smem + S * kMBytes;
  uint8_t* smem_epi = smem + S * Cfg::kStageBytes;
  const Barriers<S, PAIR> bar(smem_epi + kEpiWarps * Cfg::kSlotBytes);
  const Table table(smem_epi + kEpiWarps * Cfg::kSlotBytes + Barriers<S, PAIR>::kBytes);

  // A stage is full when each CTA has arrived and the bytes are there: those of
  // both CTAs count on CTA 0's barrier, or, for a stage whose foreign rows are to be
  // zeroed, each CTA's on its own tail barrier, and the zeroing warps arrive.
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_l);
    tma_prefetch_desc(&map_r);
  }
  const uint32_t tmem_base = set_up<S, PAIR>(bar, warp, Cfg::kTmemCols, PAIR ? 2 : 1);
  // A tile's cost is its group's rows, in 31sts of a group twice as large as the mean.
  const int per_group = shape.tiles_m * shape.tiles_n;
  if (warp == 0) {
    const float unit = 31.0f * groups.count / (2.0f * groups.rows);
    fill_table(
        table, groups, lane, tile_step, per_group, [](int) { return Cut{1, 0}; },
        [&](int rows, int) { return min(31, static_cast<int>(rows * unit)); });
  }
  __syncthreads();
  const int tiles = per_group * groups.count;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = PAIR ? cluster_addr(&bar.full[0], 0) : 0u;
      const uint32_t tail_own = PAIR ? cluster_addr(&bar.tail[0], rank) : 0u;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const int place = t / per_group, l = t - place * per_group;
        const int e = table.order[place];
        const int begin = table.first_row[e], rows = table.first_row[e + 1] - begin;
        const int i = l / shape.tiles_n, j = l - i * shape.tiles_n;
        const int m0 = i * Cfg::kTileM + static_cast<int>(rank) * kBM;
        const int n0 = j * kReduceN + static_cast<int>(rank) * Cfg::kNRows;
        const Blocks blocks(rows);
        for (int at = 0; at < blocks.count; ++at) {
          if (!mbar_wait_bounded(&bar.empty[st], ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusProducerTimeout)) {
            ok = false;
            break;
          }
          uint8_t* sm = smem_m + st * kMBytes;
          uint8_t* sn = smem_n + st * Cfg::kNBytes;
          const int kb = blocks.block_at(at);
          const int row = begin + kb * kBK;
          const bool whole = kb + 1 < blocks.count || rows % 16 == 0;  // no foreign rows in a 16-row step
          if (!whole) mbar_arrive_expect_tx(&bar.tail[st], Cfg::kStageBytes);
          if (PAIR) {
            uint32_t fb = tail_own + static_cast<uint32_t>(st) * 8u;
            if (whole) {
              fb = full0 + static_cast<uint32_t>(st) * 8u;
              if (rank == 0)
                mbar_arrive_expect_tx(&bar.full[st], 2 * Cfg::kStageBytes);
              else
                mbar_arrive_cluster(fb);
            }
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_3d_pair(sm + c * 8192, &map_l, fb, m0 + 64 * c, row, 0);
#pragma unroll
            for (int c = 0; c < Cfg::kNRows / 64; ++c) tma_load_3d_pair(sn + c * 8192, &map_r, fb, n0 + 64 * c, row, 0);
          } else {
            uint64_t* landed = whole ? &bar.full[st] : &bar.tail[st];
            if (whole) mbar_arrive_expect_tx(landed, Cfg::kStageBytes);
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_3d(sm + c * 8192, &map_l, landed, m0 + 64 * c, row, 0);
#pragma unroll
            for (int c = 0; c < Cfg::kNRows / 64; ++c) tma_load_3d(sn + c * 8192, &map_r, landed, n0 + 64 * c, row, 0);
          }
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
      drain<S, PAIR>(bar, st, ph, ok);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = make_idesc_f16(ab_bf16, 1, 1, Cfg::kTileM, kReduceN);
      const uint64_t desc_t = make_smem_desc_sw128(0, 8192, 1024);
      const uint32_t empty0 = PAIR ? cluster_addr(&bar.empty[0], 0) : 0u;
      const uint32_t empty1 = PAIR ? cluster_addr(&bar.empty[0], 1) : 0u;
      const uint32_t tfull0 = PAIR ? cluster_addr(&bar.tfull[0], 0) : 0u;
      const uint32_t tfull1 = PAIR ? cluster_addr(&bar.tfull[0], 1) : 0u;
      int st = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const int e = table.order[t / per_group];
        const int rows = table.first_row[e + 1] - table.first_row[e];
        if (rows == 0) continue;
        if (!mbar_wait_bounded(&bar.tempty[acc], acc_ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kReduceN);
        const Blocks blocks(rows);
        // Steps of the ring's current stage into the accumulator; `steps` 16-row steps.
        auto multiply = [&](int at, uint32_t at_ph, int steps, uint32_t more) {
          if (!mbar_wait_bounded(&bar.full[at], at_ph, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) return false;
          tc_fence_after();
          const uint64_t m0 = desc_t + ((smem_u32(smem_m + at * kMBytes) >> 4) & 0x3FFFu);
          const uint64_t n0 = desc_t + ((smem_u32(smem_n + at * Cfg::kNBytes) >> 4) & 0x3FFFu);
          auto step = [&](int kk, uint32_t add) {
            if (PAIR)
              tc_mma_f16_pair(d_tmem, m0 + kk * 128u, n0 + kk * 128u, idesc, add);
            else
              tc_mma_f16(d_tmem, m0 + kk * 128u, n0 + kk * 128u, idesc, add);
          };
          step(0, more);
          if (steps == kBK / 16) {
#pragma unroll
            for (int kk = 1; kk < kBK / 16; ++kk) step(kk, 1u);
          } else {
            for (int kk = 1; kk < steps; ++kk) step(kk, 1u);
          }
          if (PAIR) {
            tc_commit_pair(empty0 + static_cast<uint32_t>(at) * 8u);
            tc_commit_pair(empty1 + static_cast<uint32_t>(at) * 8u);
          } else {
            tc_commit(&bar.empty[at]);
          }
          return true;
        };
        auto advance = [&]() {
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        };
        // The whole blocks in the ring's order, past the last one, which follows them.
        const int whole = blocks.count - (rows % kBK == 0 ? 0 : 1);
        const int skip = whole < blocks.count ? blocks.last_place() : -1;
        int last = 0;
        uint32_t last_ph = 0u, more = 0u;
        for (int i = 0; i < whole; ++i) {
          if (i == skip) {
            last = st;
            last_ph = ph;
            advance();
          }
          ok = multiply(st, ph, kBK / 16, more);
          if (!ok) break;
          more = 1u;
          advance();
        }
        if (ok && whole < blocks.count) {
          if (skip >= whole) {
            last = st;
            last_ph = ph;
            advance();
          }
          ok = multiply(last, last_ph, (rows % kBK + 15) / 16, more);
        }
        if (!ok) break;
        if (PAIR) {
          tc_commit_pair(tfull0 + static_cast<uint32_t>(acc) * 8u);
          tc_commit_pair(tfull1 + static_cast<uint32_t>(acc) * 8u);
        } else {
          tc_commit(&bar.tfull[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
    }
  } else if (warp == kReduceThreads / 32 - 1) {
    // Zeroes the foreign rows of a group's last 16-row step. Row r of a 64 x 64 box is
    // bytes [128 r, 128 r + 128) of it (the swizzle stays within a row).
    const uint32_t full0 = PAIR ? cluster_addr(&bar.full[0], 0) : 0u;
    int st = 0;
    uint32_t phases = 0;  // bit s: parity of the next use of tail[s]
    for (int t = tile_begin; t < tiles; t += tile_step) {
      const int e = table.order[t / per_group];
      const int rows = table.first_row[e + 1] - table.first_row[e];
      const Blocks blocks(rows);
      const int last = (st + blocks.last_place()) % S;
      st = (st + blocks.count) % S;
      if (rows % 16 == 0) continue;
      const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bar.tail[last], (phases >> last) & 1u, bar.abort_flag,
                                                                &g_grouped_status, kStatusProducerTimeout));
      if (!ok) break;
      phases ^= 1u << last;
      // Four rows at a time, eight lanes each, from the first row of the last step on.
      const int step_row = rows % kBK / 16 * 16;
      constexpr int kBoxes = (kBM + Cfg::kNRows) / 64;
#pragma unroll
      for (int box = 0; box < kBoxes; ++box) {
        uint8_t* at = (box < kBM / 64 ? smem_m + last * kMBytes + box * 8192
                                      : smem_n + last * Cfg::kNBytes + (box - kBM / 64) * 8192) +
                      step_row * 128 + lane * 16;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (4 * q + lane / 8 >= rows % 16) *reinterpret_cast<uint4*>(at + q * 512) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();  // the zeros are written before the MMA reads them
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          mbar_arrive_release_cluster(full0 + static_cast<uint32_t>(last) * 8u);
        else
          mbar_arrive(&bar.full[last]);
      }
    }
  } else {
    const int ew = warp - 2;
    const int quarter = warp & 3;
    const int half = ew >> 2;
    uint8_t* slot = smem_epi + ew * Cfg::kSlotBytes;
    const uint32_t tempty0 = PAIR ? cluster_addr(&bar.tempty[0], 0) : 0u;
    int acc = 0;
    uint32_t acc_ph = 0;
    for (int t = tile_begin; t < tiles; t += tile_step) {
      const int place = t / per_group, l = t - place * per_group;
      const int e = table.order[place];
      const int i = l / shape.tiles_n, j = l - i * shape.tiles_n;
      const int r0 = i * Cfg::kTileM + static_cast<int>(rank) * kBM + quarter * 32;
      const int live = min(32, shape.m - r0);
      const int64_t base = e * out.bstride + static_cast<int64_t>(r0) * out.ldd;
      const bool empty = table.first_row[e + 1] == table.first_row[e];
      if (empty && out.linear) {
        // A group without rows: each of its tiles fills an equal stretch of the matrix
        // (as tiles of unaligned rows, element by element, 65 matrices of 216 x 7201 took
        // 5 times their floor).
        constexpr int es = OUT_F32 ? 4 : 2;
        const int64_t all = static_cast<int64_t>(shape.m) * shape.n;
        const int64_t share = ((all + per_group - 1) / per_group + 63) / 64 * 64;
        const int64_t from = min(all, l * share), to = min(all, from + share);
        zero_fill(static_cast<uint8_t*>(out.d) + (e * out.bstride + from) * es, (to - from) * es,
                  (static_cast<int>(rank) * kEpiWarps + ew) * 32 + lane, (PAIR ? 2 : 1) * kEpiWarps * 32);
        continue;
      }
      if (!empty) {
        if (!mbar_wait_bounded(&bar.tfull[acc], acc_ph, bar.abort_flag, &g_grouped_status, kStatusEpilogueTimeout)) break;
        __syncwarp();
        tc_fence_after();
      }
      const uint32_t at = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kReduceN);
#pragma unroll 1
      for (int c = 32 * half; c < kReduceN; c += 64) {
        const int c0 = j * kReduceN + c;
        if (live <= 0 || c0 >= shape.n) break;
        float v[32];
        __syncwarp();
        if (empty) {
#pragma unroll
          for (int q = 0; q < 32; ++q) v[q] = 0.0f;
        } else {
          tmem_load_32cols(at + c, v);
        }
        XRow<OUT_F32> x;
        round_row<OUT_F32>(v, out.bf16, x);
        stage_write_row<OUT_F32>(slot, lane, x);
        __syncwarp();
        store_rows<OUT_F32>(slot, out, base + c0, live, shape.n - c0, lane);
        __syncwarp();
      }
      if (empty) continue;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          mbar_arrive_cluster(tempty0 + static_cast<uint32_t>(acc) * 8u);
        else
          mbar_arrive(&bar.tempty[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
  }
  tear_down<S, PAIR>(bar, warp, tmem_base, Cfg::kTmemCols);
}

// ------------------------------------------------------- rows for the copies
// Copies 16-bit rows that start anywhere into rows that start on 16 bytes, the rows
// that TMA can read. A thread writes 16 bytes: it reads the two aligned 16-byte words
// that hold them (the second only if the row reaches into it) and shifts. Bound by
// HBM; a strided copy by single elements moved 1.2 TB/s (32 x 2048 x 1025). With
// `ends`, matrices of groups without rows are left out: nothing reads them.
constexpr int kPadThreads = 256;
constexpr int kPadItems = 4;  // of a thread

__global__ void __launch_bounds__(kPadThreads) pad_rows_kernel(const uint16_t* src, int64_t src_bstride,
                                                               int64_t src_rstride, uint16_t* dst, int64_t dst_bstride,
                                                               int64_t dst_rstride, uint32_t cols, uint32_t words,
                                                               uint32_t items, const Groups groups) {
  // A CTA works on one matrix. (Whatever the ends are, a group with rows ends behind
  // the one before it.)
  const int e = static_cast<int>(blockIdx.y);
  if (groups.ends != nullptr && group_end(groups, e) <= (e > 0 ? group_end(groups, e - 1) : 0)) return;
  uint4 lo[kPadItems], hi[kPadItems];
  uint32_t shift[kPadItems];
  uint16_t* to[kPadItems];
  const uint32_t first = blockIdx.x * (kPadThreads * kPadItems) + threadIdx.x;
#pragma unroll
  for (int q = 0; q < kPadItems; ++q) {
    const uint32_t item = first + q * kPadThreads;
    to[q] = nullptr;
    if (item >= items) continue;
    const uint32_t r = item / words, word = item - r * words;
    const uintptr_t row = reinterpret_cast<uintptr_t>(src + e * src_bstride + r * src_rstride);
    const uintptr_t at = row + word * 16u, end = row + static_cast<uintptr_t>(cols) * 2u;
    const uint4* from = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
    lo[q] = from[0];
    hi[q] = reinterpret_cast<uintptr_t>(from + 1) < end ? from[1] : make_uint4(0u, 0u, 0u, 0u);
    shift[q] = static_cast<uint32_t>(at & 15u);
    to[q] = dst + e * dst_bstride + r * dst_rstride + word * 8u;
  }
#pragma unroll
  for (int q = 0; q < kPadItems; ++q) {
    if (to[q] == nullptr) continue;
    uint32_t w[8] = {lo[q].x, lo[q].y, lo[q].z, lo[q].w, hi[q].x, hi[q].y, hi[q].z, hi[q].w};
    // Bytes `shift` and on: by 8, by 4, then by 2 (shift is even).
    if (shift[q] & 8u) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift[q] & 4u) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (shift[q] & 2u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    *reinterpret_cast<uint4*>(to[q]) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// -------------------------------------------------------------------- launch
std::mutex g_mutex;
constexpr int kDevices = 64, kSlots = 32;
int g_resident[kDevices][kSlots] = {};  // co-resident clusters of an instantiation

// Launches a persistent grid of at most `wanted` clusters of `kernel`, of `cluster` CTAs each.
template <typename... Params, typename... Args>
int launch_persistent(void (*kernel)(Params...), int cluster, int threads, int slot, size_t smem, int64_t wanted,
                      cudaStream_t stream, Args... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kDevices) return fail(GNS_ERR_DEVICE, "device index out of range");
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  int resident = 0;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    resident = g_resident[dev][slot];
    if (resident == 0) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      resident = device_sm_count();
      if (cluster > 1) {
        cfg.gridDim = dim3(static_cast<unsigned>(resident / cluster * cluster), 1, 1);
        e = cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg);
        if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
        if (resident < 1) return fail(GNS_ERR_UNSUPPORTED, "no cluster of the grouped product fits on the device");
      }
      g_resident[dev][slot] = resident;
    }
  }
  const int64_t units = std::max<int64_t>(1, std::min<int64_t>(wanted, resident));
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * units), 1, 1);
  e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "grouped product launch");
}

struct RowsCall {
  CUtensorMap right;
  RowMaps maps;
  Groups groups;
  RowsShape shape;
  Output out;
  int bf16;
  int64_t row_tiles;  // at most
  int split;          // CTAs that share a tile's contraction
};

template <bool F_MN, int TOK, bool OUT_F32, bool PAIR, bool SPLIT>
int launch_rows(RowsCall& c, int slot, cudaStream_t stream) {
  using Cfg = RowsConfig<TOK, OUT_F32, PAIR, SPLIT>;
  c.shape.feature_tiles = (c.shape.n + Cfg::kFeatures - 1) / Cfg::kFeatures;
  return launch_persistent(grouped_rows_kernel<F_MN, TOK, OUT_F32, PAIR, SPLIT>, SPLIT ? c.split : (PAIR ? 2 : 1), kThreads,
                           slot, Cfg::kSmemBytes, c.row_tiles * c.shape.feature_tiles, stream, c.right, c.maps, c.groups,
                           c.shape, c.out, c.bf16);
}

template <int TOK, bool PAIR, bool SPLIT = false>
int launch_rows_any(bool mn, bool f32, RowsCall& c, int slot, cudaStream_t stream) {
  if (mn) {
    if (f32) return launch_rows<true, TOK, true, PAIR, SPLIT>(c, slot + 3, stream);
    return launch_rows<true, TOK, false, PAIR, SPLIT>(c, slot + 2, stream);
  }
  if (f32) return launch_rows<false, TOK, true, PAIR, SPLIT>(c, slot + 1, stream);
  return launch_rows<false, TOK, false, PAIR, SPLIT>(c, slot, stream);
}

// Rows of a tile: 64 or 128 (a CTA, 128 features), 256 or 512 (a pair, 256 features).
// The time of a call goes in turns of all SMs, so the choice is the one with the
// least turns times the cost of its tile. The groups' sizes are not known here: T
// rows in E groups make about T / tile + E / 2 parts, one for each group at least.
// Costs of a tile, measured with one turn and with many: 1, 1.08, 1.3 (64, 128,
// 256). Microseconds measured for 64 / 128 / 256, ragged groups of g rows on average:
//   5 x (1000 x 1501)   g = 96: 13.8 / 15.0 / 18.6   g = 128: 19.4 / 15.5 / 20.0
//   8 x (2048 x 2048)   g = 48: 30.3 / 22.3 / 23.7   g = 96: 28.4 / 31.7 / 25.1
//   64 x (1024 x 4096)  g = 32: 107 / 107 / 111      g = 128: 209 / 135 / 123
// Tiles of 512 rows load the features half as often, but both accumulators belong
// to one tile, so the epilogue does not overlap the next one: for long products of
// large groups only (256 against 512: 8 groups of 2048 rows, 4096 x 14336, 1441
// and 1390 us; 64 of 1024, 4096 x 1024: 455 and 413; but 64 of 640, 1024 x 4096:
// 350 and 383, and 8 of 1024 with few tiles, 4096 x 4096: 211 and 218).
int rows_tile_choice(int64_t rows, int64_t n, int64_t k, int64_t groups) {
  const int sms = device_sm_count();
  const double t = static_cast<double>(rows), e = static_cast<double>(groups);
  if (rows >= 1024 * groups && k >= 2048 && (t / 512) * static_cast<double>((n + 255) / 256) >= 6.0 * (sms / 2)) return 512;
  int best = 64;
  double least = 0.0;
  for (int tile : {64, 128, 256}) {
    const int features = tile == 256 ? 256 : 128, workers = tile == 256 ? sms / 2 : sms;
    const double parts = std::max(std::min(e, t), t / tile + e / 2);
    const double turns = std::ceil(parts * static_cast<double>((n + features - 1) / features) / workers);
    const double cost = turns * (tile == 64 ? 1.0 : (tile == 128 ? 1.08 : 1.3));
    if (tile == 64 || cost < least) {
      best = tile;
      least = cost;
    }
  }
  return best;
}

// CTAs that share a tile of 64 rows: 1, 2, 4 or 8. Where tiles are fewer than SMs, or
// a last turn has few of them, the contraction is cut. The unit is a block of 64 of
// the contraction (0.28 us of a CTA): a turn of a split tile costs its share and 2
// blocks, 12 at least (the join of the tile before must be through: 3 us), and the
// last join 4 more. Clusters of 4 and 8 leave some SMs of a GPC unused. Microseconds
// measured for 1 / 2 / 4 / 8 (bf16, rows of the call in all):
//   1 row, 1 x (8192 x 1024)      40.4 / 23.2 / 14.4 / 10.5
//   1 row, 1 x (4096 x 4096)      22.7 / 15.0 / 12.3 / 15.2
//   8 rows, 8 x (1024 x 4096)     17.4 / 20.3 / 28.1 / 53.1
//   98 rows, 10 x (8192 x 2048)   91.4 / 75.1 / 61.4 / 68.7
//   34 rows, 25 x (8192 x 512)    44.5 / 52.6 / 48.3 / 46.7
//   192 rows, 64 x (4096 x 1024)  98.0 / 89.7 / 97.3 / 140
int rows_split(int64_t rows, int64_t n, int64_t k_blocks, int64_t groups) {
  const double t = static_cast<double>(rows), e = static_cast<double>(groups), depth = static_cast<double>(k_blocks);
  const double tiles = std::max(std::min(e, t), t / 64 + e / 2) * static_cast<double>((n + kBM - 1) / kBM);
  const int sms = device_sm_count();
  int best = 1;
  double least = std::ceil(tiles / sms) * depth;
  for (int split : {2, 4, 8}) {
    const int clusters = (split == 2 ? sms : sms * 9 / 10) / split;
    if (clusters < 1 || k_blocks < split) break;
    const double cost = std::ceil(tiles / clusters) * std::max(depth / split + 2.0, 12.0) + 4.0;
    if (cost < least) {
      best = split;
      least = cost;
    }
  }
  return best;
}

int check_groups(int ab_dtype, int ends_bits, int64_t groups, int64_t rows, int64_t a, int64_t b, int d_dtype) {
  if (ab_dtype != kF16 && ab_dtype != kBF16) return fail(GNS_ERR_ARGUMENT, "left and right must be F16 or BF16");
  if (d_dtype < 0 || d_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad output dtype");
  if (ends_bits != 32 && ends_bits != 64) return fail(GNS_ERR_ARGUMENT, "ends must have 32 or 64 bits");
  if (groups < 0 || rows < 0 || a < 0 || b < 0) return fail(GNS_ERR_ARGUMENT, "negative dimension");
  if (groups > kMaxGroups) return fail(GNS_ERR_UNSUPPORTED, "at most 1024 groups are supported");
  if (rows > (1 << 30) || a > (1 << 24) || b > (1 << 24)) return fail(GNS_ERR_UNSUPPORTED, "dimension beyond kernel limits");
  return GNS_OK;
}

bool aligned_rows(const void* d, int64_t ldd, int64_t bstride, int dtype) {
  const int es = dtype_size(dtype);
  return reinterpret_cast<uintptr_t>(d) % 16 == 0 && (ldd * es) % 16 == 0 && (bstride * es) % 16 == 0;
}

}  // namespace

int grouped_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_grouped_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_grouped_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "grouped product status");
}

}  // namespace gns

using namespace gns;

extern "C" {

int gns_grouped_gemm(int ab_dtype, int64_t rows, int64_t n, int64_t k, int64_t groups, const void* left,
                     int64_t left_rstride, const void* right, int64_t right_gstride, int64_t right_rstride,
                     int64_t right_cstride, const void* ends, int ends_bits, void* out, int out_dtype,
                     int64_t out_rstride, gns_stream_t stream) {
  clear_error();
  int rc = check_groups(ab_dtype, ends_bits, groups, rows, n, k, out_dtype);
  if (rc != GNS_OK) return rc;
  if (rows == 0 || n == 0) return GNS_OK;
  if (groups == 0 || k == 0) return fail(GNS_ERR_UNSUPPORTED, "a grouped product needs a group and k > 0");
  if (left == nullptr || right == nullptr || ends == nullptr || out == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (rows > 1 && out_rstride < n) return fail(GNS_ERR_LAYOUT, "rows of the output overlap");
  const bool k_unit = right_rstride == 1 || k == 1;  // right is [group][k][n]
  const bool n_unit = right_cstride == 1 || n == 1;
  const bool k_major = k_unit && ((right_cstride * 2) % 16 == 0 || n == 1);
  if (!k_major && !(n_unit && ((right_rstride * 2) % 16 == 0 || k == 1)))
    return fail(GNS_ERR_LAYOUT, "right needs a unit stride along rows or columns and 16-byte multiples along the other");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  RowsCall c{};
  const int tile = rows_tile_choice(rows, n, k, groups);
  rc = k_major ? encode_tiles(&c.right, ab_dtype, right, k, n, groups, right_cstride, right_gstride, kBM)
               : encode_tiles(&c.right, ab_dtype, right, n, k, groups, right_rstride, right_gstride, 64);
  for (int i = 0; i < (tile == 64 ? 2 : 4) && rc == GNS_OK; ++i)
    rc = encode_tiles(&c.maps.box[i], ab_dtype, left, k, rows, 1, left_rstride, 0, 32 * (i + 1));
  if (rc != GNS_OK) return rc;
  c.groups = {ends, ends_bits == 64 ? 1 : 0, static_cast<int>(groups), static_cast<int>(rows)};
  c.shape.n = static_cast<int>(n);
  c.shape.k_blocks = static_cast<int>((k + kBK - 1) / kBK);
  c.out = {out, out_rstride, 0, out_dtype == kBF16 ? 1 : 0, aligned_rows(out, out_rstride, 0, out_dtype) ? 1 : 0, 0};
  c.bf16 = ab_dtype == kBF16 ? 1 : 0;
  c.row_tiles = rows / (tile == 64 ? 32 : 64) + std::min(groups, rows);
  if (c.row_tiles * ((n + kBM - 1) / kBM) > (1ll << 30)) return fail(GNS_ERR_UNSUPPORTED, "too many tiles");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool f32 = out_dtype == kF32;
  c.split = tile == 64 ? rows_split(rows, n, c.shape.k_blocks, groups) : 1;
  if (c.split > 1) return launch_rows_any<64, false, true>(!k_major, f32, c, c.split == 2 ? 20 : (c.split == 4 ? 24 : 28), st);
  if (tile == 64) return launch_rows_any<64, false>(!k_major, f32, c, 0, st);
  if (tile == 128) return launch_rows_any<128, false>(!k_major, f32, c, 4, st);
  if (tile == 256) return launch_rows_any<256, true>(!k_major, f32, c, 8, st);
  return launch_rows_any<512, true>(!k_major, f32, c, 12, st);
}

int gns_grouped_gemm_plan(int64_t rows, int64_t n, int64_t k, int64_t groups, int* tile_rows, int* split) {
  clear_error();
  int rc = check_groups(kBF16, 32, groups, rows, n, k, kBF16);
  if (rc != GNS_OK) return rc;
  if (rows == 0 || n == 0 || k == 0 || groups == 0) return fail(GNS_ERR_UNSUPPORTED, "an empty product has no plan");
  if (tile_rows == nullptr || split == nullptr) return fail(GNS_ERR_ARGUMENT, "null result");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  *tile_rows = rows_tile_choice(rows, n, k, groups);
  *split = *tile_rows == 64 ? rows_split(rows, n, (k + kBK - 1) / kBK, groups) : 1;
  return GNS_OK;
}

int gns_align_rows(int64_t batch, int64_t rows, int64_t cols, const void* src, int64_t src_bstride, int64_t src_rstride,
                   const void* ends, int ends_bits, void* dst, int64_t dst_bstride, int64_t dst_rstride,
                   gns_stream_t stream) {
  clear_error();
  if (ends != nullptr && ends_bits != 32 && ends_bits != 64) return fail(GNS_ERR_ARGUMENT, "ends must have 32 or 64 bits");
  if (ends != nullptr && batch > kMaxGroups) return fail(GNS_ERR_UNSUPPORTED, "at most 1024 groups are supported");
  if (batch < 0 || rows < 0 || cols < 0) return fail(GNS_ERR_ARGUMENT, "negative dimension");
  if (batch == 0 || rows == 0 || cols == 0) return GNS_OK;
  if (cols > (1ll << 30)) return fail(GNS_ERR_UNSUPPORTED, "dimension beyond kernel limits");
  if (src == nullptr || dst == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  const int64_t words = (cols + 7) / 8;
  if (reinterpret_cast<uintptr_t>(src) % 2 != 0) return fail(GNS_ERR_LAYOUT, "source must be aligned to its elements");
  if (reinterpret_cast<uintptr_t>(dst) % 16 != 0 || dst_rstride % 8 != 0 || dst_bstride % 8 != 0 || dst_rstride < words * 8)
    return fail(GNS_ERR_LAYOUT, "destination rows must start on 16 bytes and hold whole 16-byte words");
  int rc = check_device();
  if (rc != GNS_OK) return rc;
  // Up to 65535 matrices and 2^30 words of each a launch.
  const auto* from = static_cast<const uint16_t*>(src);
  auto* to = static_cast<uint16_t*>(dst);
  const int64_t most_rows = std::max<int64_t>(1, (1ll << 30) / words);
  for (int64_t b0 = 0; b0 < batch; b0 += 65535) {
    const int64_t nb = std::min<int64_t>(batch - b0, 65535);
    for (int64_t r0 = 0; r0 < rows; r0 += most_rows) {
      const int64_t items = std::min(rows - r0, most_rows) * words;
      const dim3 grid(static_cast<unsigned>((items + kPadThreads * kPadItems - 1) / (kPadThreads * kPadItems)),
                      static_cast<unsigned>(nb));
      pad_rows_kernel<<<grid, kPadThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
          from + b0 * src_bstride + r0 * src_rstride, src_bstride, src_rstride, to + b0 * dst_bstride + r0 * dst_rstride,
          dst_bstride, dst_rstride, static_cast<uint32_t>(cols), static_cast<uint32_t>(words), static_cast<uint32_t>(items),
          Groups{ends, ends_bits == 64 ? 1 : 0, static_cast<int>(nb), 0});
    }
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "align rows kernel");
}

int gns_grouped_gemm_reduce(int ab_dtype, int64_t rows, int64_t m, int64_t n, int64_t groups, const void* left,
                            int64_t left_rstride, const void* right, int64_t right_rstride, const void* ends,
                            int ends_bits, void* out, int out_dtype, int64_t out_gstride, int64_t out_rstride,
                            gns_stream_t stream) {
  clear_error();
  int rc = check_groups(ab_dtype, ends_bits, groups, rows, m, n, out_dtype);
  if (rc != GNS_OK) return rc;
  if (groups == 0 || m == 0 || n == 0) return GNS_OK;
  if (rows == 0) return fail(GNS_ERR_UNSUPPORTED, "a reduced product needs rows");
  if (left == nullptr || right == nullptr || ends == nullptr || out == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if ((m > 1 && out_rstride < n) || (groups > 1 && out_gstride < (m > 1 ? (m - 1) * out_rstride : 0) + n))
    return fail(GNS_ERR_LAYOUT, "rows or groups of the output overlap");
  const bool pair = m > kBM;
  const int64_t tiles_m = (m + (pair ? 2 * kBM : kBM) - 1) / (pair ? 2 * kBM : kBM);
  const int64_t tiles_n = (n + kReduceN - 1) / kReduceN;
  if (tiles_m * tiles_n * groups > (1ll << 30)) return fail(GNS_ERR_UNSUPPORTED, "too many tiles");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  CUtensorMap map_l, map_r;
  rc = encode_tiles(&map_l, ab_dtype, left, m, rows, 1, left_rstride, 0, 64);
  if (rc == GNS_OK) rc = encode_tiles(&map_r, ab_dtype, right, n, rows, 1, right_rstride, 0, 64);
  if (rc != GNS_OK) return rc;
  const Groups g{ends, ends_bits == 64 ? 1 : 0, static_cast<int>(groups), static_cast<int>(rows)};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const ReduceShape shape{static_cast<int>(m), static_cast<int>(n), static_cast<int>(tiles_m), static_cast<int>(tiles_n)};
  const Output o{out, out_rstride, out_gstride, out_dtype == kBF16 ? 1 : 0,
                 aligned_rows(out, out_rstride, out_gstride, out_dtype) ? 1 : 0,
                 out_rstride == n && out_gstride == m * n ? 1 : 0};
  const int bf16 = ab_dtype == kBF16 ? 1 : 0;
  const int64_t tiles = tiles_m * tiles_n * groups;
  if (pair) {
    if (out_dtype == kF32)
      return launch_persistent(grouped_reduce_kernel<true, true>, 2, kReduceThreads, 16, ReduceConfig<true, true>::kSmemBytes, tiles, st,
                                     map_l, map_r, g, shape, o, bf16);
    return launch_persistent(grouped_reduce_kernel<false, true>, 2, kReduceThreads, 17, ReduceConfig<false, true>::kSmemBytes, tiles, st,
                                   map_l, map_r, g, shape, o, bf16);
  }
  if (out_dtype == kF32)
    return launch_persistent(grouped_reduce_kernel<true, false>, 1, kReduceThreads, 18, ReduceConfig<true, false>::kSmemBytes, tiles, st,
                                    map_l, map_r, g, shape, o, bf16);
  return launch_persistent(grouped_reduce_kernel<false, false>, 1, kReduceThreads, 19, ReduceConfig<false, false>::kSmemBytes, tiles, st,
                                  map_l, map_r, g, shape, o, bf16);
}

}  // extern "C"
