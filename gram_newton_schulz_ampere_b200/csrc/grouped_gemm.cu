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
// enter. Each group gets its own tensor maps (written by a small kernel) whose row
// extent ends with the group; TMA fills zeros behind it.
//
// Sums are fp32 in TMEM, rounded once at the store. Every wait is bounded.
#include <algorithm>
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

// Row range of group e = base + lane for the 32 lanes of a warp: ends clamped to
// [0, rows] and to the largest end before them (`carry`, updated for the next 32).
__device__ __forceinline__ void group_rows(const Groups& g, int e, int lane, int& carry, int& begin, int& end) {
  end = 0;
  if (e < g.count) {
    const int64_t v = group_end(g, e);
    end = static_cast<int>(v < 0 ? 0 : (v > g.rows ? g.rows : v));
  }
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

// A group of `rows` rows is cut into `parts` parts of `size` rows (the last may be
// shorter): as few as the tile allows, equal up to the MMA's granularity.
struct Cut {
  int parts, size;
};

__device__ __forceinline__ Cut cut_group(int rows, int tile, int unit) {
  if (rows == 0) return {0, unit};
  const int least = (rows + tile - 1) / tile;
  const int size = ((rows + least - 1) / least + unit - 1) / unit * unit;
  return {(rows + size - 1) / size, size};
}

struct Output {
  void* d;
  int64_t ldd, bstride;
  int bf16;  // 16-bit outputs: 1 = bf16, 0 = fp16
  int vec;   // base, row and group strides are multiples of 16 bytes
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
#pragma unroll 1
  for (int r = 0; r < live; ++r) {
    const int64_t i = at + r * out.ldd + lane;
    if (OUT_F32)
      static_cast<uint32_t*>(out.d)[i] = *reinterpret_cast<const uint32_t*>(slot + stage_off<true>(r, 4u * lane));
    else
      static_cast<uint16_t*>(out.d)[i] = *reinterpret_cast<const uint16_t*>(slot + stage_off<false>(r, 2u * lane));
  }
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
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  static constexpr uint32_t kBytes = (2 * S + 4) * 8 + 16;

  __device__ __forceinline__ explicit Barriers(uint8_t* at) {
    full = reinterpret_cast<uint64_t*>(at);
    empty = full + S;
    tfull = full + 2 * S;
    tempty = full + 2 * S + 2;
    tmem_slot = reinterpret_cast<uint32_t*>(full + 2 * S + 4);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }

  __device__ __forceinline__ void init() {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
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

template <bool PAIR>
__device__ __forceinline__ void meet() {
  if (PAIR)
    cluster_sync_all();
  else
    __syncthreads();
}

// Set-up common to both kernels: barriers, TMEM, and the wait for the stream's
// previous kernel. Returns the TMEM base.
template <int S, bool PAIR>
__device__ __forceinline__ uint32_t set_up(const Barriers<S, PAIR>& bar, int warp, uint32_t tmem_cols) {
  if (threadIdx.x == 0) const_cast<Barriers<S, PAIR>&>(bar).init();
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
  meet<PAIR>();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_predecessor();
  return *bar.tmem_slot;
}

// Teardown: all roles meet; after an abort, copies and MMAs in flight get time to
// land before TMEM and shared memory are released.
template <int S, bool PAIR>
__device__ __forceinline__ void tear_down(const Barriers<S, PAIR>& bar, int warp, uint32_t tmem_base,
                                          uint32_t tmem_cols) {
  tc_fence_before();
  meet<PAIR>();
  if (*bar.abort_flag) settle_for_ns(2000000ull);
  meet<PAIR>();
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

template <int TOK, bool OUT_F32, bool PAIR>
struct RowsConfig {
  static constexpr int kStages = (PAIR ? 6 : 8) - (OUT_F32 ? 1 : 0);
  static constexpr int kFeatures = PAIR ? 2 * kBM : kBM;   // features of a tile
  static constexpr int kTokRows = PAIR ? TOK / 2 : TOK;    // rows that one CTA loads, at most
  static constexpr int kUnit = PAIR ? 32 : 16;             // granularity of N
  static constexpr uint32_t kTokBytes = kTokRows * kBK * 2;
  static constexpr uint32_t kStageBytes = kMBytes + kTokBytes;
  static constexpr uint32_t kSlotBytes = 32 * (OUT_F32 ? 128 : 64);
  static constexpr uint32_t kTmemCols = 2 * TOK;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes +
                                       2 * (kMaxGroups + 1) * 4 + 8 + Barriers<kStages, PAIR>::kBytes;
};

// A tile: `rows` rows from `row0` of group e, feature tile `f`.
struct RowsTile {
  int e, row0, rows, f;
};

template <int TOK, int UNIT>
__device__ __forceinline__ RowsTile rows_tile(const int* first_tile, const int* first_row, int t, int& e) {
  while (t >= first_tile[e + 1]) ++e;
  const int begin = first_row[e], rows = first_row[e + 1] - begin;
  const Cut cut = cut_group(rows, TOK, UNIT);
  const int l = t - first_tile[e];
  RowsTile tile;
  tile.e = e;
  tile.f = l / cut.parts;  // a group's row parts are neighbours: they share the expert's columns in L2
  const int part = l - tile.f * cut.parts;
  tile.row0 = begin + part * cut.size;
  tile.rows = min(cut.size, rows - part * cut.size);
  return tile;
}

template <bool F_MN, int TOK, bool OUT_F32, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_rows_kernel(const __grid_constant__ CUtensorMap map_right, const __grid_constant__ CUtensorMap map_full,
                        const __grid_constant__ CUtensorMap map_part, const Groups groups, const RowsShape shape,
                        const Output out, const int ab_bf16) {
  using Cfg = RowsConfig<TOK, OUT_F32, PAIR>;
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
  int* first_tile = reinterpret_cast<int*>(smem_epi + kEpiWarps * Cfg::kSlotBytes + Barriers<S, PAIR>::kBytes);
  int* first_row = first_tile + kMaxGroups + 1;

  const uint32_t tmem_base = set_up<S, PAIR>(bar, warp, Cfg::kTmemCols);

  // Tiles and rows before each group.
  if (warp == 0) {
    int row_carry = 0, tile_carry = 0;
    for (int base = 0; base < groups.count; base += 32) {
      const int e = base + lane;
      int begin, end;
      group_rows(groups, e, lane, row_carry, begin, end);
      const int tiles = cut_group(end - begin, TOK, Cfg::kUnit).parts * shape.feature_tiles;
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
      }
      if (e < groups.count) {
        first_row[e] = begin;
        first_tile[e] = tile_carry + sum - tiles;
      }
      tile_carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
      first_row[groups.count] = row_carry;
      first_tile[groups.count] = tile_carry;
    }
  }
  __syncthreads();
  const int tiles = first_tile[groups.count];

  if (warp == 0) {
    if (lane == 0) {
      int st = 0, e = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = PAIR ? cluster_addr(&bar.full[0], 0) : 0u;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const RowsTile tile = rows_tile<TOK, Cfg::kUnit>(first_tile, first_row, t, e);
        const int width = (tile.rows + Cfg::kUnit - 1) / Cfg::kUnit * Cfg::kUnit;  // N of the MMA
        const int mine = PAIR ? width / 2 : width;                                  // rows this CTA loads
        const int row0 = tile.row0 + static_cast<int>(rank) * mine;
        const int f0 = tile.f * Cfg::kFeatures + static_cast<int>(rank) * kBM;
        const bool whole = mine == Cfg::kTokRows;
        const int boxes = (mine + 31) / 32;
        const uint32_t bytes = kMBytes + (whole ? Cfg::kTokBytes : static_cast<uint32_t>(boxes) * 32u * kBK * 2u);
        for (int kb = 0; kb < shape.k_blocks; ++kb) {
          if (!mbar_wait_bounded(&bar.empty[st], ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusProducerTimeout)) {
            ok = false;
            break;
          }
          const int k0 = kb * kBK;
          uint8_t* sm = smem_m + st * kMBytes;
          uint8_t* sn = smem_n + st * Cfg::kTokBytes;
          if (PAIR) {
            if (rank == 0) mbar_arrive_expect_tx(&bar.full[st], 2 * bytes);
            const uint32_t fb = full0 + static_cast<uint32_t>(st) * 8u;
            if (!F_MN) {
              tma_load_3d_pair(sm, &map_right, fb, k0, f0, tile.e);
            } else {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c) tma_load_3d_pair(sm + c * 8192, &map_right, fb, f0 + 64 * c, k0, tile.e);
            }
            if (whole)
              tma_load_3d_pair(sn, &map_full, fb, k0, row0, 0);
            else
              for (int c = 0; c < boxes; ++c) tma_load_3d_pair(sn + c * 4096, &map_part, fb, k0, row0 + 32 * c, 0);
          } else {
            mbar_arrive_expect_tx(&bar.full[st], bytes);
            if (!F_MN) {
              tma_load_3d(sm, &map_right, &bar.full[st], k0, f0, tile.e);
            } else {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c) tma_load_3d(sm + c * 8192, &map_right, &bar.full[st], f0 + 64 * c, k0, tile.e);
            }
            if (whole)
              tma_load_3d(sn, &map_full, &bar.full[st], k0, row0, 0);
            else
              for (int c = 0; c < boxes; ++c) tma_load_3d(sn + c * 4096, &map_part, &bar.full[st], k0, row0 + 32 * c, 0);
          }
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint64_t desc_k = make_smem_desc_sw128(0, 16, 1024);
      const uint64_t desc_t = make_smem_desc_sw128(0, 8192, 1024);
      const uint32_t empty0 = PAIR ? cluster_addr(&bar.empty[0], 0) : 0u;
      const uint32_t empty1 = PAIR ? cluster_addr(&bar.empty[0], 1) : 0u;
      const uint32_t tfull0 = PAIR ? cluster_addr(&bar.tfull[0], 0) : 0u;
      const uint32_t tfull1 = PAIR ? cluster_addr(&bar.tfull[0], 1) : 0u;
      int st = 0, e = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const RowsTile tile = rows_tile<TOK, Cfg::kUnit>(first_tile, first_row, t, e);
        const int width = (tile.rows + Cfg::kUnit - 1) / Cfg::kUnit * Cfg::kUnit;
        const uint32_t idesc = make_idesc_f16(ab_bf16, F_MN ? 1 : 0, 0, Cfg::kFeatures, width);
        if (!mbar_wait_bounded(&bar.tempty[acc], acc_ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * TOK);
        for (int kb = 0; kb < shape.k_blocks; ++kb) {
          if (!mbar_wait_bounded(&bar.full[st], ph, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t m0 = (F_MN ? desc_t : desc_k) + ((smem_u32(smem_m + st * kMBytes) >> 4) & 0x3FFFu);
          const uint64_t n0 = desc_k + ((smem_u32(smem_n + st * Cfg::kTokBytes) >> 4) & 0x3FFFu);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            const uint32_t more = (kb > 0 || kk > 0) ? 1u : 0u;
            if (PAIR)
              tc_mma_f16_pair(d_tmem, m0 + kk * (F_MN ? 128u : 2u), n0 + kk * 2u, idesc, more);
            else
              tc_mma_f16(d_tmem, m0 + kk * (F_MN ? 128u : 2u), n0 + kk * 2u, idesc, more);
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
  } else {
    const int ew = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    const int half = ew >> 2;      // even (0) or odd (1) blocks of 32 rows
    uint8_t* slot = smem_epi + ew * Cfg::kSlotBytes;
    const uint32_t tempty0 = PAIR ? cluster_addr(&bar.tempty[0], 0) : 0u;
    int e = 0, acc = 0;
    uint32_t acc_ph = 0;
    for (int t = tile_begin; t < tiles; t += tile_step) {
      const RowsTile tile = rows_tile<TOK, Cfg::kUnit>(first_tile, first_row, t, e);
      if (!mbar_wait_bounded(&bar.tfull[acc], acc_ph, bar.abort_flag, &g_grouped_status, kStatusEpilogueTimeout)) break;
      __syncwarp();
      tc_fence_after();
      const int f0 = tile.f * Cfg::kFeatures + static_cast<int>(rank) * kBM + quarter * 32;
      const uint32_t at = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * TOK);
#pragma unroll 1
      for (int c = 32 * half; c < tile.rows && f0 < shape.n; c += 64) {
        float v[32];
        __syncwarp();
        tmem_load_32cols(at + c, v);
        XRow<OUT_F32> x;
        round_row<OUT_F32>(v, out.bf16, x);
        // Lane = feature, value = row of the output: the block is turned in its slot.
        stage_write_col<OUT_F32>(slot, lane, x);
        __syncwarp();
        store_rows<OUT_F32>(slot, out, static_cast<int64_t>(tile.row0 + c) * out.ldd + f0, min(32, tile.rows - c),
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
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    // Rows that no group owns.
    for (int r = first_row[groups.count] + static_cast<int>(blockIdx.x) * kEpiWarps + ew; r < groups.rows;
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
  tear_down<S, PAIR>(bar, warp, tmem_base, Cfg::kTmemCols);
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
      1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes + (kMaxGroups + 1) * 4 + 4 + Barriers<kStages, PAIR>::kBytes;
};

// The tensor maps of a group's rows of both operands, from maps of the whole
// operands: base address at the group's first row, row extent to its last.
// One warp; maps [count][2] of 128 bytes each.
__global__ void __launch_bounds__(32) group_maps_kernel(const __grid_constant__ CUtensorMap left,
                                                        const __grid_constant__ CUtensorMap right, const Groups groups,
                                                        const void* left_base, const void* right_base,
                                                        int64_t left_pitch, int64_t right_pitch, CUtensorMap* maps) {
  pdl_launch_dependents();
  const int lane = threadIdx.x;
  int carry = 0;
  for (int base = 0; base < groups.count; base += 32) {
    const int e = base + lane;
    int begin, end;
    group_rows(groups, e, lane, carry, begin, end);
    if (e >= groups.count || end == begin) continue;  // no map is read for an empty group
    for (int which = 0; which < 2; ++which) {
      CUtensorMap* to = maps + 2 * e + which;
      const uint4* from = reinterpret_cast<const uint4*>(which ? &right : &left);
#pragma unroll
      for (int q = 0; q < 8; ++q) reinterpret_cast<uint4*>(to)[q] = from[q];
      const uint64_t address = reinterpret_cast<uint64_t>(which ? right_base : left_base) +
                               static_cast<uint64_t>(begin) * static_cast<uint64_t>(which ? right_pitch : left_pitch);
      asm volatile("tensormap.replace.tile.global_address.global.b1024.b64 [%0], %1;" ::"l"(to), "l"(address) : "memory");
      asm volatile("tensormap.replace.tile.global_dim.global.b1024.b32 [%0], 1, %1;" ::"l"(to), "r"(end - begin) : "memory");
    }
  }
  asm volatile("fence.proxy.tensormap::generic.release.gpu;" ::: "memory");
}

__device__ __forceinline__ void acquire_map(const CUtensorMap* map) {
  asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(map) : "memory");
}

template <bool OUT_F32, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_reduce_kernel(const CUtensorMap* __restrict__ maps, const Groups groups, const ReduceShape shape,
                          const Output out, const int ab_bf16) {
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
  int* first_row = reinterpret_cast<int*>(smem_epi + kEpiWarps * Cfg::kSlotBytes + Barriers<S, PAIR>::kBytes);

  const uint32_t tmem_base = set_up<S, PAIR>(bar, warp, Cfg::kTmemCols);
  if (warp == 0) {
    int carry = 0;
    for (int base = 0; base < groups.count; base += 32) {
      int begin, end;
      group_rows(groups, base + lane, lane, carry, begin, end);
      if (base + lane < groups.count) first_row[base + lane] = begin;
    }
    if (lane == 0) first_row[groups.count] = carry;
  }
  __syncthreads();
  const int per_group = shape.tiles_m * shape.tiles_n;
  const int tiles = per_group * groups.count;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0, have = -1;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full0 = PAIR ? cluster_addr(&bar.full[0], 0) : 0u;
      for (int t = tile_begin; t < tiles && ok; t += tile_step) {
        const int e = t / per_group, l = t - e * per_group;
        const int k_blocks = (first_row[e + 1] - first_row[e] + kBK - 1) / kBK;
        if (k_blocks == 0) continue;
        const CUtensorMap* map_l = maps + 2 * e;
        const CUtensorMap* map_r = map_l + 1;
        if (e != have) {
          acquire_map(map_l);
          acquire_map(map_r);
          have = e;
        }
        const int i = l / shape.tiles_n, j = l - i * shape.tiles_n;
        const int m0 = i * Cfg::kTileM + static_cast<int>(rank) * kBM;
        const int n0 = j * kReduceN + static_cast<int>(rank) * Cfg::kNRows;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(&bar.empty[st], ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusProducerTimeout)) {
            ok = false;
            break;
          }
          uint8_t* sm = smem_m + st * kMBytes;
          uint8_t* sn = smem_n + st * Cfg::kNBytes;
          if (PAIR) {
            if (rank == 0) mbar_arrive_expect_tx(&bar.full[st], 2 * Cfg::kStageBytes);
            const uint32_t fb = full0 + static_cast<uint32_t>(st) * 8u;
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_3d_pair(sm + c * 8192, map_l, fb, m0 + 64 * c, kb * kBK, 0);
#pragma unroll
            for (int c = 0; c < Cfg::kNRows / 64; ++c) tma_load_3d_pair(sn + c * 8192, map_r, fb, n0 + 64 * c, kb * kBK, 0);
          } else {
            mbar_arrive_expect_tx(&bar.full[st], Cfg::kStageBytes);
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_3d(sm + c * 8192, map_l, &bar.full[st], m0 + 64 * c, kb * kBK, 0);
#pragma unroll
            for (int c = 0; c < Cfg::kNRows / 64; ++c) tma_load_3d(sn + c * 8192, map_r, &bar.full[st], n0 + 64 * c, kb * kBK, 0);
          }
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
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
        const int e = t / per_group;
        const int rows = first_row[e + 1] - first_row[e];
        const int k_blocks = (rows + kBK - 1) / kBK;
        if (k_blocks == 0) continue;
        if (!mbar_wait_bounded(&bar.tempty[acc], acc_ph ^ 1u, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kReduceN);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(&bar.full[st], ph, bar.abort_flag, &g_grouped_status, kStatusMmaTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t m0 = desc_t + ((smem_u32(smem_m + st * kMBytes) >> 4) & 0x3FFFu);
          const uint64_t n0 = desc_t + ((smem_u32(smem_n + st * Cfg::kNBytes) >> 4) & 0x3FFFu);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            const uint32_t more = (kb > 0 || kk > 0) ? 1u : 0u;
            if (PAIR)
              tc_mma_f16_pair(d_tmem, m0 + kk * 128u, n0 + kk * 128u, idesc, more);
            else
              tc_mma_f16(d_tmem, m0 + kk * 128u, n0 + kk * 128u, idesc, more);
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
  } else {
    const int ew = warp - 2;
    const int quarter = warp & 3;
    const int half = ew >> 2;
    uint8_t* slot = smem_epi + ew * Cfg::kSlotBytes;
    const uint32_t tempty0 = PAIR ? cluster_addr(&bar.tempty[0], 0) : 0u;
    int acc = 0;
    uint32_t acc_ph = 0;
    for (int t = tile_begin; t < tiles; t += tile_step) {
      const int e = t / per_group, l = t - e * per_group;
      const int i = l / shape.tiles_n, j = l - i * shape.tiles_n;
      const int r0 = i * Cfg::kTileM + static_cast<int>(rank) * kBM + quarter * 32;
      const int live = min(32, shape.m - r0);
      const int64_t base = e * out.bstride + static_cast<int64_t>(r0) * out.ldd;
      const bool empty = first_row[e + 1] == first_row[e];
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

// -------------------------------------------------------------------- launch
std::mutex g_mutex;
constexpr int kDevices = 64, kSlots = 32;
int g_resident[kDevices][kSlots] = {};  // co-resident CTAs (or CTAs of pairs) of an instantiation

// Launches a persistent grid of at most `wanted` CTAs (or pairs) of `kernel`.
template <bool PAIR, typename... Params, typename... Args>
int launch_persistent(void (*kernel)(Params...), int slot, size_t smem, int64_t wanted, cudaStream_t stream, Args... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kDevices) return fail(GNS_ERR_DEVICE, "device index out of range");
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  int resident = 0;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    resident = g_resident[dev][slot];
    if (resident == 0) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      resident = device_sm_count();
      if (PAIR) {
        cfg.gridDim = dim3(static_cast<unsigned>(2 * (resident / 2)), 1, 1);
        e = cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg);
        if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
        if (resident < 1) return fail(GNS_ERR_UNSUPPORTED, "no CTA pair of the grouped product fits on an SM pair");
      }
      g_resident[dev][slot] = resident;
    }
  }
  const int64_t units = std::max<int64_t>(1, std::min<int64_t>(wanted, resident));
  cfg.gridDim = dim3(static_cast<unsigned>(PAIR ? 2 * units : units), 1, 1);
  e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "grouped product launch");
}

struct RowsCall {
  CUtensorMap right, full, part;
  Groups groups;
  RowsShape shape;
  Output out;
  int bf16;
  int64_t row_tiles;  // at most
};

template <bool F_MN, int TOK, bool OUT_F32, bool PAIR>
int launch_rows(RowsCall& c, int slot, cudaStream_t stream) {
  using Cfg = RowsConfig<TOK, OUT_F32, PAIR>;
  c.shape.feature_tiles = (c.shape.n + Cfg::kFeatures - 1) / Cfg::kFeatures;
  return launch_persistent<PAIR>(grouped_rows_kernel<F_MN, TOK, OUT_F32, PAIR>, slot, Cfg::kSmemBytes,
                                 c.row_tiles * c.shape.feature_tiles, stream, c.right, c.full, c.part, c.groups,
                                 c.shape, c.out, c.bf16);
}

template <int TOK, bool PAIR>
int launch_rows_any(bool mn, bool f32, RowsCall& c, int slot, cudaStream_t stream) {
  if (mn) {
    if (f32) return launch_rows<true, TOK, true, PAIR>(c, slot + 3, stream);
    return launch_rows<true, TOK, false, PAIR>(c, slot + 2, stream);
  }
  if (f32) return launch_rows<false, TOK, true, PAIR>(c, slot + 1, stream);
  return launch_rows<false, TOK, false, PAIR>(c, slot, stream);
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

size_t reduce_workspace(int64_t groups) { return 128 + static_cast<size_t>(groups) * 2 * sizeof(CUtensorMap); }

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
  const bool k_unit = right_rstride == 1 || k == 1;  // right is [group][k][n]
  const bool n_unit = right_cstride == 1 || n == 1;
  const bool k_major = k_unit && ((right_cstride * 2) % 16 == 0 || n == 1);
  if (!k_major && !(n_unit && ((right_rstride * 2) % 16 == 0 || k == 1)))
    return fail(GNS_ERR_LAYOUT, "right needs a unit stride along rows or columns and 16-byte multiples along the other");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  RowsCall c{};
  // Groups of up to 64 rows on average are bound by reading the experts' matrices:
  // narrow row tiles leave the shared memory to more stages of them.
  const bool small = rows <= 64 * groups;
  const int box = small ? 64 : 128;
  rc = k_major ? encode_tiles(&c.right, ab_dtype, right, k, n, groups, right_cstride, right_gstride, kBM)
               : encode_tiles(&c.right, ab_dtype, right, n, k, groups, right_rstride, right_gstride, 64);
  if (rc == GNS_OK) rc = encode_tiles(&c.full, ab_dtype, left, k, rows, 1, left_rstride, 0, box);
  if (rc == GNS_OK) rc = encode_tiles(&c.part, ab_dtype, left, k, rows, 1, left_rstride, 0, 32);
  if (rc != GNS_OK) return rc;
  c.groups = {ends, ends_bits == 64 ? 1 : 0, static_cast<int>(groups), static_cast<int>(rows)};
  c.shape.n = static_cast<int>(n);
  c.shape.k_blocks = static_cast<int>((k + kBK - 1) / kBK);
  c.out = {out, out_rstride, 0, out_dtype == kBF16 ? 1 : 0, aligned_rows(out, out_rstride, 0, out_dtype) ? 1 : 0};
  c.bf16 = ab_dtype == kBF16 ? 1 : 0;
  c.row_tiles = rows / (small ? 32 : 128) + std::min(groups, rows);
  if (c.row_tiles * ((n + kBM - 1) / kBM) > (1ll << 30)) return fail(GNS_ERR_UNSUPPORTED, "too many tiles");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (small) return launch_rows_any<64, false>(!k_major, out_dtype == kF32, c, 0, st);
  return launch_rows_any<256, true>(!k_major, out_dtype == kF32, c, 4, st);
}

size_t gns_grouped_gemm_reduce_workspace_size(int64_t groups) { return groups < 1 ? 0 : reduce_workspace(groups); }

int gns_grouped_gemm_reduce(int ab_dtype, int64_t rows, int64_t m, int64_t n, int64_t groups, const void* left,
                            int64_t left_rstride, const void* right, int64_t right_rstride, const void* ends,
                            int ends_bits, void* out, int out_dtype, int64_t out_gstride, int64_t out_rstride,
                            void* workspace, size_t workspace_bytes, gns_stream_t stream) {
  clear_error();
  int rc = check_groups(ab_dtype, ends_bits, groups, rows, m, n, out_dtype);
  if (rc != GNS_OK) return rc;
  if (groups == 0 || m == 0 || n == 0) return GNS_OK;
  if (rows == 0) return fail(GNS_ERR_UNSUPPORTED, "a reduced product needs rows");
  if (left == nullptr || right == nullptr || ends == nullptr || out == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (workspace == nullptr || workspace_bytes < reduce_workspace(groups))
    return fail(GNS_ERR_WORKSPACE, "grouped reduction workspace too small");
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
  auto* maps = reinterpret_cast<CUtensorMap*>((reinterpret_cast<uintptr_t>(workspace) + 127) & ~uintptr_t(127));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  group_maps_kernel<<<1, 32, 0, st>>>(map_l, map_r, g, left, right, left_rstride * 2, right_rstride * 2, maps);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "group maps kernel");
  const ReduceShape shape{static_cast<int>(m), static_cast<int>(n), static_cast<int>(tiles_m), static_cast<int>(tiles_n)};
  const Output o{out, out_rstride, out_gstride, out_dtype == kBF16 ? 1 : 0,
                 aligned_rows(out, out_rstride, out_gstride, out_dtype) ? 1 : 0};
  const int bf16 = ab_dtype == kBF16 ? 1 : 0;
  const int64_t tiles = tiles_m * tiles_n * groups;
  if (pair) {
    if (out_dtype == kF32)
      return launch_persistent<true>(grouped_reduce_kernel<true, true>, 8, ReduceConfig<true, true>::kSmemBytes, tiles, st,
                                     static_cast<const CUtensorMap*>(maps), g, shape, o, bf16);
    return launch_persistent<true>(grouped_reduce_kernel<false, true>, 9, ReduceConfig<false, true>::kSmemBytes, tiles, st,
                                   static_cast<const CUtensorMap*>(maps), g, shape, o, bf16);
  }
  if (out_dtype == kF32)
    return launch_persistent<false>(grouped_reduce_kernel<true, false>, 10, ReduceConfig<true, false>::kSmemBytes, tiles, st,
                                    static_cast<const CUtensorMap*>(maps), g, shape, o, bf16);
  return launch_persistent<false>(grouped_reduce_kernel<false, false>, 11, ReduceConfig<false, false>::kSmemBytes, tiles, st,
                                  static_cast<const CUtensorMap*>(maps), g, shape, o, bf16);
}

}  // extern "C"
