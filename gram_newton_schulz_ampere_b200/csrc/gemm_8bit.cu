// Products of e4m3 matrices with fp32 scales for blocks of 128 of the contraction.
//
//   out[i, j] = sum over blocks b of  l[i, b] r[b, j / 128]  sum over k in b of  left[i, k] right[k, j]
//
// left has a scale for each row and block, right one for each 128 x 128 block. The inner
// sums are the tensor cores' (tcgen05 kind::f8f6f4, fp32 accumulators in TMEM); after
// each block of 128 its partial sum leaves TMEM, is scaled and added to an fp32 sum in
// registers, while the tensor cores work on the next block in the other accumulator.
// Rounded once, at the store.
//
// Two kernels. Many rows: a CTA pair computes 256 x 256 tiles of the output, rows of left
// on the MMA's M side, so that a thread's scale is one number a block (its row's, times
// the right block's). Few rows: right's columns (a layer's features) are the M side and up
// to 128 rows of left the N side, whose width follows the rows; a cluster of CTAs shares a
// tile's contraction and joins the fp32 sums out of shared memory in a fixed order.
//
// Every wait is bounded.
#include <algorithm>
#include <mutex>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"
#include "staging.cuh"

namespace gns {
namespace {

__device__ int g_gemm8_status = 0;

constexpr int kBlock = 128;  // contraction of a stage and of a scale: 128 bytes
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr uint32_t kTileBytes = 128 * kBlock;  // 128 rows or columns of a block
constexpr int kTile = 256;                     // rows and columns of a pair's tile

struct Scales {
  const float* left;   // [m][blocks]
  const float* right;  // [blocks][n / 128]
  int64_t left_rstride, left_cstride, right_rstride, right_cstride;
};

struct Shape8 {
  int m, n, blocks;
};

struct Out8 {
  void* d;
  int64_t ldd;
  int bf16;  // 16-bit outputs: 1 = bf16, 0 = fp16
  int tma;   // the output's rows can be written by TMA
};

// D (+)= A . B, 8-bit floating point operands (e4m3: format 0 in the instruction descriptor).
__device__ __forceinline__ void mma_8bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_8bit_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The instruction descriptor's fields are those of kind::f16, with format 0 = e4m3.
__device__ __forceinline__ uint32_t idesc_8bit(bool a_mn, bool b_mn, int m, int n) {
  return make_idesc_f16(0, a_mn ? 1 : 0, b_mn ? 1 : 0, m, n);
}

// A stage's tile of 128 x 128 bytes: K-major, eight rows of 128 bytes follow one another
// and a step of 32 along k is 32 bytes; MN-major, the same with k as the rows, so a step
// is 32 rows.
__device__ __forceinline__ uint64_t tile_desc(const uint8_t* tile) { return make_smem_desc_sw128(smem_u32(tile), 16, 1024); }
constexpr uint64_t step_of(bool mn) { return mn ? 32 * 128 / 16 : 32 / 16; }
constexpr int kSteps = kBlock / 32;

// Barriers. `done` says both that a stage may be filled again and that its partial sum is in
// its accumulator: one commit a block, which the producer and the summing warps wait for (a
// commit costs the issuing thread about 60 cycles, a block's products take 512). In a pair
// the `full` and `read` barriers of CTA 0 serve both CTAs, and each CTA has its own `done`.
template <int S, bool PAIR>
struct Pipe {
  uint64_t* full;  // a stage has landed
  uint64_t* done;  // its products are done
  uint64_t* read;  // the accumulator has been read
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  static constexpr uint32_t kBytes = (2 * S + 2) * 8 + 8;

  __device__ __forceinline__ explicit Pipe(uint8_t* at) {
    full = reinterpret_cast<uint64_t*>(at);
    done = full + S;
    read = done + S;
    tmem_slot = reinterpret_cast<uint32_t*>(read + 2);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }

  __device__ __forceinline__ void init() const {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    for (int a = 0; a < 2; ++a) mbar_init(&read[a], (PAIR ? 2 : 1) * kEpiWarps);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }

  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int code) const {
    return mbar_wait_bounded(bar, parity, abort_flag, &g_gemm8_status, code);
  }

  // The producer's end: the products of every stage that it filled are done, so that no
  // arrival is on its way when the CTA leaves.
  __device__ __forceinline__ void drain(int st, uint32_t ph, bool ok) const {
    for (int i = 0; i < S && ok; ++i) {
      ok = wait(&done[st], ph ^ 1u, kStatusProducerTimeout);
      if (++st == S) {
        st = 0;
        ph ^= 1u;
      }
    }
  }
};

// Arrives on the barrier at the same place in both CTAs of the pair once every earlier pair
// MMA of this thread has completed.
__device__ __forceinline__ void commit_to_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

template <bool CLUSTER>
__device__ __forceinline__ void meet() {
  if (CLUSTER)
    cluster_sync_all();
  else
    __syncthreads();
}

// 32 columns of a thread's TMEM lane on their way to registers: they hold nothing of use
// until land(), which waits for every load that the thread has issued.
struct TmemPiece {
  uint32_t r[32];

  __device__ __forceinline__ void issue(uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
  }

  // The registers are operands, so that nothing that reads them moves above the wait.
  __device__ __forceinline__ void land() {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
  }

  __device__ __forceinline__ void add_to(Pair* sum, Pair scale) const {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      sum[e] = fma2(Pair(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), scale, sum[e]);
  }
};

// ------------------------------------------------------------------ many rows
// Warps 0 to 3 load and issue (two of them idle), 4 to 11 sum. The sums take 128 registers of a
// thread and two pieces on their way another 64, so the four leave registers to the eight:
// 40 and twice 232 of the 168 a thread at launch (3 x 168 = 40 + 2 x 232).
constexpr int kPairThreads = 32 * (4 + kEpiWarps);

template <bool OUT_F32>
struct PairConfig {
  static constexpr int kStages = 5;
  static constexpr uint32_t kStageBytes = 2 * kTileBytes;
  // A warp's part of the output on its way to memory: 32 rows in two boxes of 128 bytes a row.
  static constexpr uint32_t kBoxBytes = 32 * 128;
  static constexpr uint32_t kSlotBytes = 2 * kBoxBytes;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes + Pipe<kStages, true>::kBytes;
};

// Tiles in bands of eight rows of tiles, column by column: the tiles that run at one time
// share their operands in L2.
struct Tiling {
  int rows, cols;
  __device__ __forceinline__ void place(int t, int& i, int& j) const {
    constexpr int kBand = 8;
    const int band = t / (kBand * cols);
    const int high = min(kBand, rows - band * kBand);
    const int l = t - band * kBand * cols;
    j = l / high;
    i = band * kBand + l - j * high;
  }
};

template <bool B_MN, bool OUT_F32>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm8_pair_kernel(const __grid_constant__ CUtensorMap map_left, const __grid_constant__ CUtensorMap map_right,
                      const __grid_constant__ CUtensorMap map_out, const Scales scales, const Shape8 shape,
                      const Tiling tiling, const Out8 out) {
  using Cfg = PairConfig<OUT_F32>;
  constexpr int S = Cfg::kStages;
  const uint32_t rank = cluster_ctarank();
  const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
  const int tiles = tiling.rows * tiling.cols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_out = smem + S * Cfg::kStageBytes;
  const Pipe<S, true> pipe(smem_out + kEpiWarps * Cfg::kSlotBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_left);
    tma_prefetch_desc(&map_right);
    pipe.init();
  }
  if (warp == 1) {
    tmem_alloc_pair(pipe.tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_predecessor();
  const uint32_t tmem = *pipe.tmem_slot;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && lane == 0) {
      const uint32_t full0 = cluster_addr(&pipe.full[0], 0);
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int i, j;
        tiling.place(t, i, j);
        const int row = i * kTile + static_cast<int>(rank) * 128, col = j * kTile + static_cast<int>(rank) * 128;
        for (int b = 0; b < shape.blocks; ++b) {
          ok = pipe.wait(&pipe.done[st], ph ^ 1u, kStatusProducerTimeout);
          if (!ok) break;
          uint8_t* at = smem + st * Cfg::kStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(&pipe.full[st], 2 * Cfg::kStageBytes);
          const uint32_t fb = full0 + static_cast<uint32_t>(st) * 8u;
          tma_load_3d_pair(at, &map_left, fb, b * kBlock, row, 0);
          if (B_MN)
            tma_load_3d_pair(at + kTileBytes, &map_right, fb, col, b * kBlock, 0);
          else
            tma_load_3d_pair(at + kTileBytes, &map_right, fb, b * kBlock, col, 0);
          if (++st == S) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
      pipe.drain(st, ph, ok);
    }
    // Two warps issue the products, one the even blocks into the first accumulator, the other
    // the odd ones into the second: what a block costs its thread beside the products (two
    // waits and a commit, 300 cycles; 512 for the products, of which few are queued ahead)
    // passes while the other's run.
    if ((warp == 1 || warp == 2) && lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_8bit(false, B_MN, kTile, kTile);
      const int acc = warp - 1;
      const int mine = first < tiles ? (tiles - first + step - 1) / step : 0;
      const int64_t count = static_cast<int64_t>(mine) * shape.blocks;
      int st = acc;
      uint32_t ph = 0, acc_ph = 0;
      for (int64_t i = acc; i < count; i += 2) {
        if (!pipe.wait(&pipe.full[st], ph, kStatusMmaTimeout) ||
            !pipe.wait(&pipe.read[acc], acc_ph ^ 1u, kStatusMmaTimeout))
          break;
        tc_fence_after();
        const uint8_t* at = smem + st * Cfg::kStageBytes;
        const uint64_t left = tile_desc(at), right = tile_desc(at + kTileBytes);
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          mma_8bit_pair(tmem + static_cast<uint32_t>(acc * kTile), left + k * step_of(false), right + k * step_of(B_MN),
                        idesc, k > 0 ? 1u : 0u);
        commit_to_both(&pipe.done[st]);
        acc_ph ^= 1u;
        st += 2;
        if (st >= S) {
          st -= S;
          ph ^= 1u;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // A warp has 32 rows (its quarter of the TMEM lanes) and 128 columns of the CTA's tile:
    // 128 fp32 sums a thread, and one scale a block.
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint8_t* slot = smem_out + (warp - 4) * Cfg::kSlotBytes;
    const uint32_t read0 = cluster_addr(&pipe.read[0], 0);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(128 * half);
    int st = 0, acc = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int i, j;
      tiling.place(t, i, j);
      const int row0 = i * kTile + static_cast<int>(rank) * 128 + quarter * 32, col0 = j * kTile + 128 * half;
      const float* ls = scales.left + min(row0 + lane, shape.m - 1) * scales.left_rstride;
      const float* rs = scales.right + min(col0, shape.n - 1) / kBlock * scales.right_cstride;
      Pair sum[64];
#pragma unroll
      for (int q = 0; q < 64; ++q) sum[q] = Pair(0.0f);
      // Scales are loaded two blocks ahead of their use.
      float l0 = *ls, r0 = *rs, l1 = l0, r1 = r0;
      if (shape.blocks > 1) {
        ls += scales.left_cstride;
        rs += scales.right_rstride;
        l1 = *ls;
        r1 = *rs;
      }
      for (int b = 0; b < shape.blocks; ++b) {
        const Pair scale(l0 * r0);
        l0 = l1;
        r0 = r1;
        if (b + 2 < shape.blocks) {
          ls += scales.left_cstride;
          rs += scales.right_rstride;
          l1 = *ls;
          r1 = *rs;
        }
        ok = __all_sync(0xffffffffu, pipe.wait(&pipe.done[st], ph, kStatusEpilogueTimeout));
        if (!ok) break;
        tc_fence_after();
        // Two pieces are on their way at a time, and the accumulator is handed back as soon
        // as the last two have landed: their additions run beside the next products.
        const uint32_t at = lanes + static_cast<uint32_t>(acc * kTile);
        TmemPiece even, odd;
        even.issue(at);
        odd.issue(at + 32);
        even.land();
        odd.land();
        even.add_to(sum, scale);
        even.issue(at + 64);
        odd.add_to(sum + 16, scale);
        odd.issue(at + 96);
        even.land();
        odd.land();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(read0 + static_cast<uint32_t>(acc) * 8u);
        even.add_to(sum + 32, scale);
        odd.add_to(sum + 48, scale);
        acc ^= 1;
        if (++st == S) {
          st = 0;
          ph ^= 1u;
        }
      }
      if (!ok) break;
      // To memory by way of shared memory: boxes of 32 rows of 128 bytes, in TMA's 128-byte swizzle.
      constexpr int kCols = OUT_F32 ? 32 : 64;  // of a box
#pragma unroll
      for (int box = 0; box < 128 / kCols; ++box) {
        uint8_t* at = slot + (box % 2) * Cfg::kBoxBytes;
        if (box % 2 == 0) {  // the slot's earlier contents have left it
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float x, y;
            if (OUT_F32) {
              sum[(box * kCols + 4 * c + q) / 2].get(x, y);
              w[q] = __float_as_uint(q % 2 ? y : x);
            } else {
              sum[(box * kCols + 8 * c) / 2 + q].get(x, y);
              w[q] = pack_pair(x, y, out.bf16);
            }
          }
          *reinterpret_cast<uint4*>(at + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const int col = col0 + box * kCols;
        if (out.tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row0 < shape.m && col < shape.n) tma_store_3d(&map_out, at, col, row0, 0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
          constexpr int es = OUT_F32 ? 4 : 2;
          for (int q = 0; q < min(32, shape.m - row0); ++q) {
            const int64_t to = static_cast<int64_t>(row0 + q) * out.ldd + col;
            for (int c = lane; c < min(kCols, shape.n - col); c += 32) {
              const uint8_t* from = at + q * 128 + (((c * es / 16) ^ (q & 7)) << 4) + c * es % 16;
              if (OUT_F32)
                static_cast<uint32_t*>(out.d)[to + c] = *reinterpret_cast<const uint32_t*>(from);
              else
                static_cast<uint16_t*>(out.d)[to + c] = *reinterpret_cast<const uint16_t*>(from);
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  // All roles meet; after an abort, copies and MMAs in flight get time to land.
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (*pipe.abort_flag) settle_for_ns(2000000ull);
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------- few rows
// A tile: 128 features and up to TOK rows of left.
template <int TOK>
struct RowConfig {
  static constexpr uint32_t kRowBytes = TOK * kBlock;
  static constexpr uint32_t kStageBytes = kTileBytes + kRowBytes;
  static constexpr int kStages = 6 * 32768 / kStageBytes;
  static constexpr int kHalf = TOK / 2;  // rows of left that a warp sums
  static constexpr uint32_t kTmemCols = 2 * TOK < 32 ? 32 : 2 * TOK;
  static constexpr uint32_t kScaleBytes = kEpiWarps * 2 * kHalf * 4;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kScaleBytes + Pipe<kStages, false>::kBytes;
  static_assert(kStages * kStageBytes >= TOK * 128 * 4, "the partial sums take the stages' place");
};

// Columns of the thread's TMEM lane, 8, 16 or 32.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "");
  uint32_t r[N];
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
  else if constexpr (N == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
  if constexpr (N < 32) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
  } else {
    tmem_load_32cols(at, v);
  }
}

template <bool M_MN, int TOK, bool OUT_F32>
__global__ void __launch_bounds__(kThreads, 1)
    gemm8_rows_kernel(const __grid_constant__ CUtensorMap map_left, const __grid_constant__ CUtensorMap map_right,
                      const Scales scales, const Shape8 shape, const Out8 out) {
  using Cfg = RowConfig<TOK>;
  constexpr int S = Cfg::kStages;
  // blockIdx.x: the CTA's place in its cluster; y: features; z: rows of left.
  const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
  const int f0 = static_cast<int>(blockIdx.y) * 128, row0 = static_cast<int>(blockIdx.z) * TOK;
  const int rows = min(TOK, shape.m - row0);
  const int b_begin = static_cast<int>(static_cast<int64_t>(part) * shape.blocks / parts);
  const int b_end = static_cast<int>(static_cast<int64_t>(part + 1) * shape.blocks / parts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* smem_scales = reinterpret_cast<float*>(smem + S * Cfg::kStageBytes);
  const Pipe<S, false> pipe(smem + S * Cfg::kStageBytes + Cfg::kScaleBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_left);
    tma_prefetch_desc(&map_right);
    pipe.init();
  }
  if (warp == 1) {
    tmem_alloc(pipe.tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_predecessor();
  const uint32_t tmem = *pipe.tmem_slot;
  const int quarter = warp & 3, half = (warp - 2) >> 2;
  constexpr int kPiece = Cfg::kHalf < 32 ? Cfg::kHalf : 32;  // columns of one TMEM load
  Pair sum[Cfg::kHalf / 2];

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int b = b_begin; b < b_end; ++b) {
        ok = pipe.wait(&pipe.done[st], ph ^ 1u, kStatusProducerTimeout);
        if (!ok) break;
        uint8_t* at = smem + st * Cfg::kStageBytes;
        mbar_arrive_expect_tx(&pipe.full[st], Cfg::kStageBytes);
        if (M_MN)
          tma_load_3d(at, &map_right, &pipe.full[st], f0, b * kBlock, 0);
        else
          tma_load_3d(at, &map_right, &pipe.full[st], b * kBlock, f0, 0);
        tma_load_3d(at + kTileBytes, &map_left, &pipe.full[st], b * kBlock, row0, 0);
        if (++st == S) {
          st = 0;
          ph ^= 1u;
        }
      }
      pipe.drain(st, ph, ok);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_8bit(M_MN, false, 128, (rows + 15) / 16 * 16);
      int st = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      for (int b = b_begin; b < b_end; ++b) {
        if (!pipe.wait(&pipe.full[st], ph, kStatusMmaTimeout) ||
            !pipe.wait(&pipe.read[acc], acc_ph ^ 1u, kStatusMmaTimeout))
          break;
        tc_fence_after();
        const uint8_t* at = smem + st * Cfg::kStageBytes;
        const uint64_t features = tile_desc(at), tokens = tile_desc(at + kTileBytes);
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          mma_8bit(tmem + static_cast<uint32_t>(acc * TOK), features + k * step_of(M_MN), tokens + k * step_of(false), idesc,
                   k > 0 ? 1u : 0u);
        tc_commit(&pipe.done[st]);
        if (++st == S) {
          st = 0;
          ph ^= 1u;
        }
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
    }
  } else {
    // A thread sums a feature for half of the tile's rows of left. The scales of those rows
    // (times the block's own) go to the warp's threads through shared memory.
    float* mine = smem_scales + (warp - 2) * 2 * Cfg::kHalf;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(Cfg::kHalf * half);
    const float* rs = scales.right + f0 / kBlock * scales.right_cstride;
    constexpr int kEach = (Cfg::kHalf + 31) / 32, kAhead = 4;
    const float* ls[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      ls[e] = scales.left + min(row0 + half * Cfg::kHalf + min(32 * e + lane, Cfg::kHalf - 1), shape.m - 1) * scales.left_rstride;
    float l[kAhead][kEach], r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int b = min(b_begin + q, shape.blocks - 1);
      r[q] = rs[b * scales.right_rstride];
#pragma unroll
      for (int e = 0; e < kEach; ++e) l[q][e] = ls[e][b * scales.left_cstride];
    }
#pragma unroll
    for (int q = 0; q < Cfg::kHalf / 2; ++q) sum[q] = Pair(0.0f);
    int st = 0, acc = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int b0 = b_begin; b0 < b_end && ok; b0 += kAhead) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (b0 + q >= b_end || !ok) continue;
        float* now = mine + (q & 1) * Cfg::kHalf;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (32 * e + lane < Cfg::kHalf) now[32 * e + lane] = l[q][e] * r[q];
        const int next = min(b0 + q + kAhead, shape.blocks - 1);
        r[q] = rs[next * scales.right_rstride];
#pragma unroll
        for (int e = 0; e < kEach; ++e) l[q][e] = ls[e][next * scales.left_cstride];
        ok = __all_sync(0xffffffffu, pipe.wait(&pipe.done[st], ph, kStatusEpilogueTimeout));
        if (!ok) continue;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < Cfg::kHalf; c += kPiece) {
          float v[kPiece];
          tmem_load<kPiece>(lanes + static_cast<uint32_t>(acc * TOK + c), v);
#pragma unroll
          for (int e = 0; e < kPiece; e += 4) {
            const float4 s = *reinterpret_cast<const float4*>(now + c + e);
            sum[(c + e) / 2] = fma2(Pair(v[e], v[e + 1]), Pair(s.x, s.y), sum[(c + e) / 2]);
            sum[(c + e) / 2 + 1] = fma2(Pair(v[e + 2], v[e + 3]), Pair(s.z, s.w), sum[(c + e) / 2 + 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pipe.read[acc]);
        acc ^= 1;
        if (++st == S) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
  }
  // Every stage has been multiplied; the sums take their place, a row of left after another.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*pipe.abort_flag) settle_for_ns(2000000ull);
  tc_fence_after();
  float* joined = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
#pragma unroll
    for (int q = 0; q < Cfg::kHalf / 2; ++q) {
      float x, y;
      sum[q].get(x, y);
      float* to = joined + (half * Cfg::kHalf + 2 * q) * 128 + quarter * 32 + lane;
      to[0] = x;
      to[128] = y;
    }
  }
  meet<true>();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
  // The CTAs of the cluster take the rows in turn; a thread adds up two features, the parts
  // in their order.
  if (warp >= 2) {
    const int f = 2 * (threadIdx.x & 63);
    for (int c = part + parts * ((static_cast<int>(threadIdx.x) - 64) >> 6); c < rows; c += parts * (kEpiWarps / 2)) {
      float x = 0.0f, y = 0.0f;
      for (int p = 0; p < parts; ++p) {
        float u, v;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                     : "=f"(u), "=f"(v)
                     : "r"(cluster_addr(joined + c * 128 + f, static_cast<uint32_t>(p)))
                     : "memory");
        x += u;
        y += v;
      }
      const int left = shape.n - f0 - f;
      const int64_t at = static_cast<int64_t>(row0 + c) * out.ldd + f0 + f;
      if (OUT_F32) {
        float* d = static_cast<float*>(out.d) + at;
        if (left > 0) d[0] = x;
        if (left > 1) d[1] = y;
      } else {
        uint16_t* d = static_cast<uint16_t*>(out.d) + at;
        const uint32_t two = pack_pair(x, y, out.bf16);
        if (out.tma && left > 1) {
          *reinterpret_cast<uint32_t*>(d) = two;
        } else {
          if (left > 0) d[0] = static_cast<uint16_t>(two);
          if (left > 1) d[1] = static_cast<uint16_t>(two >> 16);
        }
      }
    }
  }
  meet<true>();  // no CTA leaves while another reads its sums
}

// -------------------------------------------------------------------- launch
std::mutex g_mutex;
constexpr int kDevices = 64, kSlots = 32;
int g_resident[kDevices][kSlots] = {};

template <typename... Params>
int prepare_kernel(void (*kernel)(Params...), int slot, size_t smem, bool pair, int* resident) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kDevices) return fail(GNS_ERR_DEVICE, "device index out of range");
  std::lock_guard<std::mutex> lock(g_mutex);
  int& known = g_resident[dev][slot];
  if (known == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
    int n = device_sm_count();
    if (pair) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.blockDim = dim3(kPairThreads, 1, 1);
      cfg.gridDim = dim3(static_cast<unsigned>(n / 2 * 2), 1, 1);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
      if (n < 1) return fail(GNS_ERR_UNSUPPORTED, "no CTA pair of the 8-bit product fits on the device");
    }
    known = n;
  }
  *resident = known;
  return GNS_OK;
}

struct Call8 {
  CUtensorMap left, right, out_map;
  Scales scales;
  Shape8 shape;
  Out8 out;
};

template <typename... Params, typename... Args>
int launch8(void (*kernel)(Params...), dim3 grid, int threads, int cluster, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
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
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "8-bit product launch");
}

template <bool B_MN, bool OUT_F32>
int launch_pair(const Call8& c, cudaStream_t stream) {
  auto kernel = gemm8_pair_kernel<B_MN, OUT_F32>;
  constexpr size_t smem = PairConfig<OUT_F32>::kSmemBytes;
  int resident = 0;
  const int rc = prepare_kernel(kernel, (B_MN ? 2 : 0) + (OUT_F32 ? 1 : 0), smem, true, &resident);
  if (rc != GNS_OK) return rc;
  const Tiling tiling{(c.shape.m + kTile - 1) / kTile, (c.shape.n + kTile - 1) / kTile};
  const int tiles = tiling.rows * tiling.cols;
  return launch8(kernel, dim3(2u * static_cast<unsigned>(std::min(tiles, resident))), kPairThreads, 2, smem, stream, c.left, c.right,
                 c.out_map, c.scales, c.shape, tiling, c.out);
}

template <bool M_MN, int TOK, bool OUT_F32>
int launch_rows(const Call8& c, int parts, int slot, cudaStream_t stream) {
  auto kernel = gemm8_rows_kernel<M_MN, TOK, OUT_F32>;
  constexpr size_t smem = RowConfig<TOK>::kSmemBytes;
  int resident = 0;
  const int rc = prepare_kernel(kernel, 4 + slot + (M_MN ? 8 : 0) + (OUT_F32 ? 16 : 0), smem, false, &resident);
  if (rc != GNS_OK) return rc;
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>((c.shape.n + 127) / 128),
                  static_cast<unsigned>((c.shape.m + TOK - 1) / TOK));
  return launch8(kernel, grid, kThreads, parts, smem, stream, c.left, c.right, c.scales, c.shape, c.out);
}

template <bool MN, bool F32>
int launch_rows_any(const Call8& c, int tok, int parts, cudaStream_t stream) {
  if (tok == 16) return launch_rows<MN, 16, F32>(c, parts, 0, stream);
  if (tok == 32) return launch_rows<MN, 32, F32>(c, parts, 1, stream);
  if (tok == 64) return launch_rows<MN, 64, F32>(c, parts, 2, stream);
  return launch_rows<MN, 128, F32>(c, parts, 3, stream);
}

struct Plan8 {
  int tok;    // rows of left of a tile of the few-rows kernel; 0: the many-rows kernel
  int parts;  // CTAs that share a tile's contraction
};

Plan8 plan8(int64_t m, int64_t n, int64_t blocks) {
  if (m > 128) return {0, 1};
  const int tok = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128));
  const int64_t tiles = (n + 127) / 128;
  const int sms = device_sm_count();
  int parts = 1;
  while (parts < 8 && tiles * parts * 2 <= sms && blocks >= 2 * parts) parts *= 2;
  return {tok, parts};
}

}  // namespace

int gemm8_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_gemm8_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_gemm8_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "8-bit product status");
}

}  // namespace gns

using namespace gns;

extern "C" {

int gns_gemm_8bit(int64_t m, int64_t n, int64_t k, const void* left, int64_t left_rstride, const float* left_scales,
                  int64_t left_scale_rstride, int64_t left_scale_cstride, const void* right, int64_t right_rstride,
                  int64_t right_cstride, const float* right_scales, int64_t right_scale_rstride,
                  int64_t right_scale_cstride, void* out, int out_dtype, int64_t out_rstride, gns_stream_t stream) {
  clear_error();
  if (out_dtype < 0 || out_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad output dtype");
  if (m < 0 || n < 0 || k < 0) return fail(GNS_ERR_ARGUMENT, "negative dimension");
  if (m > (1 << 30) || n > (1 << 24) || k > (1 << 24)) return fail(GNS_ERR_UNSUPPORTED, "dimension beyond kernel limits");
  if (m == 0 || n == 0) return GNS_OK;
  if (k == 0) return fail(GNS_ERR_UNSUPPORTED, "an 8-bit product needs k > 0");
  if (left == nullptr || right == nullptr || left_scales == nullptr || right_scales == nullptr || out == nullptr)
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (m > 1 && out_rstride < n) return fail(GNS_ERR_LAYOUT, "rows of the output overlap");
  const bool k_major = (right_rstride == 1 || k == 1) && (right_cstride % 16 == 0 || n == 1);
  if (!k_major && !((right_cstride == 1 || n == 1) && (right_rstride % 16 == 0 || k == 1)))
    return fail(GNS_ERR_LAYOUT, "right needs a unit stride along rows or columns and 16-byte multiples along the other");
  int rc = check_device();
  if (rc != GNS_OK) return rc;
  Call8 c{};
  c.scales = {left_scales, right_scales, left_scale_rstride, left_scale_cstride, right_scale_rstride, right_scale_cstride};
  c.shape = {static_cast<int>(m), static_cast<int>(n), static_cast<int>((k + kBlock - 1) / kBlock)};
  c.out = {out, out_rstride, out_dtype == kBF16 ? 1 : 0, 0};
  const Plan8 plan = plan8(m, n, c.shape.blocks);
  rc = encode_byte_tiles(&c.left, left, k, m, left_rstride, plan.tok > 0 ? plan.tok : 128);
  if (rc == GNS_OK)
    rc = k_major ? encode_byte_tiles(&c.right, right, k, n, right_cstride, 128)
                 : encode_byte_tiles(&c.right, right, n, k, right_rstride, 128);
  if (rc != GNS_OK) return rc;
  const int es = dtype_size(out_dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool f32 = out_dtype == kF32;
  if (plan.tok > 0) {
    // Pairs of 16-bit values are stored as one word where rows start on words.
    c.out.tma = reinterpret_cast<uintptr_t>(out) % 4 == 0 && (out_rstride * es) % 4 == 0;
    if (k_major) return f32 ? launch_rows_any<false, true>(c, plan.tok, plan.parts, st) : launch_rows_any<false, false>(c, plan.tok, plan.parts, st);
    return f32 ? launch_rows_any<true, true>(c, plan.tok, plan.parts, st) : launch_rows_any<true, false>(c, plan.tok, plan.parts, st);
  }
  c.out.tma = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (out_rstride * es) % 16 == 0;
  if (c.out.tma) {
    rc = encode_store_tiles(&c.out_map, out_dtype, out, n, m, out_rstride, 32);
    if (rc != GNS_OK) return rc;
  }
  if (k_major) return f32 ? launch_pair<false, true>(c, st) : launch_pair<false, false>(c, st);
  return f32 ? launch_pair<true, true>(c, st) : launch_pair<true, false>(c, st);
}

}  // extern "C"
