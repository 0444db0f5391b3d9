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
// Three kernels. Many rows: a CTA pair computes 256 x 256 tiles of the output, rows of left
// on the MMA's M side, so that a thread's scale is one number a block (its row's, times
// the right block's). Fewer rows: 128 x 128 tiles of a CTA, alike. Up to 32 rows: right's
// columns (a layer's features) are the M side and the rows of left the N side, whose width
// follows them. In the last two a cluster of CTAs may share a tile's contraction; it joins the
// fp32 sums out of shared memory in a fixed order.
//
// The pair kernel, 16384 x 4096 x 14336: 861 us, 2.23 PFLOP/s, at the power cap (1.67 GHz; in a
// run of seconds 1030 us at 1.44 GHz); 717 us, 2.68 PFLOP/s, with operands of zeros, which leave
// the clock at 1.965 GHz: 900 cycles a block of 256 x 256 x 128 a pair. Without the summing it is
// 750, near the 730 that twice the measured rate of a bf16 library product gives (the nominal rate
// gives 512; what keeps either product from it was not found). The other 150 are the hand-over:
// a block's way from its last product to the first one that may overwrite its accumulator is
// 980 cycles of signals between the CTAs and 310 of reading, more than the one block that the
// second accumulator (all of TMEM is two) gives time for.
// Measured and not kept: halves of 128 columns with four accumulators (950 without the summing:
// products 128 wide read the left operand twice as often), sixteen summing warps of 64
// columns (1046 against 962 under the profiler: twice the instructions beside the sums), sums
// one at a time instead of in pairs (1106). A library product with one scale for all, which
// adds nothing up outside of TMEM: 670 us.
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
  int whole; // the output's rows start on 16 bytes (few rows: on words)
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
template <int S, int ACC>
struct Pipe {
  uint64_t* full;  // a stage has landed
  uint64_t* done;  // its products are done
  uint64_t* read;  // the accumulator has been read
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  static constexpr uint32_t kBytes = (2 * S + ACC) * 8 + 8;

  __device__ __forceinline__ explicit Pipe(uint8_t* at) {
    full = reinterpret_cast<uint64_t*>(at);
    done = full + S;
    read = done + S;
    tmem_slot = reinterpret_cast<uint32_t*>(read + ACC);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }

  // readers: the warps that read an accumulator.
  __device__ __forceinline__ void init(uint32_t readers) const {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    for (int a = 0; a < ACC; ++a) mbar_init(&read[a], readers);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }

  // Waits that are not over at once are left to the hardware first, for up to 100 us: lanes that
  // poll take power and issue slots from those that work (operands of zeros 720 -> 705 us).
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int code) const {
    uint32_t over;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(over)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
        : "memory");
    return over != 0 || mbar_wait_bounded(bar, parity, abort_flag, &g_gemm8_status, code);
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

struct PairConfig {
  static constexpr int kStages = 5;
  static constexpr uint32_t kStageBytes = 2 * kTileBytes;
  // A warp's part of the output on its way to memory: 32 rows in two boxes of 128 bytes a row.
  static constexpr uint32_t kBoxBytes = 32 * 128;
  static constexpr uint32_t kSlotBytes = 2 * kBoxBytes;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kSlotBytes + Pipe<kStages, 2>::kBytes;
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
  using Cfg = PairConfig;
  constexpr int S = Cfg::kStages;
  const uint32_t rank = cluster_ctarank();
  const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
  const int tiles = tiling.rows * tiling.cols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_out = smem + S * Cfg::kStageBytes;
  const Pipe<S, 2> pipe(smem_out + kEpiWarps * Cfg::kSlotBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_left);
    tma_prefetch_desc(&map_right);
    pipe.init(2 * kEpiWarps);
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
      for (int left = shape.blocks; left > 0; --left) {
        const Pair scale(l0 * r0);
        l0 = l1;
        r0 = r1;
        if (left > 2) {
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
        if (out.whole) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row0 < shape.m && col < shape.n) tma_store_3d(&map_out, at, col, row0, 0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
          constexpr int es = OUT_F32 ? 4 : 2;
          const int rows = min(32, shape.m - row0), cols = shape.n - col;
          uint8_t* to = static_cast<uint8_t*>(out.d) + (static_cast<int64_t>(row0) * out.ldd + col + lane) * es;
#pragma unroll 8
          for (int q = 0; q < rows; ++q, to += out.ldd * es) {
#pragma unroll
            for (int c = lane; c < lane + kCols; c += 32) {
              if (c >= cols) continue;
              const uint8_t* from = at + q * 128 + (((c * es / 16) ^ (q & 7)) << 4) + c * es % 16;
              if (OUT_F32)
                *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
              else
                *reinterpret_cast<uint16_t*>(to + (c - lane) * es) = *reinterpret_cast<const uint16_t*>(from);
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

// ---------------------------------------------------------------- some rows
// Tiles of 128 rows of left and 128 columns of right, a CTA each, for products whose pair
// tiles would leave SMs idle. As above a thread sums a row of left, 64 columns of it, with one
// scale a block. A cluster of up to 8 CTAs shares a tile's contraction: the partial sums
// are left in shared memory and added up, by rows, in the parts' order.
struct TileConfig {
  static constexpr int kStages = 6;
  static constexpr uint32_t kStageBytes = 2 * kTileBytes;
  // Four accumulators: a block's way from its products through the summing warps and back
  // takes longer than the next one's products.
  static constexpr int kAcc = 4;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + Pipe<kStages, kAcc>::kBytes;
  static_assert(kStages * kStageBytes >= 128 * 128 * 4, "the partial sums take the stages' place");
};

constexpr int kTileThreads = kThreads + 32;

template <bool B_MN, bool OUT_F32>
__global__ void __launch_bounds__(kTileThreads, 1)
    gemm8_tile_kernel(const __grid_constant__ CUtensorMap map_left, const __grid_constant__ CUtensorMap map_right,
                      const Scales scales, const Shape8 shape, const Out8 out) {
  using Cfg = TileConfig;
  constexpr int S = Cfg::kStages;
  // blockIdx.x: the CTA's part of the contraction; y: columns of right; z: rows of left.
  const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
  const int row0 = static_cast<int>(blockIdx.z) * 128, col0 = static_cast<int>(blockIdx.y) * 128;
  // Its blocks are every parts-th, so that what the cluster reads at a time lies together in
  // memory, and tiles begin at different ones, so that not all of them read the same columns
  // of right, which lie in few of the memory's channels.
  const int count = (shape.blocks - part + parts - 1) / parts;
  const int turned = static_cast<int>(blockIdx.y * static_cast<unsigned>(count) / gridDim.y);
  auto block = [&](int i) {
    i += turned;
    return part + (i < count ? i : i - count) * parts;
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const Pipe<S, Cfg::kAcc> pipe(smem + S * Cfg::kStageBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_left);
    tma_prefetch_desc(&map_right);
    pipe.init(kEpiWarps);
  }
  if (warp == 1) {
    tmem_alloc(pipe.tmem_slot, Cfg::kAcc * 128);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait_predecessor();
  const uint32_t tmem = *pipe.tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; i < count; ++i) {
        const int b = block(i);
        ok = pipe.wait(&pipe.done[st], ph ^ 1u, kStatusProducerTimeout);
        if (!ok) break;
        uint8_t* at = smem + st * Cfg::kStageBytes;
        mbar_arrive_expect_tx(&pipe.full[st], Cfg::kStageBytes);
        tma_load_3d(at, &map_left, &pipe.full[st], b * kBlock, row0, 0);
        if (B_MN)
          tma_load_3d(at + kTileBytes, &map_right, &pipe.full[st], col0, b * kBlock, 0);
        else
          tma_load_3d(at + kTileBytes, &map_right, &pipe.full[st], b * kBlock, col0, 0);
        if (++st == S) {
          st = 0;
          ph ^= 1u;
        }
      }
      pipe.drain(st, ph, ok);
    }
  } else if (warp == 1 || warp == 2 + kEpiWarps) {
    // Two warps issue the blocks' products in turn.
    if (lane == 0) {
      const uint32_t idesc = idesc_8bit(false, B_MN, 128, 128);
      const int turn = warp == 1 ? 0 : 1;
      int st = turn, acc = turn;
      uint32_t ph = 0, acc_ph = 0;
      for (int i = turn; i < count; i += 2) {
        if (!pipe.wait(&pipe.full[st], ph, kStatusMmaTimeout) ||
            !pipe.wait(&pipe.read[acc], acc_ph ^ 1u, kStatusMmaTimeout))
          break;
        tc_fence_after();
        const uint8_t* at = smem + st * Cfg::kStageBytes;
        const uint64_t left = tile_desc(at), right = tile_desc(at + kTileBytes);
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          mma_8bit(tmem + static_cast<uint32_t>(acc * 128), left + k * step_of(false), right + k * step_of(B_MN), idesc,
                   k > 0 ? 1u : 0u);
        tc_commit(&pipe.done[st]);
        st += 2;
        if (st >= S) {
          st -= S;
          ph ^= 1u;
        }
        acc += 2;
        if (acc >= Cfg::kAcc) {
          acc -= Cfg::kAcc;
          acc_ph ^= 1u;
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(64 * half);
    const int mine = quarter * 32 + lane;
    const float* ls = scales.left + min(row0 + mine, shape.m - 1) * scales.left_rstride;
    const float* rs = scales.right + col0 / kBlock * scales.right_cstride;
    Pair sum[32];
#pragma unroll
    for (int q = 0; q < 32; ++q) sum[q] = Pair(0.0f);
    // Scales are loaded two blocks ahead of their use.
    float l0 = ls[block(0) * scales.left_cstride], r0 = rs[block(0) * scales.right_rstride], l1 = l0, r1 = r0;
    if (count > 1) {
      l1 = ls[block(1) * scales.left_cstride];
      r1 = rs[block(1) * scales.right_rstride];
    }
    int st = 0, acc = 0;
    uint32_t ph = 0;
    for (int i = 0; i < count; ++i) {
      const Pair scale(l0 * r0);
      l0 = l1;
      r0 = r1;
      if (i + 2 < count) {
        l1 = ls[block(i + 2) * scales.left_cstride];
        r1 = rs[block(i + 2) * scales.right_rstride];
      }
      if (!__all_sync(0xffffffffu, pipe.wait(&pipe.done[st], ph, kStatusEpilogueTimeout))) break;
      tc_fence_after();
      const uint32_t at = lanes + static_cast<uint32_t>(acc * 128);
      TmemPiece even, odd;
      even.issue(at);
      odd.issue(at + 32);
      even.land();
      odd.land();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pipe.read[acc]);
      even.add_to(sum, scale);
      odd.add_to(sum + 16, scale);
      if (++acc == Cfg::kAcc) acc = 0;
      if (++st == S) {
        st = 0;
        ph ^= 1u;
      }
    }
    // Every stage has been multiplied: the sums take their place, rows of 512 bytes whose
    // 16-byte pieces are turned by the row within each 128 bytes.
    uint8_t* to = smem + mine * 512 + half * 256;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      float v[4];
      sum[2 * c].get(v[0], v[1]);
      sum[2 * c + 1].get(v[2], v[3]);
      *reinterpret_cast<float4*>(to + (c / 8) * 128 + (((c % 8) ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*pipe.abort_flag) settle_for_ns(2000000ull);
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, Cfg::kAcc * 128);
  }
  // The cluster's CTAs take the rows in turn, a warp a row, four rows on their way together.
  if (warp >= 2 && warp < 2 + kEpiWarps) {
    const int rows = min(128, shape.m - row0);
    const int col = col0 + lane * 4, left = shape.n - col;
    constexpr int kDeep = 4;
    for (int r0 = part + parts * (warp - 2); r0 < rows; r0 += parts * kEpiWarps * kDeep) {
      float4 v[kDeep];
#pragma unroll
      for (int q = 0; q < kDeep; ++q) v[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int p = 0; p < parts; ++p) {
        float4 u[kDeep];
#pragma unroll
        for (int q = 0; q < kDeep; ++q) {
          const int r = r0 + q * parts * kEpiWarps;
          u[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (r >= rows) continue;
          const uint8_t* at = smem + r * 512 + (lane / 8) * 128 + (((lane % 8) ^ (r & 7)) << 4);
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(u[q].x), "=f"(u[q].y), "=f"(u[q].z), "=f"(u[q].w)
                       : "r"(cluster_addr(at, static_cast<uint32_t>(p)))
                       : "memory");
        }
#pragma unroll
        for (int q = 0; q < kDeep; ++q)
          v[q] = make_float4(v[q].x + u[q].x, v[q].y + u[q].y, v[q].z + u[q].z, v[q].w + u[q].w);
      }
#pragma unroll
      for (int q = 0; q < kDeep; ++q) {
        const int r = r0 + q * parts * kEpiWarps;
        if (r >= rows) continue;
        const int64_t at = static_cast<int64_t>(row0 + r) * out.ldd + col;
        const float one[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        if (OUT_F32) {
          float* d = static_cast<float*>(out.d) + at;
          if (out.whole && left >= 4) {
            *reinterpret_cast<float4*>(d) = v[q];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < left) d[e] = one[e];
          }
        } else {
          uint16_t* d = static_cast<uint16_t*>(out.d) + at;
          if (out.whole && left >= 4) {
            *reinterpret_cast<uint2*>(d) = make_uint2(pack_pair(one[0], one[1], out.bf16), pack_pair(one[2], one[3], out.bf16));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < left) d[e] = float_to_half_bits(one[e], out.bf16);
          }
        }
      }
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
}

// ------------------------------------------------------------------- few rows
// A tile: 128 features and up to TOK rows of left.
template <int TOK>
struct RowConfig {
  static constexpr uint32_t kRowBytes = TOK * kBlock;
  static constexpr uint32_t kStageBytes = kTileBytes + kRowBytes;
  static constexpr int kStages = 3 * 32768 / kStageBytes;  // two CTAs on an SM
  static constexpr int kHalf = TOK / 2;  // rows of left that a warp sums
  // Four accumulators: a block's way from its products through the summing warps and back
  // takes longer than the next one's products.
  static constexpr int kAcc = 4;
  static constexpr uint32_t kTmemCols = kAcc * TOK;
  static constexpr uint32_t kScaleBytes = kEpiWarps * 2 * kHalf * 4;
  static constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kScaleBytes + Pipe<kStages, kAcc>::kBytes;
  static_assert(kStages * kStageBytes >= TOK * 128 * 4, "the partial sums take the stages' place");
};

// Columns of the thread's TMEM lane, 8 or 16.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[N]) {
  static_assert(N == 8 || N == 16, "");
  uint32_t r[N];
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}

template <bool M_MN, int TOK, bool OUT_F32>
__global__ void __launch_bounds__(kThreads, 2)
    gemm8_rows_kernel(const __grid_constant__ CUtensorMap map_left, const __grid_constant__ CUtensorMap map_right,
                      const Scales scales, const Shape8 shape, const Out8 out) {
  using Cfg = RowConfig<TOK>;
  constexpr int S = Cfg::kStages;
  // blockIdx.x: the CTA's place in its cluster; y: features; z: rows of left.
  const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
  const int f0 = static_cast<int>(blockIdx.y) * 128, row0 = static_cast<int>(blockIdx.z) * TOK;
  const int rows = min(TOK, shape.m - row0);
  // Its blocks are every parts-th, so that what the cluster reads at a time lies together in
  // memory, and tiles begin at different ones, so that not all of them read the same columns
  // of right, which lie in few of the memory's channels.
  const int count = (shape.blocks - part + parts - 1) / parts;
  const int turned = static_cast<int>(blockIdx.y * static_cast<unsigned>(count) / gridDim.y);
  auto block = [&](int i) {
    i += turned;
    return part + (i < count ? i : i - count) * parts;
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* smem_scales = reinterpret_cast<float*>(smem + S * Cfg::kStageBytes);
  const Pipe<S, Cfg::kAcc> pipe(smem + S * Cfg::kStageBytes + Cfg::kScaleBytes);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_left);
    tma_prefetch_desc(&map_right);
    pipe.init(kEpiWarps);
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
  constexpr int kHalf = Cfg::kHalf;
  Pair sum[kHalf / 2];

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; i < count; ++i) {
        const int b = block(i);
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
      for (int i = 0; i < count; ++i) {
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
        if (++acc == Cfg::kAcc) {
          acc = 0;
          acc_ph ^= 1u;
        }
      }
    }
  } else {
    // A thread sums a feature for half of the tile's rows of left. The scales of those rows
    // (times the block's own) go to the warp's threads through shared memory.
    float* mine = smem_scales + (warp - 2) * 2 * kHalf;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(kHalf * half);
    const float* rs = scales.right + f0 / kBlock * scales.right_cstride;
    constexpr int kAhead = 4;
    const float* ls = scales.left + min(row0 + half * kHalf + min(lane, kHalf - 1), shape.m - 1) * scales.left_rstride;
    float l[kAhead], r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int b = block(min(q, count - 1));
      r[q] = rs[b * scales.right_rstride];
      l[q] = ls[b * scales.left_cstride];
    }
#pragma unroll
    for (int q = 0; q < kHalf / 2; ++q) sum[q] = Pair(0.0f);
    int st = 0, acc = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int i0 = 0; i0 < count && ok; i0 += kAhead) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (i0 + q >= count || !ok) continue;
        float* now = mine + (q & 1) * kHalf;
        if (lane < kHalf) now[lane] = l[q] * r[q];
        const int next = block(min(i0 + q + kAhead, count - 1));
        r[q] = rs[next * scales.right_rstride];
        l[q] = ls[next * scales.left_cstride];
        ok = __all_sync(0xffffffffu, pipe.wait(&pipe.done[st], ph, kStatusEpilogueTimeout));
        if (!ok) continue;
        __syncwarp();
        tc_fence_after();
        float v[kHalf];
        tmem_load<kHalf>(lanes + static_cast<uint32_t>(acc * TOK), v);
#pragma unroll
        for (int e = 0; e < kHalf; e += 4) {
          const float4 s = *reinterpret_cast<const float4*>(now + e);
          sum[e / 2] = fma2(Pair(v[e], v[e + 1]), Pair(s.x, s.y), sum[e / 2]);
          sum[e / 2 + 1] = fma2(Pair(v[e + 2], v[e + 3]), Pair(s.z, s.w), sum[e / 2 + 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pipe.read[acc]);
        if (++acc == Cfg::kAcc) acc = 0;
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
    for (int q = 0; q < kHalf / 2; ++q) {
      float x, y;
      sum[q].get(x, y);
      float* to = joined + (half * kHalf + 2 * q) * 128 + quarter * 32 + lane;
      to[0] = x;
      to[128] = y;
    }
  }
  cluster_sync_all();
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
        if (out.whole && left > 1) {
          *reinterpret_cast<uint32_t*>(d) = two;
        } else {
          if (left > 0) d[0] = static_cast<uint16_t>(two);
          if (left > 1) d[1] = static_cast<uint16_t>(two >> 16);
        }
      }
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
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
  constexpr size_t smem = PairConfig::kSmemBytes;
  int resident = 0;
  const int rc = prepare_kernel(kernel, (B_MN ? 2 : 0) + (OUT_F32 ? 1 : 0), smem, true, &resident);
  if (rc != GNS_OK) return rc;
  const Tiling tiling{(c.shape.m + kTile - 1) / kTile, (c.shape.n + kTile - 1) / kTile};
  const int tiles = tiling.rows * tiling.cols;
  return launch8(kernel, dim3(2u * static_cast<unsigned>(std::min(tiles, resident))), kPairThreads, 2, smem, stream, c.left,
                 c.right, c.out_map, c.scales, c.shape, tiling, c.out);
}

template <bool M_MN, int TOK, bool OUT_F32>
int launch_rows(const Call8& c, int parts, int slot, cudaStream_t stream) {
  auto kernel = gemm8_rows_kernel<M_MN, TOK, OUT_F32>;
  constexpr size_t smem = RowConfig<TOK>::kSmemBytes;
  int resident = 0;
  const int rc = prepare_kernel(kernel, 4 + slot + (M_MN ? 4 : 0) + (OUT_F32 ? 8 : 0), smem, false, &resident);
  if (rc != GNS_OK) return rc;
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>((c.shape.n + 127) / 128),
                  static_cast<unsigned>((c.shape.m + TOK - 1) / TOK));
  return launch8(kernel, grid, kThreads, parts, smem, stream, c.left, c.right, c.scales, c.shape, c.out);
}

template <bool MN, bool F32>
int launch_rows_any(const Call8& c, int tok, int parts, cudaStream_t stream) {
  if (tok == 16) return launch_rows<MN, 16, F32>(c, parts, 0, stream);
  return launch_rows<MN, 32, F32>(c, parts, 1, stream);
}

template <bool B_MN, bool OUT_F32>
int launch_tiles(const Call8& c, int parts, cudaStream_t stream) {
  auto kernel = gemm8_tile_kernel<B_MN, OUT_F32>;
  constexpr size_t smem = TileConfig::kSmemBytes;
  int resident = 0;
  const int rc = prepare_kernel(kernel, 20 + (B_MN ? 2 : 0) + (OUT_F32 ? 1 : 0), smem, false, &resident);
  if (rc != GNS_OK) return rc;
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>((c.shape.n + 127) / 128),
                  static_cast<unsigned>((c.shape.m + 127) / 128));
  return launch8(kernel, grid, kTileThreads, parts, smem, stream, c.left, c.right, c.scales, c.shape, c.out);
}

struct Plan8 {
  int rows;   // of left in a tile: 16, 32 (few rows), 128 (a CTA) or 256 (a pair)
  int parts;  // CTAs that share a tile's contraction
};

// Which kernel, and how many CTAs share a tile. Microseconds measured on one B200, captured
// calls whose weights come from HBM, m x k x n:
//   up to 32 rows, parts 1 / 2 / 4 / 8: doubled while the CTAs are at most two an SM and each
//   part has two blocks
//     1 x 4096 x 14336   19.0 / 13.3 / 17.8 / 24.5     1 x 14336 x 4096   49.8 / 27.8 / 17.2 / 14.1
//     1 x 1024 x 4096    6.2 / 4.9 / 4.2 / 5.0         32 x 8192 x 512    30.9 / 17.4 / 10.5 / 7.3
//   128-row tiles where there is an SM for each, parts 1 / 2 / 4 against pair tiles: doubled
//   while there are SMs, to four (clusters of 8 leave SMs of a GPC unused, and the join reads
//   the sums at 17 bytes a cycle), and each part has four blocks
//     96 x 14336 x 4096  42.9 / 25.0 / 17.4, 51.7      96 x 4096 x 14336  17.8 / 24.5 / -, 20.2
//     256 x 4096 x 4096  16.8 / 12.2 / 19.6, 18.9      256 x 1024 x 4096  7.9 / 7.2 / 14.4, 8.0
//     96 x 2048 x 512    9.6 / 7.4 / 6.4, 10.4         1024 x 2048 x 2048 11.3 / 16.5 / -, 11.5
//     1024 x 4096 x 4096 34.1 / - / -, 20.2
Plan8 plan8(int64_t m, int64_t n, int64_t blocks) {
  const int sms = device_sm_count();
  const int64_t tiles = (n + 127) / 128;
  int parts = 1;
  if (m <= 32) {
    while (parts < 8 && tiles * parts * 2 <= 2 * sms && blocks >= 4 * parts) parts *= 2;
    return {m <= 16 ? 16 : 32, parts};
  }
  const int64_t all = tiles * ((m + 127) / 128);
  if (all > sms) return {256, 1};
  while (parts < 4 && all * parts * 2 <= sms && blocks >= 8 * parts) parts *= 2;
  return {128, parts};
}

int check_sizes(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(GNS_ERR_ARGUMENT, "negative dimension");
  // A grid has at most 65535 tiles of 128 columns.
  if (m > (1 << 30) || n > 65535 * 128 || k > (1 << 24) || (m + 255) / 256 * ((n + 255) / 256) > (1 << 30))
    return fail(GNS_ERR_UNSUPPORTED, "dimension beyond kernel limits");
  return GNS_OK;
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

int gns_gemm_8bit_plan(int64_t m, int64_t n, int64_t k, int* tile_rows, int* parts) {
  clear_error();
  int rc = check_sizes(m, n, k);
  if (rc != GNS_OK) return rc;
  if (m == 0 || n == 0 || k == 0) return fail(GNS_ERR_UNSUPPORTED, "an empty product has no plan");
  if (tile_rows == nullptr || parts == nullptr) return fail(GNS_ERR_ARGUMENT, "null result");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  const Plan8 plan = plan8(m, n, (k + kBlock - 1) / kBlock);
  *tile_rows = plan.rows;
  *parts = plan.parts;
  return GNS_OK;
}

int gns_gemm_8bit(int64_t m, int64_t n, int64_t k, const void* left, int64_t left_rstride, const float* left_scales,
                  int64_t left_scale_rstride, int64_t left_scale_cstride, const void* right, int64_t right_rstride,
                  int64_t right_cstride, const float* right_scales, int64_t right_scale_rstride,
                  int64_t right_scale_cstride, void* out, int out_dtype, int64_t out_rstride, gns_stream_t stream) {
  clear_error();
  if (out_dtype < 0 || out_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad output dtype");
  int rc = check_sizes(m, n, k);
  if (rc != GNS_OK || m == 0 || n == 0) return rc;
  if (k == 0) return fail(GNS_ERR_UNSUPPORTED, "an 8-bit product needs k > 0");
  if (left == nullptr || right == nullptr || left_scales == nullptr || right_scales == nullptr || out == nullptr)
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (m > 1 && out_rstride < n) return fail(GNS_ERR_LAYOUT, "rows of the output overlap");
  const bool k_major = (right_rstride == 1 || k == 1) && (right_cstride % 16 == 0 || n == 1);
  if (!k_major && !((right_cstride == 1 || n == 1) && (right_rstride % 16 == 0 || k == 1)))
    return fail(GNS_ERR_LAYOUT, "right needs a unit stride along rows or columns and 16-byte multiples along the other");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  Call8 c{};
  c.scales = {left_scales, right_scales, left_scale_rstride, left_scale_cstride, right_scale_rstride, right_scale_cstride};
  c.shape = {static_cast<int>(m), static_cast<int>(n), static_cast<int>((k + kBlock - 1) / kBlock)};
  c.out = {out, out_rstride, out_dtype == kBF16 ? 1 : 0, 0};
  const Plan8 plan = plan8(m, n, c.shape.blocks);
  rc = encode_byte_tiles(&c.left, left, k, m, left_rstride, std::min(plan.rows, 128));
  if (rc == GNS_OK)
    rc = k_major ? encode_byte_tiles(&c.right, right, k, n, right_cstride, 128)
                 : encode_byte_tiles(&c.right, right, n, k, right_rstride, 128);
  if (rc != GNS_OK) return rc;
  const int es = dtype_size(out_dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool f32 = out_dtype == kF32;
  if (plan.rows <= 32) {
    // Pairs of 16-bit values are stored as one word where rows start on words.
    c.out.whole = reinterpret_cast<uintptr_t>(out) % 4 == 0 && (out_rstride * es) % 4 == 0;
    if (k_major) return f32 ? launch_rows_any<false, true>(c, plan.rows, plan.parts, st) : launch_rows_any<false, false>(c, plan.rows, plan.parts, st);
    return f32 ? launch_rows_any<true, true>(c, plan.rows, plan.parts, st) : launch_rows_any<true, false>(c, plan.rows, plan.parts, st);
  }
  c.out.whole = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (out_rstride * es) % 16 == 0;
  if (plan.rows == 128) {
    if (k_major) return f32 ? launch_tiles<false, true>(c, plan.parts, st) : launch_tiles<false, false>(c, plan.parts, st);
    return f32 ? launch_tiles<true, true>(c, plan.parts, st) : launch_tiles<true, false>(c, plan.parts, st);
  }
  if (c.out.whole) {
    rc = encode_store_tiles(&c.out_map, out_dtype, out, n, m, out_rstride, 32);
    if (rc != GNS_OK) return rc;
  }
  if (k_major) return f32 ? launch_pair<false, true>(c, st) : launch_pair<false, false>(c, st);
  return f32 ? launch_pair<true, true>(c, st) : launch_pair<true, false>(c, st);
}

}  // extern "C"
