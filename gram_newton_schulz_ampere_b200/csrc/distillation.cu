// Distillation from a teacher's top logits: the loss of each row and its gradient.
//
//   p = softmax over the row's entries of t / T        q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_j p_j (log p_j - log q[i_j])
//   dz_i = g T (q_i - sum of the p_j whose index is i)
//
// An entry whose index is not in the vocabulary has no part in a row; a row without entries
// (or whose entries' logits are all -inf) has a loss and a gradient of zero, whatever its
// logits hold.
//
// One pass over a row finds its largest logit m and s = sum exp((z - m) / T) together (each
// thread rescales its sum when its maximum grows); a second one writes the gradient. z - m is
// formed before it is scaled: z / T would lose the digits that large logits have in common.
//
// A CTA has a row, so that both passes of a call with a gradient run while the row is in L2 and
// it comes from memory once. Rows of more than 160 KB then have an SM each, of 32 warps: with
// two CTAs an SM, 296 rows on their way, a third of the logits came from memory twice (4096 x
// 131072 bf16 499 us against 434 then; 4096 x 65536 the other way round: 233 against 270). Many rows of
// up to 64 KB have CTAs of four warps (8192 x 8192 bf16, loss alone, 37 us; eight warps 54, sixteen 88).
// Few rows: a cluster of CTAs shares a row and exchanges (m, s) through shared memory (1 x
// 131072 bf16: 7 us).
//
// Logits reach the registers through rings in shared memory, one of each warp, that bulk
// copies fill two slots of two kilobytes ahead, over the ends of passes and rows. Under way on an
// SM, whatever the warps wait for: 124 KB with a CTA of thirty-two warps, 120 with two of sixteen,
// 96 with eight of four (of which the lists of 1024 entries a row, 48 KB a CTA, leave room for
// three: 36). Loaded to registers four pieces ahead: 4096 x 131072 551 us. Three slots instead of
// two: 2368 x 131072 fp32, loss alone, 210 us against 181.
//
// What a row's entries ask for is a warp's own work, beside the other warps' passes: read and
// turned into shares two rows ahead, the loss, and the gradient's corrections (with the teacher
// and the logits at the entries read when they are needed: 475 us against 434 then). For each
// entry the gradient's part walks the row's list, top^2 / 128 steps a lane: hidden behind
// the passes up to some 64 entries, the bound beyond (8192 x 4096 bf16, loss and gradient, 16, 64,
// 256 and 1024 entries a row: 59, 70, 303 and 9900 us; 8192 x 32000: 231, 240, 420 and 10060).
//
// Bound by HBM: loss alone 5.6 TB/s (bf16) to 7 (fp32), 4096 x 131072 with the gradient 428 us
// (2.15 GB, 5.0 TB/s): between its two passes a row's SM has less than the rings hold to wait
// for. (The next row brought into L2 during the second pass: 474 us.)
//
// The gradient at the row's entries is written over the dense one behind a barrier, the
// entries of one index added up by the first of them in the list's order: no atomics.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

__device__ int g_loss_status = 0;

constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kSlots = 2;                      // of a warp's ring
constexpr int kSlotPieces = 128;               // 16-byte pieces of a slot
constexpr int kEach = kSlotPieces / 32;        // of a lane
constexpr uint32_t kSlotBytes = kSlotPieces * 16;
constexpr int kWarpsPerSm = 32;

struct LossArgs {
  const void* z;
  int64_t z_stride;
  const void* index;
  const void* teacher;
  int64_t index_stride, teacher_stride;
  const float* grad;     // null without a gradient
  float* loss;           // null in a backward pass
  float2* stats;         // (m, s): written with the loss (may be null), read by a backward pass
  void* dz;
  int64_t dz_stride;
  int64_t rows;
  int vocabulary, top, index64, teacher_dt;
  float temperature, scale;  // scale: log2(e) / T
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A largest value and the sum of exp((z - m) / T) of some logits.
struct Stat {
  float m, s;
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.0f : m; }
  __device__ __forceinline__ void join(float m2, float s2, float scale) {
    const float top = fmaxf(m, m2);
    const float at = top == -INFINITY ? 0.0f : top;
    s = s * exp2_approx((m - at) * scale) + s2 * exp2_approx((m2 - at) * scale);
    m = top;
  }
};

// Sixteen bytes of logits.
template <int XD>
struct Logits {
  static constexpr int kN = XD == kF32 ? 4 : 8;
  uint4 u;

  __device__ __forceinline__ Pair pair(int q) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (XD == kF32) return Pair(__uint_as_float(w[2 * q % 4]), __uint_as_float(w[(2 * q + 1) % 4]));
    const uint32_t two = w[q % 4];
    if (XD == kBF16) return Pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
    return Pair(f.x, f.y);
  }

  static __device__ __forceinline__ uint4 minus_infinity() {
    const uint32_t w = XD == kF32 ? 0xff800000u : (XD == kBF16 ? 0xff80ff80u : 0xfc00fc00u);
    return make_uint4(w, w, w, w);
  }
};

// The largest of K pieces' elements that is not a NaN.
template <int XD, int K>
__device__ __forceinline__ float largest(const Logits<XD> (&p)[K]) {
  if (XD == kF32) {
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < K; ++q)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(p[q].u.x), __uint_as_float(p[q].u.y)),
                         fmaxf(__uint_as_float(p[q].u.z), __uint_as_float(p[q].u.w))));
    return m;
  }
  using Two = typename std::conditional<XD == kBF16, __nv_bfloat162, __half2>::type;
  Two m = *reinterpret_cast<const Two*>(&p[0].u.x);
#pragma unroll
  for (int q = 0; q < K; ++q) {
    const Two* h = reinterpret_cast<const Two*>(&p[q].u);
    m = __hmax2(m, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  }
  return fmaxf(static_cast<float>(m.x), static_cast<float>(m.y));
}

template <int XD>
__device__ __forceinline__ uint4 packed(const float (&v)[XD == kF32 ? 4 : 8]) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    constexpr int kN = XD == kF32 ? 4 : 8;
    if (XD == kF32) {
      w[q] = __float_as_uint(v[q]);
    } else if (XD == kBF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * q % kN], v[(2 * q + 1) % kN]);
      w[q] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * q % kN], v[(2 * q + 1) % kN]);
      w[q] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The lanes' statistics as one: the largest value first, then the sums relative to it. The
// product is rounded before it is added, so that all lanes come to the same bits.
__device__ __forceinline__ Stat warp_join(Stat st, float scale) {
  const Stat all{warp_max(st.m), 0.0f};
  return {all.m, warp_add(__fmul_rn(st.s, exp2_approx((st.m - all.base()) * scale)))};
}

// A row's entries in shared memory: the index (-1: left out), the share p, d = t - the largest
// t, and the logit z. The gradient at the entries takes the places of d and z once the loss
// is formed: its index (-1: none to be written) and its value.
struct Entries {
  int* index;
  float* p;
  float* d;
  float* z;
  float* log_sum;  // of exp(d / T); behind it whether any entry counts
  static __host__ __device__ constexpr int padded(int top) { return (top + 3) / 4 * 4; }
  static __host__ __device__ constexpr uint32_t bytes(int top) { return static_cast<uint32_t>(padded(top) * 16 + 16); }
  __device__ __forceinline__ Entries(uint8_t* at, int top)
      : index(reinterpret_cast<int*>(at)),
        p(reinterpret_cast<float*>(at) + padded(top)),
        d(p + padded(top)),
        z(d + padded(top)),
        log_sum(z + padded(top)) {}
  __device__ __forceinline__ int& some() const { return reinterpret_cast<int*>(log_sum)[1]; }
  __device__ __forceinline__ int* where() const { return reinterpret_cast<int*>(d); }
};

// One warp fills a row's entries, four of a lane's on their way together.
template <int XD>
__device__ __forceinline__ void fill_entries(const Entries& e, const LossArgs& a, int64_t row, int lane) {
  constexpr int kTogether = 4;
  const uint8_t* z = static_cast<const uint8_t*>(a.z) + row * a.z_stride * (XD == kF32 ? 4 : 2);
  float top = -INFINITY;
  bool some = false;
  for (int j0 = lane; j0 < e.padded(a.top); j0 += 32 * kTogether) {
    int index[kTogether];
    float t[kTogether], at[kTogether];
#pragma unroll
    for (int q = 0; q < kTogether; ++q) {
      const int j = j0 + 32 * q;
      index[q] = -1;
      if (j >= a.top) continue;
      const int64_t place = row * a.index_stride + j;
      const int64_t i = a.index64 ? static_cast<const int64_t*>(a.index)[place] : static_cast<const int32_t*>(a.index)[place];
      if (i >= 0 && i < a.vocabulary) index[q] = static_cast<int>(i);
    }
#pragma unroll
    for (int q = 0; q < kTogether; ++q) {
      t[q] = index[q] >= 0 ? load_as_float(a.teacher, row * a.teacher_stride + j0 + 32 * q, a.teacher_dt) : -INFINITY;
      at[q] = index[q] >= 0 ? load_as_float(z, index[q], XD) : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < kTogether; ++q) {
      const int j = j0 + 32 * q;
      if (j >= e.padded(a.top)) continue;
      e.index[j] = t[q] == -INFINITY ? -1 : index[q];  // a share of zero
      e.d[j] = t[q];
      e.z[j] = at[q];
      top = fmaxf(top, t[q]);
      some |= !(t[q] == -INFINITY);  // a NaN counts
    }
  }
  top = warp_max(top);
  some = __any_sync(0xffffffffu, some);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int j = lane; j < e.padded(a.top); j += 32) {
    const float d = e.d[j] - base, p = exp2_approx(d * a.scale);
    e.d[j] = d;
    e.p[j] = p;
    sum += p;
  }
  sum = warp_add(sum);
  const float inv = __fdiv_rn(1.0f, sum);
  for (int j = lane; j < e.padded(a.top); j += 32) e.p[j] *= inv;
  if (lane == 0) {
    *e.log_sum = logf(sum);
    e.some() = some ? 1 : 0;
  }
  __syncwarp();
}

// What a CTA has of a row: `head` elements up to a multiple of 16 bytes (CTA 0), the pieces
// [lo, hi) behind them, and what is left at the end (the last CTA).
template <int XD>
struct Share {
  static constexpr int es = XD == kF32 ? 4 : 2;
  const uint8_t* z;
  int head, pieces, lo, hi;

  __device__ __forceinline__ Share(const LossArgs& a, int64_t row, uint32_t rank, uint32_t ctas) {
    z = static_cast<const uint8_t*>(a.z) + row * a.z_stride * es;
    head = min(a.vocabulary, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(z) & 15u)) & 15u) / es);
    pieces = (a.vocabulary - head) / (16 / es);
    // At most 2^26 pieces and 8 CTAs.
    lo = ctas == 1 ? 0 : static_cast<int>(rank * static_cast<uint32_t>(pieces) / ctas);
    hi = ctas == 1 ? pieces : static_cast<int>((rank + 1) * static_cast<uint32_t>(pieces) / ctas);
  }
  __device__ __forceinline__ const uint8_t* body() const { return z + head * es; }
  __device__ __forceinline__ int slots() const { return (hi - lo + kSlotPieces - 1) / kSlotPieces; }
};

// A bulk load of what is not read again: the first to leave L2.
__device__ __forceinline__ void bulk_load_last(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b64 policy;\n\t"
      "createpolicy.fractional.L2::evict_first.b64 policy, 1.0;\n\t"
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], policy;\n\t"
      "}\n" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// A warp's ring. It asks for what the warp will read, in that order: its slots of a row (every
// S-th), as often as there are passes, then the next row's.
template <int XD, int S, int PASSES, bool LEAVE>
struct WarpRing {
  uint64_t* full;
  uint8_t* slots;
  volatile int* abort_flag;
  int next = 0, last = 0, under_way = 0;  // slot to be read, slot to be filled, copies not yet read
  uint32_t phase = 0;
  // What is asked for next.
  int64_t row, step;
  int pass = 0, at, count;
  const uint8_t* from;
  int left;  // pieces from `from` on to the end of the CTA's share

  __device__ __forceinline__ void enter(const LossArgs& a, uint32_t rank, uint32_t ctas, int warp) {
    pass = 0;
    at = warp;
    count = 0;
    if (row >= a.rows) return;
    const Share<XD> s(a, row, rank, ctas);
    count = s.slots();
    from = s.body() + static_cast<int64_t>(s.lo) * 16;
    left = s.hi - s.lo;
  }

  // Asks for the next slot; every lane keeps count, the first one copies.
  __device__ __forceinline__ void fetch(const LossArgs& a, uint32_t rank, uint32_t ctas, int warp, int lane) {
    while (row < a.rows && at >= count) {
      at = warp;
      if (++pass == PASSES || count <= warp) {
        row += step;
        enter(a, rank, ctas, warp);
      }
    }
    if (row >= a.rows) return;
    if (lane == 0) {
      const uint32_t bytes = static_cast<uint32_t>(min(kSlotPieces, left - at * kSlotPieces)) * 16u;
      mbar_arrive_expect_tx(&full[last], bytes);
      const uint8_t* piece = from + static_cast<int64_t>(at) * kSlotBytes;
      if (LEAVE && pass == 1)
        bulk_load_last(slots + last * kSlotBytes, piece, bytes, &full[last]);
      else
        bulk_load(slots + last * kSlotBytes, piece, bytes, &full[last]);
    }
    last = last + 1 == kSlots ? 0 : last + 1;
    ++under_way;
    at += S;
  }

  __device__ __forceinline__ void wait() const {
    mbar_wait_bounded(&full[next], (phase >> next) & 1u, abort_flag, &g_loss_status, kStatusProducerTimeout);
  }

  // The lane's pieces of the slot, of which the first `live` are the row's: the others -inf.
  __device__ __forceinline__ void read(Logits<XD> (&p)[kEach], int live, int lane) const {
    wait();
    const uint4* slot = reinterpret_cast<const uint4*>(slots + next * kSlotBytes);
    if (live >= kSlotPieces) {
#pragma unroll
      for (int q = 0; q < kEach; ++q) p[q].u = slot[lane + 32 * q];
    } else {
#pragma unroll
      for (int q = 0; q < kEach; ++q) p[q].u = lane + 32 * q < live ? slot[lane + 32 * q] : Logits<XD>::minus_infinity();
    }
    __syncwarp();
  }

  __device__ __forceinline__ void done() {
    phase ^= 1u << next;
    next = next + 1 == kSlots ? 0 : next + 1;
    --under_way;
  }

  // Leaves a row out: what has come of it is thrown away, what has not been asked for is not.
  __device__ __forceinline__ void skip(const LossArgs& a, int64_t of, int slots_of_row, uint32_t rank, uint32_t ctas, int warp,
                                       int lane) {
    int mine = PASSES * (slots_of_row > warp ? (slots_of_row - warp + S - 1) / S : 0);
    const bool here = row == of;
    if (here) mine = under_way;
    for (int i = 0; i < mine; ++i) {
      wait();
      done();
      __syncwarp();
      if (!here) fetch(a, rank, ctas, warp, lane);
    }
    if (here) {
      row += step;
      enter(a, rank, ctas, warp);
      for (int i = 0; i < kSlots; ++i) fetch(a, rank, ctas, warp, lane);
    }
  }
};

// Barrier `id` of the CTA's named ones: both halves, or the arrival alone.
template <int THREADS>
__device__ __forceinline__ void named_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void named_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}

// MODE 1: loss. 2: gradient from the statistics of an earlier call. 3: both.
// LEAVE: what the second pass has read leaves L2 first.
// W: warps of a CTA. All but the last stream the logits; the last one has the rows' entries: it
// reads those of the row after the next, forms the loss, and corrects the gradient at the
// entries, while the others are at work. They meet once a row, between its passes (kMeet):
// there the row's statistics are complete, and the next row's entries in place. The streaming
// warps do not wait for the corrections; they tell when a row's gradient is written (kWritten),
// and the next meeting comes after its corrections.
template <int XD, int MODE, int W, bool LEAVE>
__global__ void __launch_bounds__(32 * W, kWarpsPerSm / W) distillation_kernel(const LossArgs a) {
  constexpr bool kLoss = (MODE & 1) != 0, kGrad = (MODE & 2) != 0;
  constexpr int kPasses = MODE == 3 ? 2 : 1, S = W - 1, kThreads = 32 * W;
  constexpr int kMeet = 1, kWritten = 2;
  using L = Logits<XD>;
  constexpr int N = L::kN;
  constexpr int es = XD == kF32 ? 4 : 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 warps[2][S];
  __shared__ float2 parts[kMaxCluster];
  __shared__ int aborted;
  const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
  const int64_t step = gridDim.x / ctas, first = blockIdx.x / ctas;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  uint64_t* barriers = reinterpret_cast<uint64_t*>(smem + S * kSlots * kSlotBytes);
  uint8_t* lists = smem + S * kSlots * kSlotBytes + (S * kSlots * 8 + 15) / 16 * 16;
  auto list = [&](int which) { return Entries(lists + which * Entries::bytes(a.top), a.top); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < S * kSlots; ++i) mbar_init(&barriers[i], 1);
    aborted = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  // In a cluster, every CTA has begun before another writes to its shared memory.
  if (ctas > 1)
    cluster_sync_all();
  else
    __syncthreads();
  WarpRing<XD, S, kPasses, LEAVE> ring;
  if (warp == S) {
    if (first < a.rows) fill_entries<XD>(list(0), a, first, lane);
  } else {
    ring.full = barriers + warp * kSlots;
    ring.slots = smem + warp * kSlots * kSlotBytes;
    ring.abort_flag = &aborted;
    ring.row = first;
    ring.step = step;
    ring.enter(a, rank, ctas, warp);
    for (int i = 0; i < kSlots; ++i) ring.fetch(a, rank, ctas, warp, lane);
  }
  __syncthreads();
  int turn = 0, which = 0;
  // A row's statistics from the streaming warps' and, in a cluster, the CTAs'. A cluster has one
  // row (row_cluster), so the exchange is made once.
  auto joined = [&]() {
    const float2 one = lane < S ? warps[turn][lane] : make_float2(-INFINITY, 0.0f);
    Stat st = warp_join(Stat{one.x, one.y}, a.scale);
    if (ctas > 1) {
      if (threadIdx.x < ctas)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr(&parts[rank], threadIdx.x)),
                     "f"(st.m), "f"(st.s)
                     : "memory");
      __syncwarp();
      cluster_sync_all();
      st = {-INFINITY, 0.0f};
      for (uint32_t c = 0; c < ctas; ++c) st.join(parts[c].x, parts[c].y, a.scale);
    }
    return st;
  };

  if (warp == S) {
    if (first + step < a.rows) fill_entries<XD>(list(1), a, first + step, lane);
    for (int64_t row = first; row < a.rows; row += step, turn ^= 1, which = which == 2 ? 0 : which + 1) {
      const Share<XD> share(a, row, rank, ctas);
      const Entries e = list(which);
      const bool some = e.some() != 0;
      Stat st{-INFINITY, 0.0f};
      const float2 known = !kLoss && some ? a.stats[row] : make_float2(0.0f, 0.0f);
      const float g = kGrad && some ? a.grad[row] * a.temperature : 0.0f;
      named_sync<kThreads>(kMeet);
      if (!some) {
        if (kLoss && rank == 0 && lane == 0) {
          a.loss[row] = 0.0f;
          if (a.stats != nullptr) a.stats[row] = make_float2(0.0f, 0.0f);
        }
      } else if (kLoss) {
        st = joined();
        if (rank == 0) {
          // log2(e) / T times T is log2(e): exponents are differences over T.
          const float inv_t = 1.0f / a.temperature, log_s = logf(st.s);
          float sum = 0.0f;
          for (int j = lane; j < a.top; j += 32) {
            if (e.index[j] < 0) continue;
            const float log_p = e.d[j] * inv_t - *e.log_sum;
            const float log_q = (e.z[j] - st.m) * inv_t - log_s;
            if (e.p[j] != 0.0f) sum = fmaf(e.p[j], log_p - log_q, sum);
          }
          sum = warp_add(sum);
          if (lane == 0) {
            a.loss[row] = a.temperature * a.temperature * sum;
            if (a.stats != nullptr) a.stats[row] = make_float2(st.m, st.s);
          }
        }
      } else {
        st = {known.x, known.y};
      }
      if (kGrad && some) {
        // The gradient at the entries of this CTA's stretch, each by its first place in the list.
        __syncwarp();
        const float at = st.base(), inverse = __fdiv_rn(1.0f, st.s);
        const int begin = rank == 0 ? 0 : share.head + share.lo * N;
        const int end = rank + 1 == ctas ? a.vocabulary : share.head + share.hi * N;
        for (int j = lane; j < a.top; j += 32) {
          const int i = e.index[j];
          const bool mine = i >= begin && i < end;
          int first_place = j;
          float p = 0.0f;
          for (int k = 0; k < e.padded(a.top); k += 4) {
            const int4 four = *reinterpret_cast<const int4*>(e.index + k);
            if (four.x != i && four.y != i && four.z != i && four.w != i) continue;
            const int other[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (other[q] != i) continue;
              first_place = min(first_place, k + q);
              p += e.p[k + q];
            }
          }
          const float q = exp2_approx((e.z[j] - at) * a.scale) * inverse;
          e.where()[j] = mine && first_place == j ? i : -1;
          e.z[j] = (q - p) * g;
        }
      }
      if (row + 2 * step < a.rows) fill_entries<XD>(list(which == 0 ? 2 : which - 1), a, row + 2 * step, lane);
      if (!kGrad) continue;
      named_sync<kThreads>(kWritten);
      if (!some) continue;
      uint8_t* dz = static_cast<uint8_t*>(a.dz) + row * a.dz_stride * es;
      for (int j = lane; j < a.top; j += 32)
        if (e.where()[j] >= 0) store_from_float(dz, e.where()[j], XD, e.z[j]);
    }
  } else {
    for (int64_t row = first; row < a.rows; row += step, turn ^= 1, which = which == 2 ? 0 : which + 1) {
      const Share<XD> share(a, row, rank, ctas);
      const uint8_t* z = share.z;
      const int slots = share.slots();
      // This thread's element outside the pieces: of the head (CTA 0) or the rest (the last CTA).
      const int rest = share.head + share.pieces * N + static_cast<int>(threadIdx.x) - 32;
      const int lone = rank == 0 && threadIdx.x < static_cast<unsigned>(share.head) ? static_cast<int>(threadIdx.x)
                       : rank + 1 == ctas && threadIdx.x >= 32 && rest < a.vocabulary ? rest
                                                                                      : -1;
      const float alone = lone >= 0 ? load_as_float(z, lone, XD) : 0.0f;
      const float grad = kGrad ? a.grad[row] : 0.0f;
      const bool some = list(which).some() != 0;
      Stat st{-INFINITY, 0.0f};
      if (!kLoss) {
        const float2 known = a.stats[row];
        st = {known.x, known.y};
      }
      if (!some) ring.skip(a, row, slots, rank, ctas, warp, lane);
      if (kLoss && some) {
        for (int c = warp; c < slots; c += S) {
          L now[kEach];
          ring.read(now, share.hi - share.lo - c * kSlotPieces, lane);
          ring.done();
          ring.fetch(a, rank, ctas, warp, lane);
          const float top = largest<XD, kEach>(now);
          if (top > st.m) {
            st.s *= exp2_approx((st.m - top) * a.scale);
            st.m = top;
          }
          const Pair at(-st.base());
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int q = 0; q < kEach; ++q)
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
              float x, y;
              mul2(add2(now[q].pair(k), at), Pair(a.scale)).get(x, y);
              sum[2 * (q % 2)] += exp2_approx(x);
              sum[2 * (q % 2) + 1] += exp2_approx(y);
            }
          st.s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        // A NaN leaves the maximum and makes the sum one.
        if (lone >= 0) st.join(alone == alone ? alone : -INFINITY, alone == alone ? 1.0f : alone, a.scale);
        st = warp_join(st, a.scale);
        if (lane == 0) warps[turn][warp] = make_float2(st.m, st.s);
      }
      named_sync<kThreads>(kMeet);
      if (kLoss && some) st = joined();
      if (!kGrad) continue;
      uint8_t* dz = static_cast<uint8_t*>(a.dz) + row * a.dz_stride * es;
      const float at = st.base(), factor = some ? __fdiv_rn(1.0f, st.s) * (grad * a.temperature) : 0.0f;
      // Pieces of the gradient lie on 16 bytes where its rows start as the logits' do.
      const bool alike = ((reinterpret_cast<uintptr_t>(dz) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
      for (int c = warp; c < slots; c += S) {
        const int live = share.hi - share.lo - c * kSlotPieces;
        uint8_t* to = dz + share.head * es + (static_cast<int64_t>(share.lo) + c * kSlotPieces + lane) * 16;
        if (!some) {
#pragma unroll
          for (int q = 0; q < kEach; ++q) {
            if (lane + 32 * q >= live) continue;
            if (alike) {
              __stcs(reinterpret_cast<uint4*>(to + 512 * q), make_uint4(0u, 0u, 0u, 0u));
            } else {
#pragma unroll
              for (int k = 0; k < N; ++k) store_from_float(to + 512 * q, k, XD, 0.0f);
            }
          }
          continue;
        }
        L now[kEach];
        ring.read(now, live, lane);
        ring.done();
        ring.fetch(a, rank, ctas, warp, lane);
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          float v[N];
#pragma unroll
          for (int k = 0; k < N; k += 2) {
            float x, y;
            mul2(add2(now[q].pair(k / 2), Pair(-at)), Pair(a.scale)).get(x, y);
            mul2(Pair(exp2_approx(x), exp2_approx(y)), Pair(factor)).get(v[k], v[k + 1]);
          }
          if (lane + 32 * q >= live) continue;
          if (alike) {
            // Written for a later kernel: the rows that are read again are to stay in L2.
            __stcs(reinterpret_cast<uint4*>(to + 512 * q), packed<XD>(v));
          } else {
#pragma unroll
            for (int k = 0; k < N; ++k) store_from_float(to + 512 * q, k, XD, v[k]);
          }
        }
      }
      if (lone >= 0) store_from_float(dz, lone, XD, some ? exp2_approx((alone - at) * a.scale) * factor : 0.0f);
      __threadfence_block();
      named_arrive<kThreads>(kWritten);
    }
  }
  __syncthreads();
  if (aborted) settle_for_ns(2000000ull);
}

// CTAs that share a row: one where there are rows for all CTAs that fit; else up to eight, each
// with 8 KB of it at least. Where more than one shares a row, every row has a cluster of its own.
int row_cluster(int64_t rows, int64_t vocabulary, int dt, int ctas) {
  const int64_t bytes = vocabulary * dtype_size(dt);
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= ctas && bytes / (2 * c) >= 8192) c *= 2;
  return c;
}

// Bytes of rows under way at one time: beyond this L2 has too little room for their gradients,
// unless what the second pass has read goes first. 2000 x 131072 fp32 (76 MB under way) 458 -> 403
// us, 2000 x 100000 320 -> 295, 5000 x 32000 bf16 (76 MB) 162 -> 143; below it the hint costs: 4000
// x 65536 fp32 (38 MB) 377 us, with it 388, 4096 x 131072 bf16 (38 MB) 428 and 434.
constexpr int64_t kUnderWay = 48ll << 20;

std::mutex g_mutex;

template <int XD, int MODE, int W, bool LEAVE>
int launch_kernel(const LossArgs& a, int ctas, int cluster, cudaStream_t stream) {
  auto kernel = distillation_kernel<XD, MODE, W, LEAVE>;
  constexpr size_t rings = (W - 1) * kSlots * kSlotBytes + ((W - 1) * kSlots * 8 + 15) / 16 * 16;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(GNS_ERR_DEVICE, "device index out of range");
  {
    static bool ready[64] = {};
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!ready[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(rings + 3 * Entries::bytes(kMaxTop)));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      ready[dev] = true;
    }
  }
  const int resident = ctas / cluster;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * std::min<int64_t>(a.rows, std::max(1, resident))));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = rings + 3 * Entries::bytes(a.top);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "distillation loss kernel");
}

template <int XD, int MODE, int W>
int launch(const LossArgs& a, cudaStream_t stream) {
  const int ctas = kWarpsPerSm / W * device_sm_count();
  const int cluster = W == 4 ? 1 : row_cluster(a.rows, a.vocabulary, XD, ctas);
  // Two CTAs of sixteen warps an SM, with rows of at most 160 KB, stay below on 148 SMs (46 MB).
  if constexpr (MODE == 3 && W != 16) {
    if (std::min<int64_t>(a.rows, ctas / cluster) * a.vocabulary * dtype_size(XD) > kUnderWay)
      return launch_kernel<XD, MODE, W, true>(a, ctas, cluster, stream);
  }
  return launch_kernel<XD, MODE, W, false>(a, ctas, cluster, stream);
}

// Warps of a CTA by the row's length (measured at the top of this file).
template <int XD, int MODE>
int launch_rows(const LossArgs& a, cudaStream_t stream) {
  if (a.vocabulary * dtype_size(XD) <= 65536 && a.rows > 2 * device_sm_count()) return launch<XD, MODE, 4>(a, stream);
  if constexpr (MODE == 3) {
    if (a.vocabulary * dtype_size(XD) > 160 * 1024) return launch<XD, MODE, 32>(a, stream);
  }
  return launch<XD, MODE, 16>(a, stream);
}

template <int MODE>
int launch_any(int dt, const LossArgs& a, cudaStream_t stream) {
  if (dt == kBF16) return launch_rows<kBF16, MODE>(a, stream);
  if (dt == kF16) return launch_rows<kF16, MODE>(a, stream);
  return launch_rows<kF32, MODE>(a, stream);
}

}  // namespace

int loss_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_loss_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_loss_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "distillation loss status");
}

}  // namespace gns

using namespace gns;

extern "C" int gns_distillation_loss(int z_dtype, int64_t rows, int64_t vocabulary, int64_t top, const void* logits,
                                     int64_t logits_rstride, const void* indices, int index_bits, int64_t indices_rstride,
                                     const void* teacher, int teacher_dtype, int64_t teacher_rstride, float temperature,
                                     const float* grad, float* loss, float* stats, void* dlogits, int64_t dlogits_rstride,
                                     gns_stream_t stream) {
  clear_error();
  if (z_dtype < 0 || z_dtype > 2 || teacher_dtype < 0 || teacher_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad dtype");
  if (index_bits != 32 && index_bits != 64) return fail(GNS_ERR_ARGUMENT, "indices must have 32 or 64 bits");
  if (rows < 0 || vocabulary < 1 || top < 0) return fail(GNS_ERR_ARGUMENT, "a loss needs rows >= 0, a vocabulary and top >= 0");
  if (top > kMaxTop) return fail(GNS_ERR_UNSUPPORTED, "at most 1024 top logits a row are supported");
  if (vocabulary > (1 << 28)) return fail(GNS_ERR_UNSUPPORTED, "vocabulary too large");
  if (!(temperature >= 1e-4f && temperature <= 1e4f)) return fail(GNS_ERR_ARGUMENT, "temperature must be in [1e-4, 1e4]");
  if (rows == 0) return GNS_OK;
  if (logits == nullptr || (top > 0 && (indices == nullptr || teacher == nullptr))) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (loss == nullptr && (dlogits == nullptr || stats == nullptr))
    return fail(GNS_ERR_ARGUMENT, "a call returns a loss, or a gradient from an earlier call's statistics");
  if ((dlogits == nullptr) != (grad == nullptr)) return fail(GNS_ERR_ARGUMENT, "grad and dlogits come together");
  // A row's pair is one access.
  if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) return fail(GNS_ERR_LAYOUT, "statistics must start on 8 bytes");
  if (rows > 1 && (logits_rstride < vocabulary || (dlogits != nullptr && dlogits_rstride < vocabulary)))
    return fail(GNS_ERR_LAYOUT, "row stride below the row length");
  const int rc = check_device();
  if (rc != GNS_OK) return rc;
  LossArgs a{};
  a.z = logits;
  a.z_stride = logits_rstride;
  a.index = indices;
  a.index_stride = indices_rstride;
  a.index64 = index_bits == 64 ? 1 : 0;
  a.teacher = teacher;
  a.teacher_stride = teacher_rstride;
  a.teacher_dt = teacher_dtype;
  a.grad = grad;
  a.loss = loss;
  a.stats = reinterpret_cast<float2*>(stats);
  a.dz = dlogits;
  a.dz_stride = dlogits_rstride;
  a.rows = rows;
  a.vocabulary = static_cast<int>(vocabulary);
  a.top = static_cast<int>(top);
  a.temperature = temperature;
  a.scale = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (loss == nullptr) return launch_any<2>(z_dtype, a, st);
  if (dlogits == nullptr) return launch_any<1>(z_dtype, a, st);
  return launch_any<3>(z_dtype, a, st);
}
