// Layer norm over the last dimension, forward and backward.
//
//   forward   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//             y = (x - mu) r w + b;  mu and r are kept in fp32 for the backward pass
//   backward  h = (x - mu) r,  a = w dy,  c1 = mean(a h),  c2 = mean(a)
//             dx = r (a - c2 - h c1);  dw = sum over rows of dy h;  db = sum of dy
//
// A row is held in the registers of TPR threads, 16 elements each (32 in the forward
// ring kernel), so x (and dy) are read once: the mean is subtracted before the squares
// are summed, which costs a second reduction but no second read. Rows go to the groups of a
// persistent grid round robin. Each thread keeps the same columns for all its
// rows: w and b stay in registers, and dw and db are summed there over the rows,
// written once per CTA and joined by a second kernel in a fixed order (no
// atomics, the same bits on every run).
//
// Rows reach the registers in one of two ways. Rows of more than 512 elements come
// through a ring of rows in shared memory, filled by bulk copies several rows ahead
// (ring kernels); the bytes in flight do not depend on registers or occupancy. Rows
// that start anywhere are copied from the multiple of 16 bytes before them and read
// out of the ring element by element (read directly from global memory, 20157 bf16
// rows of 2337 took 166 us forward and 424 backward, now 93 and 99; fp32 rows 104 and
// 162, now 86 and 92). Shorter rows are loaded directly, a row a warp, the next row
// before the current row's reduction (direct kernels). Rows that have no place there go
// to the wide kernels, element by element from global memory in three passes: rows of
// more than 16384 elements, and in the backward pass fp32 rows from 12801 elements on
// (fewer by a few where they start anywhere), of which a stage of x and dy does not fit a
// ring twice (4096 fp32 rows backward: 12800 elements 183 us through the ring, 12808
// elements 339 without; 20480 bf16 elements 283 us forward and 472 backward).
// Statistics, sums and all arithmetic are fp32; y, dx, dw and db are rounded
// once, at their stores. Bound by HBM: 2 elements moved forward, 3 backward.
#include <algorithm>
#include <mutex>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kPer = 16;        // elements of a row per thread
constexpr int kDirectTPR = 32;  // the direct kernels: a row a warp
constexpr int kMaxTPR = 1024;   // threads of a row; wider rows have kernels of their own
constexpr int kWideThreads = 1024;
constexpr int kColThreads = 256;

struct NormArgs {
  const void* x;
  const void* dy;
  int64_t x_stride, dy_stride;
  const void* w;
  const void* b;
  void* y;  // dx in the backward pass
  float* mean;
  float* rstd;
  float* partial;  // [CTA][2][cols]: sums of dy h and of dy
  void* dw;        // not null: the grid is one CTA, which writes dw and db (may be null) itself
  void* db;
  int64_t rows;
  int cols, w_dt, parts;
  float eps;
};

// One thread's 16 elements of a row as loaded. VEC: 16-byte pieces, V elements
// each, piece j of thread t at element (j TPR + t) V; otherwise element i of
// thread t is i TPR + t.
template <int XD, int TPR, bool VEC, int E = kPer>
struct Piece {
  static constexpr int kV = XD == kF32 ? 4 : 8;
  static constexpr int kWords = XD == kF32 ? E : E / 2;
  uint32_t w[kWords];

  static __device__ __forceinline__ int col(int t, int i) {
    return VEC ? ((i / kV) * TPR + t) * kV + i % kV : i * TPR + t;
  }

  __device__ __forceinline__ void load(const void* base, int64_t row, int64_t stride, int t, int cols, bool live) {
    constexpr int es = XD == kF32 ? 4 : 2;
    const uint8_t* p = static_cast<const uint8_t*>(base) + row * stride * es;
    if (VEC) {
#pragma unroll
      for (int j = 0; j < E / kV; ++j) {
        const int c = (j * TPR + t) * kV;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (live && c < cols) u = *reinterpret_cast<const uint4*>(p + static_cast<int64_t>(c) * es);
        w[4 * j] = u.x; w[4 * j + 1] = u.y; w[4 * j + 2] = u.z; w[4 * j + 3] = u.w;
      }
    } else if (XD == kF32) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = i * TPR + t;
        w[i % kWords] = (live && c < cols) ? reinterpret_cast<const uint32_t*>(p)[c] : 0u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const int c = i * TPR + t;
        const uint32_t lo = (live && c < cols) ? reinterpret_cast<const uint16_t*>(p)[c] : 0u;
        const uint32_t hi = (live && c + TPR < cols) ? reinterpret_cast<const uint16_t*>(p)[c + TPR] : 0u;
        w[i / 2] = lo | (hi << 16);
      }
    }
  }

  __device__ __forceinline__ float get(int i) const {
    if (XD == kF32) return __uint_as_float(w[i % kWords]);
    const uint32_t two = w[i / 2 % kWords];
    if (XD == kBF16) return __uint_as_float((i & 1) ? (two & 0xffff0000u) : (two << 16));
    return __half2float(__ushort_as_half(static_cast<uint16_t>((i & 1) ? (two >> 16) : two)));
  }
};

template <int XD, int TPR, bool VEC, int E>
__device__ __forceinline__ void store_row(void* base, int64_t row, int cols, int t, const float (&v)[E]) {
  using P = Piece<XD, TPR, VEC, E>;
  constexpr int es = XD == kF32 ? 4 : 2;
  uint8_t* p = static_cast<uint8_t*>(base) + row * cols * es;
  if (VEC) {
#pragma unroll
    for (int j = 0; j < E / P::kV; ++j) {
      const int c = (j * TPR + t) * P::kV;
      if (c >= cols) continue;
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (XD == kF32) {
          o[q] = __float_as_uint(v[j * P::kV + q]);
        } else if (XD == kBF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[(j * P::kV + 2 * q) % E], v[(j * P::kV + 2 * q + 1) % E]);
          o[q] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[(j * P::kV + 2 * q) % E], v[(j * P::kV + 2 * q + 1) % E]);
          o[q] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(p + static_cast<int64_t>(c) * es) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = i * TPR + t;
      if (c < cols) store_from_float(p, c, XD, v[i]);
    }
  }
}

// Sums of (a, b) over the TPR threads of each row group, in every thread of it.
// `slot` alternates between two buffers, so one barrier per call is enough: a
// buffer is written again only after the other buffer's barrier, which every
// reader of it has passed.
template <int TPR, int THREADS, bool BOTH = true>
__device__ __forceinline__ float2 group_sum(float a, float b, float2 (*slots)[THREADS / 32], int& slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    if (BOTH) b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (TPR == 32) return make_float2(a, b);
  float2* buf = slots[slot];
  slot ^= 1;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) buf[warp] = make_float2(a, b);
  __syncthreads();
  constexpr int kW = TPR / 32;  // warps of a group
  const int first = warp / kW * kW;
  a = 0.0f;
  b = 0.0f;
  if (kW <= 8) {
#pragma unroll
    for (int q = 0; q < kW; ++q) {
      a += buf[first + q].x;
      b += buf[first + q].y;
    }
  } else {
    // 16 or 32 partial sums: one per lane, joined by shuffles.
    const float2 mine = (threadIdx.x & 31) < kW ? buf[first + (threadIdx.x & 31)] : make_float2(0.0f, 0.0f);
    a = mine.x;
    b = mine.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (BOTH) b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
  return make_float2(a, b);
}

template <int TPR>
constexpr int threads_of() {
  return TPR < 256 ? 256 : TPR;
}

template <int XD, bool VEC>
__global__ void __launch_bounds__(threads_of<kDirectTPR>()) norm_forward_kernel(const NormArgs a) {
  constexpr int TPR = kDirectTPR;
  constexpr int kThreads = threads_of<TPR>();
  constexpr int kGroups = kThreads / TPR;
  using P = Piece<XD, TPR, VEC>;
  __shared__ float2 slots[2][kThreads / 32];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  float w[kPer], b[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = P::col(t, i);
    w[i] = c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f;
    b[i] = (a.b != nullptr && c < a.cols) ? load_as_float(a.b, c, a.w_dt) : 0.0f;
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  P next;
  next.load(a.x, first, a.x_stride, t, a.cols, first < a.rows);
  // Every group of the CTA makes the same number of turns (the barriers are CTA-wide).
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < a.rows;
    float v[kPer];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = next.get(i);
      sum += v[i];
    }
    next.load(a.x, row + step, a.x_stride, t, a.cols, row + step < a.rows);
    const float mu = group_sum<TPR, kThreads, false>(sum, 0.0f, slots, slot).x * inv_n;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] -= mu;
      if (P::col(t, i) < a.cols) sq = fmaf(v[i], v[i], sq);
    }
    const float var = group_sum<TPR, kThreads, false>(sq, 0.0f, slots, slot).x * inv_n;
    const float r = rsqrtf(var + a.eps);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = fmaf(v[i] * r, w[i], b[i]);
    if (live) {
      store_row<XD, TPR, VEC, kPer>(a.y, row, a.cols, t, v);
      if (t == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
  }
}

// A CTA's column sums: its groups' are joined in `joined` (kThreads kPer floats,
// unused with one group), in a fixed order.
template <int TPR, class P>
__device__ __forceinline__ void write_partial(const NormArgs& a, const float (&dw)[kPer], const float (&db)[kPer],
                                              float* joined, int t, int group) {
  constexpr int kGroups = threads_of<TPR>() / TPR;
  auto put = [&](int which, int c, float sum) {
    if (a.dw == nullptr)
      a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * a.cols + c] = sum;
    else if (which == 0)
      store_from_float(a.dw, c, a.w_dt, sum);
    else if (a.db != nullptr)
      store_from_float(a.db, c, a.w_dt, sum);
  };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (kGroups > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) joined[(group * kPer + i) * TPR + t] = which ? db[i] : dw[i];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          float sum = 0.0f;
          for (int q = 0; q < kGroups; ++q) sum += joined[(q * kPer + i) * TPR + t];
          const int c = P::col(t, i);
          if (c < a.cols) put(which, c, sum);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = P::col(t, i);
        if (c < a.cols) put(which, c, which ? db[i] : dw[i]);
      }
    }
  }
}

template <int XD, bool VEC>
__global__ void __launch_bounds__(threads_of<kDirectTPR>()) norm_backward_kernel(const NormArgs a) {
  constexpr int TPR = kDirectTPR;
  pdl_launch_dependents();
  constexpr int kThreads = threads_of<TPR>();
  constexpr int kGroups = kThreads / TPR;
  using P = Piece<XD, TPR, VEC>;
  __shared__ float2 slots[2][kThreads / 32];
  __shared__ float joined[kGroups > 1 ? kThreads * kPer : 1];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  float w[kPer], dw[kPer], db[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = P::col(t, i);
    w[i] = c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f;
    dw[i] = 0.0f;
    db[i] = 0.0f;
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  P nx, ng;
  nx.load(a.x, first, a.x_stride, t, a.cols, first < a.rows);
  ng.load(a.dy, first, a.dy_stride, t, a.cols, first < a.rows);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < a.rows;
    const float mu = live ? a.mean[row] : 0.0f;
    const float r = live ? a.rstd[row] : 0.0f;
    float h[kPer], g[kPer];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      g[i] = ng.get(i);
      // Columns past the end hold zeros and have no place in the sums: g is zero there.
      h[i] = (nx.get(i) - mu) * r;
      dw[i] = fmaf(g[i], h[i], dw[i]);
      db[i] += g[i];
      g[i] *= w[i];
      s1 = fmaf(g[i], h[i], s1);
      s2 += g[i];
    }
    nx.load(a.x, row + step, a.x_stride, t, a.cols, row + step < a.rows);
    ng.load(a.dy, row + step, a.dy_stride, t, a.cols, row + step < a.rows);
    const float2 c = group_sum<TPR, kThreads>(s1, s2, slots, slot);
    const float c1 = c.x * inv_n, c2 = c.y * inv_n;
#pragma unroll
    for (int i = 0; i < kPer; ++i) g[i] = (g[i] - fmaf(h[i], c1, c2)) * r;
    if (live) store_row<XD, TPR, VEC, kPer>(a.y, row, a.cols, t, g);
  }
  write_partial<TPR, P>(a, dw, db, joined, t, group);
}

// ------------------------------------------------------------- ring kernels
__device__ int g_norm_status = 0;

constexpr int kMaxStages = 8;

// Ring of row slots: a stage holds one row of each group (and of dy behind it).
struct Ring {
  uint64_t* full;             // one barrier per stage, an arrival per group
  volatile int* abort_flag;
  uint8_t* rows;              // [stage][group][tensors][row]
  int stages, stage = 0;
  uint32_t phase = 0;
  uint32_t row_bytes, stage_bytes;

  __device__ __forceinline__ Ring(uint8_t* smem, int stages_, int groups, int tensors, uint32_t bytes)
      : full(reinterpret_cast<uint64_t*>(smem)),
        abort_flag(reinterpret_cast<volatile int*>(smem + 8 * kMaxStages)),
        rows(smem + 128),
        stages(stages_),
        row_bytes(bytes),
        stage_bytes(bytes * static_cast<uint32_t>(tensors * groups)) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&full[i], static_cast<uint32_t>(groups));
      *abort_flag = 0;
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    __syncthreads();
  }

  __device__ __forceinline__ uint8_t* slot(int st, int group, int tensors) {
    return rows + st * stage_bytes + static_cast<uint32_t>(group * tensors) * row_bytes;
  }

  // A wait that runs out sets the status word and lets the loop go on with what the
  // slot holds, so that the CTA's barriers stay matched; every later wait returns at
  // once.
  __device__ __forceinline__ void wait() {
    mbar_wait_bounded(&full[stage], phase, abort_flag, &g_norm_status, kStatusProducerTimeout);
  }

  __device__ __forceinline__ void advance() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }

  // After an aborted wait, copies in flight get time to land before the CTA ends.
  __device__ __forceinline__ void finish() {
    __syncthreads();
    if (*abort_flag) settle_for_ns(2000000ull);
  }
};

// Bytes of a row behind a multiple of 16.
template <int XD, bool VEC>
__device__ __forceinline__ uint32_t row_shift(const void* base, int64_t row, int64_t stride) {
  constexpr int es = XD == kF32 ? 4 : 2;
  return VEC ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base) + row * stride * es) & 15u;
}

// A row into its slot. A row that starts anywhere is copied from the multiple of 16
// before it to the one behind it: every 16 bytes read hold one of the row.
template <int XD, bool VEC>
__device__ __forceinline__ uint32_t row_span(const NormArgs& a, uint32_t shift) {
  const uint32_t bytes = static_cast<uint32_t>(a.cols) * (XD == kF32 ? 4u : 2u);
  return VEC ? bytes : (bytes + shift + 15u) & ~15u;
}

// One row of each tensor into a stage, by one thread of each group.
template <int XD, int TENSORS, bool VEC>
__device__ __forceinline__ void fetch(Ring& ring, int st, int group, const NormArgs& a, int64_t row) {
  constexpr int es = XD == kF32 ? 4 : 2;
  if (row >= a.rows) {
    mbar_arrive(&ring.full[st]);
    return;
  }
  uint8_t* slot = ring.slot(st, group, TENSORS);
  const uint32_t x_shift = row_shift<XD, VEC>(a.x, row, a.x_stride);
  const uint32_t dy_shift = TENSORS == 2 ? row_shift<XD, VEC>(a.dy, row, a.dy_stride) : 0u;
  const uint32_t x_span = row_span<XD, VEC>(a, x_shift), dy_span = row_span<XD, VEC>(a, dy_shift);
  mbar_arrive_expect_tx(&ring.full[st], x_span + (TENSORS == 2 ? dy_span : 0u));
  bulk_load(slot, static_cast<const uint8_t*>(a.x) + row * a.x_stride * es - x_shift, x_span, &ring.full[st]);
  if (TENSORS == 2)
    bulk_load(slot + ring.row_bytes, static_cast<const uint8_t*>(a.dy) + row * a.dy_stride * es - dy_shift, dy_span,
              &ring.full[st]);
}

// Slot of a row in a ring.
__host__ __device__ constexpr uint32_t slot_bytes(bool vec, int64_t cols, int es) {
  return static_cast<uint32_t>(vec ? cols * es : (cols * es + 15) / 16 * 16 + 16);
}

// Elements of a row per thread in the forward ring kernel: a reduction over a row
// costs each thread the same whatever it holds, so 32 elements halve its share
// (with 16, two reductions of two values and 256 threads for 4096 columns, the
// kernel issued 20 instructions an element and took 57 us for 16384 bf16 rows).
constexpr int kFwdPer = 32;

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Mean and variance of a row take one barrier: each warp finds the sum and the
// squared deviations from its own mean, S_w and Q_w, and over the warps
//   mu = sum S_w / n,   n var = sum Q_w + n_w (S_w / n_w - mu)^2,
// which loses nothing to cancellation, unlike sums of squares.
//
// The grid has two CTAs of 256 threads an SM, so registers are held to 128: left alone, the
// compiler takes up to 148 for 256 threads a row, and the second CTA waits (8192 rows of
// 8192 bf16 elements 68 us, now 51; 5001 fp16 elements 98, now 78). Not so for aligned
// fp32 rows, whose longer pieces then spill (8192 elements 90 us against 98).
template <int XD, int TPR, bool VEC>
__global__ void __launch_bounds__(threads_of<TPR>(), threads_of<TPR>() > 256 || (XD == kF32 && VEC) ? 0 : 2)
    norm_forward_ring_kernel(const NormArgs a, int stages) {
  constexpr int kThreads = threads_of<TPR>();
  constexpr int kGroups = kThreads / TPR;
  constexpr int kW = TPR / 32;
  constexpr int E = kFwdPer;
  using P = Piece<XD, TPR, VEC, E>;
  constexpr int kStep = VEC ? P::kV : 1;  // columns that are in or out together
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 slots[2][kThreads / 32];  // S_w, Q_w
  __shared__ float2 sizes[kThreads / 32];     // n_w, 1 / n_w
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int mine = 0;
#pragma unroll
  for (int i = 0; i < E; i += kStep) mine += P::col(t, i) < a.cols ? kStep : 0;
  const float n_w = warp_total(static_cast<float>(mine));
  const float inv_w = n_w > 0.0f ? 1.0f / n_w : 0.0f;
  if (lane == 0) sizes[warp] = make_float2(n_w, inv_w);
  Ring ring(smem, stages, kGroups, 1, slot_bytes(VEC, a.cols, XD == kF32 ? 4 : 2));
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups;
  if (t == 0)
    for (int i = 0; i < stages; ++i) fetch<XD, 1, VEC>(ring, i, group, a, base + group + i * step);
  float w[E], b[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = P::col(t, i);
    w[i] = c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f;
    b[i] = (a.b != nullptr && c < a.cols) ? load_as_float(a.b, c, a.w_dt) : 0.0f;
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  for (int64_t first = base; first < a.rows; first += step) {
    const int64_t row = first + group;
    ring.wait();
    P p;
    p.load(ring.slot(ring.stage, group, 1) + row_shift<XD, VEC>(a.x, row, a.x_stride), 0, 0, t, a.cols, true);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) sum += p.get(i);
    sum = warp_total(sum);
    const float mean_w = sum * inv_w;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i += kStep) {
      if (P::col(t, i) >= a.cols) continue;
#pragma unroll
      for (int q = 0; q < kStep; ++q) {
        const float d = p.get(i + q) - mean_w;
        sq = fmaf(d, d, sq);
      }
    }
    sq = warp_total(sq);
    float mu = mean_w, var = sq;
    if (kW > 1) {
      float2* buf = slots[slot];
      slot ^= 1;
      if (lane == 0) buf[warp] = make_float2(sum, sq);
      __syncthreads();
      const int w0 = group * kW;
      float total = 0.0f, rest = 0.0f;
      if (kW <= 8) {
#pragma unroll
        for (int q = 0; q < kW; ++q) total += buf[w0 + q].x;
        mu = total * inv_n;
#pragma unroll
        for (int q = 0; q < kW; ++q) {
          const float d = fmaf(buf[w0 + q].x, sizes[w0 + q].y, -mu);
          rest += fmaf(d * d, sizes[w0 + q].x, buf[w0 + q].y);
        }
      } else {
        // 16 partial sums: one per lane, joined by shuffles.
        const bool has = lane < kW;
        const float2 one = has ? buf[w0 + lane] : make_float2(0.0f, 0.0f);
        const float2 size = has ? sizes[w0 + lane] : make_float2(0.0f, 0.0f);
        mu = warp_total(one.x) * inv_n;
        const float d = fmaf(one.x, size.y, -mu);
        rest = warp_total(fmaf(d * d, size.x, one.y));
      }
      var = rest;
    } else {
      __syncwarp();
    }
    // Every thread of the group has read the slot: it is filled again.
    if (t == 0) fetch<XD, 1, VEC>(ring, ring.stage, group, a, row + stages * step);
    ring.advance();
    const float r = rsqrtf(fmaf(var, inv_n, a.eps));
    if (row < a.rows) {
      // The mean is taken off before the scaling: x r - mu r would round mu r, which shows
      // where the mean is large beside the deviations (a row of 1000s came out 0.01 off).
      float v[E];
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const Pair h = mul2(add2(Pair(p.get(i), p.get(i + 1)), Pair(-mu)), Pair(r));
        fma2(h, Pair(w[i], w[i + 1]), Pair(b[i], b[i + 1])).get(v[i], v[i + 1]);
      }
      store_row<XD, TPR, VEC, E>(a.y, row, a.cols, t, v);
      if (t == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
  }
  ring.finish();
}

template <int XD, int TPR, bool VEC>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_backward_ring_kernel(const NormArgs a, int stages) {
  pdl_launch_dependents();
  constexpr int kThreads = threads_of<TPR>();
  constexpr int kGroups = kThreads / TPR;
  using P = Piece<XD, TPR, VEC>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 slots[2][kThreads / 32];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  Ring ring(smem, stages, kGroups, 2, slot_bytes(VEC, a.cols, XD == kF32 ? 4 : 2));
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups;
  if (t == 0)
    for (int i = 0; i < stages; ++i) fetch<XD, 2, VEC>(ring, i, group, a, base + group + i * step);
  // Elements go two to an instruction (one at a time the kernel took 77 us for 16384
  // bf16 rows of 4096).
  Pair w[kPer / 2], dw[kPer / 2], db[kPer / 2];
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    const int c = P::col(t, i), d = P::col(t, i + 1);
    w[i / 2] = Pair(c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f, d < a.cols ? load_as_float(a.w, d, a.w_dt) : 0.0f);
    dw[i / 2] = Pair(0.0f);
    db[i / 2] = Pair(0.0f);
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  // A row's mean and rstd are loaded a turn ahead, as their rows are.
  float next_mu = 0.0f, next_r = 0.0f;
  if (base + group < a.rows) {
    next_mu = a.mean[base + group];
    next_r = a.rstd[base + group];
  }
  for (int64_t first = base; first < a.rows; first += step) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    const float mu = next_mu, r = live ? next_r : 0.0f;
    if (row + step < a.rows) {
      next_mu = a.mean[row + step];
      next_r = a.rstd[row + step];
    }
    ring.wait();
    const uint8_t* at = ring.slot(ring.stage, group, 2);
    P px, pg;
    px.load(at + row_shift<XD, VEC>(a.x, row, a.x_stride), 0, 0, t, a.cols, live);
    pg.load(at + ring.row_bytes + row_shift<XD, VEC>(a.dy, row, a.dy_stride), 0, 0, t, a.cols, live);
    Pair h[kPer / 2], g[kPer / 2], s1(0.0f), s2(0.0f);
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
      const Pair dy(pg.get(2 * i), pg.get(2 * i + 1));
      h[i] = mul2(add2(Pair(px.get(2 * i), px.get(2 * i + 1)), Pair(-mu)), Pair(r));
      dw[i] = fma2(dy, h[i], dw[i]);
      db[i] = add2(db[i], dy);
      g[i] = mul2(dy, w[i]);
      s1 = fma2(g[i], h[i], s1);
      s2 = add2(s2, g[i]);
    }
    float s1a, s1b, s2a, s2b;
    s1.get(s1a, s1b);
    s2.get(s2a, s2b);
    const float2 c = group_sum<TPR, kThreads>(s1a + s1b, s2a + s2b, slots, slot);
    if (t == 0) fetch<XD, 2, VEC>(ring, ring.stage, group, a, row + stages * step);
    ring.advance();
    const Pair c1(-c.x * inv_n), c2(-c.y * inv_n);
    float out[kPer];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) mul2(add2(fma2(h[i], c1, c2), g[i]), Pair(r)).get(out[2 * i], out[2 * i + 1]);
    if (live) store_row<XD, TPR, VEC, kPer>(a.y, row, a.cols, t, out);
  }
  float dws[kPer], dbs[kPer];
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) {
    dw[i].get(dws[2 * i], dws[2 * i + 1]);
    db[i].get(dbs[2 * i], dbs[2 * i + 1]);
  }
  ring.finish();
  write_partial<TPR, P>(a, dws, dbs, reinterpret_cast<float*>(ring.rows), t, group);
}

// Rows that no ring holds: a CTA per row. Forward x is read three times (sum, squares,
// result), backward x and dy twice for dx and once more for the sums over the rows.
__device__ __forceinline__ float2 cta_sum(float a, float b, float2 (*slots)[kWideThreads / 32], int& slot) {
  return group_sum<kWideThreads, kWideThreads>(a, b, slots, slot);
}

__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const NormArgs a, int x_dt) {
  __shared__ float2 slots[2][kWideThreads / 32];
  int slot = 0;
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.x_stride;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) sum += load_as_float(a.x, at + c, x_dt);
    const float mu = cta_sum(sum, 0.0f, slots, slot).x * inv_n;
    float sq = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      const float d = load_as_float(a.x, at + c, x_dt) - mu;
      sq = fmaf(d, d, sq);
    }
    const float r = rsqrtf(cta_sum(sq, 0.0f, slots, slot).x * inv_n + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      const float h = (load_as_float(a.x, at + c, x_dt) - mu) * r;
      const float b = a.b != nullptr ? load_as_float(a.b, c, a.w_dt) : 0.0f;
      store_from_float(a.y, row * a.cols + c, x_dt, fmaf(h, load_as_float(a.w, c, a.w_dt), b));
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mu;
      a.rstd[row] = r;
    }
  }
}

__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(const NormArgs a, int x_dt) {
  __shared__ float2 slots[2][kWideThreads / 32];
  int slot = 0;
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t xa = row * a.x_stride, ga = row * a.dy_stride;
    const float mu = a.mean[row], r = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      const float h = (load_as_float(a.x, xa + c, x_dt) - mu) * r;
      const float g = load_as_float(a.dy, ga + c, x_dt) * load_as_float(a.w, c, a.w_dt);
      s1 = fmaf(g, h, s1);
      s2 += g;
    }
    const float2 s = cta_sum(s1, s2, slots, slot);
    const float c1 = s.x * inv_n, c2 = s.y * inv_n;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      const float h = (load_as_float(a.x, xa + c, x_dt) - mu) * r;
      const float g = load_as_float(a.dy, ga + c, x_dt) * load_as_float(a.w, c, a.w_dt);
      store_from_float(a.y, row * a.cols + c, x_dt, (g - fmaf(h, c1, c2)) * r);
    }
  }
}

// Column sums over every parts-th row, for the wide rows.
__global__ void __launch_bounds__(kColThreads) norm_columns_wide_kernel(const NormArgs a, int x_dt) {
  pdl_launch_dependents();
  const int c = blockIdx.x * kColThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += a.parts) {
    const float g = load_as_float(a.dy, row * a.dy_stride + c, x_dt);
    dw = fmaf(g, (load_as_float(a.x, row * a.x_stride + c, x_dt) - a.mean[row]) * a.rstd[row], dw);
    db += g;
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
  out[c] = dw;
  out[a.cols + c] = db;
}

// dw and db from the CTAs' sums, 32 columns a CTA, in a fixed order.
constexpr int kJoinRows = 16;
__global__ void __launch_bounds__(32 * kJoinRows) norm_join_kernel(const float* partial, int parts, int cols, void* dw,
                                                                   void* db, int dt) {
  __shared__ float sums[kJoinRows][33];
  pdl_wait_predecessor();  // launched while the sums are still being made
  const int64_t both = 2 * static_cast<int64_t>(cols);
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < both)
    for (int q = threadIdx.y; q < parts; q += kJoinRows) s += partial[q * both + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || c >= both) return;
  s = 0.0f;
#pragma unroll
  for (int q = 0; q < kJoinRows; ++q) s += sums[q][threadIdx.x];
  if (c < cols)
    store_from_float(dw, c, dt, s);
  else if (db != nullptr)
    store_from_float(db, c - cols, dt, s);
}

// Threads of a row: the fewest that hold it at `per` elements each, a warp at least.
int threads_per_row(int64_t cols, int per) {
  int t = 32;
  while (t < kMaxTPR && static_cast<int64_t>(t) * per < cols) t *= 2;
  return t;
}

// How a call runs: `stages` > 0, the ring kernels; else the direct kernels for rows of
// up to 512 elements, or the wide ones for rows that no ring holds in two stages.
struct Plan {
  bool wide;
  int stages, grid, tpr;
  size_t smem;
};

// Shared memory for rings on an SM, and the stages that one is given at most. Each
// CTA's share is divided into stages; below two there is nothing to overlap.
constexpr int kRingBytes = 200 * 1024;

Plan plan_norm(bool backward, bool vec, int x_dt, int64_t rows, int64_t cols) {
  Plan p{};
  const bool ring = cols > 32 * kPer && cols <= static_cast<int64_t>(kMaxTPR) * kPer;
  const int tpr = threads_per_row(cols, ring && !backward ? kFwdPer : kPer);
  const int threads = tpr < 256 ? 256 : tpr;
  const int groups = threads / tpr;
  const int64_t turns = (rows + groups - 1) / groups;
  const int sms = device_sm_count();
  p.tpr = tpr;
  if (ring) {
    const int ctas = threads > 256 ? 1 : 2;  // per SM: what the registers allow
    const int64_t stage = static_cast<int64_t>(slot_bytes(vec, cols, dtype_size(x_dt))) * groups * (backward ? 2 : 1);
    const int64_t stages = kRingBytes / ctas / stage;
    if (stages >= 2) {
      p.stages = static_cast<int>(stages < kMaxStages ? stages : kMaxStages);
      p.grid = static_cast<int>(turns < static_cast<int64_t>(sms) * ctas ? turns : static_cast<int64_t>(sms) * ctas);
      p.smem = 128 + static_cast<size_t>(stage) * p.stages;
      // The backward pass joins its groups' sums in the ring's memory.
      if (backward && groups > 1 && p.smem < 128 + sizeof(float) * threads * kPer) p.smem = 128 + sizeof(float) * threads * kPer;
      return p;
    }
  }
  p.tpr = threads_per_row(cols, kPer);
  p.wide = p.tpr > 32;
  if (p.wide) {
    const int64_t most = 2 * static_cast<int64_t>(sms);
    p.grid = static_cast<int>(rows < most ? rows : most);
  } else {
    const int direct = p.tpr < 256 ? 256 : p.tpr;
    const int64_t needed = (rows + direct / p.tpr - 1) / (direct / p.tpr);
    const int64_t most = static_cast<int64_t>(sms) * (768 / direct);
    p.grid = static_cast<int>(needed < most ? needed : most);
  }
  return p;
}

// A backward pass of up to four turns runs in one CTA, which writes the weight's and
// bias's gradients itself: one launch less, against turns of about a microsecond.
constexpr int kLoneTurns = 4;

bool is_lone(const Plan& p, int64_t rows) {
  const int groups = (p.tpr < 256 ? 256 : p.tpr) / p.tpr;
  return !p.wide && rows <= static_cast<int64_t>(kLoneTurns) * groups;
}

// Partial sums of a backward pass: one of each CTA, or of each of 64 sets of rows.
int backward_parts(const Plan& p, int64_t rows) { return p.wide ? static_cast<int>(rows < 64 ? rows : 64) : p.grid; }

std::mutex g_mutex;
bool g_ready[64][128] = {};

template <int XD, int TPR, bool VEC>
int launch_ring(bool backward, const Plan& p, int slot, cudaStream_t st, const NormArgs& a) {
  // The forward kernel's 32 elements a thread need no more than 512 threads, and the
  // backward kernel's 16 no fewer than 64.
  constexpr int kForward = TPR > 512 ? 512 : TPR, kBackward = TPR < 64 ? 64 : TPR;
  auto kernel = backward ? norm_backward_ring_kernel<XD, kBackward, VEC> : norm_forward_ring_kernel<XD, kForward, VEC>;
  const int threads = backward ? threads_of<kBackward>() : threads_of<kForward>();
  if (p.tpr != (backward ? kBackward : kForward)) return fail(GNS_ERR_UNSUPPORTED, "no ring kernel has these threads a row");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(GNS_ERR_DEVICE, "device index out of range");
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    bool& ready = g_ready[dev][slot + (backward ? 32 : 0) + (VEC ? 0 : 64)];
    if (!ready) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes + 1024);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      ready = true;
    }
  }
  kernel<<<p.grid, threads, p.smem, st>>>(a, p.stages);
  return GNS_OK;
}

template <int XD, bool VEC>
int launch_direct(bool backward, const Plan& p, cudaStream_t st, const NormArgs& a) {
  if (backward)
    norm_backward_kernel<XD, VEC><<<p.grid, threads_of<kDirectTPR>(), 0, st>>>(a);
  else
    norm_forward_kernel<XD, VEC><<<p.grid, threads_of<kDirectTPR>(), 0, st>>>(a);
  return GNS_OK;
}

template <int XD, bool VEC>
int launch_type(bool backward, const Plan& p, cudaStream_t st, const NormArgs& a) {
  if (p.stages == 0) return launch_direct<XD, VEC>(backward, p, st, a);
  switch (p.tpr) {
    case 32: return launch_ring<XD, 32, VEC>(backward, p, 8 * XD + 5, st, a);
    case 64: return launch_ring<XD, 64, VEC>(backward, p, 8 * XD, st, a);
    case 128: return launch_ring<XD, 128, VEC>(backward, p, 8 * XD + 1, st, a);
    case 256: return launch_ring<XD, 256, VEC>(backward, p, 8 * XD + 2, st, a);
    case 512: return launch_ring<XD, 512, VEC>(backward, p, 8 * XD + 3, st, a);
    default: return launch_ring<XD, 1024, VEC>(backward, p, 8 * XD + 4, st, a);
  }
}

template <int XD>
int launch_rows(bool backward, bool vec, const Plan& p, cudaStream_t st, const NormArgs& a) {
  return vec ? launch_type<XD, true>(backward, p, st, a) : launch_type<XD, false>(backward, p, st, a);
}

int launch_any(bool backward, bool vec, int x_dt, const Plan& p, cudaStream_t st, const NormArgs& a) {
  if (x_dt == kBF16) return launch_rows<kBF16>(backward, vec, p, st, a);
  if (x_dt == kF16) return launch_rows<kF16>(backward, vec, p, st, a);
  return launch_rows<kF32>(backward, vec, p, st, a);
}

// Rows that 16-byte pieces can be read from: every piece aligned and none past the end.
bool rows_vector(const void* p, int64_t stride, int64_t cols, int dt) {
  const int es = dtype_size(dt);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * es) % 16 == 0 && (cols * es) % 16 == 0;
}

int check_norm(int x_dtype, int w_dtype, int64_t rows, int64_t cols, int64_t stride) {
  if (x_dtype < 0 || x_dtype > 2 || w_dtype < 0 || w_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad dtype");
  if (rows < 0 || cols < 1) return fail(GNS_ERR_ARGUMENT, "layer norm needs rows >= 0 and cols >= 1");
  if (cols > (1 << 30)) return fail(GNS_ERR_UNSUPPORTED, "row too wide");
  if (rows > 1 && stride < cols) return fail(GNS_ERR_LAYOUT, "row stride below the row length");
  return GNS_OK;
}

}  // namespace

int norm_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_norm_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_norm_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "layer norm status");
}

}  // namespace gns

using namespace gns;

extern "C" {

int gns_layer_norm_forward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                           const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                           gns_stream_t stream) {
  clear_error();
  int rc = check_norm(x_dtype, w_dtype, rows, cols, x_rstride);
  if (rc != GNS_OK) return rc;
  if (rows == 0) return GNS_OK;
  if (x == nullptr || weight == nullptr || y == nullptr || mean == nullptr || rstd == nullptr)
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  NormArgs a{};
  a.x = x;
  a.x_stride = x_rstride;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.w_dt = w_dtype;
  a.eps = eps;
  const bool vec = rows_vector(x, x_rstride, cols, x_dtype) && rows_vector(y, cols, cols, x_dtype);
  const Plan plan = plan_norm(false, vec, x_dtype, rows, cols);
  if (plan.wide)
    norm_forward_wide_kernel<<<plan.grid, kWideThreads, 0, st>>>(a, x_dtype);
  else
    rc = launch_any(false, vec, x_dtype, plan, st, a);
  if (rc != GNS_OK) return rc;
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "layer norm forward kernel");
}

size_t gns_layer_norm_backward_workspace_size(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  // The most that any type and alignment takes.
  int parts = 0;
  for (int dt : {kF16, kF32})
    for (bool vec : {false, true}) {
      const Plan p = plan_norm(true, vec, dt, rows, cols);
      if (!is_lone(p, rows)) parts = std::max(parts, backward_parts(p, rows));
    }
  return static_cast<size_t>(parts) * 2 * static_cast<size_t>(cols) * sizeof(float);
}

int gns_layer_norm_backward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* grad, int64_t grad_rstride,
                            const void* x, int64_t x_rstride, const void* weight, const float* mean, const float* rstd,
                            void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                            gns_stream_t stream) {
  clear_error();
  int rc = check_norm(x_dtype, w_dtype, rows, cols, x_rstride);
  if (rc == GNS_OK) rc = check_norm(x_dtype, w_dtype, rows, cols, grad_rstride);
  if (rc != GNS_OK) return rc;
  if (dweight == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (rows > 0 && (grad == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr ||
                   dx == nullptr))
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  const size_t needed = gns_layer_norm_backward_workspace_size(rows, cols);
  if (workspace_bytes < needed || (needed > 0 && workspace == nullptr))
    return fail(GNS_ERR_WORKSPACE, "layer norm backward workspace too small");
  if (needed > 0 && reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
    return fail(GNS_ERR_WORKSPACE, "layer norm backward workspace must be aligned to 4 bytes");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  NormArgs a{};
  a.x = x;
  a.dy = grad;
  a.x_stride = x_rstride;
  a.dy_stride = grad_rstride;
  a.w = weight;
  a.y = dx;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.partial = static_cast<float*>(workspace);
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.w_dt = w_dtype;
  if (rows > 0) {
    const bool vec = rows_vector(x, x_rstride, cols, x_dtype) && rows_vector(grad, grad_rstride, cols, x_dtype) &&
                     rows_vector(dx, cols, cols, x_dtype);
    Plan plan = plan_norm(true, vec, x_dtype, rows, cols);
    if (is_lone(plan, rows)) {
      plan.grid = 1;
      a.dw = dweight;
      a.db = dbias;
    }
    a.parts = backward_parts(plan, rows);
    if (plan.wide) {
      norm_backward_wide_kernel<<<plan.grid, kWideThreads, 0, st>>>(a, x_dtype);
      const dim3 grid(static_cast<unsigned>((cols + kColThreads - 1) / kColThreads), static_cast<unsigned>(a.parts));
      norm_columns_wide_kernel<<<grid, kColThreads, 0, st>>>(a, x_dtype);
    } else {
      rc = launch_any(true, vec, x_dtype, plan, st, a);
      if (rc != GNS_OK) return rc;
    }
  }
  if (a.dw != nullptr) {
    const cudaError_t lone = cudaGetLastError();
    return lone == cudaSuccess ? GNS_OK : cuda_fail(lone, "layer norm backward kernel");
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>((2 * cols + 31) / 32), 1, 1);
  cfg.blockDim = dim3(32, kJoinRows, 1);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, norm_join_kernel, static_cast<const float*>(a.partial), a.parts, a.cols,
                                     dweight, dbias, w_dtype);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "layer norm backward kernels");
}

}  // extern "C"
