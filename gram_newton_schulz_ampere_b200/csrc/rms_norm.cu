// Root-mean-square norm over the last dimension of a residual stream, forward and backward.
//
//   forward   t = x + residual (rounded to the stream's type, and kept; x itself without one)
//             r = 1 / sqrt(mean(t^2) + eps),  y = t r w
//             y in t's type, or in 8 bits with a scale for each 128 columns
//   backward  h = t r,  a = w dy,  c = mean(a h)
//             dx = r (a - h c) + (the stream's own gradient);  dw = sum over rows of dy h
//
// Rows come through a ring of rows in shared memory that bulk copies fill some rows ahead, and
// are held in the registers of a group of threads: 32 elements each forward, 16 backward. A
// row costs one reduction and one barrier of its group; groups of a CTA do not wait for one
// another. The backward pass sums dw in registers over a group's rows; the sums are joined in
// a fixed order by a second kernel. Rows of more than 16384 elements go to kernels that read
// them from global memory element by element.
//
// Rows that start on 16 bytes are read in pieces of 16 bytes: thread t of a group has the
// pieces t, t + T, ... of its row, so that a scale's 128 columns lie in 16 neighbouring lanes
// (32 with fp32). Rows that start anywhere are copied from the multiple of 16 before them to
// the one behind them: every 16 bytes read hold an element of the row, so none lie in another
// page, and the others are not used. A warp has a stretch of such a row, its lanes neighbouring
// elements.
//
// Sums, statistics and all arithmetic are fp32. Bound by HBM: 16384 rows of 4096 bf16 elements with
// a residual and 8-bit output take 71 us forward (470 MB, 6.6 TB/s) and, with the stream's
// gradient, 79 us backward (537 MB, 6.8 TB/s) and 5 for the join. Rows that start anywhere cost
// a load from shared memory and a store for each element: 4099 x 1111 fp32 11 us forward and
// 14 backward (36 and 55 MB).
#include <algorithm>
#include <mutex>

#include "../../include/gns_b200.h"
#include "blocks_8bit.cuh"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

__device__ int g_rms_status = 0;

constexpr int kFwd = 32, kBwd = 16;  // elements of a row per thread
constexpr int kMaxCols = 16384;      // of a row in a ring
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 200 * 1024;  // of shared memory on an SM
constexpr int kWideThreads = 1024;

struct RmsArgs {
  const void* x;         // backward: the stream t
  const void* second;    // forward: the residual or null; backward: dy
  const void* third;     // backward: the stream's gradient or null
  int64_t x_stride, second_stride, third_stride;
  const void* w;
  void* y;               // forward: y, or null with 8-bit output; backward: dx
  void* total;           // forward, with a residual: t
  float* rstd;
  float* partial;        // backward: [group][cols]
  CodesOut out8;
  int64_t rows;
  int cols, w_dt;
  float eps;
};

// One thread's E elements of a row (above).
template <int XD, int T, bool VEC, int E>
struct Piece {
  static constexpr int kV = XD == kF32 ? 4 : 8;
  static constexpr int kWords = XD == kF32 ? E : E / 2;
  uint32_t w[kWords];

  static __device__ __forceinline__ int col(int t, int i) {
    return VEC ? ((i / kV) * T + t) * kV + i % kV : (t & ~31) * E + i * 32 + (t & 31);
  }

  __device__ __forceinline__ void load(const uint8_t* p, int t, int cols) {
    if (VEC) {
#pragma unroll
      for (int j = 0; j < E / kV; ++j) {
        const int c = (j * T + t) * kV;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (c < cols) u = *reinterpret_cast<const uint4*>(p + c * (16 / kV));
        w[4 * j] = u.x; w[4 * j + 1] = u.y; w[4 * j + 2] = u.z; w[4 * j + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = col(t, i);
        if (XD == kF32) {
          w[i % kWords] = c < cols ? reinterpret_cast<const uint32_t*>(p)[c] : 0u;
        } else {
          const uint32_t one = c < cols ? reinterpret_cast<const uint16_t*>(p)[c] : 0u;
          if (i & 1)
            w[i / 2 % kWords] |= one << 16;
          else
            w[i / 2 % kWords] = one;
        }
      }
    }
  }

  __device__ __forceinline__ void store(void* base, int t, int cols) const {
    uint8_t* p = static_cast<uint8_t*>(base);
    if (VEC) {
#pragma unroll
      for (int j = 0; j < E / kV; ++j) {
        const int c = (j * T + t) * kV;
        if (c < cols) *reinterpret_cast<uint4*>(p + c * (16 / kV)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = col(t, i);
        if (c >= cols) continue;
        if (XD == kF32)
          reinterpret_cast<uint32_t*>(p)[c] = w[i % kWords];
        else
          reinterpret_cast<uint16_t*>(p)[c] = static_cast<uint16_t>(w[i / 2 % kWords] >> (16 * (i & 1)));
      }
    }
  }

  // Elements 2q and 2q + 1.
  __device__ __forceinline__ Pair get(int q) const {
    if (XD == kF32) return Pair(__uint_as_float(w[2 * q % kWords]), __uint_as_float(w[(2 * q + 1) % kWords]));
    const uint32_t two = w[q % kWords];
    if (XD == kBF16) return Pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
    return Pair(__half2float(__ushort_as_half(static_cast<uint16_t>(two))),
                __half2float(__ushort_as_half(static_cast<uint16_t>(two >> 16))));
  }

  __device__ __forceinline__ void put(int q, Pair v) {
    float a, b;
    v.get(a, b);
    if (XD == kF32) {
      w[2 * q % kWords] = __float_as_uint(a);
      w[(2 * q + 1) % kWords] = __float_as_uint(b);
    } else if (XD == kBF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[q % kWords] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(a, b);
      w[q % kWords] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A barrier of the T threads of a group; number 0 is the CTA's own.
template <int T>
__device__ __forceinline__ void group_barrier(int group) {
  if (T == 32)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(T) : "memory");
}

// The sum over a group, in each of its threads, behind a barrier of the group, on which the
// refilling of the ring relies. `slot` alternates between two buffers, so that one barrier is
// enough: a buffer is written again only behind the other's barrier.
template <int T>
__device__ __forceinline__ float group_sum(float v, float* slots, int group, int& slot) {
  v = warp_sum(v);
  if (T == 32) {
    // Shuffles order no accesses to shared memory, and the backward pass reads a third row of
    // the slot that does not enter the sum: every lane has read the slot only behind this.
    group_barrier<T>(group);
    return v;
  }
  constexpr int kW = T / 32;
  float* buf = slots + slot * 32 + group * kW;
  slot ^= 1;
  const int warp = (threadIdx.x % T) / 32, lane = threadIdx.x & 31;
  if (lane == 0) buf[warp] = v;
  group_barrier<T>(group);
  if (kW <= 8) {
    v = 0.0f;
#pragma unroll
    for (int q = 0; q < kW; ++q) v += buf[q];
    return v;
  }
  return warp_sum(lane < kW ? buf[lane] : 0.0f);
}

template <int T>
constexpr int threads_of() {
  return T < 256 ? 256 : T;
}

template <int XD>
constexpr int size_of() {
  return XD == kF32 ? 4 : 2;
}

// Bytes of a row behind a multiple of 16.
template <int XD, bool VEC>
__device__ __forceinline__ uint32_t row_shift(const void* base, int64_t row, int64_t stride) {
  return VEC ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base) + row * stride * size_of<XD>()) & 15u;
}

__host__ __device__ constexpr uint32_t slot_bytes(bool vec, int64_t cols, int es) {
  return static_cast<uint32_t>(vec ? cols * es : (cols * es + 15) / 16 * 16 + 16);
}

// A group's ring: each stage holds a row of each tensor. The group's first thread fills it.
template <int XD, bool VEC>
struct Ring {
  uint64_t* full;
  volatile int* abort_flag;
  uint8_t* rows;
  uint32_t row_bytes;
  int stages, tensors, stage = 0;
  uint32_t phase = 0;

  __device__ __forceinline__ Ring(uint8_t* smem, int group, int groups, int stages_, int tensors_, int cols)
      : full(reinterpret_cast<uint64_t*>(smem) + group * kMaxStages),
        abort_flag(reinterpret_cast<volatile int*>(smem + 8 * kMaxStages * 8)),
        row_bytes(slot_bytes(VEC, cols, size_of<XD>())),
        stages(stages_),
        tensors(tensors_) {
    rows = smem + 640 + static_cast<uint32_t>(group * stages * tensors) * row_bytes;
    if (threadIdx.x == 0) {
      for (int i = 0; i < groups * kMaxStages; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem) + i, 1);
      *abort_flag = 0;
      fence_barrier_init();
      fence_proxy_async_smem();
    }
    __syncthreads();
  }

  __device__ __forceinline__ uint8_t* slot(int st, int tensor) const {
    return rows + static_cast<uint32_t>(st * tensors + tensor) * row_bytes;
  }

  __device__ __forceinline__ uint32_t span(int cols, uint32_t shift) const {
    const uint32_t bytes = static_cast<uint32_t>(cols) * size_of<XD>();
    return VEC ? bytes : (bytes + shift + 15u) & ~15u;
  }

  // One row of each tensor into stage st, by one thread.
  __device__ __forceinline__ void fetch(int st, const RmsArgs& a, int64_t row) const {
    if (row >= a.rows) return;
    const void* base[3] = {a.x, a.second, a.third};
    const int64_t stride[3] = {a.x_stride, a.second_stride, a.third_stride};
    uint32_t shift[3], bytes = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i >= tensors) break;
      shift[i] = row_shift<XD, VEC>(base[i], row, stride[i]);
      bytes += span(a.cols, shift[i]);
    }
    mbar_arrive_expect_tx(&full[st], bytes);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i >= tensors) break;
      bulk_load(slot(st, i), static_cast<const uint8_t*>(base[i]) + row * stride[i] * size_of<XD>() - shift[i],
                span(a.cols, shift[i]), &full[st]);
    }
  }

  // A wait that runs out sets the status word and goes on with what the slot holds, so that
  // the barriers stay matched; later waits return at once.
  __device__ __forceinline__ void wait() const {
    mbar_wait_bounded(&full[stage], phase, abort_flag, &g_rms_status, kStatusProducerTimeout);
  }

  __device__ __forceinline__ void advance() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

template <int XD, int T, bool VEC, bool EIGHT>
__global__ void __launch_bounds__(threads_of<T>(), threads_of<T>() > 256 ? 1 : 2)
    rms_forward_kernel(const RmsArgs a, int stages) {
  constexpr int kGroups = threads_of<T>() / T;
  constexpr int E = kFwd;
  using P = Piece<XD, T, VEC, E>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float slots[64];
  int slot = 0;
  const int t = threadIdx.x % T, group = threadIdx.x / T;
  const bool both = a.second != nullptr;
  Ring<XD, VEC> ring(smem, group, kGroups, stages, both ? 2 : 1, a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  if (t == 0)
    for (int i = 0; i < stages; ++i) ring.fetch(i, a, first + i * step);
  Pair w[E / 2];
#pragma unroll
  for (int q = 0; q < E / 2; ++q) {
    const int c = P::col(t, 2 * q), d = P::col(t, 2 * q + 1);
    w[q] = Pair(c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f, d < a.cols ? load_as_float(a.w, d, a.w_dt) : 0.0f);
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = first; row < a.rows; row += step) {
    ring.wait();
    P p;
    p.load(ring.slot(ring.stage, 0) + row_shift<XD, VEC>(a.x, row, a.x_stride), t, a.cols);
    if (both) {
      P other;
      other.load(ring.slot(ring.stage, 1) + row_shift<XD, VEC>(a.second, row, a.second_stride), t, a.cols);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) p.put(q, add2(p.get(q), other.get(q)));
      p.store(static_cast<uint8_t*>(a.total) + row * a.cols * size_of<XD>(), t, a.cols);
    }
    Pair sum(0.0f);
#pragma unroll
    for (int q = 0; q < E / 2; ++q) sum = fma2(p.get(q), p.get(q), sum);
    float s0, s1;
    sum.get(s0, s1);
    const float sq = group_sum<T>(s0 + s1, slots, group, slot);
    // Every thread of the group has read the slot: it is filled again.
    if (t == 0) ring.fetch(ring.stage, a, row + stages * step);
    ring.advance();
    const float r = rsqrtf(fmaf(sq, inv_n, a.eps));
    if (t == 0) a.rstd[row] = r;
    if (!EIGHT) {
#pragma unroll
      for (int q = 0; q < E / 2; ++q) p.put(q, mul2(mul2(p.get(q), Pair(r)), w[q]));
      p.store(static_cast<uint8_t*>(a.y) + row * a.cols * size_of<XD>(), t, a.cols);
      continue;
    }
    uint8_t* codes = a.out8.codes + row * a.out8.ld;
    float* scales = a.out8.scales + row * a.out8.srow;
    constexpr int kV = P::kV;
    constexpr int kPer = VEC ? kV : 4;             // elements of a thread in a block of 128
    constexpr int kLanes = VEC ? 128 / kV : 32;    // lanes of a block
#pragma unroll
    for (int j = 0; j < E / kPer; ++j) {
      const int c0 = P::col(t, j * kPer);  // of the thread's first element in this block
      if (P::col(t & ~31, j * kPer) >= a.out8.width) continue;  // the warp has none
      float v[kPer];
      float top = 0.0f;
#pragma unroll
      for (int q = 0; q < kPer / 2; ++q) {
        mul2(mul2(p.get(j * kPer / 2 + q), Pair(r)), w[j * kPer / 2 + q]).get(v[2 * q], v[2 * q + 1]);
        top = fmaxf(top, fmaxf(fabsf(v[2 * q]), fabsf(v[2 * q + 1])));
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const BlockScale s(top);
      if (c0 / kScaleBlock * kScaleBlock < a.cols && threadIdx.x % kLanes == 0) scales[c0 / kScaleBlock * a.out8.scol] = s.scale;
      if (VEC) {
        if (c0 < a.out8.width) {
          const uint32_t low = e4m3_four(v[0] * s.factor, v[1] * s.factor, v[2] * s.factor, v[3] * s.factor);
          if (kV == 4)
            *reinterpret_cast<uint32_t*>(codes + c0) = low;
          else
            *reinterpret_cast<uint2*>(codes + c0) =
                make_uint2(low, e4m3_four(v[4 % kPer] * s.factor, v[5 % kPer] * s.factor, v[6 % kPer] * s.factor, v[7 % kPer] * s.factor));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + 32 * i < a.out8.width) codes[c0 + 32 * i] = static_cast<uint8_t>(e4m3_pair(v[i % kPer] * s.factor, 0.0f));
      }
    }
  }
  __syncthreads();
  if (*ring.abort_flag) settle_for_ns(2000000ull);
}

template <int XD, int T, bool VEC>
__global__ void __launch_bounds__(threads_of<T>(), threads_of<T>() > 256 ? 1 : 2)
    rms_backward_kernel(const RmsArgs a, int stages) {
  pdl_launch_dependents();
  constexpr int kGroups = threads_of<T>() / T;
  constexpr int E = kBwd;
  using P = Piece<XD, T, VEC, E>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float slots[64];
  int slot = 0;
  const int t = threadIdx.x % T, group = threadIdx.x / T;
  const bool more = a.third != nullptr;
  Ring<XD, VEC> ring(smem, group, kGroups, stages, more ? 3 : 2, a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  if (t == 0)
    for (int i = 0; i < stages; ++i) ring.fetch(i, a, first + i * step);
  Pair w[E / 2], dw[E / 2];
#pragma unroll
  for (int q = 0; q < E / 2; ++q) {
    const int c = P::col(t, 2 * q), d = P::col(t, 2 * q + 1);
    w[q] = Pair(c < a.cols ? load_as_float(a.w, c, a.w_dt) : 0.0f, d < a.cols ? load_as_float(a.w, d, a.w_dt) : 0.0f);
    dw[q] = Pair(0.0f);
  }
  const float inv_n = 1.0f / static_cast<float>(a.cols);
  float next_r = first < a.rows ? a.rstd[first] : 0.0f;  // loaded a turn ahead, as the rows are
  for (int64_t row = first; row < a.rows; row += step) {
    const float r = next_r;
    if (row + step < a.rows) next_r = a.rstd[row + step];
    ring.wait();
    P pt, pg, pm;
    pt.load(ring.slot(ring.stage, 0) + row_shift<XD, VEC>(a.x, row, a.x_stride), t, a.cols);
    pg.load(ring.slot(ring.stage, 1) + row_shift<XD, VEC>(a.second, row, a.second_stride), t, a.cols);
    if (more) pm.load(ring.slot(ring.stage, 2) + row_shift<XD, VEC>(a.third, row, a.third_stride), t, a.cols);
    Pair h[E / 2], g[E / 2], sum(0.0f);
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      const Pair dy = pg.get(q);
      h[q] = mul2(pt.get(q), Pair(r));
      dw[q] = fma2(dy, h[q], dw[q]);
      g[q] = mul2(dy, w[q]);
      sum = fma2(g[q], h[q], sum);
    }
    float s0, s1;
    sum.get(s0, s1);
    const float c = group_sum<T>(s0 + s1, slots, group, slot) * inv_n;
    if (t == 0) ring.fetch(ring.stage, a, row + stages * step);
    ring.advance();
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      const Pair inner = fma2(h[q], Pair(-c), g[q]);
      pt.put(q, more ? fma2(inner, Pair(r), pm.get(q)) : mul2(inner, Pair(r)));
    }
    pt.store(static_cast<uint8_t*>(a.y) + row * a.cols * size_of<XD>(), t, a.cols);
  }
  __syncthreads();
  if (*ring.abort_flag) settle_for_ns(2000000ull);
  // The groups' sums, joined in the ring's place.
  float* joined = reinterpret_cast<float*>(smem + 640);
  float* to = a.partial + static_cast<int64_t>(blockIdx.x) * a.cols;
  float* mine = kGroups == 1 ? to : joined + group * a.cols;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    float x, y;
    dw[i / 2].get(x, y);
    const int c = P::col(t, i), d = P::col(t, i + 1);
    if (c < a.cols) mine[c] = x;
    if (d < a.cols) mine[d] = y;
  }
  if constexpr (kGroups > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += threads_of<T>()) {
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) sum += joined[q * a.cols + c];
      to[c] = sum;
    }
  }
}

// Rows that no ring holds: a CTA a row, element by element.
__device__ __forceinline__ float cta_sum(float v, float* slots, int& slot) {
  return group_sum<kWideThreads>(v, slots, 0, slot);
}

template <bool EIGHT>
__global__ void __launch_bounds__(kWideThreads) rms_forward_wide_kernel(const RmsArgs a, int dt) {
  __shared__ float slots[64];
  int slot = 0;
  const int lane = threadIdx.x & 31;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t xa = row * a.x_stride, ra = row * a.second_stride, to = row * a.cols;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      float v = load_as_float(a.x, xa + c, dt);
      if (a.second != nullptr) {
        v = round_to(v + load_as_float(a.second, ra + c, dt), dt);
        store_from_float(a.total, to + c, dt, v);
      }
      sum = fmaf(v, v, sum);
    }
    const float r = rsqrtf(fmaf(cta_sum(sum, slots, slot), 1.0f / static_cast<float>(a.cols), a.eps));
    if (threadIdx.x == 0) a.rstd[row] = r;
    auto value = [&](int c) {
      float v = load_as_float(a.x, xa + c, dt);
      if (a.second != nullptr) v = round_to(v + load_as_float(a.second, ra + c, dt), dt);
      return v * r * load_as_float(a.w, c, a.w_dt);
    };
    if (!EIGHT) {
      for (int c = threadIdx.x; c < a.cols; c += kWideThreads) store_from_float(a.y, to + c, dt, value(c));
      continue;
    }
    // A warp a block of 128 columns.
    for (int c0 = threadIdx.x / 32 * kScaleBlock; c0 < a.cols; c0 += kWideThreads / 32 * kScaleBlock) {
      float v[4], top = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 4 * lane + i;
        v[i] = c < a.cols ? value(c) : 0.0f;
        top = fmaxf(top, fabsf(v[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const BlockScale s(top);
      if (lane == 0) a.out8.scales[row * a.out8.srow + c0 / kScaleBlock * a.out8.scol] = s.scale;
      if (c0 + 4 * lane < a.out8.width)
        *reinterpret_cast<uint32_t*>(a.out8.codes + row * a.out8.ld + c0 + 4 * lane) =
            e4m3_four(v[0] * s.factor, v[1] * s.factor, v[2] * s.factor, v[3] * s.factor);
    }
  }
}

__global__ void __launch_bounds__(kWideThreads) rms_backward_wide_kernel(const RmsArgs a, int dt) {
  __shared__ float slots[64];
  int slot = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t xa = row * a.x_stride, ga = row * a.second_stride, ma = row * a.third_stride;
    const float r = a.rstd[row];
    float sum = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads)
      sum = fmaf(load_as_float(a.second, ga + c, dt) * load_as_float(a.w, c, a.w_dt), load_as_float(a.x, xa + c, dt) * r, sum);
    const float mean = cta_sum(sum, slots, slot) / static_cast<float>(a.cols);
    for (int c = threadIdx.x; c < a.cols; c += kWideThreads) {
      const float h = load_as_float(a.x, xa + c, dt) * r;
      const float inner = fmaf(h, -mean, load_as_float(a.second, ga + c, dt) * load_as_float(a.w, c, a.w_dt));
      store_from_float(a.y, row * a.cols + c, dt, a.third != nullptr ? fmaf(inner, r, load_as_float(a.third, ma + c, dt)) : inner * r);
    }
  }
}

// Column sums over every parts-th row, for those rows.
constexpr int kColThreads = 256;
__global__ void __launch_bounds__(kColThreads) rms_columns_wide_kernel(const RmsArgs a, int dt) {
  pdl_launch_dependents();
  const int c = blockIdx.x * kColThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
    dw = fmaf(load_as_float(a.second, row * a.second_stride + c, dt), load_as_float(a.x, row * a.x_stride + c, dt) * a.rstd[row], dw);
  a.partial[static_cast<int64_t>(blockIdx.y) * a.cols + c] = dw;
}

// dw from the CTAs' sums, 32 columns a CTA, in a fixed order.
constexpr int kJoinRows = 32;
__global__ void __launch_bounds__(32 * kJoinRows) rms_join_kernel(const float* partial, int parts, int cols, void* dw, int dt) {
  __shared__ float sums[kJoinRows][33];
  pdl_wait_predecessor();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 5
    for (int q = threadIdx.y; q < parts; q += kJoinRows) s += partial[static_cast<int64_t>(q) * cols + c];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || c >= cols) return;
  s = 0.0f;
#pragma unroll
  for (int q = 0; q < kJoinRows; ++q) s += sums[q][threadIdx.x];
  store_from_float(dw, c, dt, s);
}

// How a call runs: with stages through rings, else by the wide kernels. A single stage hides
// little, but the wide kernels read twice and element by element (4096 fp32 rows with a
// residual or the stream's gradient, one stage against none: 8192 elements forward 94 us and
// 252, 14336 forward 151 and 458, backward 222 and 470).
struct Plan {
  int stages, grid, threads;
  size_t smem;
};

Plan plan_rms(int per, int tensors, bool vec, int dt, int64_t rows, int64_t cols) {
  Plan p{};
  const int sms = device_sm_count();
  if (cols <= kMaxCols) {
    int t = 32;
    while (static_cast<int64_t>(t) * per < cols) t *= 2;
    const int threads = t < 256 ? 256 : t, groups = threads / t;
    const int ctas = threads > 256 ? 1 : 2;  // of an SM
    const int64_t stage = static_cast<int64_t>(slot_bytes(vec, cols, dtype_size(dt))) * groups * tensors;
    const int64_t stages = kRingBytes / ctas / stage;
    if (stages > 0) {
      p.threads = t;
      p.stages = static_cast<int>(std::min<int64_t>(stages, kMaxStages));
      p.grid = static_cast<int>(std::min<int64_t>((rows + groups - 1) / groups, static_cast<int64_t>(sms) * ctas));
      p.smem = 640 + static_cast<size_t>(stage) * p.stages;
      // The backward pass joins its groups' sums in the ring's memory.
      p.smem = std::max(p.smem, static_cast<size_t>(640 + (per == kBwd && groups > 1 ? 4 * groups * cols : 0)));
      return p;
    }
  }
  p.grid = static_cast<int>(std::min<int64_t>(rows, 2 * static_cast<int64_t>(sms)));
  return p;
}

int wide_parts(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, 64)); }

std::mutex g_mutex;

template <typename Kernel>
int launch_ring(Kernel kernel, bool (&ready)[64], const Plan& p, int threads, cudaStream_t st, const RmsArgs& a) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(GNS_ERR_DEVICE, "device index out of range");
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!ready[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes + 1024);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      ready[dev] = true;
    }
  }
  kernel<<<p.grid, threads, p.smem, st>>>(a, p.stages);
  return GNS_OK;
}

template <int XD, int T, bool VEC>
int launch_one(bool backward, const Plan& p, cudaStream_t st, const RmsArgs& a) {
  static bool ready[3][64] = {};
  // Forward groups have 32 to 512 threads, backward ones to 1024.
  if constexpr (T <= 512) {
    if (!backward && a.out8.codes != nullptr)
      return launch_ring(rms_forward_kernel<XD, T, VEC, true>, ready[0], p, threads_of<T>(), st, a);
    if (!backward) return launch_ring(rms_forward_kernel<XD, T, VEC, false>, ready[1], p, threads_of<T>(), st, a);
  }
  if (backward) return launch_ring(rms_backward_kernel<XD, T, VEC>, ready[2], p, threads_of<T>(), st, a);
  return fail(GNS_ERR_UNSUPPORTED, "no ring kernel has these threads a row");
}

template <int XD, bool VEC>
int launch_type(bool backward, const Plan& p, cudaStream_t st, const RmsArgs& a) {
  switch (p.threads) {
    case 32: return launch_one<XD, 32, VEC>(backward, p, st, a);
    case 64: return launch_one<XD, 64, VEC>(backward, p, st, a);
    case 128: return launch_one<XD, 128, VEC>(backward, p, st, a);
    case 256: return launch_one<XD, 256, VEC>(backward, p, st, a);
    case 512: return launch_one<XD, 512, VEC>(backward, p, st, a);
    default: return launch_one<XD, 1024, VEC>(backward, p, st, a);
  }
}

int launch_any(bool backward, bool vec, int dt, const Plan& p, cudaStream_t st, const RmsArgs& a) {
  if (dt == kBF16) return vec ? launch_type<kBF16, true>(backward, p, st, a) : launch_type<kBF16, false>(backward, p, st, a);
  if (dt == kF16) return vec ? launch_type<kF16, true>(backward, p, st, a) : launch_type<kF16, false>(backward, p, st, a);
  return vec ? launch_type<kF32, true>(backward, p, st, a) : launch_type<kF32, false>(backward, p, st, a);
}

// Rows that 16-byte pieces can be read from or written to, none past the end.
bool vector_rows(const void* p, int64_t stride, int64_t cols, int dt) {
  const int es = dtype_size(dt);
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * es) % 16 == 0 && (cols * es) % 16 == 0);
}

int check_rms(int x_dtype, int w_dtype, int64_t rows, int64_t cols) {
  if (x_dtype < 0 || x_dtype > 2 || w_dtype < 0 || w_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad dtype");
  if (rows < 0 || cols < 1) return fail(GNS_ERR_ARGUMENT, "a norm needs rows >= 0 and cols >= 1");
  if (cols > (1 << 30)) return fail(GNS_ERR_UNSUPPORTED, "row too wide");
  return GNS_OK;
}

int forward(int x_dtype, int w_dtype, const RmsArgs& given, int64_t rows, int64_t cols, cudaStream_t st) {
  RmsArgs a = given;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.w_dt = w_dtype;
  const bool vec = vector_rows(a.x, a.x_stride, cols, x_dtype) && vector_rows(a.second, a.second_stride, cols, x_dtype) &&
                   vector_rows(a.total, cols, cols, x_dtype) && vector_rows(a.y, cols, cols, x_dtype);
  const Plan plan = plan_rms(kFwd, a.second != nullptr ? 2 : 1, vec, x_dtype, rows, cols);
  if (plan.stages > 0) {
    const int rc = launch_any(false, vec, x_dtype, plan, st, a);
    if (rc != GNS_OK) return rc;
  } else if (a.out8.codes != nullptr) {
    rms_forward_wide_kernel<true><<<plan.grid, kWideThreads, 0, st>>>(a, x_dtype);
  } else {
    rms_forward_wide_kernel<false><<<plan.grid, kWideThreads, 0, st>>>(a, x_dtype);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "RMS norm forward kernel");
}

int check_inputs(int64_t rows, int64_t cols, const void* x, int64_t x_rstride, const void* residual, int64_t residual_rstride,
                 const void* weight, const void* total, const float* rstd) {
  if (rows > 1 && (x_rstride < cols || (residual != nullptr && residual_rstride < cols)))
    return fail(GNS_ERR_LAYOUT, "row stride below the row length");
  if (x == nullptr || weight == nullptr || rstd == nullptr || (residual != nullptr && total == nullptr))
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  return check_device();
}

}  // namespace

int rms_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_rms_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_rms_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "RMS norm status");
}

}  // namespace gns

using namespace gns;

extern "C" {

int gns_rms_norm_forward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                         const void* residual, int64_t residual_rstride, const void* weight, float eps, void* y,
                         void* total, float* rstd, gns_stream_t stream) {
  clear_error();
  int rc = check_rms(x_dtype, w_dtype, rows, cols);
  if (rc != GNS_OK || rows == 0) return rc;
  if (y == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  rc = check_inputs(rows, cols, x, x_rstride, residual, residual_rstride, weight, total, rstd);
  if (rc != GNS_OK) return rc;
  RmsArgs a{};
  a.x = x;
  a.x_stride = x_rstride;
  a.second = residual;
  a.second_stride = residual_rstride;
  a.w = weight;
  a.y = y;
  a.total = residual != nullptr ? total : nullptr;
  a.rstd = rstd;
  a.eps = eps;
  return forward(x_dtype, w_dtype, a, rows, cols, reinterpret_cast<cudaStream_t>(stream));
}

int gns_rms_norm_forward_8bit(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                              const void* residual, int64_t residual_rstride, const void* weight, float eps, void* codes,
                              int64_t codes_rstride, float* scales, int64_t scale_rstride, int64_t scale_cstride,
                              void* total, float* rstd, gns_stream_t stream) {
  clear_error();
  int rc = check_rms(x_dtype, w_dtype, rows, cols);
  if (rc != GNS_OK || rows == 0) return rc;
  if (codes == nullptr || scales == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || codes_rstride % 16 != 0 || codes_rstride < cols)
    return fail(GNS_ERR_LAYOUT, "rows of codes must start on 16 bytes and hold a row");
  rc = check_inputs(rows, cols, x, x_rstride, residual, residual_rstride, weight, total, rstd);
  if (rc != GNS_OK) return rc;
  RmsArgs a{};
  a.x = x;
  a.x_stride = x_rstride;
  a.second = residual;
  a.second_stride = residual_rstride;
  a.w = weight;
  a.total = residual != nullptr ? total : nullptr;
  a.rstd = rstd;
  a.eps = eps;
  a.out8 = {static_cast<uint8_t*>(codes), codes_rstride, static_cast<int>(round_up(cols, 16)), scales, scale_rstride, scale_cstride};
  return forward(x_dtype, w_dtype, a, rows, cols, reinterpret_cast<cudaStream_t>(stream));
}

size_t gns_rms_norm_backward_workspace_size(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  // The most that any type, alignment and number of tensors takes.
  int parts = 0;
  for (int dt : {kF16, kF32})
    for (bool vec : {false, true})
      for (int tensors : {2, 3}) {
        const Plan p = plan_rms(kBwd, tensors, vec, dt, rows, cols);
        parts = std::max(parts, p.stages > 0 ? p.grid : wide_parts(rows));
      }
  return static_cast<size_t>(parts) * static_cast<size_t>(cols) * sizeof(float);
}

int gns_rms_norm_backward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* grad, int64_t grad_rstride,
                          const void* total, int64_t total_rstride, const void* weight, const float* rstd,
                          const void* grad_total, int64_t grad_total_rstride, void* dx, void* dweight, void* workspace,
                          size_t workspace_bytes, gns_stream_t stream) {
  clear_error();
  int rc = check_rms(x_dtype, w_dtype, rows, cols);
  if (rc != GNS_OK) return rc;
  if (dweight == nullptr || (rows > 0 && (grad == nullptr || total == nullptr || weight == nullptr || rstd == nullptr || dx == nullptr)))
    return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (rows > 1 && (grad_rstride < cols || total_rstride < cols || (grad_total != nullptr && grad_total_rstride < cols)))
    return fail(GNS_ERR_LAYOUT, "row stride below the row length");
  const size_t needed = gns_rms_norm_backward_workspace_size(rows, cols);
  if (workspace_bytes < needed || (needed > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 != 0)))
    return fail(GNS_ERR_WORKSPACE, "RMS norm backward workspace too small or not aligned to 4 bytes");
  rc = check_device();
  if (rc != GNS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  RmsArgs a{};
  a.x = total;
  a.x_stride = total_rstride;
  a.second = grad;
  a.second_stride = grad_rstride;
  a.third = grad_total;
  a.third_stride = grad_total_rstride;
  a.w = weight;
  a.y = dx;
  a.rstd = const_cast<float*>(rstd);
  a.partial = static_cast<float*>(workspace);
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.w_dt = w_dtype;
  int parts = 0;
  if (rows > 0) {
    const bool vec = vector_rows(total, total_rstride, cols, x_dtype) && vector_rows(grad, grad_rstride, cols, x_dtype) &&
                     vector_rows(grad_total, grad_total_rstride, cols, x_dtype) && vector_rows(dx, cols, cols, x_dtype);
    const Plan plan = plan_rms(kBwd, grad_total != nullptr ? 3 : 2, vec, x_dtype, rows, cols);
    if (plan.stages > 0) {
      parts = plan.grid;
      rc = launch_any(true, vec, x_dtype, plan, st, a);
      if (rc != GNS_OK) return rc;
    } else {
      parts = wide_parts(rows);
      rms_backward_wide_kernel<<<plan.grid, kWideThreads, 0, st>>>(a, x_dtype);
      const dim3 grid(static_cast<unsigned>((cols + kColThreads - 1) / kColThreads), static_cast<unsigned>(parts));
      rms_columns_wide_kernel<<<grid, kColThreads, 0, st>>>(a, x_dtype);
    }
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>((cols + 31) / 32), 1, 1);
  cfg.blockDim = dim3(32, kJoinRows, 1);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, rms_join_kernel, static_cast<const float*>(a.partial), parts, a.cols, dweight, w_dtype);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "RMS norm backward kernels");
}

}  // extern "C"
