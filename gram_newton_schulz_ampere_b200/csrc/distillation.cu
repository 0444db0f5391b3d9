// Distillation from a teacher's top logits: the loss of each row and its gradient.
//
//   p = softmax over the row's entries of t / T        q = softmax(z / T) over the vocabulary
//   loss = T^2 sum_j p_j (log p_j - log q[i_j])
//   dz_i = g T (q_i - sum of the p_j whose index is i)
//
// An entry whose index is not in the vocabulary has no part in a row; a row without entries
// (or whose entries' logits are all -inf) has a loss and a gradient of zero, whatever its
// logits hold, and they are not read.
//
// One pass over a row finds its largest logit m and s = sum exp((z - m) / T) together (each
// thread rescales its sum when its maximum grows); a second one writes the gradient. A CTA
// has a row, so that both passes of a call with a gradient run while the row is in L2: it
// comes from memory once. Few rows: a cluster of CTAs shares a row and exchanges (m, s)
// through shared memory. z - m is formed before it is scaled: z / T would lose the digits
// that large logits have in common.
//
// The gradient at the row's entries is written over the dense one behind a barrier, the
// entries of one index added up by the first of them in the list's order: no atomics.
#include <algorithm>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;
constexpr int kDeep = 4;  // pieces that a thread loads at once
constexpr int kMaxCluster = 8;

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
    // Not fused, so that both sides of an exchange come to the same bits.
    s = __fadd_rn(__fmul_rn(s, exp2_approx((m - at) * scale)), __fmul_rn(s2, exp2_approx((m2 - at) * scale)));
    m = top;
  }
};

// Sixteen bytes of logits.
template <int XD>
struct Logits {
  static constexpr int kN = XD == kF32 ? 4 : 8;
  uint4 u;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (XD == kF32) return __uint_as_float(w[i % 4]);
    const uint32_t two = w[i / 2 % 4];
    if (XD == kBF16) return __uint_as_float((i & 1) ? (two & 0xffff0000u) : (two << 16));
    return __half2float(__ushort_as_half(static_cast<uint16_t>((i & 1) ? (two >> 16) : two)));
  }
};

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

// A row's entries in shared memory: the index (-1: left out) and its share p.
struct Entries {
  int index[kMaxTop];
  float p[kMaxTop];
  float top, log_sum;  // largest t, log of the sum of exp((t - top) / T)
  int some;            // whether any entry counts
};

// One warp fills a row's entries.
__device__ __forceinline__ void fill_entries(Entries& e, const LossArgs& a, int64_t row, int lane) {
  float top = -INFINITY;
  bool some = false;
  for (int j = lane; j < a.top; j += 32) {
    const int64_t at = row * a.index_stride + j;
    const int64_t i = a.index64 ? static_cast<const int64_t*>(a.index)[at] : static_cast<const int32_t*>(a.index)[at];
    const bool there = i >= 0 && i < a.vocabulary;
    const float t = there ? load_as_float(a.teacher, row * a.teacher_stride + j, a.teacher_dt) : -INFINITY;
    e.index[j] = there ? static_cast<int>(i) : -1;
    e.p[j] = t;
    top = fmaxf(top, t);
    some |= !(t == -INFINITY);  // a NaN counts
  }
  top = warp_max(top);
  some = __any_sync(0xffffffffu, some);
  const float at = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int j = lane; j < a.top; j += 32) sum += exp2_approx((e.p[j] - at) * a.scale);
  sum = warp_add(sum);
  const float inv = __fdiv_rn(1.0f, sum);
  for (int j = lane; j < a.top; j += 32) {
    if (!some || e.p[j] == -INFINITY) e.index[j] = -1;  // a share of zero
    e.p[j] = exp2_approx((e.p[j] - at) * a.scale) * inv;
  }
  if (lane == 0) {
    e.top = at;
    e.log_sum = logf(sum);
    e.some = some ? 1 : 0;
  }
}

// MODE 1: loss. 2: gradient from the statistics of an earlier call. 3: both.
template <int XD, int MODE>
__global__ void __launch_bounds__(kThreads, 2) distillation_kernel(const LossArgs a) {
  constexpr bool kLoss = (MODE & 1) != 0, kGrad = (MODE & 2) != 0;
  using L = Logits<XD>;
  constexpr int N = L::kN;
  constexpr int es = XD == kF32 ? 4 : 2;
  __shared__ Entries entries[2];
  __shared__ float2 warps[2][kWarps];
  __shared__ float2 parts[2][kMaxCluster];
  const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
  const int64_t step = gridDim.x / ctas;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  int turn = 0, exchange = 0;
  for (int64_t row = blockIdx.x / ctas; row < a.rows; row += step, turn ^= 1) {
    const uint8_t* z = static_cast<const uint8_t*>(a.z) + row * a.z_stride * es;
    // The row: `head` elements up to a multiple of 16 bytes, pieces of 16 bytes, the rest.
    const int head = min(a.vocabulary, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(z) & 15u)) & 15u) / es);
    const int pieces = (a.vocabulary - head) / N;
    const int lo = static_cast<int>(static_cast<int64_t>(rank) * pieces / ctas), hi = static_cast<int>(static_cast<int64_t>(rank + 1) * pieces / ctas);
    const uint4* body = reinterpret_cast<const uint4*>(z + head * es);
    // This thread's element outside the pieces: of the head (CTA 0) or the rest (the last CTA).
    const int rest = head + pieces * N + static_cast<int>(threadIdx.x) - 32;
    const int lone = rank == 0 && threadIdx.x < static_cast<unsigned>(head) ? static_cast<int>(threadIdx.x)
                     : rank + 1 == ctas && threadIdx.x >= 32 && rest < a.vocabulary ? rest
                                                                                    : -1;
    Entries& e = entries[turn];
    L first[kDeep];
    if (kLoss) {
#pragma unroll
      for (int q = 0; q < kDeep; ++q) {
        const int i = lo + q * kThreads + static_cast<int>(threadIdx.x);
        if (i < hi) first[q].u = body[i];
      }
    }
    if (warp == 0) fill_entries(e, a, row, lane);
    __syncthreads();
    const bool some = e.some != 0;
    Stat st{-INFINITY, 0.0f};
    if (!some) {
      if (kLoss && rank == 0 && threadIdx.x == 0) {
        a.loss[row] = 0.0f;
        if (a.stats != nullptr) a.stats[row] = make_float2(0.0f, 0.0f);
      }
    } else if (kLoss) {
      for (int i0 = lo; i0 < hi; i0 += kDeep * kThreads) {
        L now[kDeep];
#pragma unroll
        for (int q = 0; q < kDeep; ++q) {
          now[q] = first[q];
          const int i = i0 + (kDeep + q) * kThreads + static_cast<int>(threadIdx.x);
          if (i < hi) first[q].u = body[i];
        }
#pragma unroll
        for (int q = 0; q < kDeep; ++q) {
          if (i0 + q * kThreads + static_cast<int>(threadIdx.x) >= hi) continue;
          float top = now[q].get(0);
#pragma unroll
          for (int k = 1; k < N; ++k) top = fmaxf(top, now[q].get(k));
          if (top > st.m) {
            st.s *= exp2_approx((st.m - top) * a.scale);
            st.m = top;
          }
          const float at = st.base();
#pragma unroll
          for (int k = 0; k < N; ++k) st.s += exp2_approx((now[q].get(k) - at) * a.scale);
        }
      }
      if (lone >= 0) {
        const float v = load_as_float(z, lone, XD);
        // A NaN leaves the maximum and makes the sum one.
        st.join(v == v ? v : -INFINITY, v == v ? 1.0f : v, a.scale);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), a.scale);
      if (lane == 0) warps[turn][warp] = make_float2(st.m, st.s);
      __syncthreads();
      const float2 one = lane < kWarps ? warps[turn][lane] : make_float2(-INFINITY, 0.0f);
      st = {one.x, one.y};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), a.scale);
      if (ctas > 1) {
        // Two buffers in turn: a CTA writes to one again only behind the barrier of the other's
        // exchange, which every reader of it has passed.
        if (threadIdx.x < ctas)
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr(&parts[exchange][rank], threadIdx.x)),
                       "f"(st.m), "f"(st.s)
                       : "memory");
        __syncwarp();
        cluster_sync_all();
        st = {-INFINITY, 0.0f};
        for (uint32_t c = 0; c < ctas; ++c) st.join(parts[exchange][c].x, parts[exchange][c].y, a.scale);
        exchange ^= 1;
      }
      if (rank == 0 && warp == 0) {
        // log2(e) / T times T is log2(e): exponents are differences over T.
        const float inv_t = 1.0f / a.temperature, log_s = logf(st.s);
        float sum = 0.0f;
        for (int j = lane; j < a.top; j += 32) {
          const int i = e.index[j];
          if (i < 0) continue;
          const float t = load_as_float(a.teacher, row * a.teacher_stride + j, a.teacher_dt);
          const float log_p = (t - e.top) * inv_t - e.log_sum;
          const float log_q = (load_as_float(z, i, XD) - st.m) * inv_t - log_s;
          if (e.p[j] != 0.0f) sum = fmaf(e.p[j], log_p - log_q, sum);
        }
        sum = warp_add(sum);
        if (lane == 0) {
          a.loss[row] = a.temperature * a.temperature * sum;
          if (a.stats != nullptr) a.stats[row] = make_float2(st.m, st.s);
        }
      }
    } else {
      const float2 known = a.stats[row];
      st = {known.x, known.y};
    }
    if (!kGrad) continue;
    uint8_t* dz = static_cast<uint8_t*>(a.dz) + row * a.dz_stride * es;
    const float g = some ? a.grad[row] * a.temperature : 0.0f;
    const float at = st.base(), share = some ? __fdiv_rn(1.0f, st.s) : 0.0f, factor = share * g;
    auto value = [&](float v) { return exp2_approx((v - at) * a.scale) * factor; };
    // Pieces of the gradient lie on 16 bytes where its rows start as the logits' do.
    const bool alike = ((reinterpret_cast<uintptr_t>(dz) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
    for (int i0 = lo; i0 < hi; i0 += kDeep * kThreads) {
      L now[kDeep];
#pragma unroll
      for (int q = 0; q < kDeep; ++q) {
        const int i = i0 + q * kThreads + static_cast<int>(threadIdx.x);
        if (i < hi && some) now[q].u = body[i];
      }
#pragma unroll
      for (int q = 0; q < kDeep; ++q) {
        const int i = i0 + q * kThreads + static_cast<int>(threadIdx.x);
        if (i >= hi) continue;
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = some ? value(now[q].get(k)) : 0.0f;
        if (alike) {
          *reinterpret_cast<uint4*>(dz + head * es + static_cast<int64_t>(i) * 16) = packed<XD>(v);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) store_from_float(dz, head + static_cast<int64_t>(i) * N + k, XD, v[k]);
        }
      }
    }
    if (lone >= 0) store_from_float(dz, lone, XD, some ? value(load_as_float(z, lone, XD)) : 0.0f);
    __syncthreads();
    if (!some) continue;
    // Entries of this CTA's stretch, each by its first place in the list.
    const int begin = rank == 0 ? 0 : head + lo * N, end = rank + 1 == ctas ? a.vocabulary : head + hi * N;
    for (int j = threadIdx.x; j < a.top; j += kThreads) {
      const int i = e.index[j];
      if (i < begin || i >= end) continue;
      float p = 0.0f;
      bool is_first = true;
      for (int k = 0; k < a.top; ++k) {
        if (e.index[k] != i) continue;
        is_first &= k >= j;
        p += e.p[k];
      }
      if (is_first) {
        const float q = exp2_approx((load_as_float(z, i, XD) - at) * a.scale) * share;
        store_from_float(dz, i, XD, (q - p) * g);
      }
    }
  }
}

// CTAs that share a row: with rows for all SMs, one; else up to eight, each with 8 KB of it at least.
int row_cluster(int64_t rows, int64_t vocabulary, int dt) {
  const int sms = device_sm_count();
  const int64_t bytes = vocabulary * dtype_size(dt);
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= 2 * sms && bytes / (2 * c) >= 8192) c *= 2;
  return c;
}

template <int XD, int MODE>
int launch(const LossArgs& a, cudaStream_t stream) {
  const int cluster = row_cluster(a.rows, a.vocabulary, XD);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * std::min<int64_t>(a.rows, std::max(1, 2 * device_sm_count() / cluster))));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, distillation_kernel<XD, MODE>, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "distillation loss kernel");
}

template <int MODE>
int launch_any(int dt, const LossArgs& a, cudaStream_t stream) {
  if (dt == kBF16) return launch<kBF16, MODE>(a, stream);
  if (dt == kF16) return launch<kF16, MODE>(a, stream);
  return launch<kF32, MODE>(a, stream);
}

}  // namespace
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
