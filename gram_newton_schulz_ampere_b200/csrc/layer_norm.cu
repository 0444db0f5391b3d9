// Layer norm over the last dimension, forward and backward.
//
//   forward   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//             y = (x - mu) r w + b;  mu and r are kept in fp32 for the backward pass
//   backward  h = (x - mu) r,  a = w dy,  c1 = mean(a h),  c2 = mean(a)
//             dx = r (a - c2 - h c1);  dw = sum over rows of dy h;  db = sum of dy
//
// A row is held in the registers of TPR threads, 16 elements each, so x (and dy)
// are read once: the mean is subtracted before the squares are summed, which
// costs a second reduction but no second read. Rows go to the groups of a
// persistent grid round robin; the next row's loads are issued before the
// current row's reduction, so that memory does not wait for the barrier. Each
// thread keeps the same columns for all its rows: w and b stay in registers, and
// dw and db are summed there over the rows, written once per CTA and joined by a
// second kernel in a fixed order (no atomics, the same bits on every run).
// Statistics, sums and all arithmetic are fp32; y, dx, dw and db are rounded
// once, at their stores. Bound by HBM: 2 elements moved forward, 3 backward.
#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kPer = 16;        // elements of a row per thread
constexpr int kMaxTPR = 1024;   // threads of a row; wider rows are read twice (the wide kernels)
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
  int64_t rows;
  int cols, w_dt, parts;
  float eps;
};

// One thread's 16 elements of a row as loaded. VEC: 16-byte pieces, V elements
// each, piece j of thread t at element (j TPR + t) V; otherwise element i of
// thread t is i TPR + t.
template <int XD, int TPR, bool VEC>
struct Piece {
  static constexpr int kV = XD == kF32 ? 4 : 8;
  static constexpr int kWords = XD == kF32 ? 16 : 8;
  uint32_t w[kWords];

  static __device__ __forceinline__ int col(int t, int i) {
    return VEC ? ((i / kV) * TPR + t) * kV + i % kV : i * TPR + t;
  }

  __device__ __forceinline__ void load(const void* base, int64_t row, int64_t stride, int t, int cols, bool live) {
    constexpr int es = XD == kF32 ? 4 : 2;
    const uint8_t* p = static_cast<const uint8_t*>(base) + row * stride * es;
    if (VEC) {
#pragma unroll
      for (int j = 0; j < kPer / kV; ++j) {
        const int c = (j * TPR + t) * kV;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (live && c < cols) u = *reinterpret_cast<const uint4*>(p + static_cast<int64_t>(c) * es);
        w[4 * j] = u.x; w[4 * j + 1] = u.y; w[4 * j + 2] = u.z; w[4 * j + 3] = u.w;
      }
    } else if (XD == kF32) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = i * TPR + t;
        w[i % kWords] = (live && c < cols) ? reinterpret_cast<const uint32_t*>(p)[c] : 0u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
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

template <int XD, int TPR, bool VEC>
__device__ __forceinline__ void store_row(void* base, int64_t row, int cols, int t, const float (&v)[kPer]) {
  using P = Piece<XD, TPR, VEC>;
  constexpr int es = XD == kF32 ? 4 : 2;
  uint8_t* p = static_cast<uint8_t*>(base) + row * cols * es;
  if (VEC) {
#pragma unroll
    for (int j = 0; j < kPer / P::kV; ++j) {
      const int c = (j * TPR + t) * P::kV;
      if (c >= cols) continue;
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (XD == kF32) {
          o[q] = __float_as_uint(v[j * P::kV + q]);
        } else if (XD == kBF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[(j * P::kV + 2 * q) % kPer], v[(j * P::kV + 2 * q + 1) % kPer]);
          o[q] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[(j * P::kV + 2 * q) % kPer], v[(j * P::kV + 2 * q + 1) % kPer]);
          o[q] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(p + static_cast<int64_t>(c) * es) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i * TPR + t;
      if (c < cols) store_from_float(p, c, XD, v[i]);
    }
  }
}

// Sums of (a, b) over the TPR threads of each row group, in every thread of it.
// `slot` alternates between two buffers, so one barrier per call is enough: a
// buffer is written again only after the other buffer's barrier, which every
// reader of it has passed.
template <int TPR, int THREADS>
__device__ __forceinline__ float2 group_sum(float a, float b, float2 (*slots)[THREADS / 32], int& slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
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
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
  return make_float2(a, b);
}

template <int TPR>
constexpr int threads_of() {
  return TPR < 256 ? 256 : TPR;
}

template <int XD, int TPR, bool VEC>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_forward_kernel(const NormArgs a) {
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
    const float mu = group_sum<TPR, kThreads>(sum, 0.0f, slots, slot).x * inv_n;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] -= mu;
      if (P::col(t, i) < a.cols) sq = fmaf(v[i], v[i], sq);
    }
    const float var = group_sum<TPR, kThreads>(sq, 0.0f, slots, slot).x * inv_n;
    const float r = rsqrtf(var + a.eps);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = fmaf(v[i] * r, w[i], b[i]);
    if (live) {
      store_row<XD, TPR, VEC>(a.y, row, a.cols, t, v);
      if (t == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
  }
}

template <int XD, int TPR, bool VEC>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_backward_kernel(const NormArgs a) {
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
    if (live) store_row<XD, TPR, VEC>(a.y, row, a.cols, t, g);
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
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
          if (c < a.cols) out[which * a.cols + c] = sum;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = P::col(t, i);
        if (c < a.cols) out[which * a.cols + c] = which ? db[i] : dw[i];
      }
    }
  }
}

// Rows too wide for the registers of a CTA: a CTA per row, read again for each pass.
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

// Threads of a row: the fewest that hold it at 16 elements each, a warp at least.
int threads_per_row(int64_t cols) {
  int t = 32;
  while (t < kMaxTPR && static_cast<int64_t>(t) * kPer < cols) t *= 2;
  return t;
}

bool is_wide(int64_t cols) { return cols > static_cast<int64_t>(kMaxTPR) * kPer; }

// CTAs of the persistent grids: enough for two thirds of an SM's threads, and no
// more than there are rows for.
int norm_grid(int64_t rows, int64_t cols) {
  const int tpr = threads_per_row(cols);
  const int threads = tpr < 256 ? 256 : tpr;
  const int64_t turns = (rows + threads / tpr - 1) / (threads / tpr);
  const int64_t most = static_cast<int64_t>(device_sm_count()) * (threads >= 1024 ? 1 : 768 / threads);
  return static_cast<int>(turns < most ? turns : most);
}

int backward_parts(int64_t rows, int64_t cols) {
  if (!is_wide(cols)) return norm_grid(rows, cols);
  return static_cast<int>(rows < 64 ? rows : 64);
}

template <int XD, int TPR, bool VEC>
void launch_norm(bool backward, int grid, cudaStream_t st, const NormArgs& a) {
  if (backward)
    norm_backward_kernel<XD, TPR, VEC><<<grid, threads_of<TPR>(), 0, st>>>(a);
  else
    norm_forward_kernel<XD, TPR, VEC><<<grid, threads_of<TPR>(), 0, st>>>(a);
}

template <int XD, bool VEC>
void launch_rows(bool backward, int grid, cudaStream_t st, const NormArgs& a) {
  switch (threads_per_row(a.cols)) {
    case 32: return launch_norm<XD, 32, VEC>(backward, grid, st, a);
    case 64: return launch_norm<XD, 64, VEC>(backward, grid, st, a);
    case 128: return launch_norm<XD, 128, VEC>(backward, grid, st, a);
    case 256: return launch_norm<XD, 256, VEC>(backward, grid, st, a);
    case 512: return launch_norm<XD, 512, VEC>(backward, grid, st, a);
    default: return launch_norm<XD, 1024, VEC>(backward, grid, st, a);
  }
}

void launch_any(bool backward, bool vec, int x_dt, int grid, cudaStream_t st, const NormArgs& a) {
  if (x_dt == kBF16)
    vec ? launch_rows<kBF16, true>(backward, grid, st, a) : launch_rows<kBF16, false>(backward, grid, st, a);
  else if (x_dt == kF16)
    vec ? launch_rows<kF16, true>(backward, grid, st, a) : launch_rows<kF16, false>(backward, grid, st, a);
  else
    vec ? launch_rows<kF32, true>(backward, grid, st, a) : launch_rows<kF32, false>(backward, grid, st, a);
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
  if (is_wide(cols)) {
    const int64_t most = 2 * static_cast<int64_t>(device_sm_count());
    norm_forward_wide_kernel<<<static_cast<int>(rows < most ? rows : most), kWideThreads, 0, st>>>(a, x_dtype);
  } else {
    const bool vec = rows_vector(x, x_rstride, cols, x_dtype) && rows_vector(y, cols, cols, x_dtype);
    launch_any(false, vec, x_dtype, norm_grid(rows, cols), st, a);
  }
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "layer norm forward kernel");
}

size_t gns_layer_norm_backward_workspace_size(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  return static_cast<size_t>(backward_parts(rows, cols)) * 2 * static_cast<size_t>(cols) * sizeof(float);
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
  if (workspace_bytes < gns_layer_norm_backward_workspace_size(rows, cols) || (rows > 0 && workspace == nullptr))
    return fail(GNS_ERR_WORKSPACE, "layer norm backward workspace too small");
  if (rows > 0 && reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
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
  a.parts = rows > 0 ? backward_parts(rows, cols) : 0;
  if (rows > 0) {
    if (is_wide(cols)) {
      const int64_t most = 2 * static_cast<int64_t>(device_sm_count());
      norm_backward_wide_kernel<<<static_cast<int>(rows < most ? rows : most), kWideThreads, 0, st>>>(a, x_dtype);
      const dim3 grid(static_cast<unsigned>((cols + kColThreads - 1) / kColThreads), static_cast<unsigned>(a.parts));
      norm_columns_wide_kernel<<<grid, kColThreads, 0, st>>>(a, x_dtype);
    } else {
      const bool vec = rows_vector(x, x_rstride, cols, x_dtype) && rows_vector(grad, grad_rstride, cols, x_dtype) &&
                       rows_vector(dx, cols, cols, x_dtype);
      launch_any(true, vec, x_dtype, a.parts, st, a);
    }
  }
  const int join = static_cast<int>((2 * cols + 31) / 32);
  norm_join_kernel<<<join, dim3(32, kJoinRows), 0, st>>>(a.partial, a.parts, a.cols, dweight, dbias, w_dtype);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "layer norm backward kernels");
}

}  // extern "C"
