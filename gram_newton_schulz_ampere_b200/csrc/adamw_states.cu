// AdamW over many tensors at once, with its two moments in 32 bits or in 8.
//
//   g' = s g            (s: an optional scale read from device memory)
//   m  = b1 m + (1 - b1) g'          v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All arithmetic is fp32; the parameter is rounded once, at its store. (The
// other AdamW entry point, adamw_kernel, rounds after every step as the torch
// sequence it replaces does.) sqrt and the division use the approximate
// instructions: their error of about 2^-22 is of the update, far below the
// rounding of the parameter it is added to.
//
// 8-bit states hold e4m3 values with one fp32 scale for each block of 256
// consecutive elements of a tensor, scale = max|m| / 448, so that the block's
// largest value is exact and the codes cover a range of 2^17.8 below it. The
// update uses the new moments before they are rounded. Rounding is to nearest
// even, except that a second moment above zero never rounds to zero: it stays at
// the smallest code, which makes that element's step smaller instead of letting
// m / (0 + eps) make it huge. A warp holds a block in registers (8 elements a
// lane), so the maximum is 8 integer maxima and one warp reduction, and the
// block is read and written once.
//
// Bound by HBM: 10 bytes an element for bf16 parameters and gradients with
// 8-bit states, 22 with 32-bit states.
#include <cuda_fp8.h>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kBlockElems = 256;   // elements that share a scale: 8 for each lane of a warp
constexpr float kE4M3Max = 448.0f;
constexpr float kE4M3Tiny = 0.001953125f;  // 2^-9, the smallest e4m3 value above zero
constexpr float kFlushBelow = 1e-30f;      // a block whose maximum is not above this is held as zeros
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 16384;  // elements of a tensor that one CTA steps
constexpr int kTensors = 128;  // tensors of one launch (8.7 KB of kernel arguments)

struct StateArgs {
  void* p[kTensors];
  const void* g[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  float* m_scale[kTensors];
  float* v_scale[kTensors];
  int64_t numel[kTensors];
  float lr_bc1[kTensors];   // lr / (1 - b1^t)
  float inv_bc2[kTensors];  // 1 / sqrt(1 - b2^t)
  int block_start[kTensors + 1];
  int count;
};

struct StateScalars {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon, decay;
  const float* grad_scale;  // nullptr: 1
};

// The tensor whose CTAs hold `blk`: block_start ascends, and tensors without
// elements have none.
__device__ __forceinline__ int owner_of(const StateArgs& a, int blk) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.block_start[mid] <= blk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void unpack8(const uint4& u, int dt, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t x = w[e];
    const float2 t = (dt == kBF16) ? __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&x))
                                   : __half22float2(*reinterpret_cast<__half2*>(&x));
    f[2 * e] = t.x;
    f[2 * e + 1] = t.y;
  }
}

// 8 consecutive elements; the address is a multiple of 16 bytes.
__device__ __forceinline__ void load8(const void* base, int64_t i, int dt, float (&f)[8]) {
  if (dt == kF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const float4 a = q[0], b = q[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i), dt, f);
  }
}

__device__ __forceinline__ void store8(void* base, int64_t i, int dt, const float (&f)[8]) {
  if (dt == kF32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (dt == kBF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void decode8(uint2 codes, float scale, float (&f)[8]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(w[h >> 1] >> (16 * (h & 1)));
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
    const float2 t = __half22float2(__half2(r));
    f[2 * h] = t.x * scale;
    f[2 * h + 1] = t.y * scale;
  }
}

__device__ __forceinline__ uint2 encode8(const float (&f)[8]) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * h], f[2 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    w[h >> 1] |= two << (16 * (h & 1));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void adamw_math(float g, float& p, float& m, float& v, const StateScalars& k, float scale,
                                           float lr_bc1, float inv_bc2) {
  g *= scale;
  m = fmaf(k.one_minus_beta1, g, m * k.beta1);
  v = fmaf(k.one_minus_beta2, g * g, v * k.beta2);
  const float u = __fdividef(m, fmaf(sqrt_approx(v), inv_bc2, k.epsilon));
  p = fmaf(-lr_bc1, u, p * k.decay);
}

// The largest magnitude of the block, in every lane. Magnitudes order as their
// bits do, and a NaN is above all of them, so it reaches the scale.
__device__ __forceinline__ float block_max(const float (&f)[8]) {
  uint32_t top = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}

__device__ __forceinline__ float inverse_scale(float top) {
  return top <= kFlushBelow ? 0.0f : __fdividef(kE4M3Max, top);
}

// One warp steps one block of 256 elements at `i` whose 8-bit states it decodes,
// updates and encodes. VEC: lane L holds elements 8 L .. 8 L + 7, all in range and
// aligned; otherwise lane L holds L, L + 32, ..., with `left` elements in range.
template <bool VEC>
__device__ __forceinline__ void step_block(void* p, const void* g, void* m, void* v, float* m_scale, float* v_scale,
                                           int64_t i, int left, int lane, int p_dt, int g_dt, const StateScalars& k,
                                           float scale, float lr_bc1, float inv_bc2) {
  const int64_t block = i / kBlockElems;
  float pf[8], gf[8], mf[8], vf[8];
  const float ms = m_scale[block], vs = v_scale[block];
  uint8_t* mq = static_cast<uint8_t*>(m) + i;
  uint8_t* vq = static_cast<uint8_t*>(v) + i;
  if (VEC) {
    load8(g, i + 8 * lane, g_dt, gf);
    load8(p, i + 8 * lane, p_dt, pf);
    const uint2 mc = reinterpret_cast<const uint2*>(mq)[lane];
    const uint2 vc = reinterpret_cast<const uint2*>(vq)[lane];
    decode8(mc, ms, mf);
    decode8(vc, vs, vf);
  } else {
    uint2 mc = make_uint2(0u, 0u), vc = make_uint2(0u, 0u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = lane + 32 * e;
      const bool in = at < left;
      gf[e] = in ? load_as_float(g, i + at, g_dt) : 0.0f;
      pf[e] = in ? load_as_float(p, i + at, p_dt) : 0.0f;
      const uint32_t a = in ? mq[at] : 0u, b = in ? vq[at] : 0u;
      (e < 4 ? mc.x : mc.y) |= a << (8 * (e & 3));
      (e < 4 ? vc.x : vc.y) |= b << (8 * (e & 3));
    }
    decode8(mc, ms, mf);
    decode8(vc, vs, vf);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) adamw_math(gf[e], pf[e], mf[e], vf[e], k, scale, lr_bc1, inv_bc2);
  const float m_top = block_max(mf), v_top = block_max(vf);
  const float m_inv = inverse_scale(m_top), v_inv = inverse_scale(v_top);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    mf[e] *= m_inv;
    const float y = vf[e] * v_inv;
    vf[e] = (vf[e] > 0.0f && y < kE4M3Tiny) ? kE4M3Tiny : y;
  }
  const uint2 mc = encode8(mf), vc = encode8(vf);
  if (VEC) {
    store8(p, i + 8 * lane, p_dt, pf);
    reinterpret_cast<uint2*>(mq)[lane] = mc;
    reinterpret_cast<uint2*>(vq)[lane] = vc;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = lane + 32 * e;
      if (at >= left) continue;
      store_from_float(p, i + at, p_dt, pf[e]);
      mq[at] = static_cast<uint8_t>((e < 4 ? mc.x : mc.y) >> (8 * (e & 3)));
      vq[at] = static_cast<uint8_t>((e < 4 ? vc.x : vc.y) >> (8 * (e & 3)));
    }
  }
  if (lane == 0) {
    m_scale[block] = m_top * (1.0f / kE4M3Max);
    v_scale[block] = v_top * (1.0f / kE4M3Max);
  }
}

// P, G >= 0 fix the types at compile time (the common combinations); -1 takes
// them from the arguments.
template <int P, int G>
__global__ void __launch_bounds__(kThreads) adamw_8bit_kernel(const __grid_constant__ StateArgs args, int p_rt, int g_rt,
                                                              const StateScalars k) {
  const int p_dt = P >= 0 ? P : p_rt;
  const int g_dt = G >= 0 ? G : g_rt;
  const int t = owner_of(args, blockIdx.x);
  const int64_t n = args.numel[t];
  const int64_t start = static_cast<int64_t>(blockIdx.x - args.block_start[t]) * kChunk;
  const int64_t end = min(n, start + kChunk);
  void* p = args.p[t];
  const void* g = args.g[t];
  void* m = args.m[t];
  void* v = args.v[t];
  float* ms = args.m_scale[t];
  float* vs = args.v_scale[t];
  const float lr_bc1 = args.lr_bc1[t], inv_bc2 = args.inv_bc2[t];
  const float scale = k.grad_scale != nullptr ? *k.grad_scale : 1.0f;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g);
  const uintptr_t half = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  const bool vec = wide % 16 == 0 && half % 8 == 0;
  const int lane = threadIdx.x & 31;
  for (int64_t i = start + static_cast<int64_t>(threadIdx.x >> 5) * kBlockElems; i < end;
       i += kWarps * kBlockElems) {
    if (vec && i + kBlockElems <= end)
      step_block<true>(p, g, m, v, ms, vs, i, kBlockElems, lane, p_dt, g_dt, k, scale, lr_bc1, inv_bc2);
    else
      step_block<false>(p, g, m, v, ms, vs, i, static_cast<int>(min(static_cast<int64_t>(kBlockElems), end - i)), lane,
                        p_dt, g_dt, k, scale, lr_bc1, inv_bc2);
  }
}

template <int P, int G>
__global__ void __launch_bounds__(kThreads) adamw_32bit_kernel(const __grid_constant__ StateArgs args, int p_rt,
                                                               int g_rt, const StateScalars k) {
  const int p_dt = P >= 0 ? P : p_rt;
  const int g_dt = G >= 0 ? G : g_rt;
  const int t = owner_of(args, blockIdx.x);
  const int64_t n = args.numel[t];
  const int64_t start = static_cast<int64_t>(blockIdx.x - args.block_start[t]) * kChunk;
  const int64_t end = min(n, start + kChunk);
  void* p = args.p[t];
  const void* g = args.g[t];
  void* m = args.m[t];
  void* v = args.v[t];
  const float lr_bc1 = args.lr_bc1[t], inv_bc2 = args.inv_bc2[t];
  const float scale = k.grad_scale != nullptr ? *k.grad_scale : 1.0f;
  const uintptr_t all = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
                        reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  int64_t i = start;
  if (all % 16 == 0) {
    const int64_t vend = start + (end - start) / 8 * 8;
#pragma unroll 2
    for (i = start + threadIdx.x * 8; i < vend; i += kThreads * 8) {
      float pf[8], gf[8], mf[8], vf[8];
      load8(g, i, g_dt, gf);
      load8(p, i, p_dt, pf);
      load8(m, i, kF32, mf);
      load8(v, i, kF32, vf);
#pragma unroll
      for (int e = 0; e < 8; ++e) adamw_math(gf[e], pf[e], mf[e], vf[e], k, scale, lr_bc1, inv_bc2);
      store8(p, i, p_dt, pf);
      store8(m, i, kF32, mf);
      store8(v, i, kF32, vf);
    }
    i = vend;
  }
  for (int64_t j = i + threadIdx.x; j < end; j += kThreads) {
    float pf = load_as_float(p, j, p_dt), mf = static_cast<float*>(m)[j], vf = static_cast<float*>(v)[j];
    adamw_math(load_as_float(g, j, g_dt), pf, mf, vf, k, scale, lr_bc1, inv_bc2);
    store_from_float(p, j, p_dt, pf);
    static_cast<float*>(m)[j] = mf;
    static_cast<float*>(v)[j] = vf;
  }
}

template <int P, int G>
void launch(int bits, int blocks, cudaStream_t st, const StateArgs& a, int p_dt, int g_dt, const StateScalars& k) {
  if (bits == 8)
    adamw_8bit_kernel<P, G><<<blocks, kThreads, 0, st>>>(a, p_dt, g_dt, k);
  else
    adamw_32bit_kernel<P, G><<<blocks, kThreads, 0, st>>>(a, p_dt, g_dt, k);
}

}  // namespace
}  // namespace gns

using namespace gns;

extern "C" int gns_adamw_states_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs,
                                     void* const* exp_avg_sqs, float* const* exp_avg_scales,
                                     float* const* exp_avg_sq_scales, const int64_t* numel, int p_dtype, int g_dtype,
                                     int state_bits, const float* lr_bc1, const float* inv_bc2, float beta1,
                                     float one_minus_beta1, float beta2, float one_minus_beta2, float epsilon,
                                     float decay, const float* grad_scale, gns_stream_t stream) {
  clear_error();
  if (state_bits != 8 && state_bits != 32) return fail(GNS_ERR_ARGUMENT, "state_bits must be 8 or 32");
  for (int dt : {p_dtype, g_dtype})
    if (dt < 0 || dt > 2) return fail(GNS_ERR_ARGUMENT, "bad dtype");
  if (count < 0 || (count > 0 && (params == nullptr || grads == nullptr || exp_avgs == nullptr ||
                                  exp_avg_sqs == nullptr || numel == nullptr || lr_bc1 == nullptr ||
                                  inv_bc2 == nullptr)))
    return fail(GNS_ERR_ARGUMENT, "bad tensor list");
  if (count > 0 && state_bits == 8 && (exp_avg_scales == nullptr || exp_avg_sq_scales == nullptr))
    return fail(GNS_ERR_ARGUMENT, "8-bit states need their scales");
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0) return fail(GNS_ERR_ARGUMENT, "negative numel");
    if (numel[i] == 0) continue;
    if (params[i] == nullptr || grads[i] == nullptr || exp_avgs[i] == nullptr || exp_avg_sqs[i] == nullptr ||
        (state_bits == 8 && (exp_avg_scales[i] == nullptr || exp_avg_sq_scales[i] == nullptr)))
      return fail(GNS_ERR_ARGUMENT, "null tensor pointer");
    if (numel[i] > (1ll << 44)) return fail(GNS_ERR_UNSUPPORTED, "tensor too large");
  }
  if (count == 0) return GNS_OK;
  int rc = check_device();
  if (rc != GNS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const StateScalars k{beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon, decay, grad_scale};
  int i = 0;
  while (i < count) {
    StateArgs a;
    a.count = 0;
    int64_t blocks = 0;
    for (; i < count && a.count < kTensors; ++i) {
      if (numel[i] == 0) continue;
      const int64_t nb = (numel[i] + kChunk - 1) / kChunk;
      if (blocks > 0 && blocks + nb > (1ll << 30)) break;  // next launch
      const int j = a.count++;
      a.p[j] = params[i];
      a.g[j] = grads[i];
      a.m[j] = exp_avgs[i];
      a.v[j] = exp_avg_sqs[i];
      a.m_scale[j] = state_bits == 8 ? exp_avg_scales[i] : nullptr;
      a.v_scale[j] = state_bits == 8 ? exp_avg_sq_scales[i] : nullptr;
      a.numel[j] = numel[i];
      a.lr_bc1[j] = lr_bc1[i];
      a.inv_bc2[j] = inv_bc2[i];
      a.block_start[j] = static_cast<int>(blocks);
      blocks += nb;
    }
    if (a.count == 0) break;
    a.block_start[a.count] = static_cast<int>(blocks);
    const int grid = static_cast<int>(blocks);
    if (p_dtype == kBF16 && g_dtype == kBF16)
      launch<kBF16, kBF16>(state_bits, grid, st, a, p_dtype, g_dtype, k);
    else if (p_dtype == kF32 && g_dtype == kF32)
      launch<kF32, kF32>(state_bits, grid, st, a, p_dtype, g_dtype, k);
    else if (p_dtype == kF16 && g_dtype == kF16)
      launch<kF16, kF16>(state_bits, grid, st, a, p_dtype, g_dtype, k);
    else if (p_dtype == kBF16 && g_dtype == kF32)
      launch<kBF16, kF32>(state_bits, grid, st, a, p_dtype, g_dtype, k);
    else
      launch<-1, -1>(state_bits, grid, st, a, p_dtype, g_dtype, k);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "adamw states kernel");
  }
  return GNS_OK;
}
