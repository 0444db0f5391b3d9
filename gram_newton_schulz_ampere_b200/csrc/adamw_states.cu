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
// m / (0 + eps) make it huge. Rounding to nearest has no memory: a moment that decays
// by less than half a code a step stays where it is, and a second moment above its
// exact value comes down only as its block's scale does. UNBIASED instead rounds up or
// down with the probabilities that make the mean right, by bits that follow from the step
// number and the element's place (3000 steps at b2 = 0.95, elements a tenth of their
// block's largest: sqrt(v) 1.45 times the exact one to nearest, 0.997 unbiased). It costs
// three instructions an element: 323M bf16 elements 501 us to nearest, 562 unbiased.
// A warp holds a block in registers (8 elements a
// lane), so the maximum is 8 integer maxima and one warp reduction, and the
// block is read and written once.
//
// Bound by HBM: 10 bytes an element for bf16 parameters and gradients with
// 8-bit states, 22 with 32-bit states.
#include <cuda_fp8.h>

#include <mutex>

#include "../../include/gns_b200.h"
#include "gns_common.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kBlockElems = 256;   // elements that share a scale: 8 for each lane of a warp
constexpr float kE4M3Max = 448.0f;
constexpr float kFlushBelow = 1e-30f;      // a block whose maximum is not above this is held as zeros
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunkMin = kWarps * kBlockElems;  // elements of a tensor that one CTA steps, at least
constexpr int kChunkMax = 16 * kChunkMin;        // and at most (a warp's lanes hold its blocks' scales: 32 at most)
constexpr int kTensors = 128;  // tensors of one launch (8.7 KB of kernel arguments)

constexpr bool sixteen(int dt) { return dt == kF16 || dt == kBF16; }

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
  uint32_t key[kTensors];   // of the random bits: from the step number and the tensor's place
  int block_start[kTensors + 1];
  int count;
  int chunk;  // elements of a tensor that one CTA steps
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

__device__ __forceinline__ float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The largest magnitude of three; NaN if any is.
__device__ __forceinline__ float largest(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

// 8 consecutive elements of a type as loaded; the address is a multiple of 16 bytes.
// D < 0: the type is known at run time only.
template <int D>
struct Eight {
  uint4 u[D == kF16 || D == kBF16 ? 1 : 2];

  __device__ __forceinline__ void load(const void* base, int64_t i, int dt) {
    if (dt == kF32) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
      u[0] = q[0];
      u[sizeof(u) / sizeof(uint4) - 1] = q[1];
    } else {
      u[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
    }
  }

  __device__ __forceinline__ void get(int dt, float (&f)[8]) const {
    if (dt == kF32) {
      const uint4 a = u[0], b = u[sizeof(u) / sizeof(uint4) - 1];
      f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
      f[4] = __uint_as_float(b.x); f[5] = __uint_as_float(b.y); f[6] = __uint_as_float(b.z); f[7] = __uint_as_float(b.w);
    } else {
      unpack8(u[0], dt, f);
    }
  }
};

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

__device__ __forceinline__ void decode8(uint2 codes, float (&f)[8]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(w[h >> 1] >> (16 * (h & 1)));
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
    const float2 t = __half22float2(__half2(r));
    f[2 * h] = t.x;
    f[2 * h + 1] = t.y;
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

// Spreads differences of its argument over all bits: odd multiples of 2^32 / golden ratio,
// the upper bits folded into the lower ones.
__host__ __device__ __forceinline__ uint32_t scramble(uint32_t x) {
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x9E3779B1u;
  x ^= x >> 13;
  x *= 0x9E3779B1u;
  return x ^ (x >> 16);
}

// Rounds four values up or down to e4m3, up with the probability of their place between
// the two codes (to 16 bits: the lower 16 of `random` serve two of them, the upper the
// others). The first value is the lowest byte.
__device__ __forceinline__ uint32_t encode4_unbiased(float a, float b, float c, float d, uint32_t random) {
  uint32_t four;
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%4, %3, %2, %1}, %5;" : "=r"(four) : "f"(a), "f"(b), "f"(c), "f"(d), "r"(random));
  return four;
}

// `word`: the first of the two random words' numbers.
template <bool UNBIASED>
__device__ __forceinline__ uint2 encode(const float (&f)[8], uint32_t key, uint32_t word) {
  if (!UNBIASED) return encode8(f);
  return make_uint2(encode4_unbiased(f[0], f[1], f[2], f[3], scramble(key + word)),
                    encode4_unbiased(f[4], f[5], f[6], f[7], scramble(key + word + 1u)));
}

__device__ __forceinline__ float adamw_update(float p, float m, float v, const StateScalars& k, float lr_bc1,
                                              float inv_bc2) {
  const float u = m * reciprocal_approx(fmaf(sqrt_approx(v), inv_bc2, k.epsilon));
  return fmaf(-lr_bc1, u, p * k.decay);
}

__device__ __forceinline__ void adamw_math(float g, float& p, float& m, float& v, const StateScalars& k, float scale,
                                           float lr_bc1, float inv_bc2) {
  g *= scale;
  m = fmaf(k.one_minus_beta1, g, m * k.beta1);
  v = fmaf(k.one_minus_beta2, g * g, v * k.beta2);
  p = adamw_update(p, m, v, k, lr_bc1, inv_bc2);
}

// The largest magnitude of the block, in every lane. Magnitudes order as their
// bits do, and a NaN is above all of them, so it reaches the scale.
__device__ __forceinline__ float block_max(const float (&f)[8]) {
  const float top = largest(largest(f[0], f[1], f[2]), largest(f[3], f[4], f[5]), largest(f[6], f[7], 0.0f));
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu));
}

// 448 / top for the codes of a block; 0 for a block that is held as zeros. Correctly
// rounded, as the moments are: a code that is rounded the other way moves by 6%, so
// all that leads to it is kept free of choices.
__device__ __forceinline__ float inverse_scale(float top) {
  return top <= kFlushBelow ? 0.0f : __fmul_rn(kE4M3Max, __frcp_rn(top));
}

// Per-launch constants of one tensor.
struct Step {
  float scale, lr_bc1, inv_bc2;
  uint32_t key;

  __device__ __forceinline__ Step(const StateArgs& a, const StateScalars& k, int t)
      : scale(k.grad_scale != nullptr ? *k.grad_scale : 1.0f), lr_bc1(a.lr_bc1[t]), inv_bc2(a.inv_bc2[t]), key(a.key[t]) {}
};

__device__ __forceinline__ bool has_zero_byte(uint32_t w) { return ((w - 0x01010101u) & ~w & 0x80808080u) != 0u; }

// New moments and parameter of a lane's 8 elements of a block, the moments' codes and
// the block's scales (in every lane). `block` is the block's number in its tensor; the
// random words repeat after 2^25 blocks.
template <bool UNBIASED>
__device__ __forceinline__ void step_eight(const float (&gf)[8], float (&pf)[8], uint2& mc, uint2& vc, float& ms,
                                           float& vs, const StateScalars& k, const Step& s, uint32_t block) {
  float mf[8], vf[8];
  decode8(mc, mf);
  decode8(vc, vf);
  // Every product and sum of the moments is rounded by itself (no fma). Elements go two
  // to an instruction: one at a time, the kernel issued 38 instructions an element and
  // took 5% longer.
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const Pair g = mul2(Pair(gf[e], gf[e + 1]), Pair(s.scale));
    // (The sums are scalar: a paired add of two products is fused with one of them.)
    float m0, m1, v0, v1;
    mul2(mul2(Pair(mf[e], mf[e + 1]), Pair(ms)), Pair(k.beta1)).get(mf[e], mf[e + 1]);
    mul2(g, Pair(k.one_minus_beta1)).get(m0, m1);
    mul2(mul2(Pair(vf[e], vf[e + 1]), Pair(vs)), Pair(k.beta2)).get(vf[e], vf[e + 1]);
    mul2(mul2(g, g), Pair(k.one_minus_beta2)).get(v0, v1);
    mf[e] = __fadd_rn(mf[e], m0);
    mf[e + 1] = __fadd_rn(mf[e + 1], m1);
    vf[e] = __fadd_rn(vf[e], v0);
    vf[e + 1] = __fadd_rn(vf[e + 1], v1);
    float d0, d1;
    fma2(Pair(sqrt_approx(vf[e]), sqrt_approx(vf[e + 1])), Pair(s.inv_bc2), Pair(k.epsilon)).get(d0, d1);
    const Pair u = mul2(Pair(mf[e], mf[e + 1]), Pair(reciprocal_approx(d0), reciprocal_approx(d1)));
    fma2(Pair(-s.lr_bc1), u, mul2(Pair(pf[e], pf[e + 1]), Pair(k.decay))).get(pf[e], pf[e + 1]);
  }
  const float m_top = block_max(mf), v_top = block_max(vf);
  // One lane in two works out the inverse for m, the other for v.
  const float inverse = inverse_scale((threadIdx.x & 1) ? v_top : m_top);
  const float m_inv = __shfl_sync(0xffffffffu, inverse, 0), v_inv = __shfl_sync(0xffffffffu, inverse, 1);
  float yf[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    mul2(Pair(mf[e], mf[e + 1]), Pair(m_inv)).get(mf[e], mf[e + 1]);
    Pair y = mul2(Pair(vf[e], vf[e + 1]), Pair(v_inv));
    y.get(yf[e], yf[e + 1]);
  }
  const uint32_t word = block * 128u + (threadIdx.x & 31u) * 4u;
  mc = encode<UNBIASED>(mf, s.key, word);
  vc = encode<UNBIASED>(yf, s.key, word + 2u);
  // Codes of zero are rare: only where there is one is it seen to that its second
  // moment is zero.
  if (has_zero_byte(vc.x) || has_zero_byte(vc.y)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t& w = e < 4 ? vc.x : vc.y;
      const uint32_t byte = 0xffu << (8 * (e & 3));
      if (vf[e] > 0.0f && (w & byte) == 0u) w |= 1u << (8 * (e & 3));
    }
  }
  ms = m_top * (1.0f / kE4M3Max);
  vs = v_top * (1.0f / kE4M3Max);
}

// A lane's elements L, L + 32, ... of a block, wherever it starts: from `base` on, in
// global or shared memory.
__device__ __forceinline__ void gather8(const void* base, int lane, int left, int dt, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = lane + 32 * e < left ? load_as_float(base, lane + 32 * e, dt) : 0.0f;
}

__device__ __forceinline__ uint2 gather_codes(const uint8_t* base, int lane, int left) {
  uint2 c = make_uint2(0u, 0u);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = lane + 32 * e < left ? base[lane + 32 * e] : 0u;
    (e < 4 ? c.x : c.y) |= b << (8 * (e & 3));
  }
  return c;
}

__device__ __forceinline__ void scatter8(void* base, int lane, int left, int dt, const float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (lane + 32 * e < left) store_from_float(base, lane + 32 * e, dt, f[e]);
}

__device__ __forceinline__ void scatter_codes(uint8_t* base, int lane, int left, uint2 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (lane + 32 * e < left) base[lane + 32 * e] = static_cast<uint8_t>((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
}

// The last, incomplete block of a tensor: `left` elements at `i`.
template <bool UNBIASED>
__device__ __noinline__ void step_ragged(const StateArgs& args, int t, int64_t i, int left, int p_dt, int g_dt,
                                         const StateScalars& k) {
  const int lane = threadIdx.x & 31;
  uint8_t* p = static_cast<uint8_t*>(args.p[t]) + i * (p_dt == kF32 ? 4 : 2);
  const uint8_t* g = static_cast<const uint8_t*>(args.g[t]) + i * (g_dt == kF32 ? 4 : 2);
  uint8_t* m = static_cast<uint8_t*>(args.m[t]) + i;
  uint8_t* v = static_cast<uint8_t*>(args.v[t]) + i;
  float* m_scale = args.m_scale[t] + i / kBlockElems;
  float* v_scale = args.v_scale[t] + i / kBlockElems;
  const Step s(args, k, t);
  float pf[8], gf[8];
  gather8(p, lane, left, p_dt, pf);
  gather8(g, lane, left, g_dt, gf);
  uint2 mc = gather_codes(m, lane, left), vc = gather_codes(v, lane, left);
  float ms = *m_scale, vs = *v_scale;
  step_eight<UNBIASED>(gf, pf, mc, vc, ms, vs, k, s, static_cast<uint32_t>(i / kBlockElems));
  scatter8(p, lane, left, p_dt, pf);
  scatter_codes(m, lane, left, mc);
  scatter_codes(v, lane, left, vc);
  if (lane == 0) {
    *m_scale = ms;
    *v_scale = vs;
  }
}

__device__ int g_states_status = 0;

// Ring slots of a warp: a block's parameters, gradients and codes.
constexpr int kSlots = 4;

template <int P, int G, bool ALIGNED>
struct Slot {
  static constexpr uint32_t kP = kBlockElems * (sixteen(P) ? 2 : 4);
  static constexpr uint32_t kG = kBlockElems * (sixteen(G) ? 2 : 4);
  static constexpr uint32_t kSpare = ALIGNED ? 0 : 16;  // for what a copy starts ahead of its row
  static constexpr uint32_t kBytes = kP + kG + 2 * kBlockElems + 4 * kSpare;
  static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kSlots * kBytes;
};

// P, G >= 0 fix the types at compile time (the common combinations); -1 takes
// them from the arguments.
//
// Each warp steps consecutive blocks of the chunk. Bulk copies bring them into a
// ring of its own, four blocks ahead: 48 KB in flight a CTA and 147 KB an SM
// without a register held for it, and no barrier between warps. Loads into
// registers kept 41 KB in flight and moved 2.9 TB/s, or 4.5 TB/s with the next
// block prefetched; the ring moves 6.3 TB/s, 0.98 of the measured copy rate (323M
// bf16 elements in 1129, 717 and 508 us; four CTAs an SM at 64 registers instead of
// three: 553; a sustained run under the power cap takes 580). The scales of the warp's blocks are read and written once, a lane
// for each.
//
// ALIGNED: all rows start on multiples of 16 bytes. Otherwise the copies start at the
// multiples before and the lanes take single elements (a launch of its own: one
// kernel for both was 1.4 times as slow on aligned tensors).
template <int P, int G, bool ALIGNED, bool UNBIASED>
__global__ void __launch_bounds__(kThreads, sixteen(P) && sixteen(G) ? 3 : 2)
    adamw_8bit_kernel(const __grid_constant__ StateArgs args, int p_rt, int g_rt, const __grid_constant__ StateScalars k) {
  using S = Slot<P, G, ALIGNED>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kWarps][kSlots];
  __shared__ volatile int abort_flag;
  const int p_dt = P >= 0 ? P : p_rt;
  const int g_dt = G >= 0 ? G : g_rt;
  const int t = owner_of(args, blockIdx.x);
  const int64_t start = static_cast<int64_t>(blockIdx.x - args.block_start[t]) * args.chunk;
  const int count = static_cast<int>(min(args.numel[t] - start, static_cast<int64_t>(args.chunk)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(&full[warp][i], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  // This warp's blocks of the chunk: [first, first + whole) complete ones, and
  // perhaps one more that is not.
  const int share = args.chunk / (kWarps * kBlockElems);
  const int first = warp * share;
  const int mine = min(max(count - first * kBlockElems, 0), share * kBlockElems);
  const int whole = mine / kBlockElems;
  if (whole > 0) {
    const Step s(args, k, t);
    const int64_t at0 = start + static_cast<int64_t>(first) * kBlockElems;
    uint8_t* p = static_cast<uint8_t*>(args.p[t]) + at0 * (p_dt == kF32 ? 4 : 2);
    const uint8_t* g = static_cast<const uint8_t*>(args.g[t]) + at0 * (g_dt == kF32 ? 4 : 2);
    uint8_t* m = static_cast<uint8_t*>(args.m[t]) + at0;
    uint8_t* v = static_cast<uint8_t*>(args.v[t]) + at0;
    const uint32_t first_block = static_cast<uint32_t>(at0 / kBlockElems);
    float* m_scale = args.m_scale[t] + at0 / kBlockElems;
    float* v_scale = args.v_scale[t] + at0 / kBlockElems;
    const uint32_t p_bytes = kBlockElems * (p_dt == kF32 ? 4 : 2), g_bytes = kBlockElems * (g_dt == kF32 ? 4 : 2);
    // Bytes of each behind a multiple of 16, the same for all blocks. A copy starts at
    // that multiple and takes 16 bytes more: every 16 that it reads hold a byte of the block.
    const uint32_t p_off = ALIGNED ? 0u : reinterpret_cast<uintptr_t>(p) & 15u;
    const uint32_t g_off = ALIGNED ? 0u : reinterpret_cast<uintptr_t>(g) & 15u;
    const uint32_t m_off = ALIGNED ? 0u : reinterpret_cast<uintptr_t>(m) & 15u;
    const uint32_t v_off = ALIGNED ? 0u : reinterpret_cast<uintptr_t>(v) & 15u;
    uint8_t* ring = smem + static_cast<uint32_t>(warp * kSlots) * S::kBytes;
    // g, m, v and the next slot behind p.
    constexpr uint32_t at_g = S::kP + S::kSpare, at_m = at_g + S::kG + S::kSpare;
    constexpr uint32_t at_v = at_m + kBlockElems + S::kSpare;
    auto fetch = [&](int i, int st) {
      uint8_t* slot = ring + static_cast<uint32_t>(st) * S::kBytes;
      uint64_t* bar = &full[warp][st];
      const uint32_t pn = p_bytes + (p_off ? 16u : 0u), gn = g_bytes + (g_off ? 16u : 0u);
      const uint32_t mn = kBlockElems + (m_off ? 16u : 0u), vn = kBlockElems + (v_off ? 16u : 0u);
      mbar_arrive_expect_tx(bar, pn + gn + mn + vn);
      bulk_load(slot, p - p_off + static_cast<uint32_t>(i) * p_bytes, pn, bar);
      bulk_load(slot + at_g, g - g_off + static_cast<uint32_t>(i) * g_bytes, gn, bar);
      bulk_load(slot + at_m, m - m_off + i * kBlockElems, mn, bar);
      bulk_load(slot + at_v, v - v_off + i * kBlockElems, vn, bar);
    };
    if (lane == 0)
      for (int i = 0; i < kSlots && i < whole; ++i) fetch(i, i);
    float my_ms = 0.0f, my_vs = 0.0f;  // of block `lane` of the warp's
    if (lane < whole) {
      my_ms = m_scale[lane];
      my_vs = v_scale[lane];
    }
    uint32_t phase = 0;
    int st = 0;
    bool ok = true;
    for (int i = 0; i < whole; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][st], phase, &abort_flag, &g_states_status,
                                                     kStatusProducerTimeout));
      if (!ok) break;
      const uint8_t* slot = ring + static_cast<uint32_t>(st) * S::kBytes;
      float pf[8], gf[8];
      uint2 mc, vc;
      if (ALIGNED) {  // lane L: elements 8 L .. 8 L + 7
        Eight<P> pe;
        Eight<G> ge;
        pe.load(slot, 8 * lane, p_dt);
        ge.load(slot + at_g, 8 * lane, g_dt);
        mc = reinterpret_cast<const uint2*>(slot + at_m)[lane];
        vc = reinterpret_cast<const uint2*>(slot + at_v)[lane];
        pe.get(p_dt, pf);
        ge.get(g_dt, gf);
      } else {  // lane L: elements L, L + 32, ..
        gather8(slot + p_off, lane, kBlockElems, p_dt, pf);
        gather8(slot + at_g + g_off, lane, kBlockElems, g_dt, gf);
        mc = gather_codes(slot + at_m + m_off, lane, kBlockElems);
        vc = gather_codes(slot + at_v + v_off, lane, kBlockElems);
      }
      __syncwarp();  // every lane has read the slot: it is filled again
      if (lane == 0 && i + kSlots < whole) fetch(i + kSlots, st);
      float ms = __shfl_sync(0xffffffffu, my_ms, i), vs = __shfl_sync(0xffffffffu, my_vs, i);
      step_eight<UNBIASED>(gf, pf, mc, vc, ms, vs, k, s, first_block + static_cast<uint32_t>(i));
      uint8_t* to = p + static_cast<uint32_t>(i) * p_bytes;
      if (ALIGNED) {
        store8(to, 8 * lane, p_dt, pf);
        reinterpret_cast<uint2*>(m + i * kBlockElems)[lane] = mc;
        reinterpret_cast<uint2*>(v + i * kBlockElems)[lane] = vc;
      } else {
        scatter8(to, lane, kBlockElems, p_dt, pf);
        scatter_codes(m + i * kBlockElems, lane, kBlockElems, mc);
        scatter_codes(v + i * kBlockElems, lane, kBlockElems, vc);
      }
      if (lane == i) {
        my_ms = ms;
        my_vs = vs;
      }
      if (++st == kSlots) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (!ok) {
      settle_for_ns(2000000ull);  // copies in flight land before the CTA's memory is released
      return;
    }
    if (lane < whole) {
      m_scale[lane] = my_ms;
      v_scale[lane] = my_vs;
    }
  }
  for (int i = whole * kBlockElems; i < mine; i += kBlockElems)
    step_ragged<UNBIASED>(args, t, start + static_cast<int64_t>(first) * kBlockElems + i, min(kBlockElems, mine - i), p_dt, g_dt, k);
}

template <int P, int G>
__global__ void __launch_bounds__(kThreads) adamw_32bit_kernel(const __grid_constant__ StateArgs args, int p_rt,
                                                               int g_rt, const StateScalars k) {
  const int p_dt = P >= 0 ? P : p_rt;
  const int g_dt = G >= 0 ? G : g_rt;
  const int t = owner_of(args, blockIdx.x);
  const int64_t n = args.numel[t];
  const int64_t start = static_cast<int64_t>(blockIdx.x - args.block_start[t]) * args.chunk;
  const int64_t end = min(n, start + args.chunk);
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
      Eight<P> pe;
      Eight<G> ge;
      Eight<kF32> me, ve;
      ge.load(g, i, g_dt);
      pe.load(p, i, p_dt);
      me.load(m, i, kF32);
      ve.load(v, i, kF32);
      ge.get(g_dt, gf);
      pe.get(p_dt, pf);
      me.get(kF32, mf);
      ve.get(kF32, vf);
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

std::mutex g_mutex;
bool g_ready[64][32] = {};

template <int P, int G, bool ALIGNED, bool UNBIASED>
int launch_8bit(int blocks, cudaStream_t st, const StateArgs& a, int p_dt, int g_dt, const StateScalars& k, int slot) {
  constexpr size_t smem = Slot<P, G, ALIGNED>::kSmem;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(GNS_ERR_DEVICE, "device index out of range");
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!g_ready[dev][slot]) {
      e = cudaFuncSetAttribute(adamw_8bit_kernel<P, G, ALIGNED, UNBIASED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(smem));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(smem)");
      g_ready[dev][slot] = true;
    }
  }
  adamw_8bit_kernel<P, G, ALIGNED, UNBIASED><<<blocks, kThreads, smem, st>>>(a, p_dt, g_dt, k);
  return GNS_OK;
}

template <int P, int G>
int launch(int bits, bool unbiased, bool aligned, int blocks, cudaStream_t st, const StateArgs& a, int p_dt, int g_dt,
           const StateScalars& k, int slot) {
  int rc = GNS_OK;
  if (bits == 32)
    adamw_32bit_kernel<P, G><<<blocks, kThreads, 0, st>>>(a, p_dt, g_dt, k);
  else if (aligned)
    rc = unbiased ? launch_8bit<P, G, true, true>(blocks, st, a, p_dt, g_dt, k, 4 * slot)
                  : launch_8bit<P, G, true, false>(blocks, st, a, p_dt, g_dt, k, 4 * slot + 1);
  else
    rc = unbiased ? launch_8bit<P, G, false, true>(blocks, st, a, p_dt, g_dt, k, 4 * slot + 2)
                  : launch_8bit<P, G, false, false>(blocks, st, a, p_dt, g_dt, k, 4 * slot + 3);
  if (rc != GNS_OK) return rc;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "adamw states kernel");
}

}  // namespace

int states_status(int* status, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_states_status, sizeof(int));
  if (e == cudaSuccess && clear && *status != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_states_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "adamw states status");
}

}  // namespace gns

using namespace gns;

namespace {

// steps: nullptr, or each tensor's step number, which rounds 8-bit states without bias.
int states_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs,
                void* const* exp_avg_sqs, float* const* exp_avg_scales, float* const* exp_avg_sq_scales,
                const int64_t* numel, int p_dtype, int g_dtype, int state_bits, const uint32_t* steps,
                const float* lr_bc1, const float* inv_bc2, float beta1, float one_minus_beta1, float beta2,
                float one_minus_beta2, float epsilon, float decay, const float* grad_scale, gns_stream_t stream) {
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
  const bool unbiased = steps != nullptr;
  int rc = check_device();
  if (rc != GNS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const StateScalars k{beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon, decay, grad_scale};
  // Long chunks keep a warp's ring going; short ones give every SM work. 8-bit states:
  // up to 8 chunks an SM of the shortest kind, then longer ones (7.8M bf16 elements 34.7
  // us with up to 32, 25.0 with 8 or 12; 3M: 17.2, 14.2; 16M: 40.3, 33.6). 32-bit states
  // have no ring: up to 32 (16M: 61.8 us with 8, 56.6 with 32).
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += numel[i];
  int chunk = kChunkMin;
  while (chunk < kChunkMax && total / chunk > (state_bits == 8 ? 8 : 32) * static_cast<int64_t>(device_sm_count())) chunk *= 2;
  // 8-bit states: the tensors whose rows all start on 16 bytes, then the others.
  auto is_aligned = [&](int i) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(params[i]) | reinterpret_cast<uintptr_t>(grads[i]) |
                          reinterpret_cast<uintptr_t>(exp_avgs[i]) | reinterpret_cast<uintptr_t>(exp_avg_sqs[i]);
    return state_bits == 32 || all % 16 == 0;
  };
  for (bool aligned : {true, false}) {
    int i = 0;
    while (i < count) {
      StateArgs a;
      a.count = 0;
      a.chunk = chunk;
      int64_t blocks = 0;
      for (; i < count && a.count < kTensors; ++i) {
        if (numel[i] == 0 || is_aligned(i) != aligned) continue;
        const int64_t nb = (numel[i] + chunk - 1) / chunk;
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
        a.key[j] = unbiased ? scramble(scramble(steps[i]) + static_cast<uint32_t>(i)) : 0u;
        a.block_start[j] = static_cast<int>(blocks);
        blocks += nb;
      }
      if (a.count == 0) break;
      a.block_start[a.count] = static_cast<int>(blocks);
      const int grid = static_cast<int>(blocks);
      if (p_dtype == kBF16 && g_dtype == kBF16)
        rc = launch<kBF16, kBF16>(state_bits, unbiased, aligned, grid, st, a, p_dtype, g_dtype, k, 0);
      else if (p_dtype == kF32 && g_dtype == kF32)
        rc = launch<kF32, kF32>(state_bits, unbiased, aligned, grid, st, a, p_dtype, g_dtype, k, 1);
      else if (p_dtype == kF16 && g_dtype == kF16)
        rc = launch<kF16, kF16>(state_bits, unbiased, aligned, grid, st, a, p_dtype, g_dtype, k, 2);
      else if (p_dtype == kBF16 && g_dtype == kF32)
        rc = launch<kBF16, kF32>(state_bits, unbiased, aligned, grid, st, a, p_dtype, g_dtype, k, 3);
      else
        rc = launch<-1, -1>(state_bits, unbiased, aligned, grid, st, a, p_dtype, g_dtype, k, 4);
      if (rc != GNS_OK) return rc;
    }
  }
  return GNS_OK;
}

}  // namespace

extern "C" int gns_adamw_states_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs,
                                     void* const* exp_avg_sqs, float* const* exp_avg_scales,
                                     float* const* exp_avg_sq_scales, const int64_t* numel, int p_dtype, int g_dtype,
                                     int state_bits, const float* lr_bc1, const float* inv_bc2, float beta1,
                                     float one_minus_beta1, float beta2, float one_minus_beta2, float epsilon,
                                     float decay, const float* grad_scale, gns_stream_t stream) {
  return states_step(count, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, numel, p_dtype,
                     g_dtype, state_bits, nullptr, lr_bc1, inv_bc2, beta1, one_minus_beta1, beta2, one_minus_beta2,
                     epsilon, decay, grad_scale, stream);
}

extern "C" int gns_adamw_states_step_unbiased(int count, void* const* params, const void* const* grads,
                                              void* const* exp_avgs, void* const* exp_avg_sqs,
                                              float* const* exp_avg_scales, float* const* exp_avg_sq_scales,
                                              const int64_t* numel, int p_dtype, int g_dtype, const uint32_t* steps,
                                              const float* lr_bc1, const float* inv_bc2, float beta1,
                                              float one_minus_beta1, float beta2, float one_minus_beta2, float epsilon,
                                              float decay, const float* grad_scale, gns_stream_t stream) {
  if (count > 0 && steps == nullptr) {
    clear_error();
    return fail(GNS_ERR_ARGUMENT, "unbiased rounding needs the tensors' step numbers");
  }
  return states_step(count, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, numel, p_dtype,
                     g_dtype, 8, steps, lr_bc1, inv_bc2, beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon, decay,
                     grad_scale, stream);
}
