// Staging of 32 x 32 result blocks in shared memory between the accumulator's
// layout (a lane holds one row) and coalesced global rows; used by the epilogues
// of the tcgen05 kernels.
#pragma once

#include "gns_common.cuh"

namespace gns {

// Byte offset of (row, byte) inside a swizzled 32-row staging block. The
// pattern equals the TMA's SWIZZLE_64B (16-bit rows) / SWIZZLE_128B (fp32 rows).
template <bool OUT_F32>
__device__ __forceinline__ uint32_t stage_off(uint32_t row, uint32_t byte) {
  if (OUT_F32) return row * 128u + (byte ^ ((row & 7u) << 4));
  return row * 64u + (byte ^ (((row >> 1) & 3u) << 4));
}

// Two values rounded to 16 bits (round to nearest even), the first in the low half.
__device__ __forceinline__ uint32_t pack_pair(float a, float b, int bf16) {
  if (bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float half_bits_to_float(uint16_t bits, int bf16) {
  if (bf16) return __bfloat162float(__ushort_as_bfloat16(bits));
  return __half2float(__ushort_as_half(bits));
}

__device__ __forceinline__ uint16_t float_to_half_bits(float v, int bf16) {
  if (bf16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}

// One lane's 32 results of a chunk, already rounded to the output type: fp32
// bit patterns, or 16-bit values packed in pairs (element 2i in the low half).
template <bool OUT_F32>
struct XRow {
  uint32_t w[OUT_F32 ? 32 : 16];
};

// Writes row `row` of a swizzled staging block.
template <bool OUT_F32>
__device__ __forceinline__ void stage_write_row(uint8_t* buf, uint32_t row, const XRow<OUT_F32>& x) {
  constexpr int kVec = OUT_F32 ? 8 : 4;
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    *reinterpret_cast<uint4*>(buf + stage_off<OUT_F32>(row, 16u * k)) =
        make_uint4(x.w[4 * k], x.w[4 * k + 1], x.w[4 * k + 2], x.w[4 * k + 3]);
}

// Writes column `col` (= the lane) of a swizzled staging block: element q goes
// to (q, col). 16-bit values go as 32-bit words of two adjacent columns built
// from lane pairs: per pair of rows (q, q + 1) the even lane stores row q and
// the odd lane row q + 1, each with one value received from its partner.
template <bool OUT_F32>
__device__ __forceinline__ void stage_write_col(uint8_t* buf, uint32_t col, const XRow<OUT_F32>& x) {
  if (OUT_F32) {
#pragma unroll
    for (int q = 0; q < 32; ++q) *reinterpret_cast<uint32_t*>(buf + stage_off<true>(q, 4u * col)) = x.w[q];
  } else {
    const bool odd = (col & 1u) != 0;
    const uint32_t even_col = col & ~1u;
#pragma unroll
    for (int q = 0; q < 32; q += 2) {
      const uint32_t lo = x.w[q >> 1] & 0xffffu, hi = x.w[q >> 1] >> 16;  // elements q, q + 1
      const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
      const uint32_t row = odd ? static_cast<uint32_t>(q + 1) : static_cast<uint32_t>(q);
      const uint32_t word = odd ? (got | (hi << 16)) : (lo | (got << 16));
      *reinterpret_cast<uint32_t*>(buf + stage_off<false>(row, 2u * even_col)) = word;
    }
  }
}

template <bool OUT_F32>
__device__ __forceinline__ float stage_get(const uint8_t* buf, uint32_t row, uint32_t col, int bf16) {
  if (OUT_F32) return *reinterpret_cast<const float*>(buf + stage_off<true>(row, 4u * col));
  return half_bits_to_float(*reinterpret_cast<const uint16_t*>(buf + stage_off<false>(row, 2u * col)), bf16);
}

template <bool OUT_F32>
__device__ __forceinline__ void global_put(void* base, int64_t idx, float v, int bf16) {
  if (OUT_F32)
    static_cast<float*>(base)[idx] = v;
  else
    static_cast<uint16_t*>(base)[idx] = float_to_half_bits(v, bf16);
}

template <bool OUT_F32>
__device__ __forceinline__ float global_get(const void* base, int64_t idx, int bf16) {
  if (OUT_F32) return static_cast<const float*>(base)[idx];
  return half_bits_to_float(static_cast<const uint16_t*>(base)[idx], bf16);
}

}  // namespace gns
