// Values in 8 bits with a scale for a block of 128, as gns_gemm_8bit reads them:
//
//   top = max(largest magnitude, 448 * 2^-126),  scale = top / 448,
//   code = e4m3(x * (448 / top)), to nearest even, at most 448 in magnitude
//
// The lower bound keeps scales normal numbers (a block of zeros has codes of zero and a
// scale of 2^-126). A NaN keeps a code of NaN and does not enter the scale; an infinity
// makes its block's scale infinite, so its products are NaN.
#pragma once

#include "gns_common.cuh"

namespace gns {

constexpr int kScaleBlock = 128;
constexpr float kE4m3Top = 448.0f;
constexpr float kLeastTop = 448.0f * 1.17549435e-38f;  // 448 * 2^-126

// Two values as e4m3 codes, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  uint16_t two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(two) : "f"(a), "f"(b));
  return two;
}

__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) {
  return e4m3_pair(a, b) | (e4m3_pair(c, d) << 16);
}

// A block's scale, and the factor that its values are multiplied by, from its largest magnitude.
struct BlockScale {
  float scale, factor;
  __device__ __forceinline__ explicit BlockScale(float largest) {
    const float top = fmaxf(largest, kLeastTop);
    // top / 448 correctly rounded (Markstein's correction of a product with the reciprocal); the
    // remainder of an infinity is a NaN.
    constexpr float kInverse = 1.0f / kE4m3Top;
    const float q = top * kInverse;
    scale = top == INFINITY ? top : fmaf(fmaf(-q, kE4m3Top, top), kInverse, q);
    factor = __fdiv_rn(kE4m3Top, top);
  }
};

// Where codes and scales go: row r, column c at codes[r * ld + c]. Rows start on 16 bytes and
// are written up to `width`, the row length rounded up to 16, zeros behind the last column.
// The scale of row r (or block row) and block b: scales[r * srow + b * scol].
struct CodesOut {
  uint8_t* codes;
  int64_t ld;
  int width;
  float* scales;
  int64_t srow, scol;
};

}  // namespace gns
