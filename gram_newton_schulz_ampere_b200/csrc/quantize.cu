// A matrix in 8 bits with a scale for each block: 1 x 128 (activations and gradients, as the
// left factor of gns_gemm_8bit) or 128 x 128 (weights, as the right one).
//
// Sixteen lanes hold a row's block of 128, eight elements each, so that a block's largest
// magnitude takes four shuffles and the codes of a lane are one store of 8 bytes. Read once,
// written once: bound by HBM (3 bytes an element for 16-bit inputs).
#include "../../include/gns_b200.h"
#include "blocks_8bit.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kThreads = 256;
constexpr int kHalves = kThreads / 16;
constexpr int kRowItems = 4;  // blocks of a row kernel's half-warp, loaded together

struct QuantArgs {
  const void* x;
  int64_t stride;
  int64_t rows;
  int cols, blocks;
  CodesOut out;
};

// Eight elements from column c on, zeros past the end.
template <int XD, bool VEC>
__device__ __forceinline__ void load8(const QuantArgs& a, int64_t row, int c, float (&v)[8]) {
  constexpr int es = XD == kF32 ? 4 : 2;
  const uint8_t* p = static_cast<const uint8_t*>(a.x) + (row * a.stride + c) * es;
  if (VEC && c + 8 <= a.cols) {
    uint32_t w[XD == kF32 ? 8 : 4];
#pragma unroll
    for (int q = 0; q < (XD == kF32 ? 2 : 1); ++q) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[q];
      w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (XD == kF32) {
        v[i] = __uint_as_float(w[i % (XD == kF32 ? 8 : 4)]);
      } else if (XD == kBF16) {
        v[i] = __uint_as_float((i & 1) ? (w[i / 2] & 0xffff0000u) : (w[i / 2] << 16));
      } else {
        v[i] = __half2float(__ushort_as_half(static_cast<uint16_t>((i & 1) ? (w[i / 2] >> 16) : w[i / 2])));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < a.cols ? load_as_float(p, i, XD) : 0.0f;
  }
}

__device__ __forceinline__ float largest8(const float (&v)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
  return top;
}

__device__ __forceinline__ void store8(const QuantArgs& a, int64_t row, int c, const float (&v)[8], float factor) {
  if (c >= a.out.width) return;
  uint2 codes;
  codes.x = e4m3_four(v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor);
  codes.y = e4m3_four(v[4] * factor, v[5] * factor, v[6] * factor, v[7] * factor);
  *reinterpret_cast<uint2*>(a.out.codes + row * a.out.ld + c) = codes;
}

template <int XD, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantArgs a) {
  const int lane16 = threadIdx.x & 15;
  const int64_t items = a.rows * a.blocks;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kHalves * kRowItems) + threadIdx.x / 16;
  float v[kRowItems][8];
  int64_t row[kRowItems];
  int block[kRowItems];
#pragma unroll
  for (int q = 0; q < kRowItems; ++q) {
    const int64_t item = first + q * kHalves;
    row[q] = item / a.blocks;
    block[q] = static_cast<int>(item - row[q] * a.blocks);
    if (item >= items) continue;
    load8<XD, VEC>(a, row[q], block[q] * kScaleBlock + lane16 * 8, v[q]);
  }
#pragma unroll
  for (int q = 0; q < kRowItems; ++q) {
    const bool live = first + q * kHalves < items;
    float top = live ? largest8(v[q]) : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    const BlockScale s(top);
    store8(a, row[q], block[q] * kScaleBlock + lane16 * 8, v[q], s.factor);
    if (lane16 == 0) a.out.scales[row[q] * a.out.srow + block[q] * a.out.scol] = s.scale;
  }
}

// A block of 128 x 128 a CTA.
template <int XD, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const QuantArgs a) {
  constexpr int kRows = kScaleBlock / kHalves;
  __shared__ float tops[kThreads / 32];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / static_cast<unsigned>(a.blocks)) * kScaleBlock;
  const int block = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.blocks));
  const int c = block * kScaleBlock + (threadIdx.x & 15) * 8;
  float v[kRows][8];
  float top = 0.0f;
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const int64_t row = row0 + q * kHalves + threadIdx.x / 16;
    if (row >= a.rows) continue;
    load8<XD, VEC>(a, row, c, v[q]);
  }
#pragma unroll
  for (int q = 0; q < kRows; ++q)
    if (row0 + q * kHalves + threadIdx.x / 16 < a.rows) top = fmaxf(top, largest8(v[q]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, tops[w]);
  const BlockScale s(top);
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const int64_t row = row0 + q * kHalves + threadIdx.x / 16;
    if (row < a.rows) store8(a, row, c, v[q], s.factor);
  }
  if (threadIdx.x == 0) a.out.scales[row0 / kScaleBlock * a.out.srow + block * a.out.scol] = s.scale;
}

template <int XD>
void launch(bool vec, bool square, const QuantArgs& a, unsigned grid, cudaStream_t st) {
  if (square) {
    if (vec)
      quantize_blocks_kernel<XD, true><<<grid, kThreads, 0, st>>>(a);
    else
      quantize_blocks_kernel<XD, false><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (vec)
      quantize_rows_kernel<XD, true><<<grid, kThreads, 0, st>>>(a);
    else
      quantize_rows_kernel<XD, false><<<grid, kThreads, 0, st>>>(a);
  }
}

}  // namespace
}  // namespace gns

using namespace gns;

extern "C" int gns_quantize_8bit(int x_dtype, int block_rows, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                                 void* codes, int64_t codes_rstride, float* scales, int64_t scale_rstride,
                                 int64_t scale_cstride, gns_stream_t stream) {
  clear_error();
  if (x_dtype < 0 || x_dtype > 2) return fail(GNS_ERR_ARGUMENT, "bad dtype");
  if (block_rows != 1 && block_rows != kScaleBlock) return fail(GNS_ERR_ARGUMENT, "a block has 1 or 128 rows");
  if (rows < 0 || cols < 0) return fail(GNS_ERR_ARGUMENT, "negative dimension");
  if (rows == 0 || cols == 0) return GNS_OK;
  if (cols > (1 << 30) || rows > (1ll << 40)) return fail(GNS_ERR_UNSUPPORTED, "dimension beyond kernel limits");
  if (x == nullptr || codes == nullptr || scales == nullptr) return fail(GNS_ERR_ARGUMENT, "null tensor");
  if (rows > 1 && x_rstride < cols && x_rstride != 0) return fail(GNS_ERR_LAYOUT, "row stride below the row length");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || codes_rstride % 16 != 0 || codes_rstride < cols)
    return fail(GNS_ERR_LAYOUT, "rows of codes must start on 16 bytes and hold a row");
  const int rc = check_device();
  if (rc != GNS_OK) return rc;
  const QuantArgs a{x, x_rstride, rows, static_cast<int>(cols), static_cast<int>((cols + kScaleBlock - 1) / kScaleBlock),
              {static_cast<uint8_t*>(codes), codes_rstride, static_cast<int>(round_up(cols, 16)), scales, scale_rstride,
               scale_cstride}};
  const int es = dtype_size(x_dtype);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (x_rstride * es) % 16 == 0;
  const bool square = block_rows != 1;
  const int64_t ctas = square ? (rows + kScaleBlock - 1) / kScaleBlock * a.blocks
                              : (rows * a.blocks + kHalves * kRowItems - 1) / (kHalves * kRowItems);
  if (ctas > (1ll << 31) - 1) return fail(GNS_ERR_UNSUPPORTED, "matrix beyond kernel limits");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(ctas);
  if (x_dtype == kF32)
    launch<kF32>(vec, square, a, grid, st);
  else if (x_dtype == kBF16)
    launch<kBF16>(vec, square, a, grid, st);
  else
    launch<kF16>(vec, square, a, grid, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GNS_OK : cuda_fail(e, "8-bit quantisation kernel");
}
