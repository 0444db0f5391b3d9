// A matrix in 8 bits with a scale for each block: 1 x 128 (activations and gradients, as the
// left factor of gns_gemm_8bit) or 128 x 128 (weights, as the right one).
//
// Read once, written once: bound by HBM (3 bytes an element for 16-bit inputs) and, near it, by
// the instructions beside the conversions. So eight lanes hold a row's block of 128, twice eight
// elements each: three shuffles and one division serve 16 elements. 16384 x 4096 bf16: 33 us
// (6.1 TB/s; with sixteen lanes 43, a block at a time with its place found by divisions 81);
// 14336 x 4096 in blocks of 128 x 128 29 us (6.1 TB/s). Rows that start anywhere are loaded element
// by element: 57 us for 16384 x 4095 bf16, bound by those loads.
#include <type_traits>

#include "../../include/gns_b200.h"
#include "blocks_8bit.cuh"
#include "gns_host.h"

namespace gns {
namespace {

constexpr int kThreads = 256;
constexpr int kHalves = kThreads / 16;
constexpr int kRowLanes = 8;                    // of a block in the row kernel
constexpr int kRowGroups = kThreads / kRowLanes;
constexpr int kRowItems = 2;                    // blocks of such a group, loaded together
constexpr int kRowPieces = 16 / kRowLanes;      // of eight elements, in each

struct QuantArgs {
  const void* x;
  int64_t stride;
  int64_t rows;
  int cols, blocks;
  uint32_t tile_cols;  // row kernel: tiles of 2^shift blocks side by side
  int shift;
  CodesOut out;
};

// Eight elements as loaded.
template <int XD>
struct Eight {
  static constexpr int kWords = XD == kF32 ? 8 : 4;
  uint32_t w[kWords];

  // From column c on, zeros past the end.
  template <bool VEC>
  __device__ __forceinline__ void load(const QuantArgs& a, int64_t row, int c) {
    constexpr int es = XD == kF32 ? 4 : 2;
    const uint8_t* p = static_cast<const uint8_t*>(a.x) + (row * a.stride + c) * es;
    if (VEC && c + 8 <= a.cols) {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + q);
        w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (XD == kF32) {
          w[i % kWords] = c + i < a.cols ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
        } else {
          const uint32_t one = c + i < a.cols ? reinterpret_cast<const uint16_t*>(p)[i] : 0u;
          w[i / 2 % kWords] = i & 1 ? w[i / 2 % kWords] | one << 16 : one;
        }
      }
    }
  }

  __device__ __forceinline__ float get(int i) const {
    if (XD == kF32) return __uint_as_float(w[i % kWords]);
    const uint32_t two = w[i / 2 % kWords];
    if (XD == kBF16) return __uint_as_float((i & 1) ? (two & 0xffff0000u) : (two << 16));
    return __half2float(__ushort_as_half(static_cast<uint16_t>((i & 1) ? (two >> 16) : two)));
  }

  // The largest magnitude that is not a NaN.
  __device__ __forceinline__ float largest() const {
    if (XD != kF32) {
      using Two = typename std::conditional<XD == kBF16, __nv_bfloat162, __half2>::type;
      uint32_t m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) m[q] = w[q % kWords] & 0x7fff7fffu;
      const Two* h = reinterpret_cast<const Two*>(m);
      const Two top = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(fmaxf(static_cast<float>(top.x), static_cast<float>(top.y)), 0.0f);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(get(i)));
    return top;
  }

  __device__ __forceinline__ void store(const CodesOut& out, int64_t row, int c, float factor) const {
    if (c >= out.width) return;
    uint2 codes;
    codes.x = e4m3_four(get(0) * factor, get(1) * factor, get(2) * factor, get(3) * factor);
    codes.y = e4m3_four(get(4) * factor, get(5) * factor, get(6) * factor, get(7) * factor);
    *reinterpret_cast<uint2*>(out.codes + row * out.ld + c) = codes;
  }
};

// 64 blocks a CTA: as many of a row as fit 1024 columns, and the rows below them, so that rows
// are read in stretches of 2 KB and the scales of a block column written in sectors.
template <int XD, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantArgs a) {
  const int lane8 = threadIdx.x & (kRowLanes - 1);
  const uint32_t down = blockIdx.x / a.tile_cols, across = blockIdx.x - down * a.tile_cols;
  const int64_t row0 = static_cast<int64_t>(down) * ((kRowGroups * kRowItems) >> a.shift);
  const int block0 = static_cast<int>(across) << a.shift;
  Eight<XD> v[kRowItems][kRowPieces];
#pragma unroll
  for (int q = 0; q < kRowItems; ++q) {
    const int item = q * kRowGroups + static_cast<int>(threadIdx.x / kRowLanes);
    const int64_t row = row0 + (item >> a.shift);
    const int block = block0 + (item & ((1 << a.shift) - 1));
    if (row >= a.rows || block >= a.blocks) continue;
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) v[q][i].template load<VEC>(a, row, block * kScaleBlock + (lane8 + kRowLanes * i) * 8);
  }
#pragma unroll
  for (int q = 0; q < kRowItems; ++q) {
    const int item = q * kRowGroups + static_cast<int>(threadIdx.x / kRowLanes);
    const int64_t row = row0 + (item >> a.shift);
    const int block = block0 + (item & ((1 << a.shift) - 1));
    const bool live = row < a.rows && block < a.blocks;
    float top = 0.0f;
    if (live) {
#pragma unroll
      for (int i = 0; i < kRowPieces; ++i) top = fmaxf(top, v[q][i].largest());
    }
#pragma unroll
    for (int o = kRowLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    const BlockScale s(top);
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) v[q][i].store(a.out, row, block * kScaleBlock + (lane8 + kRowLanes * i) * 8, s.factor);
    if (lane8 == 0) a.out.scales[row * a.out.srow + block * a.out.scol] = s.scale;
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
  Eight<XD> v[kRows];
  float top = 0.0f;
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const int64_t row = row0 + q * kHalves + threadIdx.x / 16;
    if (row < a.rows) v[q].template load<VEC>(a, row, c);
  }
#pragma unroll
  for (int q = 0; q < kRows; ++q)
    if (row0 + q * kHalves + threadIdx.x / 16 < a.rows) top = fmaxf(top, v[q].largest());
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
    if (row < a.rows) v[q].store(a.out, row, c, s.factor);
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
  const int blocks = static_cast<int>((cols + kScaleBlock - 1) / kScaleBlock);
  int shift = 0;
  while (shift < 3 && (1 << shift) < blocks) ++shift;
  const int64_t tile_cols = (blocks + (1 << shift) - 1) >> shift, tile_rows = (kRowGroups * kRowItems) >> shift;
  const QuantArgs a{x, x_rstride, rows, static_cast<int>(cols), blocks, static_cast<uint32_t>(tile_cols), shift,
                    {static_cast<uint8_t*>(codes), codes_rstride, static_cast<int>(round_up(cols, 16)), scales,
                     scale_rstride, scale_cstride}};
  const int es = dtype_size(x_dtype);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (x_rstride * es) % 16 == 0;
  const bool square = block_rows != 1;
  const int64_t ctas = square ? (rows + kScaleBlock - 1) / kScaleBlock * blocks : (rows + tile_rows - 1) / tile_rows * tile_cols;
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
