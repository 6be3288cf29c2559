// Quantisation to 8 bits in blocks: of each block of 1 x 128 or 128 x 128 values the scale, max(largest magnitude / 448, 2^-126)
// (57344 for e5m2), and the values x / scale as e4m3 or e5m2; as the matrix lies, or transposed (with blocks along what were the
// columns' rows), as the products of a backward pass take their operands.
//
// Bound by HBM: every value is read once, into registers, and leaves as one byte. Blocks of one row: 16 threads a block, no shared
// memory. All else: a CTA takes 128 x 128 values, a thread 8 x 8 of them, so that it holds eight neighbouring bytes in either
// direction; transposed they change hands through shared memory.
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/kcg_b200.h"
#include "fp8_common.cuh"
#include "kernels/ptx_sm100.cuh"

namespace {

using namespace kcg;
using namespace kcg8;

struct QuantArgs {
  const void* x;
  uint8_t* q;
  float* scales;  // contiguous: a row of `blocks` scales for each block row of q
  long long ldx, ldq, rows;
  int cols, blocks;
};

// Eight values of a row from column c on; those past the row's end as zeros.
template <typename T, bool kVec>
__device__ __forceinline__ void load_piece(const T* row, int c, int cols, float (&v)[8]) {
  if (kVec && c + 8 <= cols) {
    load8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(row[c + j]) : 0.f;
  }
}

// Blocks of 1 x 128, as the matrix lies: 16 threads a block.
template <typename T, bool kVec, bool kE5M2>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const long long total = a.rows * a.blocks;
  const int part = threadIdx.x & 15;
  for (long long b = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4); b - (threadIdx.x >> 4 & 1) < total;
       b += static_cast<long long>(gridDim.x) * 16) {  // (both halves of a warp stay for the exchange)
    const bool in = b < total;
    const long long row = in ? b / a.blocks : 0;
    const int block = in ? static_cast<int>(b - row * a.blocks) : 0, c = block * 128 + part * 8;
    float v[8];
    load_piece<T, kVec>(static_cast<const T*>(a.x) + row * a.ldx, c, in ? a.cols : 0, v);
    uint32_t top = abs_max(v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = block_scale<kE5M2>(top);
    if (in && c < a.cols) {  // (rows of q are padded to whole pieces)
      *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = quantize8<kE5M2>(v, 1.f / scale);
      if (part == 0) a.scales[b] = scale;
    }
  }
}

// A CTA quantises 128 x 128 values of x; thread (g, l) rows 8 g .. 8 g + 7, columns 8 l .. 8 l + 7 of them.
template <typename T, bool kVec, bool kE5M2, bool kSquare, bool kTransposed>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantArgs a) {
  __shared__ uint32_t tops[kSquare ? 8 : 8 * 128];
  __shared__ uint2 bytes[kTransposed ? 128 * 16 : 1];  // [column of x][8 rows of x], the latter XORed with l
  griddep_launch_dependents();
  griddep_wait();
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_c = (a.cols + 127) / 128;
  const long long tile_r = blockIdx.x / tiles_c;
  const int tile_c = static_cast<int>(blockIdx.x - tile_r * tiles_c);
  const long long r0 = tile_r * 128 + g * 8;
  const int c0 = tile_c * 128 + l * 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load_piece<T, kVec>(static_cast<const T*>(a.x) + (r0 + i < a.rows ? r0 + i : 0) * a.ldx, c0, r0 + i < a.rows ? a.cols : 0, v[i]);
  float inv[8];  // of each column (kSquare: all alike)
  if constexpr (kSquare) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_max(v[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
    const float scale = block_scale<kE5M2>(top);
    if (threadIdx.x == 0) a.scales[kTransposed ? static_cast<long long>(tile_c) * a.blocks + tile_r : tile_r * a.blocks + tile_c] = scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = 1.f / scale;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
      if (lane < 16) tops[warp * 128 + l * 8 + j] = top;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, tops[i * 128 + l * 8 + j]);
      const float scale = block_scale<kE5M2>(top);
      inv[j] = 1.f / scale;
      if (g == 0 && c0 + j < a.cols) a.scales[static_cast<long long>(c0 + j) * a.blocks + tile_r] = scale;
    }
  }
  if constexpr (!kTransposed) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r0 + i < a.rows && c0 < a.cols) *reinterpret_cast<uint2*>(a.q + (r0 + i) * a.ldq + c0) = quantize8<kE5M2>(v[i], inv[0]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float column[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
      bytes[(l * 8 + j) * 16 + (g ^ l)] = quantize8<kE5M2>(column, inv[j]);
    }
    __syncthreads();
    // a row of q: 128 bytes from 8 threads
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i * 32 + (threadIdx.x >> 3), u = (threadIdx.x & 7) * 2;
      const long long r = tile_r * 128 + u * 8;
      const uint2 lo = bytes[c * 16 + (u ^ (c >> 3))], hi = bytes[c * 16 + ((u + 1) ^ (c >> 3))];
      if (tile_c * 128 + c < a.cols && r < a.rows)  // (rows of q are padded to whole 16-byte pieces)
        *reinterpret_cast<uint4*>(a.q + static_cast<long long>(tile_c * 128 + c) * a.ldq + r) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
}

template <typename T, bool kVec, bool kE5M2>
int launch_quantize(const QuantArgs& a, int block_rows, bool transposed, int sms, cudaStream_t st) {
  Launch l(st);
  if (block_rows == 1 && !transposed) {
    const long long ctas = (a.rows * a.blocks + 15) / 16, most = static_cast<long long>(sms) * 64;
    l.shape(static_cast<unsigned>(ctas < most ? ctas : most), 256);
    return l(quantize_rows_kernel<T, kVec, kE5M2>, "quantize launch", a);
  }
  const long long tiles = ((a.rows + 127) / 128) * ((a.cols + 127) / 128);
  if (tiles > 0x7fffffffLL) return fail(KCG_E_TOO_LARGE, "too many blocks for one launch");
  l.shape(static_cast<unsigned>(tiles), 256);
  if (block_rows == 1) return l(quantize_tile_kernel<T, kVec, kE5M2, false, true>, "quantize launch", a);
  if (transposed) return l(quantize_tile_kernel<T, kVec, kE5M2, true, true>, "quantize launch", a);
  return l(quantize_tile_kernel<T, kVec, kE5M2, true, false>, "quantize launch", a);
}

template <typename T>
int launch_quantize(const QuantArgs& a, int block_rows, bool transposed, bool e5m2, int sms, cudaStream_t st) {
  const bool vec = reinterpret_cast<uint64_t>(a.x) % 16 == 0 && a.ldx * static_cast<long long>(sizeof(T)) % 16 == 0;
  if (vec)
    return e5m2 ? launch_quantize<T, true, true>(a, block_rows, transposed, sms, st)
                : launch_quantize<T, true, false>(a, block_rows, transposed, sms, st);
  return e5m2 ? launch_quantize<T, false, true>(a, block_rows, transposed, sms, st)
              : launch_quantize<T, false, false>(a, block_rows, transposed, sms, st);
}

}  // namespace

extern "C" int kcg_quantize_fp8(int device, uint64_t stream, uint64_t X, int64_t ldx, uint64_t Q, int64_t ldq, uint64_t S, int64_t rows,
                                int cols, int block_rows, int transposed, int dtype, int dtype8) {
  if (!known_dtype(dtype)) return fail(KCG_E_BAD_ARG, "quantisation takes float16, bfloat16 or float32 data");
  if (dtype8 != KCG_FP8_E4M3 && dtype8 != KCG_FP8_E5M2) return fail(KCG_E_BAD_ARG, "quantisation gives e4m3 or e5m2 values");
  if (block_rows != 1 && block_rows != 128) return fail(KCG_E_BAD_ARG, "blocks have 1 or 128 rows");
  if (rows < 0 || rows > 0x7fffffffLL || cols <= 0) return fail(KCG_E_BAD_ARG, "shape out of range");
  if (rows == 0) return 0;
  if (!X || !Q || !S) return fail(KCG_E_BAD_ARG, "null matrix");
  const int64_t out_cols = transposed ? rows : cols;
  if (ldx == 0) ldx = cols;
  if (ldq == 0) ldq = out_cols;
  if (ldx < cols || ldq < out_cols) return fail(KCG_E_BAD_ARG, "leading dimension below the row length");
  if (Q % 16 || ldq % 16) return fail(KCG_E_BAD_ARG, "rows of 8-bit values must start on 16-byte boundaries");
  const int eb = dtype == KCG_DTYPE_FLOAT32 ? 4 : 2;
  if (X % eb || S % 4) return fail(KCG_E_BAD_ARG, "operands must be aligned to their values");
  int sms = 0;
  if (int e = sm_count(device, &sms)) return e;
  QuantArgs a{};
  a.x = reinterpret_cast<const void*>(X), a.q = reinterpret_cast<uint8_t*>(Q), a.scales = reinterpret_cast<float*>(S);
  a.ldx = ldx, a.ldq = ldq, a.rows = rows, a.cols = cols, a.blocks = static_cast<int>((out_cols + 127) / 128);
  DeviceGuard guard;
  const cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool e5m2 = dtype8 == KCG_FP8_E5M2, t = transposed != 0;
  if (dtype == KCG_DTYPE_FLOAT32) return launch_quantize<float>(a, block_rows, t, e5m2, sms, st);
  return dtype == KCG_DTYPE_FLOAT16 ? launch_quantize<__half>(a, block_rows, t, e5m2, sms, st)
                                    : launch_quantize<__nv_bfloat16>(a, block_rows, t, e5m2, sms, st);
}
