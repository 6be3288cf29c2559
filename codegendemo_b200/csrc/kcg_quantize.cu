// Quantisation to 8 bits in blocks: of each block of 1 x 128 or 128 x 128 values the scale, max(largest magnitude / 448, 2^-126)
// (57344 for e5m2), and the values x * (1 / scale) as e4m3 or e5m2; as the matrix lies, or transposed (with blocks along what were the
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

// Magnitudes, kept in the raw type: its bits without the sign, in whose order a NaN is the largest. Words of two 16-bit values or of
// one fp32 value; eight values are kWords of them.
template <typename T>
struct Tops {
  static constexpr int kWords = sizeof(T) == 4 ? 8 : 4;
  __device__ static __forceinline__ uint32_t word(const Raw8<T>& v, int i) { return reinterpret_cast<const uint32_t*>(&v)[i]; }
  __device__ static __forceinline__ uint32_t magnitude(uint32_t w) { return w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
      return max(a, b);
    } else {
      return __vmaxu2(a, b);
    }
  }
  // The larger of a word's values (sizeof(T) == 2: of its two), as the bits of an fp32 number.
  __device__ static __forceinline__ uint32_t f32(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
      return w;
    } else {
      return f32_of(max(w >> 16, w & 0xffffu));
    }
  }
  // A 16-bit value's bits as those of an fp32 number.
  __device__ static __forceinline__ uint32_t f32_of(uint32_t bits) {
    const uint16_t h = static_cast<uint16_t>(bits);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h)));
  }
  __device__ static __forceinline__ uint32_t of(const Raw8<T>& v) {
    uint32_t m = magnitude(word(v, 0));
#pragma unroll
    for (int i = 1; i < kWords; ++i) m = larger(m, magnitude(word(v, i)));
    return m;
  }
};

// Blocks of 1 x 128, as the matrix lies: 16 threads take four blocks at once. Issue-bound if each thread divides for each block (139
// instructions for eight values, 8192 x 4096 bf16 22.8 us): the four maxima are exchanged so that each thread ends with one block's, divides once and
// hands the reciprocal round.
template <typename T, bool kVec, bool kE5M2>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
  using Top = Tops<T>;
  griddep_launch_dependents();
  griddep_wait();
  const int part = threadIdx.x & 15;
  // A CTA takes the 64 blocks from blockIdx.x on, in the order of the rows; these 16 threads every 16th of them.
  const long long first = static_cast<long long>(blockIdx.x) * 64 + (threadIdx.x >> 4);
  const long long total = a.rows * a.blocks;
  Raw8<T> v[4];
  uint32_t top[4];
  long long row = first < total ? first <= 0x7fffffffLL ? static_cast<uint32_t>(first) / static_cast<uint32_t>(a.blocks) : first / a.blocks : 0;
  int block = static_cast<int>(first - row * a.blocks), c[4];
  const long long row0 = row;
  int rows_on[4];  // from row0
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = first + i * 16 < total;
    rows_on[i] = static_cast<int>(row - row0);
    c[i] = in ? block * 128 + part * 8 : a.cols;
    load_piece<T, kVec>(static_cast<const T*>(a.x) + (in ? row : 0) * a.ldx, c[i], a.cols, v[i]);
    block += 16;
    if (block >= a.blocks) {
      const int more = a.blocks > 15 ? 1 : block / a.blocks;
      row += more, block -= more * a.blocks;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = Top::of(v[i]);
  // Threads 8 apart share out four maxima, 4 apart two: the thread ends with that of block `mine`.
  const bool high = (part & 8) != 0, upper = (part & 4) != 0;
  uint32_t two[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    two[i] = Top::larger(high ? top[i + 2] : top[i], __shfl_xor_sync(0xffffffffu, high ? top[i] : top[i + 2], 8));
  uint32_t one = Top::larger(upper ? two[1] : two[0], __shfl_xor_sync(0xffffffffu, upper ? two[0] : two[1], 4));
  one = Top::larger(one, __shfl_xor_sync(0xffffffffu, one, 2));
  one = Top::larger(one, __shfl_xor_sync(0xffffffffu, one, 1));
  const int mine = (high ? 2 : 0) + (upper ? 1 : 0);
  const float scale = block_scale<kE5M2>(Top::f32(one)), inv = 1.f / scale;
  if ((part & 3) == 0 && first + mine * 16 < total) a.scales[first + mine * 16] = scale;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = __shfl_sync(0xffffffffu, inv, i * 4, 16);
    if (c[i] < a.cols) {  // (rows of q are padded to whole pieces)
      float2 x[4];
      pairs_of(v[i], x);
      *reinterpret_cast<uint2*>(a.q + (row0 + rows_on[i]) * a.ldq + c[i]) = quantize8<kE5M2>(x, f);
    }
  }
}

// A CTA quantises 128 x 128 values of x; thread (g, l) rows 8 g .. 8 g + 7, columns 8 l .. 8 l + 7 of them, which it keeps as they lie in
// memory (as fp32 numbers they took 93 registers, two CTAs an SM: 11008 x 4096 bf16 in 128 x 128 40 us). The columns' scales are divided for once, by
// a thread a column.
template <typename T, bool kVec, bool kE5M2, bool kSquare, bool kTransposed>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantArgs a) {
  using Top = Tops<T>;
  constexpr int kWords = Top::kWords;
  __shared__ uint32_t tops[kSquare ? 8 : 8 * 16 * kWords];
  __shared__ float invs[kSquare ? 1 : 128];
  __shared__ uint2 bytes[kTransposed ? 128 * 16 : 1];  // [column of x][8 rows of x], the latter XORed with l
  griddep_launch_dependents();
  griddep_wait();
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_c = (a.cols + 127) / 128;
  const long long tile_r = blockIdx.x / tiles_c;
  const int tile_c = static_cast<int>(blockIdx.x - tile_r * tiles_c);
  const long long r0 = tile_r * 128 + g * 8;
  const int c0 = tile_c * 128 + l * 8;
  Raw8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load_piece<T, kVec>(static_cast<const T*>(a.x) + (r0 + i < a.rows ? r0 + i : 0) * a.ldx, c0, r0 + i < a.rows ? a.cols : 0, v[i]);
  float inv[kSquare ? 1 : 8];  // of each column, or of all
  if constexpr (kSquare) {
    uint32_t top = Top::of(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = Top::larger(top, Top::of(v[i]));
    top = __reduce_max_sync(0xffffffffu, Top::f32(top));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
    const float scale = block_scale<kE5M2>(top);
    if (threadIdx.x == 0) a.scales[kTransposed ? static_cast<long long>(tile_c) * a.blocks + tile_r : tile_r * a.blocks + tile_c] = scale;
    inv[0] = 1.f / scale;
  } else {
    // columns' magnitudes: a word's over the thread's rows, the warp's two groups of rows, the CTA's warps
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      uint32_t top = Top::magnitude(Top::word(v[0], k));
#pragma unroll
      for (int i = 1; i < 8; ++i) top = Top::larger(top, Top::magnitude(Top::word(v[i], k)));
      top = Top::larger(top, __shfl_xor_sync(0xffffffffu, top, 16));
      if (lane < 16) tops[(warp * kWords + k) * 16 + l] = top;
    }
    __syncthreads();
    if (threadIdx.x < 128) {  // a column each
      constexpr int kEach = 8 / kWords;  // values of a word
      const int c = threadIdx.x, k = c % 8 / kEach;
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = Top::larger(top, tops[(i * kWords + k) * 16 + c / 8]);
      const float scale = block_scale<kE5M2>(sizeof(T) == 4 ? top : Top::f32_of(c & 1 ? top >> 16 : top & 0xffffu));
      invs[c] = 1.f / scale;
      if (tile_c * 128 + c < a.cols) a.scales[static_cast<long long>(tile_c * 128 + c) * a.blocks + tile_r] = scale;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = invs[l * 8 + j];
  }
  if constexpr (!kTransposed) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 f[4];
      pairs_of(v[i], f);
      if (r0 + i < a.rows && c0 < a.cols) *reinterpret_cast<uint2*>(a.q + (r0 + i) * a.ldq + c0) = quantize8<kE5M2>(f, inv[0]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float2 column[4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f[8];
        v[i].values(f);
        (i & 1 ? column[i / 2].y : column[i / 2].x) = f[j];
      }
      bytes[(l * 8 + j) * 16 + (g ^ l)] = quantize8<kE5M2>(column, inv[kSquare ? 0 : j]);
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
int launch_quantize(const QuantArgs& a, int block_rows, bool transposed, cudaStream_t st) {
  Launch l(st);
  if (block_rows == 1 && !transposed) {
    const long long ctas = (a.rows * a.blocks + 63) / 64;
    if (ctas > 0x7fffffffLL) return fail(KCG_E_TOO_LARGE, "too many blocks for one launch");
    l.shape(static_cast<unsigned>(ctas), 256);
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
int launch_quantize(const QuantArgs& a, int block_rows, bool transposed, bool e5m2, cudaStream_t st) {
  const bool vec = reinterpret_cast<uint64_t>(a.x) % 16 == 0 && a.ldx * static_cast<long long>(sizeof(T)) % 16 == 0;
  if (vec)
    return e5m2 ? launch_quantize<T, true, true>(a, block_rows, transposed, st)
                : launch_quantize<T, true, false>(a, block_rows, transposed, st);
  return e5m2 ? launch_quantize<T, false, true>(a, block_rows, transposed, st)
              : launch_quantize<T, false, false>(a, block_rows, transposed, st);
}

}  // namespace

extern "C" int kcg_quantize_fp8(int device, uint64_t stream, uint64_t X, int64_t ldx, uint64_t Q, int64_t ldq, uint64_t S, int64_t rows,
                                int cols, int block_rows, int transposed, int dtype, int dtype8) {
  if (!known_dtype(dtype)) return fail(KCG_E_BAD_ARG, "quantisation takes float16, bfloat16 or float32 data");
  if (dtype8 != KCG_FP8_E4M3 && dtype8 != KCG_FP8_E5M2) return fail(KCG_E_BAD_ARG, "quantisation gives e4m3 or e5m2 values");
  if (block_rows != 1 && block_rows != 128) return fail(KCG_E_BAD_ARG, "blocks have 1 or 128 rows");
  if (rows < 0 || cols <= 0) return fail(KCG_E_BAD_ARG, "shape out of range");
  if (rows > kMaxSize || cols > kMaxSize) return fail(KCG_E_TOO_LARGE, "a size of an 8-bit matrix is above 2^31 - 256");
  if (rows == 0) return 0;
  if (!X || !Q || !S) return fail(KCG_E_BAD_ARG, "null matrix");
  const int64_t out_cols = transposed ? rows : cols;
  if (ldx == 0) ldx = cols;
  if (ldq == 0) ldq = out_cols;
  if (ldx < cols || ldq < out_cols) return fail(KCG_E_BAD_ARG, "leading dimension below the row length");
  if (Q % 16 || ldq % 16) return fail(KCG_E_BAD_ARG, "rows of 8-bit values must start on 16-byte boundaries");
  const int eb = dtype == KCG_DTYPE_FLOAT32 ? 4 : 2;
  if (X % eb || S % 4) return fail(KCG_E_BAD_ARG, "operands must be aligned to their values");
  QuantArgs a{};
  a.x = reinterpret_cast<const void*>(X), a.q = reinterpret_cast<uint8_t*>(Q), a.scales = reinterpret_cast<float*>(S);
  a.ldx = ldx, a.ldq = ldq, a.rows = rows, a.cols = cols, a.blocks = static_cast<int>((out_cols + 127) / 128);
  DeviceGuard guard;
  const cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool e5m2 = dtype8 == KCG_FP8_E5M2, t = transposed != 0;
  if (dtype == KCG_DTYPE_FLOAT32) return launch_quantize<float>(a, block_rows, t, e5m2, st);
  return dtype == KCG_DTYPE_FLOAT16 ? launch_quantize<__half>(a, block_rows, t, e5m2, st)
                                    : launch_quantize<__nv_bfloat16>(a, block_rows, t, e5m2, st);
}
