// Root-mean-square norm of rows, forward (with the residual's addition in front of it, its result in the rows' type or as 8-bit
// values with a scale for each 128 of a row) and backward, for fp16, bf16 and fp32:
//     h = x + residual,   y = h * r * w,   r = 1 / sqrt(mean(h^2) + eps)
//     with g = dy * w:    dx = dh + r * g - h * r^3 * mean(g * h),   dw = sum over the rows of dy * h * r
// (dh: the gradient that reaches h past the norm, along the residual stream.) Sums and products in fp32, one rounding at the end:
// y comes from the unrounded sum h, which is rounded only where it is stored.
//
// A sum of squares past fp32's largest number makes r 0 (rows of 1.8e19 and more, a single value of that size), one below its smallest, with
// eps = 0, infinite.
//
// Bound by HBM: a row is read once, into registers, and written once, by a warp (forward, up to 1024 values) or by CTAs that walk rows. Rows
// that are no whole 16-byte pieces are read value by value, forward by a kernel of their own. Read twice, the second time from a
// cache: such rows of more than 16384 values, and h and dy of every row of more than 16384 in the gradient.
//
// Registers: the CTAs an SM were chosen for 16-bit rows. In fp32 with a residual, up to 16384 values, 72 to 160 bytes a thread are spilled, in
// every type past 16384 values 60 to 950, and by the gradient 36 to 264 in fp32 up to 8192 values and 320 to 644 in every type from there to
// 16384 (four pieces of h, dy, the weight and their shares of dw in 128 registers).
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <string>

#include "../../include/kcg_b200.h"
#include "fp8_common.cuh"
#include "kernels/ptx_sm100.cuh"

namespace {

using namespace kcg;
using namespace kcg8;

struct NormArgs {
  const void *x, *residual, *w;
  void *y, *h;       // y: 8-bit values where there are scales
  float* scales;     // rows x ceil(width / 128)
  long long ldx, ldr, ldy, ldh, rows;
  int width, blocks;  // blocks: scales of a row
  float eps;
};

// Warps of a CTA of so many threads, up to the next power of two.
__host__ __device__ constexpr int warps_of(int threads) { return threads <= 256 ? 8 : threads <= 512 ? 16 : 32; }

// Sums over the threads of a row: a warp's (kWarps = 1), or those of a CTA of kWarps warps at most (a power of two).
template <int kWarps, int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float* scratch) {
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  static_assert((kWarps & (kWarps - 1)) == 0, "lanes stand for warps");
  if constexpr (kWarps > 1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, from = lane & (kWarps - 1);
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < kN; ++n) scratch[n * kWarps + warp] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      v[n] = from < warps ? scratch[n * kWarps + from] : 0.f;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
  }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float rcp_ftz(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The end of a forward pass for one piece: h is stored, y (= h * r * w, in that order: h * w may leave fp32's range where y does not) stored
// or quantised. kFp8: the 16 neighbouring threads that hold 128 values of the row come together.
template <typename T, bool kRes, bool kFp8>
__device__ __forceinline__ void finish_piece(const NormArgs& a, long long row, int v, bool in, int tid, const float2 (&h)[4],
                                             const float2 (&w)[4], float r) {
  if (kRes && in) store8(static_cast<T*>(a.h) + row * a.ldh + 8 * v, h);
  float2 y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = __fmul2_rn(__fmul2_rn(h[j], both(r)), w[j]);
  if constexpr (kFp8) {
    uint32_t bits = in ? abs_max(y) : 0u;  // (__reduce_max_sync of a warp's halves runs them one after the other, all that follows too)
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    const float top = __uint_as_float(bits);
    // scale = top / 448 and, for 1 / scale, 448 / top, off by an ulp or two. Where one of them is no normal number (a block of next to nothing,
    // values near the largest, an infinity or a NaN in the row) by the definition.
    float scale = top * (1.f / 448.f), factor = 448.f * rcp_ftz(top);
    if (!(scale >= FLT_MIN && factor >= FLT_MIN)) {
      if (scale < FLT_MIN) scale = FLT_MIN;
      factor = 1.f / scale;
    }
    if (in) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row * a.ldy + 8 * v) = quantize8<false>(y, factor);
      if ((tid & 15) == 0) a.scales[row * a.blocks + (v >> 4)] = scale;
    }
  } else if (in) {
    store8(static_cast<T*>(a.y) + row * a.ldy + 8 * v, y);
  }
}

// h = x + residual of a piece, and its squares on top of `sum`.
template <typename T, bool kRes>
__device__ __forceinline__ void sum_piece(const Raw8<T>& x, const Raw8<T>& res, float2 (&h)[4], float2& sum) {
  pairs_of(x, h);
  if constexpr (kRes) {
    float2 f[4];
    pairs_of(res, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __fadd2_rn(h[j], f[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sum = __ffma2_rn(h[j], h[j], sum);
}

// A warp a row, rows of up to 1024 values. kVPT: pieces of 8 values a thread holds.
template <typename T, int kVPT, bool kRes, bool kFp8>
__global__ void __launch_bounds__(256) norm_warp_kernel(const NormArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x & 31, pieces = a.width / 8;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = kRes ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  float2 h[kVPT][4], squares = both(0.f);
#pragma unroll
  for (int i = 0; i < kVPT; ++i) {
    const int v = i * 32 + tid;
    Raw8<T> p, q;
    p.zero(), q.zero();
    if (v < pieces) {
      p.load(x + 8 * v);
      if constexpr (kRes) q.load(res + 8 * v);
    }
    sum_piece<T, kRes>(p, q, h[i], squares);
  }
  float sum[1] = {squares.x + squares.y};
  row_sum<1>(sum, nullptr);
  const float r = rsqrtf(sum[0] / static_cast<float>(a.width) + a.eps);
#pragma unroll
  for (int i = 0; i < kVPT; ++i) {
    const int v = i * 32 + tid;
    Raw8<T> raw;
    raw.zero();
    if (v < pieces) raw.load(static_cast<const T*>(a.w) + 8 * v);
    float2 w[4];
    pairs_of(raw, w);
    finish_piece<T, kRes, kFp8>(a, row, v, v < pieces, tid, h[i], w, r);
  }
}

// A CTA walks rows blockIdx.x, + gridDim.x, ...; it keeps the weight, and asks for the next row before it reduces the present one (with one
// row a CTA, 5001 x 5504 fp16 into 8 bits took 37 us: loads, sum and stores of a row by turns).
template <typename T, int kVPT, bool kRes, bool kFp8, int kThreads, int kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) norm_kernel(const NormArgs a) {
  __shared__ float scratch[2][32];
  constexpr bool kAhead = kThreads <= 512;  // (registers)
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, threads = blockDim.x, pieces = a.width / 8;
  Raw8<T> w[kVPT], x[kVPT], res[kRes ? kVPT : 1];
  auto ask = [&](long long row) {
#pragma unroll
    for (int i = 0; i < kVPT; ++i) {
      const int v = i * threads + tid;
      if (v < pieces) {
        x[i].load(static_cast<const T*>(a.x) + row * a.ldx + 8 * v);
        if constexpr (kRes) res[i].load(static_cast<const T*>(a.residual) + row * a.ldr + 8 * v);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kVPT; ++i) {
    w[i].zero();
    x[i].zero();
    if constexpr (kRes) res[i].zero();
    if (kAhead && i * threads + tid < pieces) w[i].load(static_cast<const T*>(a.w) + 8 * (i * threads + tid));
  }
  long long row = blockIdx.x;
  if (kAhead && row < a.rows) ask(row);
  for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
    if constexpr (!kAhead) ask(row);
    float2 h[kVPT][4], squares = both(0.f);
#pragma unroll
    for (int i = 0; i < kVPT; ++i) sum_piece<T, kRes>(x[i], res[kRes ? i : 0], h[i], squares);
    float sum[1] = {squares.x + squares.y};
    if (kAhead && row + gridDim.x < a.rows) ask(row + gridDim.x);
    row_sum<warps_of(kThreads)>(sum, scratch[turn]);  // (two scratches: one barrier a row)
    const float r = rsqrtf(sum[0] / static_cast<float>(a.width) + a.eps);
#pragma unroll
    for (int i = 0; i < kVPT; ++i) {
      const int v = i * threads + tid;
      if constexpr (!kAhead) {
        if (v < pieces) w[i].load(static_cast<const T*>(a.w) + 8 * v);
      }
      float2 f[4];
      pairs_of(w[i], f);
      finish_piece<T, kRes, kFp8>(a, row, v, v < pieces, tid, h[i], f, r);
    }
  }
}

// Rows of any width, pitch and alignment: single values, 128 of them to a warp at a time. kB: the warp's blocks of 128, kept in registers
// with their weights; 0: any number (rows of more than 16384 values), read twice, the second time from a cache. Read twice against kept: 8192 x
// 4095 bf16 with residual 112, 66 us; 4000 x 8191 122, 77 (four blocks a warp of 16; of 32 warps, one CTA an SM, 152); 2000 x 16001 fp16 101, 70;
// 20000 x 300 33, 21.
template <typename T, int kB, bool kRes, bool kFp8, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_any_kernel(const NormArgs a) {
  __shared__ float scratch[32];
  griddep_launch_dependents();
  griddep_wait();
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = kRes ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  const T* w = static_cast<const T*>(a.w);
  auto value = [&](int c) { return kRes ? to_f32(x[c]) + to_f32(res[c]) : to_f32(x[c]); };
  float sum[1] = {0.f}, kept[kB ? kB : 1][4];
  T weight[kB ? kB : 1][4];
  if constexpr (kB > 0) {
#pragma unroll
    for (int i = 0; i < kB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = (i * kWarps + warp) * 128 + j * 32 + lane;
        kept[i][j] = c < a.width ? value(c) : 0.f;
        weight[i][j] = c < a.width ? w[c] : from_f32<T>(0.f);
      }
#pragma unroll
    for (int i = 0; i < kB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[0] = fmaf(kept[i][j], kept[i][j], sum[0]);
  } else {
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float v = value(c);
      sum[0] = fmaf(v, v, sum[0]);
    }
  }
  row_sum<kWarps>(sum, scratch);
  const float r = rsqrtf(sum[0] / static_cast<float>(a.width) + a.eps);
  auto finish = [&](int b, const float* known, const T* weights) {
    float y[4];
    uint32_t top = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = b * 128 + j * 32 + lane;
      y[j] = 0.f;
      if (c < a.width) {
        const float v = kB > 0 ? known[j] : value(c);
        y[j] = v * r * to_f32(kB > 0 ? weights[j] : w[c]);
        // (where h is written over x or the residual, each value has been read by the thread that writes it)
        if constexpr (kRes) static_cast<T*>(a.h)[row * a.ldh + c] = from_f32<T>(v);
        if constexpr (!kFp8) static_cast<T*>(a.y)[row * a.ldy + c] = from_f32<T>(y[j]);
      }
      top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
    }
    if constexpr (kFp8) {
      const float scale = block_scale<false>(__reduce_max_sync(0xffffffffu, top)), inv = 1.f / scale;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = b * 128 + j * 32 + lane;
        if (c < a.width) static_cast<uint8_t*>(a.y)[row * a.ldy + c] = quantize1<false>(y[j], inv);
      }
      if (lane == 0) a.scales[row * a.blocks + b] = scale;
    }
  };
  if constexpr (kB > 0) {
#pragma unroll
    for (int i = 0; i < kB; ++i)
      if ((i * kWarps + warp) * 128 < a.width) finish(i * kWarps + warp, kept[i], weight[i]);
  } else {
    for (int b = warp; b * 128 < a.width; b += kWarps) finish(b, nullptr, nullptr);
  }
}

struct GradArgs {
  const void *dy, *h, *w, *dh;
  void *dx, *dw;
  float* partial;  // one row of `width` sums for each CTA
  long long lddy, ldh, lddh, lddx, rows;
  int width;
  float eps;
};

// Each CTA walks rows blockIdx.x, + gridDim.x, ...; a thread keeps its columns' share of dw in registers, the row as it lies in
// memory, and (kAhead: rows of up to 8192 values) asks for the next row before it reduces the present one. !kWhole: rows that
// are no whole 16-byte pieces, value by value, a warp's side by side (8192 x 4095 bf16 104 us; eight of a row in each thread 156; dw in shared
// memory 300).
template <typename T, int kVPT, bool kDh, bool kWhole, int kThreads, int kCtas, bool kAhead>
__global__ void __launch_bounds__(kThreads, kCtas) norm_grad_kernel(const GradArgs a) {
  constexpr int kWarps = warps_of(kThreads);
  __shared__ float scratch[2][2 * kWarps];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, threads = blockDim.x;
  struct Row {
    Raw8<T> h[kVPT], dy[kVPT], dh[kDh ? kVPT : 1];
  };
  float2 dw[kVPT][4];
  Raw8<T> w[kVPT];
  Row at, next;
  // The column of a thread's piece v = i * threads + tid, whose others follow at once, or (single values) `threads` apart.
  auto first = [&](int v) { return kWhole ? 8 * v : 8 * (v - tid) + tid; };
  auto read = [&](Raw8<T>& to, const T* from, int v) {
    if constexpr (kWhole) {
      to.load(from + 8 * v);
    } else {
      load_piece<T, false>(from, first(v), a.width, to, threads);
    }
  };
  auto ask = [&](Row& to, long long row) {
#pragma unroll
    for (int i = 0; i < kVPT; ++i) {
      const int v = i * threads + tid;
      if (first(v) < a.width) {
        read(to.h[i], static_cast<const T*>(a.h) + row * a.ldh, v);
        read(to.dy[i], static_cast<const T*>(a.dy) + row * a.lddy, v);
        if constexpr (kDh) read(to.dh[i], static_cast<const T*>(a.dh) + row * a.lddh, v);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kVPT; ++i) {
    w[i].zero(), at.h[i].zero(), at.dy[i].zero(), next.h[i].zero(), next.dy[i].zero();
    if constexpr (kDh) at.dh[i].zero(), next.dh[i].zero();
    if (first(i * threads + tid) < a.width) read(w[i], static_cast<const T*>(a.w), i * threads + tid);
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i][j] = both(0.f);
  }
  const float inv = 1.f / static_cast<float>(a.width);
  long long row = blockIdx.x;
  if (kAhead && row < a.rows) ask(next, row);
  for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
    if constexpr (kAhead) {
      at = next;
      if (row + gridDim.x < a.rows) ask(next, row + gridDim.x);
    } else {
      ask(at, row);
    }
    float2 squares = both(0.f), products = both(0.f);
#pragma unroll
    for (int i = 0; i < kVPT; ++i) {
      float2 h[4], dy[4], f[4];
      pairs_of(at.h[i], h);
      pairs_of(at.dy[i], dy);
      pairs_of(w[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        squares = __ffma2_rn(h[j], h[j], squares);
        products = __ffma2_rn(__fmul2_rn(dy[j], f[j]), h[j], products);
      }
    }
    float sum[2] = {squares.x + squares.y, products.x + products.y};
    row_sum<kWarps>(sum, scratch[turn]);  // (two scratches: one barrier a row)
    const float r = rsqrtf(fmaf(sum[0], inv, a.eps));
    const float back = -r * r * (sum[1] * inv);  // dx = r * (g + h * back)
#pragma unroll
    for (int i = 0; i < kVPT; ++i) {
      const int v = i * threads + tid;
      float2 h[4], dy[4], f[4], d[4];
      pairs_of(at.h[i], h);
      pairs_of(at.dy[i], dy);
      pairs_of(w[i], f);
      if constexpr (kDh) pairs_of(at.dh[i], d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 g = __ffma2_rn(h[j], both(back), __fmul2_rn(dy[j], f[j]));
        dw[i][j] = __ffma2_rn(dy[j], __fmul2_rn(h[j], both(r)), dw[i][j]);
        d[j] = kDh ? __ffma2_rn(g, both(r), d[j]) : __fmul2_rn(g, both(r));
      }
      if (first(v) < a.width) store_piece<T, kWhole>(static_cast<T*>(a.dx) + row * a.lddx, first(v), a.width, d, threads);
    }
  }
  float* mine = a.partial + static_cast<long long>(blockIdx.x) * a.width;
#pragma unroll
  for (int i = 0; i < kVPT; ++i) {
    const int v = i * threads + tid;
    if (first(v) < a.width) store_piece<float, kWhole>(mine, first(v), a.width, dw[i], threads);
  }
}

// Rows of more than 16384 values, any pitch and alignment: the CTA's share of dw in shared memory, each value owned by one thread.
template <typename T, bool kDh>
__global__ void __launch_bounds__(512) norm_grad_any_kernel(const GradArgs a) {
  extern __shared__ float dw[];
  __shared__ float scratch[2][64];
  griddep_launch_dependents();
  griddep_wait();
  const T* w = static_cast<const T*>(a.w);
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) dw[c] = 0.f;
  int turn = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T *h = static_cast<const T*>(a.h) + row * a.ldh, *dy = static_cast<const T*>(a.dy) + row * a.lddy;
    float sum[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      const float v = to_f32(h[c]);
      sum[0] = fmaf(v, v, sum[0]);
      sum[1] = fmaf(to_f32(dy[c]) * to_f32(w[c]), v, sum[1]);
    }
    row_sum<16>(sum, scratch[turn]);
    const float inv = 1.f / static_cast<float>(a.width);
    const float r = rsqrtf(fmaf(sum[0], inv, a.eps)), back = r * r * (sum[1] * inv);
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      const float v = to_f32(h[c]), g = to_f32(dy[c]);
      float dx = r * (g * to_f32(w[c]) - v * back);
      if constexpr (kDh) dx += to_f32(static_cast<const T*>(a.dh)[row * a.lddh + c]);
      static_cast<T*>(a.dx)[row * a.lddx + c] = from_f32<T>(dx);
      dw[c] = fmaf(g, v * r, dw[c]);
    }
  }
  float* mine = a.partial + static_cast<long long>(blockIdx.x) * a.width;
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) mine[c] = dw[c];
}

// dw = sum of the CTAs' shares, in their order: 32 threads a column, each a 32nd of the shares.
template <typename T>
__global__ void __launch_bounds__(1024) norm_grad_sum_kernel(const float* partial, int parts, int width, T* dw) {
  __shared__ float sums[32][33];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int p = part; p < parts; p += 32) s += partial[static_cast<long long>(p) * width + c];
  }
  sums[part][lane] = s;
  __syncthreads();
  s = sums[lane][part];  // share `lane` of column `part`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && blockIdx.x * 32 + part < width) dw[blockIdx.x * 32 + part] = from_f32<T>(s);
}

// ------------------------------------------------------------------------------------------------ launches
// CTAs of a kernel that an SM holds at once (asked once per number of threads; one kind of GPU a process).
template <typename K>
int ctas_per_sm(K kernel, int threads, std::atomic<int> (&known)[33]) {
  int n = known[threads / 32].load();
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    known[threads / 32].store(n);
  }
  return n;
}

template <typename T, int kVPT, bool kRes, bool kFp8, int kThreads, int kCtas>
int launch_norm_rows(Launch& l, const NormArgs& a, int sms) {
  static std::atomic<int> known[33];
  const auto kernel = norm_kernel<T, kVPT, kRes, kFp8, kThreads, kCtas>;
  const int threads = ((a.width / 8 + kVPT - 1) / kVPT + 31) / 32 * 32;
  const long long most = static_cast<long long>(sms) * ctas_per_sm(kernel, threads, known);
  l.shape(static_cast<unsigned>(a.rows < most ? a.rows : most), threads);
  return l(kernel, "norm launch", a);
}

template <typename T, bool kRes, bool kFp8>
int launch_norm(const NormArgs& a, bool vectors, int sms, cudaStream_t st) {
  Launch l(st);
  if (!vectors) {
    const int blocks = (a.width + 127) / 128;
    const int threads = blocks <= 4 ? 64 : blocks <= 16 ? 256 : blocks <= 64 ? 512 : blocks <= 128 ? 1024 : 256;
    l.shape(static_cast<unsigned>(a.rows), threads);
    if (blocks <= 4) return l(norm_any_kernel<T, 2, kRes, kFp8, 64>, "norm launch", a);
    if (blocks <= 16) return l(norm_any_kernel<T, 2, kRes, kFp8, 256>, "norm launch", a);
    if (blocks <= 32) return l(norm_any_kernel<T, 2, kRes, kFp8, 512>, "norm launch", a);
    if (blocks <= 64) return l(norm_any_kernel<T, 4, kRes, kFp8, 512>, "norm launch", a);
    if (blocks <= 128) return l(norm_any_kernel<T, 4, kRes, kFp8, 1024>, "norm launch", a);
    return l(norm_any_kernel<T, 0, kRes, kFp8, 256>, "norm launch", a);
  }
  const int pieces = a.width / 8;
  if (pieces <= 128) {
    l.shape(static_cast<unsigned>((a.rows + 7) / 8), 256);
    if (pieces <= 32) return l(norm_warp_kernel<T, 1, kRes, kFp8>, "norm launch", a);
    if (pieces <= 64) return l(norm_warp_kernel<T, 2, kRes, kFp8>, "norm launch", a);
    return l(norm_warp_kernel<T, 4, kRes, kFp8>, "norm launch", a);
  }
  if (pieces <= 256) return launch_norm_rows<T, 1, kRes, kFp8, 256, 6>(l, a, sms);
  if (pieces <= 512) return launch_norm_rows<T, 2, kRes, kFp8, 256, kRes || kFp8 ? 4 : 5>(l, a, sms);
  if (!kRes && pieces <= 768) return launch_norm_rows<T, 2, kRes, kFp8, 384, 3>(l, a, sms);
  if (pieces <= 1024) return launch_norm_rows<T, 2, kRes, kFp8, 512, 2>(l, a, sms);
  if (pieces <= 2048) return launch_norm_rows<T, 4, kRes, kFp8, 512, 1>(l, a, sms);
  return launch_norm_rows<T, 4, kRes, kFp8, 1024, 1>(l, a, sms);
}

template <typename T>
int launch_norm(const NormArgs& a, bool vectors, int sms, cudaStream_t st) {
  if (a.residual) return a.scales ? launch_norm<T, true, true>(a, vectors, sms, st) : launch_norm<T, true, false>(a, vectors, sms, st);
  return a.scales ? launch_norm<T, false, true>(a, vectors, sms, st) : launch_norm<T, false, false>(a, vectors, sms, st);
}

constexpr int kMaxWidth = 32768;  // (1024 threads hold four pieces each; a CTA's share of dw takes 128 KB of shared memory)

// Threads of a CTA of the backward pass: two pieces each up to 8192 values a row, then four.
int grad_threads(int width) {
  const int pieces = (width + 7) / 8, each = pieces <= 1024 ? 2 : 4;
  return ((pieces + each - 1) / each + 31) / 32 * 32;
}
// CTAs that walk its rows, each with its own share of dw: as many as run at once (512 threads an SM, by their registers), with two rows
// each or more (513 x 1376 bf16 with one, two, four 5.3, 4.6, 6.1 us).
int grad_ctas(int sms, long long rows, int width) {
  const int per_sm = 512 / grad_threads(width);
  const long long most = static_cast<long long>(sms) * (per_sm < 1 ? 1 : per_sm), few = (rows + 1) / 2;
  return static_cast<int>(few < most ? few : most);
}

template <typename T, bool kDh, bool kWhole>
int launch_grad(const GradArgs& a, int ctas, cudaStream_t st) {
  Launch l(st);
  const int threads = grad_threads(a.width);
  l.shape(ctas, threads);
  if (a.width > 8192) return l(norm_grad_kernel<T, 4, kDh, kWhole, 512, 1, false>, "norm gradient launch", a);
  if (threads > 256) return l(norm_grad_kernel<T, 2, kDh, kWhole, 512, 1, true>, "norm gradient launch", a);
  return l(norm_grad_kernel<T, 2, kDh, kWhole, 256, 2, true>, "norm gradient launch", a);
}
template <typename T, bool kDh>
int launch_grad(const GradArgs& a, int ctas, bool whole, cudaStream_t st) {
  if (a.width <= 16384) return whole ? launch_grad<T, kDh, true>(a, ctas, st) : launch_grad<T, kDh, false>(a, ctas, st);
  Launch l(st);
  const cudaError_t e = cudaFuncSetAttribute(norm_grad_any_kernel<T, kDh>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kMaxWidth * static_cast<int>(sizeof(float)));
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  l.shape(ctas, 512, static_cast<size_t>(a.width) * sizeof(float));
  return l(norm_grad_any_kernel<T, kDh>, "norm gradient launch", a);
}

template <typename T>
int launch_grad(const GradArgs& a, int ctas, bool vectors, cudaStream_t st) {
  if (int e = a.dh ? launch_grad<T, true>(a, ctas, vectors, st) : launch_grad<T, false>(a, ctas, vectors, st)) return e;
  Launch l(st);
  l.shape((a.width + 31) / 32, 1024);
  return l(norm_grad_sum_kernel<T>, "norm gradient launch", static_cast<const float*>(a.partial), ctas, a.width,
           static_cast<T*>(a.dw));
}

// Whether all rows of a matrix start on 16-byte boundaries and hold whole pieces of 8 values.
bool pieces_of_8(uint64_t p, int64_t ld, int bytes) { return p % 16 == 0 && ld * bytes % 16 == 0; }

int norm_checks(int64_t rows, int width, int dtype, float eps) {
  if (rows < 0 || rows > 0x7fffffffLL) return fail(KCG_E_BAD_ARG, "number of rows out of range");
  if (width <= 0 || width > kMaxWidth) return fail(KCG_E_BAD_ARG, "row width must be 1 to 32768");
  if (!known_dtype(dtype)) return fail(KCG_E_BAD_ARG, "the norm takes float16, bfloat16 or float32 data");
  if (!(eps >= 0.f) || eps > 3e38f) return fail(KCG_E_BAD_ARG, "eps must be finite and not negative");
  return 0;
}

int norm_forward(int device, uint64_t stream, NormArgs a, uint64_t X, uint64_t R, uint64_t W, uint64_t Y, uint64_t H, int dtype) {
  if (int e = norm_checks(a.rows, a.width, dtype, a.eps)) return e;
  if (a.rows == 0) return 0;
  if (!X || !W || !Y || !R != !H) return fail(KCG_E_BAD_ARG, "null matrix, or a residual without a place for the sum");
  const bool fp8 = a.scales != nullptr;
  if (a.ldx == 0) a.ldx = a.width;
  if (a.ldr == 0) a.ldr = a.width;
  if (a.ldy == 0) a.ldy = a.width;
  if (a.ldh == 0) a.ldh = a.width;
  if (a.ldx < a.width || a.ldr < a.width || a.ldy < a.width || a.ldh < a.width)
    return fail(KCG_E_BAD_ARG, "leading dimension below the row length");
  const int eb = dtype == KCG_DTYPE_FLOAT32 ? 4 : 2;
  if ((X | R | W | H | (fp8 ? 0 : Y)) % eb) return fail(KCG_E_BAD_ARG, "operands must be aligned to their values");
  const bool vectors = a.width % 8 == 0 && pieces_of_8(X, a.ldx, eb) && pieces_of_8(R, a.ldr, eb) && pieces_of_8(H, a.ldh, eb) &&
                       W % 16 == 0 && (fp8 ? Y % 8 == 0 && a.ldy % 8 == 0 : pieces_of_8(Y, a.ldy, eb));
  a.x = reinterpret_cast<const void*>(X), a.residual = reinterpret_cast<const void*>(R), a.w = reinterpret_cast<const void*>(W);
  a.y = reinterpret_cast<void*>(Y), a.h = reinterpret_cast<void*>(H);
  int sms = 0;
  if (int e = sm_count(device, &sms)) return e;
  DeviceGuard guard;
  const cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == KCG_DTYPE_FLOAT32) return launch_norm<float>(a, vectors, sms, st);
  return dtype == KCG_DTYPE_FLOAT16 ? launch_norm<__half>(a, vectors, sms, st) : launch_norm<__nv_bfloat16>(a, vectors, sms, st);
}

}  // namespace

extern "C" int kcg_rms_norm(int device, uint64_t stream, uint64_t X, int64_t ldx, uint64_t R, int64_t ldr, uint64_t W, uint64_t Y,
                            int64_t ldy, uint64_t H, int64_t ldh, int64_t rows, int width, float eps, int dtype) {
  NormArgs a{};
  a.ldx = ldx, a.ldr = ldr, a.ldy = ldy, a.ldh = ldh, a.rows = rows, a.width = width, a.eps = eps;
  return norm_forward(device, stream, a, X, R, W, Y, H, dtype);
}

extern "C" int kcg_rms_norm_fp8(int device, uint64_t stream, uint64_t X, int64_t ldx, uint64_t R, int64_t ldr, uint64_t W, uint64_t Q,
                                int64_t ldq, uint64_t S, uint64_t H, int64_t ldh, int64_t rows, int width, float eps, int dtype) {
  NormArgs a{};
  if (!S || S % 4) return fail(KCG_E_BAD_ARG, "scales: null or not aligned to 4 bytes");
  a.scales = reinterpret_cast<float*>(S), a.blocks = (width + 127) / 128;
  a.ldx = ldx, a.ldr = ldr, a.ldy = ldq, a.ldh = ldh, a.rows = rows, a.width = width, a.eps = eps;
  return norm_forward(device, stream, a, X, R, W, Q, H, dtype);
}

extern "C" int64_t kcg_rms_norm_backward_workspace(int device, int64_t rows, int width) {
  if (rows <= 0 || width <= 0) return 0;
  int sms = 0;
  if (sm_count(device, &sms)) return -1;
  return static_cast<int64_t>(grad_ctas(sms, rows, width)) * width * static_cast<int64_t>(sizeof(float));
}

extern "C" int kcg_rms_norm_backward(int device, uint64_t stream, uint64_t DY, int64_t lddy, uint64_t H, int64_t ldh, uint64_t W,
                                     uint64_t DH, int64_t lddh, uint64_t DX, int64_t lddx, uint64_t DW, uint64_t workspace,
                                     int64_t workspace_bytes, int64_t rows, int width, float eps, int dtype) {
  if (int e = norm_checks(rows, width, dtype, eps)) return e;
  if (rows == 0) return fail(KCG_E_BAD_ARG, "empty shape");
  if (!DY || !H || !W || !DX || !DW || !workspace) return fail(KCG_E_BAD_ARG, "null matrix");
  if (lddy == 0) lddy = width;
  if (ldh == 0) ldh = width;
  if (lddh == 0) lddh = width;
  if (lddx == 0) lddx = width;
  if (lddy < width || ldh < width || lddh < width || lddx < width) return fail(KCG_E_BAD_ARG, "leading dimension below the row length");
  const int eb = dtype == KCG_DTYPE_FLOAT32 ? 4 : 2;
  if ((DY | H | W | DH | DX | DW) % eb || workspace % 16) return fail(KCG_E_BAD_ARG, "operands must be aligned to their values");
  int sms = 0;
  if (int e = sm_count(device, &sms)) return e;
  const int ctas = grad_ctas(sms, rows, width);
  if (workspace_bytes < static_cast<int64_t>(ctas) * width * static_cast<int64_t>(sizeof(float)))
    return fail(KCG_E_BAD_ARG, "workspace too small");
  GradArgs a{};
  a.dy = reinterpret_cast<const void*>(DY), a.h = reinterpret_cast<const void*>(H), a.w = reinterpret_cast<const void*>(W);
  a.dh = reinterpret_cast<const void*>(DH), a.dx = reinterpret_cast<void*>(DX), a.dw = reinterpret_cast<void*>(DW);
  a.partial = reinterpret_cast<float*>(workspace);
  a.lddy = lddy, a.ldh = ldh, a.lddh = lddh, a.lddx = lddx, a.rows = rows, a.width = width, a.eps = eps;
  const bool vectors = width % 8 == 0 && pieces_of_8(DY, lddy, eb) && pieces_of_8(H, ldh, eb) && pieces_of_8(DH, lddh, eb) &&
                       pieces_of_8(DX, lddx, eb) && W % 16 == 0;
  DeviceGuard guard;
  const cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == KCG_DTYPE_FLOAT32) return launch_grad<float>(a, ctas, vectors, st);
  return dtype == KCG_DTYPE_FLOAT16 ? launch_grad<__half>(a, ctas, vectors, st) : launch_grad<__nv_bfloat16>(a, ctas, vectors, st);
}
