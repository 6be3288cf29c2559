// What the kernels of the 8-bit linear layer share: loads and stores of eight values, the 8-bit values of a block and its scale,
// and the host side of a launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>
#include <string>

#include "../../include/kcg_b200.h"

extern "C" int kcg_internal_fail(int code, const char* msg);
extern "C" void kcg_internal_count_launch(void);

namespace kcg8 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8], __half) {
  const __half2* e = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(e[j]);
    v[2 * j] = f.x, v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8], __nv_bfloat16) {
  const uint32_t e[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(e[j] << 16), v[2 * j + 1] = __uint_as_float(e[j] & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight consecutive values from a 16-byte boundary, as they lie in memory: one 16-byte vector of a 16-bit type, two of fp32.
template <typename T>
struct Raw8 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void set(const T (&e)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = *reinterpret_cast<const uint16_t*>(&e[2 * j]) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&e[2 * j + 1])) << 16;
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void values(float (&f)[8]) const { unpack8(v, f, T()); }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void set(const float (&e)[8]) {
    a = make_float4(e[0], e[1], e[2], e[3]), b = make_float4(e[4], e[5], e[6], e[7]);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
};
// The same as pairs, for instructions that take two numbers at once.
template <typename T>
__device__ __forceinline__ void pairs_of(const Raw8<T>& raw, float2 (&f)[4]) {
  float v[8];
  raw.values(v);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = make_float2(v[2 * j], v[2 * j + 1]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float2 (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0].x, v[0].y, T()), pack2(v[1].x, v[1].y, T()), pack2(v[2].x, v[2].y, T()),
                                              pack2(v[3].x, v[3].y, T()));
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  Raw8<T> raw;
  raw.load(p);
  raw.values(v);
}

// Eight values of a row from column c on, as they lie in memory; those past the row's end as zeros. kVec: rows start on 16-byte
// boundaries, else the values may lie `step` apart.
template <typename T, bool kVec>
__device__ __forceinline__ void load_piece(const T* row, int c, int cols, Raw8<T>& v, int step = 1) {
  if (kVec && c + 8 <= cols) {
    v.load(row + c);
  } else {
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = c + j * step < cols ? row[c + j * step] : T(0.f);
    v.set(e);
  }
}

// Eight values to a row from column c on, as far as the row goes. kWhole: rows of whole pieces on 16-byte boundaries, else the values
// may go `step` apart.
template <typename T, bool kWhole>
__device__ __forceinline__ void store_piece(T* row, int c, int cols, const float2 (&v)[4], int step = 1) {
  if constexpr (kWhole) {
    store8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j * step < cols) row[c + j * step] = from_f32<T>(j & 1 ? v[j / 2].y : v[j / 2].x);
  }
}

// ---- 8-bit blocks. Of a block with largest magnitude top: scale = max(top / largest 8-bit value, 2^-126), values
// x * (1 / scale), reciprocal and product rounded to fp32, then to nearest even. The lower bound keeps 1 / scale finite, also for a block of
// zeros. Magnitudes are compared as integers, in which a NaN is the largest: it makes the block's scale, and with it every value of the block,
// a NaN.

// The larger magnitude of three values, a NaN if one of them is.
__device__ __forceinline__ float abs_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
__device__ __forceinline__ uint32_t abs_max(const float2 (&v)[4]) {
  const float m = abs_max3(abs_max3(v[0].x, v[0].y, v[1].x), abs_max3(v[1].y, v[2].x, v[2].y), abs_max3(v[3].x, v[3].y, v[3].y));
  return __float_as_uint(m) & 0x7fffffffu;
}
template <bool kE5M2>
__device__ __forceinline__ float block_scale(uint32_t top) {
  const float s = __uint_as_float(top) / (kE5M2 ? 57344.f : 448.f);
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;  // (a NaN stays one)
}
// Two values as 8-bit ones, `lo` in the low byte; what lies past the largest (by the rounding of 1 / scale) becomes it.
template <bool kE5M2>
__device__ __forceinline__ uint32_t pack_fp8(float lo, float hi) {
  uint16_t r;
  if constexpr (kE5M2) {
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  }
  return r;
}
template <bool kE5M2>
__device__ __forceinline__ uint2 quantize8(const float2 (&v)[4], float inv) {
  float2 y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = __fmul2_rn(v[j], make_float2(inv, inv));
  uint2 q;
  q.x = pack_fp8<kE5M2>(y[0].x, y[0].y) | pack_fp8<kE5M2>(y[1].x, y[1].y) << 16;
  q.y = pack_fp8<kE5M2>(y[2].x, y[2].y) | pack_fp8<kE5M2>(y[3].x, y[3].y) << 16;
  return q;
}
template <bool kE5M2>
__device__ __forceinline__ uint8_t quantize1(float v, float inv) {
  return static_cast<uint8_t>(pack_fp8<kE5M2>(v * inv, 0.f));
}

// ------------------------------------------------------------------------------------------------ host side
inline int fail(int code, const std::string& msg) { return kcg_internal_fail(code, msg.c_str()); }
// The error also leaves the runtime, which would give it to the next call that asks how its launch went.
inline int cuda_fail(cudaError_t e, const char* what) {
  cudaGetLastError();
  return fail(static_cast<int>(e), std::string(what) + ": " + cudaGetErrorString(e));
}
inline bool known_dtype(int dt) { return dt == KCG_DTYPE_FLOAT32 || dt == KCG_DTYPE_FLOAT16 || dt == KCG_DTYPE_BFLOAT16; }

// Rows or columns of an 8-bit matrix: rounding them up to tiles stays within 32 bits.
constexpr int kMaxSize = 0x7fffff00;

// Makes a device current, and the caller's again when it goes.
struct DeviceGuard {
  int prev = -1;
  bool switched = false;
  cudaError_t enter(int device) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e != cudaSuccess || prev == device) return e;
    e = cudaSetDevice(device);
    switched = e == cudaSuccess;
    return e;
  }
  ~DeviceGuard() {
    if (switched) cudaSetDevice(prev);
  }
};

// KCG_PDL=0 turns programmatic dependent launch off (read once, at the first launch of the process).
inline bool pdl_on() {
  static const bool on = [] {
    const char* e = getenv("KCG_PDL");
    return !(e && e[0] == '0');
  }();
  return on;
}

inline int sm_count(int device, int* out) {
  static std::atomic<int> known[64];
  if (device < 0 || device >= 64) return fail(KCG_E_BAD_ARG, "device index out of range");
  int n = known[device].load();
  if (n == 0) {
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute(MultiProcessorCount)");
    known[device].store(n);
  }
  *out = n;
  return 0;
}

// One launch, allowed to set itself up while the kernel before it in the stream drains (the kernels wait for it before their first
// access to memory).
struct Launch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  explicit Launch(cudaStream_t st) {
    cfg.stream = st;
    cfg.attrs = attr;
    if (pdl_on()) {
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.numAttrs = 1;
    }
  }
  void shape(unsigned grid, unsigned threads, size_t smem = 0, unsigned cluster = 1) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    if (cluster > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = cluster;
      attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
  }
  template <typename K, typename... A>
  int operator()(K kernel, const char* what, const A&... args) {
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return cuda_fail(e, what);
    kcg_internal_count_launch();
    return 0;
  }
};

}  // namespace kcg8
