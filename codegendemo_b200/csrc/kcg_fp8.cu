// Product of 8-bit matrices with a scale for each block of 128 values along K:
//     C[m, n] = sum over blocks kb of  sa[m, kb] * sb[n, kb] * sum over k in kb of a[m, k] * b[n, k],
// a and b in e4m3 or e5m2 (each its own), rows of K values; sa a scale per row and block; sb one per 128 rows and block (a weight's
// 128 x 128 blocks) or per row and block (both operands of a weight's gradient). fp32 accumulation, then beta * C + bias, ReLU, one
// rounding to bf16, fp16 or fp32.
//
// The scales change with every 128 values of K, so the tensor core sums 128 values only (kind::f8f6f4, four instructions of 32),
// into one of several accumulators in tensor memory; while it fills the next, warps read that one and add it to fp32 registers, times
// its scales.
//
// Error against the same sums in 64 bits, fp32 results, 4096 x 4096 x 8192: 1.5e-7 of the norm.
//
// Two kernels. Fp8Tile: one CTA a tile of 128 rows by kBN columns, K split over the CTAs of a cluster, which add their tiles through
// distributed shared memory (in the order of their ranks). With few tokens the weight's rows are the tile's rows and the tokens its
// columns, 16 to 64 of them, so that a tile streams weights and little else. Fp8Pair: CTA pairs, 256 x 256 tiles, persistent.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/kcg_b200.h"
#include "fp8_common.cuh"
#include "kernels/ptx_sm100.cuh"
#include "kernels/store_blocks.h"

namespace {

using namespace kcg;
using namespace kcg8;

__device__ unsigned int g_fp8_status[4];  // {code, block, detail, detail}; 0 = no wait ran out
enum : uint32_t { FP8_TIMEOUT_PRODUCER = 1, FP8_TIMEOUT_MMA = 2, FP8_TIMEOUT_ACCUMULATE = 3 };

// D[tmem] (+)= A[smem] * B[smem], 8-bit operands; issued by ONE thread (of the leader CTA, kCtas = 2).
template <int kCtas>
__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
#define KCG_UMMA_FP8(group)                                                                \
  asm volatile(                                                                            \
      "{\n\t"                                                                              \
      ".reg .pred p;\n\t"                                                                  \
      "setp.ne.b32 p, %4, 0;\n\t"                                                          \
      "tcgen05.mma.cta_group::" group ".kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"             \
      "}\n"                                                                                \
      :                                                                                    \
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)                   \
      : "memory")
  if constexpr (kCtas == 2) {
    KCG_UMMA_FP8("2");
  } else {
    KCG_UMMA_FP8("1");
  }
#undef KCG_UMMA_FP8
}

// TMEM -> registers: 16 consecutive columns of this thread's lane
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// The same tensor memory spread as the products of mma.sync are: of 16 lanes (rows) and 8 columns a group, register 4 g + 2 h + e of a
// thread holds row 8 h + lane / 4, column 8 g + 2 (lane % 4) + e.
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// The registers of the warps of a warpgroup, all of which come here.
template <int kRegs>
__device__ __forceinline__ void set_max_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void set_max_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
// Ties the registers of an earlier load to the wait before it: no use of them may be scheduled ahead of this.
template <int kN>
__device__ __forceinline__ void pin(uint32_t (&r)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+r"(r[i]));
}

// Completion of the pair's products issued so far -> one arrival on this barrier of both CTAs.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

struct Fp8Params {
  CUtensorMap tmP, tmQ;  // {K, rows}: the operand whose rows are the tile's rows, and the one whose rows are its columns
  CUtensorMap tmC;       // Fp8Pair, tma_store: {N, M}, blocks of 128 bytes x 32 rows
  const float *sp, *sq;  // scale of row i at block kb: s[(i >> shift) * ld + kb]
  long long ldsp, ldsq;
  int sp_shift, sq_shift;
  int rows_p, rows_q, num_kb;
  uint32_t fmt_p, fmt_q;  // 0 = e4m3, 1 = e5m2
  void* C;
  long long ldc;
  const void* bias;
  float beta;
  int relu;
  int fused;  // any of the three
  int vector_store, word_store;  // rows of C start on 16-byte boundaries, on 4-byte ones
  int tma_store;                 // and end on 16-byte ones: a TMA store writes 16 bytes or none
  int vector_sp, vector_sq;  // so do those of the scales
  int splits;        // Fp8Tile: CTAs that share a tile's K
};

// The product of two scales, of which only the result of the sum decides whether it is out of range: no 0 * infinity.
__device__ __forceinline__ float scale_product(float a, float b) {
  const float f = a * b;
  return f == INFINITY && a != INFINITY && b != INFINITY ? FLT_MAX : f;
}

// acc[i] += part[i] * f, for kN columns whose scale is the same.
template <int kN>
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&part)[kN], float f) {
#pragma unroll
  for (int i = 0; i < kN; i += 2) {
    const float2 y = __ffma2_rn(make_float2(__uint_as_float(part[i]), __uint_as_float(part[i + 1])), make_float2(f, f),
                                make_float2(acc[i], acc[i + 1]));
    acc[i] = y.x, acc[i + 1] = y.y;
  }
}
// acc[i] += part[i] * scale[i] * f, scales of the columns in shared memory. The part times its column's scale has to stay in the range of
// fp32: parts reach 57344^2 x 128 < 2^39, so scales 2^88. (The two scales multiplied first have no such bound, but 4096 x 4096 x 4096 with a
// scale for each row of b took 106 us in place of 100, and clamped against 0 x infinity 132.)
template <int kN>
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&part)[kN], const float* scale, float f) {
#pragma unroll
  for (int i = 0; i < kN; i += 4) {
    const float4 s = *reinterpret_cast<const float4*>(scale + i);
    const float2 t0 = __fmul2_rn(make_float2(__uint_as_float(part[i]), __uint_as_float(part[i + 1])), make_float2(s.x, s.y));
    const float2 t1 = __fmul2_rn(make_float2(__uint_as_float(part[i + 2]), __uint_as_float(part[i + 3])), make_float2(s.z, s.w));
    const float2 y0 = __ffma2_rn(t0, make_float2(f, f), make_float2(acc[i], acc[i + 1]));
    const float2 y1 = __ffma2_rn(t1, make_float2(f, f), make_float2(acc[i + 2], acc[i + 3]));
    acc[i] = y0.x, acc[i + 1] = y0.y, acc[i + 2] = y1.x, acc[i + 3] = y1.y;
  }
}

// A NaN stays one (fmaxf would make it 0).
__device__ __forceinline__ float relu(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}

// One value of C from its sum.
template <typename T>
__device__ __forceinline__ float finish(const Fp8Params& p, float v, const T* c, float bias) {
  if (p.beta != 0.f) v = fmaf(p.beta, to_f32(*c), v);
  v += bias;
  return p.relu ? relu(v) : v;
}
template <typename T>
__device__ __forceinline__ float bias_at(const Fp8Params& p, int n) {
  return p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.f;
}

// Unit u of 16 bytes of values of C.
template <typename T>
__device__ __forceinline__ uint4 unit16(const float* v, int u) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3]));
  } else {
    return make_uint4(pack2(v[8 * u], v[8 * u + 1], T()), pack2(v[8 * u + 2], v[8 * u + 3], T()), pack2(v[8 * u + 4], v[8 * u + 5], T()),
                      pack2(v[8 * u + 6], v[8 * u + 7], T()));
  }
}

// beta * C, bias and ReLU of kN values of row m from column n on, a row a thread, the warp's rows together (a column's bias is in
// one lane: loaded by every thread for every column it took as long as the rest of 777 x 2752 x 1488).
template <typename T, int kN>
__device__ __forceinline__ void finish_row(const Fp8Params& p, float (&v)[kN], int m, int n) {
  if (p.beta != 0.f && m < p.rows_p) {
    const T* c = static_cast<const T*>(p.C) + static_cast<long long>(m) * p.ldc + n;
#pragma unroll
    for (int i = 0; i < kN; i += 8) {
      if (p.vector_store && n + i + 8 <= p.rows_q) {
        float old[8];
        load8(c + i, old);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i + j] = fmaf(p.beta, old[j], v[i + j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n + i + j < p.rows_q) v[i + j] = fmaf(p.beta, to_f32(c[i + j]), v[i + j]);
      }
    }
  }
  if (p.bias) {
    const int lane = threadIdx.x & 31;
    float b[(kN + 31) / 32];
#pragma unroll
    for (int i = 0; i < (kN + 31) / 32; ++i) b[i] = n + i * 32 + lane < p.rows_q ? bias_at<T>(p, n + i * 32 + lane) : 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] += __shfl_sync(0xffffffffu, b[i / 32], i % 32);
  }
  if (p.relu) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = relu(v[i]);
  }
}

// 32 rows of kN values of C wait in a warp's shared memory, kPitch bytes a row (16-byte units of the rows then lie in different banks), and
// go to C row by row. (Written from the registers of a thread a row, single values of an odd N took 60 us instead of 10 at 2049 x 2305 x 304.)
template <typename T, int kN>
struct RowStore {
  static constexpr int kPitch = kN * static_cast<int>(sizeof(T)) + 16, kBytes = 32 * kPitch;
  __device__ static __forceinline__ void put_row(uint8_t* stage, const float* v) {
    uint8_t* to = stage + (threadIdx.x & 31) * kPitch;
#pragma unroll
    for (int u = 0; u < kN * static_cast<int>(sizeof(T)) / 16; ++u) *reinterpret_cast<uint4*>(to + 16 * u) = unit16<T>(v, u);
  }
  // Called by a whole warp; the rows have been put (__syncwarp) and may be overwritten afterwards.
  __device__ static __forceinline__ void copy(const Fp8Params& p, const uint8_t* stage, int row0, int col0) {
    const int lane = threadIdx.x & 31, rows = min(32, p.rows_p - row0), cols = min(kN, p.rows_q - col0);
    T* c = static_cast<T*>(p.C) + static_cast<long long>(row0) * p.ldc + col0;
    __syncwarp();
    constexpr int kEach = 16 / static_cast<int>(sizeof(T)), kUnits = kN / kEach;
    if (p.vector_store && cols % kEach == 0) {
      const int units = cols / kEach;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r = (i * 32 + lane) / kUnits, u = (i * 32 + lane) % kUnits;
        if (r < rows && u < units) reinterpret_cast<uint4*>(c + r * p.ldc)[u] = *reinterpret_cast<const uint4*>(stage + r * kPitch + u * 16);
      }
    } else if (sizeof(T) == 2 && p.word_store) {
      const int words = cols / 2;
#pragma unroll 8
      for (int r = 0; r < rows; ++r) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(stage + r * kPitch);
        uint32_t* to = reinterpret_cast<uint32_t*>(c + r * p.ldc);
        for (int i = lane; i < words; i += 32) to[i] = from[i];
        if ((cols & 1) && lane == 0) c[r * p.ldc + cols - 1] = reinterpret_cast<const T*>(from)[cols - 1];
      }
    } else {
#pragma unroll 8
      for (int r = 0; r < rows; ++r)
        for (int i = lane; i < cols; i += 32) c[r * p.ldc + i] = reinterpret_cast<const T*>(stage + r * kPitch)[i];
    }
    __syncwarp();
  }
};

template <typename Bars>
__device__ __forceinline__ void report(Bars* bars, uint32_t code, uint32_t d0, uint32_t d1) {
  bars->abort_flag = 1u;
  if (atomicCAS(&g_fp8_status[0], 0u, code) == 0u) {
    g_fp8_status[1] = blockIdx.x;
    g_fp8_status[2] = d0;
    g_fp8_status[3] = d1;
  }
}

// kBN: columns of a tile. kVector: each column has a scale of its own, else the tile's columns share one (kBN <= 128).
// kSwap: the tile's rows are columns of C (weights), its columns rows of C (tokens).
// Four accumulators in tensor memory: products, signals and additions of a block take about three times as long as the products alone, with
// two accumulators 128 x 128 tiles took 800 cycles a block.
template <int kBN, bool kVector, bool kSwap, typename T>
struct Fp8Tile {
  // producer, issuer, four accumulating warps, or eight that share the columns: four are busy 800 cycles with 128 of them
  static constexpr int GROUPS = kBN == 128 ? 2 : 1, COLS = kBN / GROUPS;
  static constexpr int NUM_THREADS = 64 + 128 * GROUPS;
  static constexpr int P_BYTES = 128 * 128, STAGE_BYTES = P_BYTES + kBN * 128;
  static constexpr int STAGES = kBN == 16 ? 6 : kBN == 32 ? 5 : kBN == 64 ? 4 : 6;
  static constexpr int CTAS_PER_SM = kBN <= 64 ? 2 : 1;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int BUFS = 4, PIECE = kBN < 32 ? 16 : 32;
  static constexpr uint32_t TMEM_COLS = BUFS * kBN;  // (a power of two; two CTAs an SM: 512 together at most)
  static constexpr int SMEM_BYTES = RING_BYTES + 1024 + 2048;
  static constexpr int PART_BYTES = kBN * 128 * 4;  // a tile in fp32
  static_assert(PART_BYTES + (kSwap ? 0 : 4 * GROUPS * RowStore<T, COLS>::kBytes) <= RING_BYTES, "a tile, and rows to store, are laid over the ring");

  struct Barriers {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t tmem_full[BUFS], tmem_empty[BUFS];
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
    alignas(16) float scale[2][kVector ? kBN : 4];
  };
  static_assert(sizeof(Barriers) <= 2048, "barrier block exceeds its shared-memory slot");

  __device__ static __forceinline__ void load(uint32_t taddr, uint32_t (&r)[PIECE]) {
    if constexpr (PIECE == 16) {
      tmem_ld_32x32b_x16(taddr, r);
    } else {
      tmem_ld_32x32b_x32(taddr, r);
    }
  }

  // kN columns of this thread's row of the tile to C. `stage`: this warp's shared memory.
  template <int kN>
  __device__ static __forceinline__ void store(const Fp8Params& p, float (&v)[kN], int gp, int gq, uint8_t* stage) {
    if constexpr (kSwap) {
      if (gp >= p.rows_p) return;
      const float bias = bias_at<T>(p, gp);
      T* out = static_cast<T*>(p.C) + static_cast<long long>(gq) * p.ldc + gp;
#pragma unroll
      for (int c = 0; c < kN; ++c, out += p.ldc)
        if (gq + c < p.rows_q) *out = from_f32<T>(finish<T>(p, v[c], out, bias));
    } else {
      const int row0 = gp - static_cast<int>(threadIdx.x & 31);
      if (row0 >= p.rows_p || gq >= p.rows_q) return;
      if (p.fused) finish_row<T, kN>(p, v, gp, gq);
      RowStore<T, kN>::put_row(stage, v);
      RowStore<T, kN>::copy(p, stage, row0, gq);
    }
  }

  // The tile from the parts of kS CTAs, in the order of their ranks; this one's share of the columns, this group's share of that.
  template <int kS>
  __device__ static __forceinline__ void join(const Fp8Params& p, const float* part, int rank, int group, int row, int p0, int q0,
                                              uint8_t* stage) {
    constexpr int kPer = kBN / kS / GROUPS, kAtOnce = kPer < 8 ? kPer : 8;
    const int first = (rank * GROUPS + group) * kPer;
    const uint32_t mine = smem_u32(part + first * 128 + row);
    uint32_t from[kS];
#pragma unroll
    for (int r = 0; r < kS; ++r) from[r] = map_to_cta(mine, r);
    float v[kPer];
#pragma unroll
    for (int c0 = 0; c0 < kPer; c0 += kAtOnce) {
      float x[kS][kAtOnce];
#pragma unroll
      for (int r = 0; r < kS; ++r)
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c) x[r][c] = ld_cluster_f32(from[r] + (c0 + c) * 512);
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) {
        v[c0 + c] = x[0][c];
#pragma unroll
        for (int r = 1; r < kS; ++r) v[c0 + c] += x[r][c];
      }
    }
    store<kPer>(p, v, p0 + row, q0 + first, stage);
  }

  __device__ static void run(const Fp8Params& p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    Barriers* bars = reinterpret_cast<Barriers*>(smem + RING_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.splits > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int tile = static_cast<int>(blockIdx.x) / p.splits;
    const int tiles_q = (p.rows_q + kBN - 1) / kBN;
    const int p0 = tile / tiles_q * 128, q0 = tile % tiles_q * kBN;
    // (splits <= num_kb: every CTA has at least one block)
    const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * rank / p.splits);
    const int n = static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / p.splits) - kb0;

    if (threadIdx.x == 0) {
      tma_prefetch_desc(&p.tmP);
      tma_prefetch_desc(&p.tmQ);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&bars->full[s], 1);
        mbar_init(&bars->empty[s], 1);
      }
      for (int b = 0; b < BUFS; ++b) {
        mbar_init(&bars->tmem_full[b], 1);
        mbar_init(&bars->tmem_empty[b], 4 * GROUPS);
      }
      bars->abort_flag = 0u;
      fence_mbar_init();
      fence_proxy_async_smem();
    }
    if (warp == 1) {
      tmem_alloc(&bars->tmem_base, TMEM_COLS);
      tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = bars->tmem_base;
    griddep_wait();

    float acc[COLS];
    // (accumulating warps) TMEM lane quarter, row of the tile, which columns
    const int q = warp & 3, row = q * 32 + lane, group = (warp - 2) >> 2;
    bool ok = true;
    if (warp == 0) {
      if (lane == 0) {
        for (int i = 0; i < n; ++i) {
          const int s = i % STAGES;
          if (!mbar_wait(&bars->empty[s], ((i / STAGES) & 1u) ^ 1u, &bars->abort_flag)) {
            report(bars, FP8_TIMEOUT_PRODUCER, i, s);
            break;
          }
          mbar_expect_tx(&bars->full[s], STAGE_BYTES);
          tma_load_2d(smem + s * STAGE_BYTES, &p.tmP, &bars->full[s], (kb0 + i) * 128, p0);
          tma_load_2d(smem + s * STAGE_BYTES + P_BYTES, &p.tmQ, &bars->full[s], (kb0 + i) * 128, q0);
        }
      }
      __syncwarp();
      griddep_launch_dependents();
    } else if (warp == 1) {
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint64_t pdesc = make_smem_desc(smem_u32(smem), 16, 1024, SWZ_128B);
      const uint64_t qdesc = make_smem_desc(smem_u32(smem) + P_BYTES, 16, 1024, SWZ_128B);
      const uint32_t idesc = make_instr_desc(0u, 0u, 0u, 128u, kBN) | p.fmt_p << 7 | p.fmt_q << 10;
      for (int i = 0; i < n; ++i) {
        const uint32_t s = i % STAGES, b = i % BUFS;
        if (!mbar_wait_warp(&bars->full[s], (i / STAGES) & 1u, &bars->abort_flag) ||
            !mbar_wait_warp(&bars->tmem_empty[b], ((i / BUFS) & 1u) ^ 1u, &bars->abort_flag)) {
          if (lane == 0) report(bars, FP8_TIMEOUT_MMA, i, s);
          break;
        }
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)  // 32 values = 32 bytes of a row
            umma_fp8<1>(tmem + b * kBN, pdesc + s * (STAGE_BYTES >> 4) + ks * 2, qdesc + s * (STAGE_BYTES >> 4) + ks * 2, idesc,
                        ks > 0 ? 1u : 0u);
          umma_commit(&bars->tmem_full[b]);
          umma_commit(&bars->empty[s]);
        }
        __syncwarp();
      }
    } else {
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
      const int t = group * COLS + (threadIdx.x - 64) % 128;  // column whose scale this thread fetches
      const float* sp = p.sp + (static_cast<long long>(min(p0 + row, p.rows_p - 1)) >> p.sp_shift) * p.ldsp + kb0;
      const float* sq = p.sq + (static_cast<long long>(min(q0 + (kVector ? t : 0), p.rows_q - 1)) >> p.sq_shift) * p.ldsq + kb0;
      const bool fetches = !kVector || (threadIdx.x - 64) % 128 < COLS;
      // the scales of four blocks at a time, four blocks ahead (by ordinary loads: the kernel before this one may have written them while
      // this one was there already, so they are not read-only for its whole life, as the non-coherent path asks)
      float next_p[4], next_q[4];
      auto fetch = [&](int i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          next_p[j] = i + j < n ? sp[i + j] : 0.f;
          next_q[j] = fetches && i + j < n ? sq[i + j] : 0.f;
        }
      };
      fetch(0);
      for (int i0 = 0; i0 < n; i0 += 4) {
        float f[4], g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = next_p[j], g[j] = next_q[j];
        if (i0 + 4 < n) fetch(i0 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j;
          if (i >= n) break;
          if constexpr (kVector) {
            // (two buffers: a thread that writes one again has passed the meeting behind which all have read it)
            if (fetches) bars->scale[j & 1][t] = g[j];
            named_bar_sync(1 + group, 128);
          }
          if (ok) {
            const bool got = mbar_wait(&bars->tmem_full[j], (i0 / 4) & 1u, &bars->abort_flag);
            if (!__all_sync(0xffffffffu, got)) {
              if (lane == 0) report(bars, FP8_TIMEOUT_ACCUMULATE, i, j);
              ok = false;
            }
          }
          if (!ok) continue;  // (the meetings go on)
          tc_fence_after_sync();
          const uint32_t col = tmem_base + j * kBN + group * COLS + (static_cast<uint32_t>(q * 32) << 16);
          const float* scale = &bars->scale[j & 1][kVector ? group * COLS : 0];
          const float factor = kVector ? f[j] : scale_product(f[j], g[j]);
          uint32_t r[2][PIECE];
          load(col, r[0]);
#pragma unroll
          for (int c = 0; c < COLS / PIECE; ++c) {
            tmem_ld_wait();
            pin(r[c & 1]);
            if (c + 1 < COLS / PIECE) {
              load(col + (c + 1) * PIECE, r[(c + 1) & 1]);
            } else {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars->tmem_empty[j]);
            }
            if constexpr (kVector) {
              add_scaled<PIECE>(acc + c * PIECE, r[c & 1], scale + c * PIECE, factor);
            } else {
              add_scaled<PIECE>(acc + c * PIECE, r[c & 1], factor);
            }
          }
        }
      }
    }

    // Every product has been read, so the ring is idle (the accumulating warps' shared memory lies behind a tile's).
    uint8_t* stage = smem + (kSwap ? 0 : PART_BYTES + (warp >= 2 ? warp - 2 : 0) * RowStore<T, COLS>::kBytes);
    if (p.splits > 1) {
      // the CTA's tile, column after column of 128 rows
      float* part = reinterpret_cast<float*>(smem);
      if (warp >= 2 && ok) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) part[(group * COLS + c) * 128 + row] = acc[c];
      }
      __syncwarp();
      cluster_sync_all();
      if (warp >= 2 && ok) {
        if (p.splits == 2) {
          join<2>(p, part, rank, group, row, p0, q0, stage);
        } else if (p.splits == 4) {
          join<4>(p, part, rank, group, row, p0, q0, stage);
        } else if constexpr (kSwap) {
          join<8>(p, part, rank, group, row, p0, q0, stage);
        }
      }
      __syncwarp();
      cluster_sync_all();  // shared memory stays until the others have read it
    } else if (warp >= 2 && ok) {
      store<COLS>(p, acc, p0 + row, q0 + group * COLS, stage);
    }

    // ---------------------------------------------------------------- common exit
    __syncwarp();
    if (bars->abort_flag != 0u) {
      // give loads / products still in flight time to land before shared memory and TMEM are released
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after_sync();
      tmem_dealloc(tmem_base, TMEM_COLS);
    }
  }
};

template <int kBN, bool kVector, bool kSwap, typename T>
__global__ void __launch_bounds__(Fp8Tile<kBN, kVector, kSwap, T>::NUM_THREADS, Fp8Tile<kBN, kVector, kSwap, T>::CTAS_PER_SM)
fp8_tile_kernel(const __grid_constant__ Fp8Params p) {
  Fp8Tile<kBN, kVector, kSwap, T>::run(p);
}

// CTA pairs, tiles of 256 x 256, one after another. Each CTA holds 128 rows of A and 128 of B a stage. Twelve warps: warp 0 waits in the
// accumulating warps' place, warp 1 of the leader issues the products, warp 2 loads the operands, warp 3 brings the scales of four
// blocks of K at a time into shared memory, warps 4-7 accumulate the first 128 columns and warps 8-11 the others.
//
// A block of K takes 512 cycles of the tensor pipe, and its accumulator has to be read, and the leader's issuer to hear of it from both
// CTAs, while the other fills. The products' operands and TMA fill the shared-memory port, where an access then takes
// hundreds of cycles, so the accumulating warps look at no mbarrier and have registers enough: warp 0 looks, and tells each half's four
// warps on a named barrier. (With mbarriers of their own a block took 1070 cycles, with a few spilled registers 1300.) The halves do not
// meet: one adds while the other waits for tensor memory, and the next 32 columns are asked for while these are added, for which the
// first four warps give up registers. 4096 x 4096 x 4096, all warps on one barrier and 32 columns at a time in 168 registers 71.2 us, the next 32 columns
// ahead in 224 65.8, a barrier a half 65.6; kVector, with its own 16 columns ahead in both, 99.8, 100.4, 94.9. (Barriers of two warps each
// are no faster.)
//
// Where the columns of a half share a scale, a thread accumulates one row of 128 columns, times one factor. Where each has its own
// (kVector), a thread takes two neighbouring columns of each eight of four rows, as tcgen05.ld.16x256b gives them: 32 scales
// of columns and four of rows, where a row a thread would take 128 from shared memory, 16 bytes a lane, which alone is 1024
// cycles of its port a block of K against 512 of the tensor pipe.
template <bool kVector, typename T>
struct Fp8Pair {
  static constexpr int NUM_THREADS = 384, kBM = 256, kBN = 256;
  // Registers: 168 a thread at launch, of which the first four warps give up what the accumulating ones take.
  static constexpr int LAUNCH_REGS = 168, FEW_REGS = 56, MANY_REGS = 224;
  static_assert(128 * FEW_REGS + 256 * MANY_REGS <= NUM_THREADS * LAUNCH_REGS, "the shares exceed what the CTA was launched with");
  static constexpr int HALF_BYTES = 128 * 128, STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int STAGES = 4;  // (three are as fast)
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int STORE_BYTES = 8 * 2 * 32 * 128;  // two blocks of 32 rows of 128 bytes for each accumulating warp
  static constexpr int SCALES = 128 + (kVector ? 256 : 4);  // of a block of K: the CTA's rows, the tile's columns (or halves)
  static constexpr int GROUP_KB = 4;                        // blocks of K whose scales come together
  // Groups in shared memory: one that the later half may still read, the next, and the one after it on its way.
  static constexpr int GROUPS = 3;
  static constexpr int SCALE_BYTES = GROUPS * GROUP_KB * SCALES * 4;
  static constexpr int SMEM_BYTES = RING_BYTES + STORE_BYTES + SCALE_BYTES + 1024 + 512;
  static constexpr int GROUP = 8;  // tile rows that are walked together, column after column
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr int COLS_BLOCK = 128 / static_cast<int>(sizeof(T));  // columns of a store

  struct Barriers {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t tmem_full[2], tmem_empty[2];
    uint64_t scale_full[GROUPS], scale_empty[GROUPS];
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
  };
  static_assert(sizeof(Barriers) <= 512, "barrier block exceeds its shared-memory slot");

  // Named barriers. At BAR_FULL warp 0 and the accumulating warps meet once: the first scales are there. At BAR_HALF + 2 half + (block & 1)
  // warp 0 arrives, without waiting, and the half's warps wait: the block's accumulator is complete, its scales and the next block's
  // are in shared memory. Warp 0 comes back to a barrier only when the accumulator of two blocks later is complete, for which all have left
  // it. Where a wait of warp 0 ran out, it does meet the halves in every block left, so that all of them end; they store nothing.
  static constexpr uint32_t BAR_HALF = 2, BAR_FULL = 1, MEETING = 32 + 256;

  // Rows and columns of C at which tile i starts.
  __device__ static __forceinline__ void tile_at(int i, int tiles_m, int tiles_n, int& m0, int& n0) {
    const int per_group = GROUP * tiles_n, group = i / per_group, first = group * GROUP;
    const int rows = min(GROUP, tiles_m - first), in = i - group * per_group;
    m0 = (first + in % rows) * kBM;
    n0 = in / rows * kBN;
  }

  // The scales of GROUP_KB blocks of K from block kb on, those of 32 kRows rows from `row` on: four of a row a lane, all rows under way at
  // once, to slot[i] of each block's place. (Ordinary loads, as in Fp8Tile.)
  template <int kRows>
  __device__ static __forceinline__ void bring(const float* s, long long ld, int shift, int row, int rows, int kb, int num_kb, bool vec,
                                               float* slot) {
    const int lane = threadIdx.x & 31, left = num_kb - kb;  // (those past the last block are not used)
    float4 v[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float* at = s + (static_cast<long long>(min(row + i * 32 + lane, rows - 1)) >> shift) * ld + kb;
      v[i] = vec && left >= 4 ? *reinterpret_cast<const float4*>(at)
                              : make_float4(at[0], left > 1 ? at[1] : 0.f, left > 2 ? at[2] : 0.f, left > 3 ? at[3] : 0.f);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float* to = slot + i * 32 + lane;
      to[0] = v[i].x, to[SCALES] = v[i].y, to[2 * SCALES] = v[i].z, to[3 * SCALES] = v[i].w;
    }
  }

  // This warp's accumulators to C: 32 rows of 128 columns, through blocks of shared memory: 16-byte units XORed with the row, the
  // swizzle of the tensor map, and TMA stores, two under way; or rows by RowStore where TMA cannot address them or would write past
  // their ends (8192 x 4095 x 4096 into rows of 4096 130 us; only the last columns of such rows by RowStore 126, which cost 8192 x 8192 x 128 with
  // no such rows 29.5 for 28.5).
  __device__ static __forceinline__ void store(const Fp8Params& p, float (&acc)[128], int row0, int col0, uint8_t* blocks) {
    using Rows = RowStore<T, COLS_BLOCK>;
    static_assert(Rows::kBytes <= 8192, "a block of rows exceeds a warp's shared memory");
    const int lane = threadIdx.x & 31;
    if (p.fused) {
      if constexpr (!kVector) {
        finish_row<T, 128>(p, acc, row0 + lane, col0);
      } else {
        // tcgen05.ld.16x256b's layout: pairs of columns, four rows
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int n = col0 + j * 8 + (lane & 3) * 2;
          float bias[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) bias[e] = n + e < p.rows_q ? bias_at<T>(p, n + e) : 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = row0 + r * 8 + (lane >> 2);
            const T* c = static_cast<const T*>(p.C) + static_cast<long long>(m) * p.ldc + n;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (m < p.rows_p && n + e < p.rows_q) acc[j * 8 + r * 2 + e] = finish<T>(p, acc[j * 8 + r * 2 + e], c + e, bias[e]);
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < 128 / COLS_BLOCK; ++b) {
      if (row0 >= p.rows_p || col0 + b * COLS_BLOCK >= p.rows_q) break;
      uint8_t* block = blocks + (p.tma_store ? store_block(b) * 4096 : 0);
      if (p.tma_store) {
        if (lane == 0) {
          if (stores_reading(b) == 0) {
            tma_store_wait_read<0>();
          } else {
            static_assert(stores_reading(1) == 1, "the wait below leaves one store reading");
            tma_store_wait_read<1>();
          }
        }
        __syncwarp();
      }
      if constexpr (!kVector) {
        const float* v = acc + b * COLS_BLOCK;
        if (p.tma_store) {
#pragma unroll
          for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(block + lane * 128 + ((u ^ (lane & 7)) << 4)) = unit16<T>(v, u);
        } else {
          Rows::put_row(block, v);
        }
      } else {
        const uint32_t x = lane >> 2, t = lane & 3;  // (row within eight, pair of columns within eight)
        const uint32_t swizzle = !p.tma_store ? 0u : (sizeof(T) == 4 ? x ^ (t >> 1) : x) << 4, pitch = p.tma_store ? 128 : Rows::kPitch;
        uint8_t* to = block + x * pitch + (sizeof(T) == 4 ? (t & 1) * 8 + (p.tma_store ? 0 : (t >> 1) * 16) : t * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r, to += 8 * pitch)
#pragma unroll
          for (int j = 0; j < COLS_BLOCK / 8; ++j) {
            const float* v = acc + (b * (COLS_BLOCK / 8) + j) * 8 + r * 2;
            uint8_t* at = to + ((j * (sizeof(T) == 4 ? 32 : 16)) ^ swizzle);
            if constexpr (sizeof(T) == 4) {
              *reinterpret_cast<float2*>(at) = make_float2(v[0], v[1]);
            } else {
              *reinterpret_cast<uint32_t*>(at) = pack2(v[0], v[1], T());
            }
          }
      }
      if (p.tma_store) {
        send(p, block, row0, col0 + b * COLS_BLOCK);
      } else {
        Rows::copy(p, block, row0, col0 + b * COLS_BLOCK);
      }
    }
  }
  __device__ static __forceinline__ void send(const Fp8Params& p, uint8_t* block, int row, int col) {
    fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      tma_store_2d(&p.tmC, block, col, row);
      tma_store_commit();
    }
  }

  __device__ static void run(const Fp8Params& p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* scales = reinterpret_cast<float*>(smem + RING_BYTES + STORE_BYTES);
    Barriers* bars = reinterpret_cast<Barriers*>(smem + RING_BYTES + STORE_BYTES + SCALE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();  // 0 = leader
    const int tiles_m = (p.rows_p + kBM - 1) / kBM, tiles_n = (p.rows_q + kBN - 1) / kBN, tiles = tiles_m * tiles_n;
    const int tile0 = static_cast<int>(blockIdx.x >> 1), stride = static_cast<int>(gridDim.x >> 1);

    if (threadIdx.x == 0) {
      tma_prefetch_desc(&p.tmP);
      tma_prefetch_desc(&p.tmQ);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&bars->full[s], 1);
        mbar_init(&bars->empty[s], 1);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->tmem_full[b], 1);
        mbar_init(&bars->tmem_empty[b], 16);  // one arrival for each accumulating warp of both CTAs
      }
      for (int g = 0; g < GROUPS; ++g) {
        mbar_init(&bars->scale_full[g], 32);
        mbar_init(&bars->scale_empty[g], 8);
      }
      bars->abort_flag = 0u;
      fence_mbar_init();
      fence_proxy_async_smem();
    }
    if (warp == 1) {
      tmem_alloc_pair(&bars->tmem_base, TMEM_COLS);
      tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // the peer's barriers exist before anyone signals them
    tc_fence_after_sync();
    const uint32_t tmem_base = bars->tmem_base;
    griddep_wait();

    if (warp >= 4) {
      set_max_registers_up<MANY_REGS>();
      const int q = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quarter of this warp, half of the tile's columns
      uint8_t* block = smem + RING_BYTES + (warp - 4) * 8192;
      // The scales of a block's rows (and of its half's columns, where they share one) are read when the block before has been added:
      // read before its additions they cost a third of the speed.
      const float* row_scales = scales + q * 32 + (kVector ? lane >> 2 : lane);
      const float* column_scales = scales + 128 + half * (kVector ? 128 : 1) + (kVector ? (lane & 3) * 2 : 0);
      const uint32_t empty_leader = map_to_cta(smem_u32(&bars->tmem_empty[0]), 0u);
      constexpr int kF = kVector ? 4 : 2;
      float f[kF];
      uint32_t at = 0, group_at = 0, it = 0;  // where the block's scales lie, and its group's
      auto fetch = [&]() {
        if constexpr (kVector) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = row_scales[at + i * 8];
        } else {
          f[0] = row_scales[at];
          f[1] = column_scales[at];
        }
      };
      named_bar_sync(BAR_FULL, MEETING);
      fetch();
      for (int tile = tile0; tile < tiles; tile += stride) {
        float acc[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] = 0.f;
        for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
          const uint32_t col = tmem_base + (it & 1u) * kBN + half * 128 + (static_cast<uint32_t>(q * 32) << 16);
          named_bar_sync(BAR_HALF + half * 2 + (it & 1u), 160);
          tc_fence_after_sync();
          auto release = [&]() {  // (the reads are complete)
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_cta(empty_leader + (it & 1u) * 8);
          };
          if constexpr (!kVector) {
            const float factor = scale_product(f[0], f[1]);
            uint32_t r[2][32];
            tmem_ld_32x32b_x32(col, r[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_ld_wait();
              pin(r[c & 1]);
              if (c < 3) {
                tmem_ld_32x32b_x32(col + (c + 1) * 32, r[(c + 1) & 1]);
              } else {
                release();
              }
              add_scaled<32>(acc + c * 32, r[c & 1], factor);
            }
          } else {
            uint32_t r[2][2][8];
            float2 s[2][2];
            auto load = [&](int c) {
              tmem_ld_16x256b_x2(col + c * 16, r[c & 1][0]);
              tmem_ld_16x256b_x2(col + c * 16 + (16u << 16), r[c & 1][1]);
#pragma unroll
              for (int j = 0; j < 2; ++j) s[c & 1][j] = *reinterpret_cast<const float2*>(column_scales + at + c * 16 + j * 8);
            };
            load(0);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              tmem_ld_wait();
              pin(r[c & 1][0]);
              pin(r[c & 1][1]);
              if (c < 7) {
                load(c + 1);
              } else {
                release();
              }
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // rows i * 8 + lane / 4
                  const uint32_t* part = &r[c & 1][i >> 1][j * 4 + (i & 1) * 2];
                  float* a = acc + (c * 2 + j) * 8 + i * 2;
                  const float2 y = __ffma2_rn(__fmul2_rn(make_float2(__uint_as_float(part[0]), __uint_as_float(part[1])), s[c & 1][j]),
                                              make_float2(f[i], f[i]), make_float2(a[0], a[1]));
                  a[0] = y.x, a[1] = y.y;
                }
            }
          }
          // the next block's place: the next of the group, or the first of the next group
          if (kb % GROUP_KB == GROUP_KB - 1 || kb == p.num_kb - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->scale_empty[group_at / (GROUP_KB * SCALES)]);
            group_at = group_at == (GROUPS - 1) * GROUP_KB * SCALES ? 0u : group_at + GROUP_KB * SCALES;
            at = group_at;
          } else {
            at += SCALES;
          }
          fetch();
        }
        if (bars->abort_flag != 0u) continue;
        int m0, n0;
        tile_at(tile, tiles_m, tiles_n, m0, n0);
        store(p, acc, m0 + static_cast<int>(rank) * 128 + q * 32, n0 + half * 128, block);
      }
      if (lane == 0) tma_store_wait_read<0>();  // shared memory outlives the stores' reads
      __syncwarp();
    } else {
      set_max_registers_down<FEW_REGS>();
      if (warp == 0) {
        // ------------------------------------------------ waits in the accumulating warps' place
        uint32_t it = 0, g = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t what) {
          if (!ok || mbar_wait_warp(bar, parity, &bars->abort_flag)) return;
          ok = false;
          if (lane == 0) report(bars, FP8_TIMEOUT_ACCUMULATE, it, what);
          for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // the halves leave the barriers at which this warp has arrived
        };
        wait(&bars->scale_full[0], 0u, 2u);
        named_bar_sync(BAR_FULL, MEETING);  // the first block's scales
        for (int tile = tile0; tile < tiles; tile += stride) {
          for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
            if (kb == p.num_kb - 1 ? tile + stride < tiles : kb % GROUP_KB == GROUP_KB - 1) {
              ++g;
              wait(&bars->scale_full[g % GROUPS], (g / GROUPS) & 1u, 2u);
            }
            wait(&bars->tmem_full[it & 1u], (it >> 1) & 1u, 0u);
            tc_fence_after_sync();
            tc_fence_before_sync();
            if (ok) {
              named_bar_arrive(BAR_HALF + (it & 1u), 160);
              named_bar_arrive(BAR_HALF + 2 + (it & 1u), 160);
            } else {
              named_bar_sync(BAR_HALF + (it & 1u), 160);
              named_bar_sync(BAR_HALF + 2 + (it & 1u), 160);
            }
          }
        }
      } else if (warp == 1) {
        if (rank == 0u) {
          const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
          const uint64_t adesc = make_smem_desc(smem_u32(smem), 16, 1024, SWZ_128B);
          const uint64_t bdesc = make_smem_desc(smem_u32(smem) + HALF_BYTES, 16, 1024, SWZ_128B);
          const uint32_t idesc = make_instr_desc(0u, 0u, 0u, 256u, kBN) | p.fmt_p << 7 | p.fmt_q << 10;
          uint32_t it = 0;
          bool ok = true;
          for (int tile = tile0; tile < tiles && ok; tile += stride) {
            for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
              const uint32_t s = it % STAGES, b = it & 1u;
              // (the operands have mostly been there for long: what is waited for is the accumulator)
              if (!mbar_wait_warp(&bars->full[s], (it / STAGES) & 1u, &bars->abort_flag) ||
                  !mbar_wait_warp(&bars->tmem_empty[b], ((it >> 1) & 1u) ^ 1u, &bars->abort_flag)) {
                if (lane == 0) report(bars, FP8_TIMEOUT_MMA, it, s);
                ok = false;
                break;
              }
              tc_fence_after_sync();
              if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                  umma_fp8<2>(tmem + b * kBN, adesc + s * (STAGE_BYTES >> 4) + ks * 2, bdesc + s * (STAGE_BYTES >> 4) + ks * 2, idesc,
                              ks > 0 ? 1u : 0u);
                umma_commit_both(&bars->tmem_full[b]);
                umma_commit_both(&bars->empty[s]);
              }
              __syncwarp();
            }
          }
        }
      } else if (warp == 2) {
        // ------------------------------------------------ operands
        uint32_t it = 0;
        bool ok = true;
        for (int tile = tile0; tile < tiles && ok; tile += stride) {
          int m0, n0;
          tile_at(tile, tiles_m, tiles_n, m0, n0);
          m0 += static_cast<int>(rank) * 128, n0 += static_cast<int>(rank) * 128;
          for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
            const uint32_t s = it % STAGES;
            ok = mbar_wait_warp(&bars->empty[s], ((it / STAGES) & 1u) ^ 1u, &bars->abort_flag);
            if (!ok) {
              if (lane == 0) report(bars, FP8_TIMEOUT_PRODUCER, it, s);
              break;
            }
            if (lane == 0) {
              // completion bytes of both CTAs land on the leader's barrier
              const uint32_t full_leader = map_to_cta(smem_u32(&bars->full[s]), 0u);
              if (rank == 0u) mbar_expect_tx(&bars->full[s], 2 * STAGE_BYTES);
              tma_load_2d_pair(smem + s * STAGE_BYTES, &p.tmP, full_leader, kb * 128, m0);
              tma_load_2d_pair(smem + s * STAGE_BYTES + HALF_BYTES, &p.tmQ, full_leader, kb * 128, n0);
            }
            __syncwarp();
          }
        }
        griddep_launch_dependents();
      } else {
        // ------------------------------------------------ scales, GROUP_KB blocks at a time, as soon as a group's place is free
        uint32_t g = 0;
        bool ok = true;
        for (int tile = tile0; tile < tiles && ok; tile += stride) {
          int m0, n0;
          tile_at(tile, tiles_m, tiles_n, m0, n0);
          m0 += static_cast<int>(rank) * 128;
          for (int kb = 0; kb < p.num_kb; kb += GROUP_KB, ++g) {
            ok = mbar_wait_warp(&bars->scale_empty[g % GROUPS], ((g / GROUPS) & 1u) ^ 1u, &bars->abort_flag);
            if (!ok) {
              if (lane == 0) report(bars, FP8_TIMEOUT_PRODUCER, g, 100u);
              break;
            }
            float* slot = scales + g % GROUPS * GROUP_KB * SCALES;
            bring<4>(p.sp, p.ldsp, p.sp_shift, m0, p.rows_p, kb, p.num_kb, p.vector_sp, slot);
            if constexpr (kVector) {
#pragma unroll 1
              for (int half = 0; half < 256; half += 128)  // (one after the other: 16 registers)
                bring<4>(p.sq, p.ldsq, p.sq_shift, n0 + half, p.rows_q, kb, p.num_kb, p.vector_sq, slot + 128 + half);
            } else if (lane < 2) {  // (lanes 0 and 1: the tile's two halves)
              bring<1>(p.sq, p.ldsq, 0, n0 >> 7, (p.rows_q + 127) / 128, kb, p.num_kb, p.vector_sq, slot + 128);
            }
            mbar_arrive(&bars->scale_full[g % GROUPS]);
            __syncwarp();
          }
        }
      }
    }

    // ------------------------------------------------------------ common exit
    __syncwarp();
    if (bars->abort_flag != 0u) {
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_before_sync();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();  // the peer's shared memory and TMEM stay valid until both CTAs are done
    if (warp == 1) {
      __syncwarp();
      tc_fence_after_sync();
      tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
  }
};

template <bool kVector, typename T>
__global__ void __launch_bounds__(384, 1) fp8_pair_kernel(const __grid_constant__ Fp8Params p) {
  Fp8Pair<kVector, T>::run(p);
}

// ------------------------------------------------------------------------------------------------ host side
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::mutex g_mutex;
EncodeFn g_encode = nullptr;

int encoder(EncodeFn* out) {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (!g_encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
      return fail(KCG_E_NO_DRIVER, "cuTensorMapEncodeTiled not available from the driver");
    g_encode = reinterpret_cast<EncodeFn>(fn);
  }
  *out = g_encode;
  return 0;
}

// Rows of K bytes, `ld` apart; boxes of 128 bytes x `box_rows` rows. What lies past the matrix reads as zero.
int encode(EncodeFn fn, CUtensorMap* tm, uint64_t ptr, int k, int64_t ld, int rows, int box_rows) {
  cuuint64_t gdim[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t gstride[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, estr[2] = {1, 1};
  const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, reinterpret_cast<void*>(ptr), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(static_cast<int>(r), "cuTensorMapEncodeTiled failed");
}

// C, for stores of 128 bytes x 32 rows; rows past it are not stored, columns past it are where they share 16 bytes with one inside.
int encode_c(EncodeFn fn, CUtensorMap* tm, uint64_t ptr, int dtype, int n, int64_t ld, int m) {
  const int eb = dtype == KCG_DTYPE_FLOAT32 ? 4 : 2;
  cuuint64_t gdim[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(m)};
  cuuint64_t gstride[1] = {static_cast<cuuint64_t>(ld) * eb};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / eb), 32}, estr[2] = {1, 1};
  const CUtensorMapDataType type = dtype == KCG_DTYPE_FLOAT32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == KCG_DTYPE_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = fn(tm, type, 2, reinterpret_cast<void*>(ptr), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(static_cast<int>(r), "cuTensorMapEncodeTiled failed");
}

// Once per device: the kernel may use more than 48 KB of shared memory.
template <typename K>
int opt_in(K kernel, int device, int smem, bool (&ready)[64]) {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (!ready[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
    ready[device] = true;
  }
  return 0;
}

struct Plan {
  int pair;    // Fp8Pair
  int swap;    // Fp8Tile: the weight's rows are the tile's rows
  int bn;      // columns of a tile
  int splits;  // CTAs that share a tile's K
};

// Which kernel takes a product. `vector`: each row of B has scales of its own.
// Up to 32 tokens (64 with `vector`, where 128 weights would be 128 columns with a scale each: 64 x 4096 x 4096 9.8 us against 11.4) the
// weight's rows are the tile's rows, and K is split until a quarter more CTAs run than there are SMs (two fit one): 1 x 4096 x 4096 in 1, 2,
// 4, 8 parts 10.9, 7.6, 5.8, 6.2 us, 1 x 14336 x 4096 13.0, 13.6, 16.5, 22.3.
// More tokens: 128 x 128 tiles, K in up to four parts while all run at once (eight: 200 x 1024 x 8192 17.4 us against 10.9), or pairs, whichever
// takes less time by {fixed, per wave and block of K, per wave, joining 2 and 4 parts}, fitted to 35 shapes of 33 to 8192 tokens x 264 to 11008 x
// 128 to 11008, 6 to 8 % rms, of which it picks one within 3 % of the fastest every time. Tiles of 128 against pairs: 128 x 4096 x 4096 in four
// parts 9.7 / 17.0 us, 512 x 4096 x 11008 33 / 39, 1444 x 1040 x 1760 8.5 / 10.6; 777 x 2752 x 1488 13.8 / 10.6, 512 x 11008 x 4096 43 / 34,
// 1204 x 6600 x 128 13.8 / 8.8.
Plan plan_of(int m, int n, int k, bool vector, int sms) {
  const int num_kb = (k - 1) / 128 + 1;
  Plan plan{0, 0, 128, 1};
  if (m <= (vector ? 64 : 32)) {
    plan.swap = 1;
    plan.bn = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    const long long tiles = (n - 1) / 128 + 1;
    while (plan.splits < 8 && 4 * tiles * 2 * plan.splits <= 5LL * sms && num_kb >= 4 * plan.splits) plan.splits *= 2;
    return plan;
  }
  const double pair_us[3] = {vector ? 3.6 : 3.0, vector ? 0.633 : 0.416, vector ? 1.9 : 1.8};
  const double tile_us[3] = {vector ? -0.4 : -0.6, vector ? 0.602 : 0.365, vector ? 3.2 : 3.4};
  const long long tiles = (static_cast<long long>(m - 1) / 128 + 1) * ((n - 1) / 128 + 1);
  const long long large = (static_cast<long long>(m - 1) / 256 + 1) * ((n - 1) / 256 + 1), pairs = sms >= 2 ? sms / 2 : 1;
  double best = pair_us[0] + static_cast<double>((large - 1) / pairs + 1) * (num_kb * pair_us[1] + pair_us[2]);
  plan.pair = 1, plan.bn = 256;
  for (int s = 1; s <= 4; s *= 2) {
    if (s > 1 && (tiles * s > sms || num_kb < 2 * s)) break;
    const double us = tile_us[0] + static_cast<double>((tiles * s - 1) / sms + 1) * (((num_kb - 1) / s + 1) * tile_us[1] + tile_us[2]) +
                      (s == 2 ? 2.2 : s == 4 ? 3.2 : 0.0);
    if (us < best) {
      best = us;
      plan = Plan{0, 0, 128, s};
    }
  }
  return plan;
}

template <int kBN, bool kVector, bool kSwap, typename T>
int launch_tile(int device, cudaStream_t st, const Fp8Params& p) {
  using Kern = Fp8Tile<kBN, kVector, kSwap, T>;
  static bool ready[64];
  const auto kernel = fp8_tile_kernel<kBN, kVector, kSwap, T>;
  if (int e = opt_in(kernel, device, Kern::SMEM_BYTES, ready)) return e;
  const long long ctas = static_cast<long long>((p.rows_p + 127) / 128) * ((p.rows_q + kBN - 1) / kBN) * p.splits;
  if (ctas > 0x7fffffffLL) return fail(KCG_E_TOO_LARGE, "too many tiles for one launch");
  Launch l(st);
  l.shape(static_cast<unsigned>(ctas), Kern::NUM_THREADS, Kern::SMEM_BYTES, p.splits);
  return l(kernel, "8-bit product launch", p);
}

template <bool kVector, typename T>
int launch_pair(int device, int sms, cudaStream_t st, const Fp8Params& p) {
  using Kern = Fp8Pair<kVector, T>;
  static bool ready[64];
  const auto kernel = fp8_pair_kernel<kVector, T>;
  if (int e = opt_in(kernel, device, Kern::SMEM_BYTES, ready)) return e;
  // the accumulating warps would wait for ever for registers that the CTA was not launched with
  static std::atomic<int> registers{0};
  if (registers.load() == 0) {
    cudaFuncAttributes attributes;
    const cudaError_t e = cudaFuncGetAttributes(&attributes, kernel);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes");
    registers.store(attributes.numRegs);
  }
  if (registers.load() < Kern::LAUNCH_REGS) return fail(KCG_E_BAD_CONFIG, "the 8-bit product was built with too few registers");
  const long long tiles = static_cast<long long>((p.rows_p + 255) / 256) * ((p.rows_q + 255) / 256);
  if (tiles > 0x3fffffffLL) return fail(KCG_E_TOO_LARGE, "too many tiles for one launch");
  const int pairs = static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
  Launch l(st);
  l.shape(2 * pairs, Kern::NUM_THREADS, Kern::SMEM_BYTES, 2);
  return l(kernel, "8-bit product launch", p);
}

template <typename T>
int launch(const Plan& plan, int device, int sms, cudaStream_t st, const Fp8Params& p, bool vector) {
  if (plan.pair) return vector ? launch_pair<true, T>(device, sms, st, p) : launch_pair<false, T>(device, sms, st, p);
  if (!plan.swap) return vector ? launch_tile<128, true, false, T>(device, st, p) : launch_tile<128, false, false, T>(device, st, p);
  switch (plan.bn) {
    case 16: return launch_tile<16, true, true, T>(device, st, p);
    case 32: return launch_tile<32, true, true, T>(device, st, p);
    default: return launch_tile<64, true, true, T>(device, st, p);
  }
}

}  // namespace

// For tests of the host logic: the plan of a product as {pair, swap, columns of a tile, splits}.
extern "C" int kcg_internal_fp8_plan(int m, int n, int k, int block_b, int sms, int out[4]) {
  const Plan plan = plan_of(m, n, k, block_b == 1, sms);
  out[0] = plan.pair, out[1] = plan.swap, out[2] = plan.bn, out[3] = plan.splits;
  return 0;
}

extern "C" int kcg_matmul_fp8(int device, uint64_t stream, const kcg_fp8_product* a) {
  if (!a) return fail(KCG_E_BAD_ARG, "null argument");
  if (a->m < 0 || a->n <= 0 || a->k <= 0) return fail(KCG_E_BAD_ARG, "shape out of range");
  if (a->m > kMaxSize || a->n > kMaxSize || a->k > kMaxSize) return fail(KCG_E_TOO_LARGE, "a size of an 8-bit matrix is above 2^31 - 256");
  if (a->m == 0) return 0;
  if (!a->A || !a->B || !a->C || !a->scale_a || !a->scale_b) return fail(KCG_E_BAD_ARG, "null device pointer");
  if ((a->dtype_a != KCG_FP8_E4M3 && a->dtype_a != KCG_FP8_E5M2) || (a->dtype_b != KCG_FP8_E4M3 && a->dtype_b != KCG_FP8_E5M2))
    return fail(KCG_E_BAD_ARG, "operands are e4m3 or e5m2");
  if (!known_dtype(a->dtype_c)) return fail(KCG_E_BAD_ARG, "the result is float16, bfloat16 or float32");
  if (a->block_b != 1 && a->block_b != 128) return fail(KCG_E_BAD_ARG, "blocks of b have 1 or 128 rows");
  const int kb = (a->k - 1) / 128 + 1;
  int64_t lda = a->lda ? a->lda : a->k, ldb = a->ldb ? a->ldb : a->k;
  if (a->m == 1) lda = (lda + 15) / 16 * 16;  // (there is no second row)
  if (a->n == 1) ldb = (ldb + 15) / 16 * 16;
  const int64_t ldc = a->ldc ? a->ldc : a->n;
  const int64_t ldsa = a->ld_scale_a ? a->ld_scale_a : kb, ldsb = a->ld_scale_b ? a->ld_scale_b : kb;
  if (lda < a->k || ldb < a->k || ldc < a->n || ldsa < kb || ldsb < kb)
    return fail(KCG_E_BAD_ARG, "leading dimension below the row length");
  if (a->A % 16 || a->B % 16 || lda % 16 || ldb % 16)
    return fail(KCG_E_BAD_ARG, "rows of 8-bit operands must start on 16-byte boundaries");
  const int eb = a->dtype_c == KCG_DTYPE_FLOAT32 ? 4 : 2;
  if (a->C % eb || a->bias % eb || a->scale_a % 4 || a->scale_b % 4) return fail(KCG_E_BAD_ARG, "operands must be aligned to their values");
  int sms = 0;
  if (int e = sm_count(device, &sms)) return e;
  DeviceGuard guard;
  const cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  EncodeFn enc = nullptr;
  if (int r = encoder(&enc)) return r;
  const Plan plan = plan_of(a->m, a->n, a->k, a->block_b == 1, sms);
  Fp8Params p{};
  const int rows_box = plan.pair ? 128 : plan.bn;
  const uint32_t fa = a->dtype_a == KCG_FP8_E5M2, fb = a->dtype_b == KCG_FP8_E5M2;
  const int shift_b = a->block_b == 128 ? 7 : 0;
  const float *sa = reinterpret_cast<const float*>(a->scale_a), *sb = reinterpret_cast<const float*>(a->scale_b);
  if (plan.swap) {
    if (int r = encode(enc, &p.tmP, a->B, a->k, ldb, a->n, 128)) return r;
    if (int r = encode(enc, &p.tmQ, a->A, a->k, lda, a->m, rows_box)) return r;
    p.sp = sb, p.ldsp = ldsb, p.sp_shift = shift_b, p.sq = sa, p.ldsq = ldsa, p.sq_shift = 0;
    p.rows_p = a->n, p.rows_q = a->m, p.fmt_p = fb, p.fmt_q = fa;
  } else {
    if (int r = encode(enc, &p.tmP, a->A, a->k, lda, a->m, 128)) return r;
    if (int r = encode(enc, &p.tmQ, a->B, a->k, ldb, a->n, rows_box)) return r;
    p.sp = sa, p.ldsp = ldsa, p.sp_shift = 0, p.sq = sb, p.ldsq = ldsb, p.sq_shift = shift_b;
    p.rows_p = a->m, p.rows_q = a->n, p.fmt_p = fa, p.fmt_q = fb;
  }
  p.num_kb = kb;
  p.C = reinterpret_cast<void*>(a->C), p.ldc = ldc, p.bias = reinterpret_cast<const void*>(a->bias);
  p.fused = a->beta != 0.f || a->bias != 0 || a->relu != 0;
  p.beta = a->beta, p.relu = a->relu, p.splits = plan.splits;
  p.vector_store = a->C % 16 == 0 && ldc * eb % 16 == 0;
  p.word_store = a->C % 4 == 0 && ldc * eb % 4 == 0;
  p.tma_store = plan.pair && p.vector_store && static_cast<int64_t>(a->n) * eb % 16 == 0;
  p.vector_sp = reinterpret_cast<uint64_t>(p.sp) % 16 == 0 && p.ldsp % 4 == 0;
  p.vector_sq = reinterpret_cast<uint64_t>(p.sq) % 16 == 0 && p.ldsq % 4 == 0;
  if (p.tma_store)
    if (int r = encode_c(enc, &p.tmC, a->C, a->dtype_c, a->n, ldc, a->m)) return r;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vector = a->block_b == 1;
  if (a->dtype_c == KCG_DTYPE_FLOAT32) return launch<float>(plan, device, sms, st, p, vector);
  return a->dtype_c == KCG_DTYPE_FLOAT16 ? launch<__half>(plan, device, sms, st, p, vector)
                                         : launch<__nv_bfloat16>(plan, device, sms, st, p, vector);
}

// Reads (and clears) the status word of the 8-bit products on `device`: out = {code, block, detail, detail}; code 0 = no bounded
// wait has run out since the last call. Synchronises the device.
extern "C" int kcg_matmul_fp8_status(int device, uint32_t out[4]) {
  if (!out) return fail(KCG_E_BAD_ARG, "null argument");
  DeviceGuard guard;
  cudaError_t e = guard.enter(device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
  e = cudaMemcpyFromSymbol(out, g_fp8_status, sizeof(uint32_t) * 4);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyFromSymbol");
  if (out[0] != 0u) {
    const uint32_t zero[4] = {0u, 0u, 0u, 0u};
    e = cudaMemcpyToSymbol(g_fp8_status, zero, sizeof(zero));
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyToSymbol");
    return fail(KCG_E_DEVICE_TIMEOUT, "a bounded wait of an 8-bit product ran out");
  }
  return 0;
}
