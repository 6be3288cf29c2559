// The paged cache of keys and values: storing a step's rows in it, with the rotation by their positions on the way.
//
// Bound by HBM: each row's heads are read once and written once (a prompt), or by the latency of three dependent loads (the row's
// sequence, its length, its page) in a decode step. A warp takes one row and four heads (d = 64: eight) at a time, a thread two
// 16-byte pieces whose values turn together, so that it reads its angles once for all heads and needs no other thread's values;
// where there are few rows, several warps share one. 12085 rows of 32 + 2 x 8 heads of 128 values, bf16: 53.6 us, 5.7 TB/s, with four CTAs an
// SM (64 registers; three of 74: 59.9, five or six, with spills, 58.8 and 62.7; the rows towards L2 while their places are looked up: 56.0);
// 32 rows 3.2 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "../../include/kcg_b200.h"
#include "attn_common.cuh"
#include "fp8_common.cuh"
#include "kernels/ptx_sm100.cuh"
#include "paged.cuh"

namespace {

using namespace kcg;
using namespace kcg8;
using namespace kcgp;

struct AppendArgs {
  Sequences seq;
  const void *k, *v, *q;
  void *k_cache, *v_cache, *qo;
  long long k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;
  long long kc[3], vc[3];  // strides of the caches
  const float *cos, *sin;
  const int32_t* positions;
  long long angles;
  int q_heads, kv_heads, rotary, warps_log2;  // warps that share a row
};

constexpr int kAppendWarps = 8;

// A thread's piece pair u of a head: halves rotary / 2 values apart (the pair turns together), neighbouring pieces when interleaved
// or past the rotated part.
template <typename T, int kD, bool kInterleaved>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) append_kv_kernel(const AppendArgs a) {
  constexpr int UNITS = kD / 16, HEADS = 32 / UNITS;  // piece pairs of a head, heads of a warp's step
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = (static_cast<int>(blockIdx.x) << (3 - a.warps_log2)) + (warp >> a.warps_log2);
  if (row >= a.seq.rows) return;
  const int u = lane % UNITS;
  const bool turned = u * 16 < a.rotary;
  const int at0 = turned && !kInterleaved ? u * 8 : u * 16;
  const int at1 = turned && !kInterleaved ? at0 + a.rotary / 2 : at0 + 8;

  const int b = sequence_of(a.seq, row);
  if (b < 0) return;
  const int n = a.seq.start(b + 1) - a.seq.start(b);
  const int position = max(a.seq.lengths[b], 0) - n + (row - a.seq.start(b));  // (of any length below 0 a negative one)
  const int page = position >= 0 && position < a.seq.capacity() ? a.seq.page_of(b, position) : -1;
  float c[8], s[8];
  if (turned) {
    const long long p = a.positions ? a.positions[row] : position;
    if (p >= 0 && p < a.angles) {
      const long long at = p * (a.rotary / 2) + u * 8;
      load8(a.cos + at, c), load8(a.sin + at, s);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
  }
  const long long slot = position & ((1 << a.seq.page_log2) - 1);
  const int heads = a.q_heads + 2 * a.kv_heads;
#pragma unroll 4
  for (int h = ((warp & ((1 << a.warps_log2) - 1)) * HEADS) + lane / UNITS; h < heads; h += HEADS << a.warps_log2) {
    const T* from;
    T* to;
    bool turn = turned;
    if (h < a.q_heads) {
      from = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
      to = static_cast<T*>(a.qo) + row * a.qo_row + h * a.qo_head;
    } else if (h < a.q_heads + a.kv_heads) {
      const int kh = h - a.q_heads;
      from = static_cast<const T*>(a.k) + row * a.k_row + kh * a.k_head;
      to = page < 0 ? nullptr : static_cast<T*>(a.k_cache) + page * a.kc[0] + kh * a.kc[1] + slot * a.kc[2];
    } else {
      const int vh = h - a.q_heads - a.kv_heads;
      from = static_cast<const T*>(a.v) + row * a.v_row + vh * a.v_head;
      to = page < 0 ? nullptr : static_cast<T*>(a.v_cache) + page * a.vc[0] + vh * a.vc[1] + slot * a.vc[2];
      turn = false;
    }
    if (!to) continue;
    Raw8<T> x, y;
    x.load(from + at0), y.load(from + at1);
    if (position < 0) {
      x.zero(), y.zero();  // (only queries come here)
    } else if (turn) {
      float p[8], q[8], e[8], f[8];
      x.values(p), y.values(q);
      if constexpr (kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[2 * i] = p[2 * i] * c[i] - p[2 * i + 1] * s[i], e[2 * i + 1] = p[2 * i + 1] * c[i] + p[2 * i] * s[i];
          f[2 * i] = q[2 * i] * c[i + 4] - q[2 * i + 1] * s[i + 4], f[2 * i + 1] = q[2 * i + 1] * c[i + 4] + q[2 * i] * s[i + 4];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i] * c[i] - q[i] * s[i], f[i] = q[i] * c[i] + p[i] * s[i];
      }
      float2 ev[4], fv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ev[i] = make_float2(e[2 * i], e[2 * i + 1]), fv[i] = make_float2(f[2 * i], f[2 * i + 1]);
      store8(to + at0, ev), store8(to + at1, fv);
      continue;
    }
    *reinterpret_cast<uint4*>(to + at0) = x.v, *reinterpret_cast<uint4*>(to + at1) = y.v;
  }
}

template <typename T>
int append(Launch& launch, const AppendArgs& a, int d, bool interleaved) {
  if (d == 128)
    return interleaved ? launch(append_kv_kernel<T, 128, true>, "append_kv launch", a) : launch(append_kv_kernel<T, 128, false>, "append_kv launch", a);
  return interleaved ? launch(append_kv_kernel<T, 64, true>, "append_kv launch", a) : launch(append_kv_kernel<T, 64, false>, "append_kv launch", a);
}

// ---------------------------------------------------------------------------------------------------- attention
__device__ unsigned int g_paged_status[4];  // {code, block, detail, detail}; 0 = no wait ran out
enum : uint32_t { PAGED_TIMEOUT_LOADS = 1, PAGED_TIMEOUT_ATTENTION = 2, PAGED_TIMEOUT_UNIT = 3 };

#include "paged_prompt.cuh"
#include "paged_tokens.cuh"

int check_query(const kcg_paged_cache* c, const kcg_paged_query* q) {
  if (!q) return fail(KCG_E_BAD_ARG, "attention_paged: null pointer");
  if (int r = check_cache(c, q->rows)) return r;
  if (q->rows > 0 && (!q->Q || !q->O)) return fail(KCG_E_BAD_ARG, "attention_paged: null pointer");
  if (q->Q % 16 || q->O % 16 || q->workspace % 16) return fail(KCG_E_BAD_ARG, "attention_paged: operands must start on 16-byte boundaries");
  if (!aligned_rows(q->q_stride, 2, c->d) || !aligned_rows(q->o_stride, 2, c->d))
    return fail(KCG_E_BAD_ARG, "attention_paged: strides are multiples of 8 values, at least a head's");
  if (q->q_heads < 1 || q->q_heads % c->kv_heads || q->q_heads / c->kv_heads > 64)
    return fail(KCG_E_BAD_ARG, "attention_paged: 1 to 64 query heads share a key head");
  if (q->window < 0 || q->sinks < 0) return fail(KCG_E_BAD_ARG, "attention_paged: negative window or sinks");
  if (!(q->scale > 0.f) || !(q->scale <= 2e38f)) return fail(KCG_E_BAD_ARG, "scale must be positive and finite");  // (times log2 e, too)
  if (static_cast<long long>(q->rows) * q->q_heads > 0x7fffff00LL) return fail(KCG_E_TOO_LARGE, "attention_paged: too many rows");
  return 0;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::mutex g_mutex;

int encoder(EncodeFn* out) {
  static EncodeFn known = nullptr;
  std::lock_guard<std::mutex> lock(g_mutex);
  if (!known) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e != cudaSuccess || found != cudaDriverEntryPointSuccess || !fn) {
      cudaGetLastError();
      return fail(KCG_E_NO_DRIVER, "cuTensorMapEncodeTiled not available from the driver");
    }
    known = reinterpret_cast<EncodeFn>(fn);
  }
  *out = known;
  return 0;
}

// {d, token of a page, head, page} view of a cache; boxes of 64 values x `box_rows` tokens of one head and page. What is outside reads as zero.
int encode_cache(EncodeFn encode, CUtensorMap* tm, const kcg_paged_cache* c, uint64_t ptr, const int64_t* stride, int box_rows) {
  cuuint64_t dim[4] = {static_cast<cuuint64_t>(c->d), static_cast<cuuint64_t>(c->page), static_cast<cuuint64_t>(c->kv_heads), static_cast<cuuint64_t>(c->pages)};
  cuuint64_t step[3] = {static_cast<cuuint64_t>(stride[2]) * 2, static_cast<cuuint64_t>(stride[1]) * 2, static_cast<cuuint64_t>(stride[0]) * 2};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = encode(tm, c->dtype == KCG_DTYPE_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                            reinterpret_cast<void*>(ptr), dim, step, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(static_cast<int>(r), "cuTensorMapEncodeTiled failed");
}

// Dynamic shared memory of a kernel, opted in to once on each device.
template <auto kKernel>
int opt_in(int device, int bytes, bool large_clusters = false) {
  static std::atomic<unsigned long long> done{0};
  if (done.load() >> device & 1ull) return 0;
  cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && large_clusters) e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
  done.fetch_or(1ull << device);
  return 0;
}

// Rows that share a key head, where every sequence has as many new tokens; those of up to 64 go by tokens (paged_tokens.cuh).
int shared_rows(const kcg_paged_cache* c, const kcg_paged_query* q) {
  if (c->starts) return 0;
  const long long n = static_cast<long long>(q->rows / c->sequences) * (q->q_heads / c->kv_heads);
  return n <= 64 ? static_cast<int>(n) : 0;
}

// How many clusters of a size run at once (asked once per device and kernel; -1: the size is not to be had).
template <auto kKernel>
int clusters_at_once(int device, int threads, int smem, int size) {
  static std::atomic<int> known[64][17];
  int n = known[device][size].load();
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(size), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.attrs = attr, cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = -1;
    }
    known[device][size].store(n);
  }
  return n;
}

// CTAs of a cluster that share the keys of one (sequence, key head) of `units`, where each has one of its own, and no second kernel joins their
// parts: where the table is so short that each has four tiles at most, and all clusters run at once; two tiles at least, if there are
// four. 0: the keys of all sequences are cut into ranges. Bf16, 32 heads over 8 of 128 values, keys that are not in L2, cluster against ranges: 1 sequence of
// 128 keys 6.5 us / 8.6, of 1024 8.8 / 10.3, of 2048 (two tiles each) 9.6 / 11.7, of 4096 (four) 11.4 / 13.4, of 5120 (five) 12.6 / 14.8, of 8192 (eight) 15.0 / 16.5, of
// 16384 22.2 / 21.0, of 32768 36 / 31; 4 of 2048 (four) 13.0 / 17.1, of 8192 28.2 / 32.1; 16 of 512 (four) 12.7 / 17.7. So four is a border on the safe side: with sequences as
// long as the table clusters win up to some eight tiles. What it keeps out is a table much wider than most of its sequences are long, whose longest one
// a cluster has to itself (and keys in L2: 1 of 8192 14.0 / 13.7).
template <typename Active>
int tokens_cluster(long long units, int max_tiles, Active&& active) {
  if (max_tiles <= 4) return 1;
  const int s = max_tiles / 2 < 16 ? max_tiles / 2 : 16, least = (max_tiles + 3) / 4;
  for (int n = s; n >= least; --n)
    if (units <= active(n)) return n;
  return 0;
}

int64_t tokens_workspace(int sms, int rows, int d) { return 2ll * sms * (2ll * rows * (d + 2) * 4 + 16); }

template <int kD, bool kBf16, int kRowGroups>
int launch_tokens(int device, int sms, cudaStream_t st, const kcg_paged_cache* c, TokensArgs& p) {
  using Kern = AttnTokens<kD, kBf16, kRowGroups, false>;
  constexpr auto ranges = attention_tokens_kernel<kD, kBf16, kRowGroups, false>;
  constexpr auto cluster = attention_tokens_kernel<kD, kBf16, kRowGroups, true>;
  if (int r = opt_in<ranges>(device, Kern::SMEM_BYTES)) return r;
  if (int r = opt_in<cluster>(device, Kern::SMEM_BYTES, true)) return r;
  const long long units = static_cast<long long>(c->sequences) * c->kv_heads;
  long long keys = static_cast<long long>(c->width) * c->page;
  if (p.window > 0) keys = std::min(keys, static_cast<long long>(p.window) + p.seq.each + p.sinks + 2 * (1 << p.box_log2));
  const int max_tiles = static_cast<int>(std::min((keys + Kern::BC - 1) / Kern::BC, 1000000LL));
  p.splits = tokens_cluster(units, max_tiles, [&](int s) { return clusters_at_once<cluster>(device, Kern::NUM_THREADS, Kern::SMEM_BYTES, s); });
  Launch launch(st);
  if (p.splits > 0) {
    if (units * p.splits > 0x7fffffffLL) return fail(KCG_E_TOO_LARGE, "attention_paged: too many rows");
    launch.shape(static_cast<unsigned>(units * p.splits), Kern::NUM_THREADS, Kern::SMEM_BYTES, p.splits);
    return launch(cluster, "attention_paged launch", p);
  }
  launch.shape(2 * sms, Kern::NUM_THREADS, Kern::SMEM_BYTES);
  if (int r = launch(ranges, "attention_paged launch", p)) return r;
  launch.shape(2 * sms, 512);
  return launch(attention_tokens_join_kernel<kD, kBf16>, "attention_paged join launch", p, 2 * sms);
}

template <int kRowGroups>
int launch_tokens_of(int device, int sms, cudaStream_t st, const kcg_paged_cache* c, TokensArgs& p) {
  if (c->d == 128)
    return c->dtype == KCG_DTYPE_BFLOAT16 ? launch_tokens<128, true, kRowGroups>(device, sms, st, c, p) : launch_tokens<128, false, kRowGroups>(device, sms, st, c, p);
  return c->dtype == KCG_DTYPE_BFLOAT16 ? launch_tokens<64, true, kRowGroups>(device, sms, st, c, p) : launch_tokens<64, false, kRowGroups>(device, sms, st, c, p);
}

int attention_tokens(int device, cudaStream_t st, const kcg_paged_cache* c, const kcg_paged_query* q, int rows) {
  int sms;
  if (int r = sm_count(device, &sms)) return r;
  if (!q->workspace || q->workspace_bytes < tokens_workspace(sms, rows, c->d)) return fail(KCG_E_BAD_ARG, "attention_paged: workspace too small");
  EncodeFn encode;
  if (int r = encoder(&encode)) return r;
  TokensArgs p{};
  const int most = q->window > 0 ? 16 : c->d == 128 ? 64 : 128, box = c->page < most ? c->page : most;  // keys of a box: see attention_prompt()
  if (int r = encode_cache(encode, &p.tmK, c, c->K, c->k_stride, box)) return r;
  if (int r = encode_cache(encode, &p.tmV, c, c->V, c->v_stride, box)) return r;
  p.seq = sequences_of(c, q->rows);
  p.q = reinterpret_cast<const void*>(q->Q), p.o = reinterpret_cast<void*>(q->O);
  p.q_row = q->q_stride[0], p.q_head = q->q_stride[1], p.o_row = q->o_stride[0], p.o_head = q->o_stride[1];
  p.parts = reinterpret_cast<float*>(q->workspace);
  p.kv_heads = c->kv_heads, p.group = q->q_heads / c->kv_heads, p.window = q->window, p.sinks = q->sinks;
  while ((1 << p.box_log2) < box) ++p.box_log2;
  p.scale_log2 = q->scale * 1.4426950408889634f;
  if (rows <= 16) return launch_tokens_of<1>(device, sms, st, c, p);
  if (rows <= 32) return launch_tokens_of<2>(device, sms, st, c, p);
  return launch_tokens_of<4>(device, sms, st, c, p);
}

template <int kD, bool kBf16>
int launch_prompt(int device, cudaStream_t st, PromptArgs& p, long long pairs, int max_steps) {
  using Kern = AttnPrompt<kD, kBf16, false>;
  constexpr auto whole = attention_prompt_kernel<kD, kBf16, false>;
  constexpr auto split = attention_prompt_kernel<kD, kBf16, true>;
  if (int r = opt_in<whole>(device, Kern::SMEM_BYTES)) return r;
  if (int r = opt_in<split>(device, Kern::SMEM_BYTES)) return r;
  const long long units = pairs * p.kv_heads;
  if (units > 0x7fffffffLL / 8) return fail(KCG_E_TOO_LARGE, "attention_paged: too many rows");
  // The largest number of CTAs, 2 to 8, that can share the keys of a pair of tiles with every cluster running at once and, where the
  // sequences are as long as the table, four tiles of keys each (joining costs what two do).
  p.splits = 1;
  for (int s = 8; s >= 2 && p.splits == 1; --s)
    if (max_steps >= 4 * s && units <= clusters_at_once<split>(device, Kern::NUM_THREADS, Kern::SMEM_BYTES, s)) p.splits = s;
  Launch launch(st);
  launch.shape(static_cast<unsigned>(units * p.splits), Kern::NUM_THREADS, Kern::SMEM_BYTES, p.splits);
  return p.splits > 1 ? launch(split, "attention_paged launch", p) : launch(whole, "attention_paged launch", p);
}

int attention_prompt(int device, cudaStream_t st, const kcg_paged_cache* c, const kcg_paged_query* q) {
  if (device < 0 || device >= 64) return fail(KCG_E_BAD_ARG, "device index out of range");
  EncodeFn encode;
  if (int r = encoder(&encode)) return r;
  PromptArgs p{};
  p.seq = sequences_of(c, q->rows);
  p.o = reinterpret_cast<void*>(q->O);
  p.o_row = q->o_stride[0], p.o_head = q->o_stride[1];
  p.kv_heads = c->kv_heads, p.group = q->q_heads / c->kv_heads, p.window = q->window, p.sinks = q->sinks;
  p.tile_tokens = 128 / p.group;
  p.scale_log2 = q->scale * 1.4426950408889634f;
  const int pair = 2 * p.tile_tokens;
  const long long pairs = AttnPrompt<128, true, false>::places(p.seq, pair);
  if (pairs > 0x7fffffffLL) return fail(KCG_E_TOO_LARGE, "attention_paged: too many rows");
  p.pairs = static_cast<int>(pairs);
  // Keys of a box: of a page, or of 32 where a window's keys begin anywhere and are laid out from a box's border on.
  const int most = q->window > 0 ? 32 : 128, box = c->page < most ? c->page : most;
  while ((1 << p.box_log2) < box) ++p.box_log2;
  const bool bf16 = c->dtype == KCG_DTYPE_BFLOAT16;
  {
    cuuint64_t dim[3] = {static_cast<cuuint64_t>(c->d), static_cast<cuuint64_t>(q->q_heads), static_cast<cuuint64_t>(q->rows)};
    cuuint64_t step[2] = {static_cast<cuuint64_t>(q->q_stride[1]) * 2, static_cast<cuuint64_t>(q->q_stride[0]) * 2};
    cuuint32_t box3[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(p.tile_tokens)}, one[3] = {1, 1, 1};
    const CUresult r = encode(&p.tmQ, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, reinterpret_cast<void*>(q->Q), dim,
                              step, box3, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(static_cast<int>(r), "cuTensorMapEncodeTiled failed");
  }
  if (int r = encode_cache(encode, &p.tmK, c, c->K, c->k_stride, box)) return r;
  if (int r = encode_cache(encode, &p.tmV, c, c->V, c->v_stride, box)) return r;
  long long keys = static_cast<long long>(c->width) * c->page;
  if (q->window > 0) keys = std::min(keys, static_cast<long long>(q->window) + pair + q->sinks);
  const int max_steps = static_cast<int>(std::min((keys + 127) / 128, 1000000LL));
  if (c->d == 128) return bf16 ? launch_prompt<128, true>(device, st, p, pairs, max_steps) : launch_prompt<128, false>(device, st, p, pairs, max_steps);
  return bf16 ? launch_prompt<64, true>(device, st, p, pairs, max_steps) : launch_prompt<64, false>(device, st, p, pairs, max_steps);
}

}  // namespace

extern "C" int kcg_append_kv(int device, uint64_t stream, const kcg_paged_cache* c, const kcg_new_rows* r) {
  if (!r) return fail(KCG_E_BAD_ARG, "append_kv: null pointer");
  if (int e = check_cache(c, r->rows)) return e;
  const bool queries = r->Q != 0;
  if (r->rows > 0 && (!r->K || !r->V)) return fail(KCG_E_BAD_ARG, "append_kv: null pointer");
  if (queries != (r->QO != 0) || (queries && (r->q_heads < 1 || r->q_heads > 65535))) return fail(KCG_E_BAD_ARG, "append_kv: queries, their heads and their results go together");
  if (!aligned_rows(r->k_stride, 2, c->d) || !aligned_rows(r->v_stride, 2, c->d) ||
      (queries && (!aligned_rows(r->q_stride, 2, c->d) || !aligned_rows(r->qo_stride, 2, c->d))))
    return fail(KCG_E_BAD_ARG, "append_kv: strides are multiples of 8 values, at least a head's");
  if (r->rotary < 0 || r->rotary > c->d || r->rotary % 16) return fail(KCG_E_BAD_ARG, "append_kv: a multiple of 16 values is turned, at most a head's");
  if (r->rotary > 0 && (!r->cos || !r->sin || r->angles < 1)) return fail(KCG_E_BAD_ARG, "append_kv: no angles");
  if (r->K % 16 || r->V % 16 || r->Q % 16 || r->QO % 16 || r->cos % 16 || r->sin % 16 || r->positions % 4)
    return fail(KCG_E_BAD_ARG, "append_kv: operands must start on 16-byte boundaries");
  if (r->rows > 0x7fffff00) return fail(KCG_E_TOO_LARGE, "append_kv: too many rows");
  if (r->rows == 0) return 0;
  DeviceGuard guard;
  if (cudaError_t e = guard.enter(device)) return cuda_fail(e, "cudaSetDevice");
  int sms;
  if (int e = sm_count(device, &sms)) return e;
  AppendArgs a{};
  a.seq = sequences_of(c, r->rows);
  a.k = reinterpret_cast<const void*>(r->K), a.v = reinterpret_cast<const void*>(r->V), a.q = reinterpret_cast<const void*>(r->Q);
  a.k_cache = reinterpret_cast<void*>(c->K), a.v_cache = reinterpret_cast<void*>(c->V), a.qo = reinterpret_cast<void*>(r->QO);
  a.k_row = r->k_stride[0], a.k_head = r->k_stride[1], a.v_row = r->v_stride[0], a.v_head = r->v_stride[1];
  a.q_row = r->q_stride[0], a.q_head = r->q_stride[1], a.qo_row = r->qo_stride[0], a.qo_head = r->qo_stride[1];
  for (int i = 0; i < 3; ++i) a.kc[i] = c->k_stride[i], a.vc[i] = c->v_stride[i];
  a.cos = reinterpret_cast<const float*>(r->cos), a.sin = reinterpret_cast<const float*>(r->sin);
  a.positions = reinterpret_cast<const int32_t*>(r->positions);
  a.angles = r->angles;
  a.q_heads = queries ? r->q_heads : 0, a.kv_heads = c->kv_heads, a.rotary = r->rotary;
  // Warps that share a row: as many as leave the GPU some 16 warps an SM, and each something to do.
  const int steps = ((a.q_heads + 2 * a.kv_heads) * (c->d / 16) + 31) / 32;
  while (a.warps_log2 < 3 && (r->rows << a.warps_log2) < sms * 16 && (1 << a.warps_log2) < steps) ++a.warps_log2;
  const int per = kAppendWarps >> a.warps_log2;
  Launch launch(reinterpret_cast<cudaStream_t>(stream));
  launch.shape(static_cast<unsigned>((static_cast<long long>(r->rows) + per - 1) / per), kAppendWarps * 32);
  return c->dtype == KCG_DTYPE_BFLOAT16 ? append<__nv_bfloat16>(launch, a, c->d, r->interleaved != 0) : append<__half>(launch, a, c->d, r->interleaved != 0);
}

extern "C" int64_t kcg_attention_paged_workspace(int device, const kcg_paged_cache* c, const kcg_paged_query* q) {
  if (int r = check_query(c, q)) return r;
  const int rows = shared_rows(c, q);
  if (rows == 0) return 0;
  int sms;
  if (int r = sm_count(device, &sms)) return r < 0 ? r : KCG_E_BAD_ARG;
  return tokens_workspace(sms, rows, c->d);
}

extern "C" int kcg_attention_paged(int device, uint64_t stream, const kcg_paged_cache* c, const kcg_paged_query* q) {
  if (int r = check_query(c, q)) return r;
  if (q->rows == 0) return 0;
  DeviceGuard guard;
  if (cudaError_t e = guard.enter(device)) return cuda_fail(e, "cudaSetDevice");
  if (const int rows = shared_rows(c, q)) return attention_tokens(device, reinterpret_cast<cudaStream_t>(stream), c, q, rows);
  return attention_prompt(device, reinterpret_cast<cudaStream_t>(stream), c, q);
}

extern "C" int kcg_attention_paged_status(int device, uint32_t out[4]) {
  if (!out) return fail(KCG_E_BAD_ARG, "null argument");
  DeviceGuard guard;
  if (cudaError_t e = guard.enter(device)) return cuda_fail(e, "cudaSetDevice");
  if (cudaError_t e = cudaDeviceSynchronize()) return cuda_fail(e, "cudaDeviceSynchronize");
  if (cudaError_t e = cudaMemcpyFromSymbol(out, g_paged_status, sizeof(uint32_t) * 4)) return cuda_fail(e, "cudaMemcpyFromSymbol");
  if (out[0] == 0u) return 0;
  const uint32_t zero[4] = {0u, 0u, 0u, 0u};
  if (cudaError_t e = cudaMemcpyToSymbol(g_paged_status, zero, sizeof(zero))) return cuda_fail(e, "cudaMemcpyToSymbol");
  return fail(KCG_E_DEVICE_TIMEOUT, "a bounded wait of the paged attention ran out");
}
