// What the kernels of the paged cache share: which sequence a row belongs to, where its positions lie, which keys it sees, and the
// host's checks of a cache.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/kcg_b200.h"
#include "fp8_common.cuh"

namespace kcgp {

// The device's view of a kcg_paged_cache's tables.
struct Sequences {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;  // or null: `each` rows a sequence
  long long table_ld;
  int pages, page_log2, width;
  int count, rows, each;

  // Rows of the step before sequence b, within the rows that there are.
  __device__ __forceinline__ int start(int b) const {
    if (!starts) return b * each;  // (at most `rows`)
    const int s = starts[b];
    return s < 0 ? 0 : s > rows ? rows : s;
  }
  // Positions that the table has pages for.
  __device__ __forceinline__ long long capacity() const { return static_cast<long long>(width) << page_log2; }
  // Keys of a sequence of length `length`.
  __device__ __forceinline__ int keys(int length) const {
    const long long cap = capacity();
    return length < 0 ? 0 : length > cap ? static_cast<int>(cap) : length;
  }
  // The page of a position that the table reaches; -1 for one that does not exist.
  __device__ __forceinline__ int page_of(int b, int position) const {
    const int p = table[b * table_ld + (position >> page_log2)];
    return p >= 0 && p < pages ? p : -1;
  }
};

// The keys that rows at positions p_lo .. see some of, laid end to end in whole boxes (parts of pages, `box` keys, a power of two): those of the first
// `sinks` keys that lie before the first row's window, then those from that window on, up to `end`. A place v below `lead` is key v, others key
// v + shift. (With a window of 1024 and 4 sinks 64 tokens see 9 tiles of 128; as tiles of a sequence's keys the same are 10 or 11.)
struct KeyList {
  int lead, shift;  // places of the sinks, when they are apart; keys between them and the others
  int lo;           // place of the first key of the first row's window: places from `sinks` to here are of no row's keys
  int count;        // places
  __device__ __forceinline__ KeyList() {}
  __device__ __forceinline__ KeyList(int end, int p_lo, int window, int sinks, int box) {
    const int first = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;
    const int from = first & -box;
    lead = sinks < from ? (sinks + box - 1) & -box : from;
    shift = from - lead;
    if (shift == 0) lead = 0;  // (one piece)
    lo = first - shift;
    count = place(end);
  }
  // Keys below x as places.
  __device__ __forceinline__ int place(int x) const { return x - shift > lead ? x - shift : min(x, lead); }
  __device__ __forceinline__ int key(int v) const { return v < lead ? v : v + shift; }
  // Whether some row may see a key of the box at place v.
  __device__ __forceinline__ bool seen(int v, int box, int sinks) const { return v < count && (v < sinks || v + box > lo); }
};

// Weights are 2^(score * scale - maximum), in one operation whose product is not rounded, where the maximum is that product rounded: half a unit of
// its last place stands in the exponent of all of a row's weights, and their sum divides it out again. From 2^27 on that would be a factor of 2^8 and more,
// which with the prompts' lagging maximum passes fp16's range, and from 2^31 on fp32's. So from this magnitude on products are rounded first, as the
// maximum is: the largest weight is 1, and what is infinite gives NaN. The two ways differ by 2^-13 of the exponent at most below it (a row's tiles
// may go either way: with 2^24, a factor of 2^0.5, equal scores had unequal weights).
constexpr float kLargeScores = 4096.f;

// The sequence whose rows hold `row`, or -1; asked by a whole (converged) warp, 32 places at a time. (The last sequence that starts at
// or before the row, if it has not ended there: empty ones start where the next one does.)
__device__ __forceinline__ int sequence_of(const Sequences& s, int row) {
  if (!s.starts) {
    const int b = row / s.each;
    return b < s.count ? b : -1;
  }
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = s.count;  // the answer is in [lo, hi), if there is one
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const unsigned there = __ballot_sync(0xffffffffu, at < hi && s.starts[at] <= row);
    if (there == 0u) return -1;
    const int last = 31 - __clz(there);
    lo += last * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return s.count > 0 && s.starts[lo] <= row && row < s.starts[lo + 1] ? lo : -1;
}

// Host side: the checks of a cache, and its tables for a launch.
inline bool aligned_rows(const int64_t* stride, int n, int d) {
  for (int i = 0; i < n; ++i)
    if (stride[i] < d || stride[i] % 8 || stride[i] >= 1LL << 39) return false;
  return true;
}

inline int check_cache(const kcg_paged_cache* c, int rows) {
  using kcg8::fail;
  if (!c || !c->K || !c->V || !c->table || !c->lengths) return fail(KCG_E_BAD_ARG, "paged cache: null pointer");
  if (c->dtype != KCG_DTYPE_BFLOAT16 && c->dtype != KCG_DTYPE_FLOAT16) return fail(KCG_E_BAD_ARG, "paged cache: float16 or bfloat16");
  if (c->d != 64 && c->d != 128) return fail(KCG_E_BAD_CONFIG, "head dimension must be 64 or 128");
  if (c->page < 8 || (c->page & (c->page - 1)) || c->page > 1 << 20) return fail(KCG_E_BAD_ARG, "pages hold a power of two of tokens, at least 8");
  if (c->pages < 1 || c->width < 1 || c->sequences < 1 || c->kv_heads < 1 || c->table_ld < c->width)
    return fail(KCG_E_BAD_ARG, "paged cache: empty or overlapping shape");
  if (static_cast<long long>(c->width) * c->page > 0x7fffff00LL) return fail(KCG_E_TOO_LARGE, "paged cache: a sequence of more than 2^31 - 256 tokens");
  if (c->kv_heads > 65535 || c->sequences > 1 << 24) return fail(KCG_E_TOO_LARGE, "paged cache: too many heads or sequences");
  if (!aligned_rows(c->k_stride, 3, c->d) || !aligned_rows(c->v_stride, 3, c->d))
    return fail(KCG_E_BAD_ARG, "paged cache: strides are multiples of 8 values, at least a head's");
  if (c->K % 16 || c->V % 16 || c->table % 4 || c->lengths % 4 || c->starts % 4) return fail(KCG_E_BAD_ARG, "paged cache: misaligned pointer");
  if (rows < 0) return fail(KCG_E_BAD_ARG, "paged cache: negative rows");
  if (!c->starts && rows % c->sequences) return fail(KCG_E_BAD_ARG, "paged cache: without row ranges every sequence has as many rows");
  return 0;
}

inline Sequences sequences_of(const kcg_paged_cache* c, int rows) {
  Sequences s{};
  s.table = reinterpret_cast<const int32_t*>(c->table);
  s.lengths = reinterpret_cast<const int32_t*>(c->lengths);
  s.starts = reinterpret_cast<const int32_t*>(c->starts);
  s.table_ld = c->table_ld;
  s.pages = c->pages;
  s.width = c->width;
  while ((1 << s.page_log2) < c->page) ++s.page_log2;
  s.count = c->sequences;
  s.rows = rows;
  s.each = c->starts ? 0 : rows / c->sequences;
  return s;
}

}  // namespace kcgp
