// Attention of one or a few new tokens of each sequence over its keys in the paged cache: up to 64 rows (tokens x query heads that share a
// key head) meet every key of a sequence and key head.
//
// Each key is read once, 2 * d values, for at most 64 rows, so HBM bounds it. Sequences differ in length, and one of them may be all there is: so
// the tiles of 64 keys (d = 64: 128) of all sequences and key heads are laid end to end, kTokensPause places apart for what the end of
// one costs, and cut into equal ranges, one for each CTA, two CTAs an SM; a range may cover the end of one (sequence, head) and the
// beginning of others. What a range covers whole leaves as a result, a part as
// unnormalised fp32 rows with their maximum and sum in a workspace; a second kernel, already on the GPU when the first one ends, joins the
// parts of a (sequence, head) in the order of its keys. No atomics: the order of every sum follows from the lengths.
// 16 sequences of 16384 keys, 8 key heads of 128 values, bf16: 174 us for 4 rows a key head (6.2 TB/s), 177 for 24, 178 for 32, but 230 for 40 (4.7 TB/s; d = 64
// 94 for 24, 137 for 40): in the form of up to 64 rows each warp reads all of K and V from shared memory, four times in all.
//   warp 4     loads: a lane a box of a page (16 keys of K, say), its page's number fetched while the tile before is waited for; tells the others
//              through the stage which rows and keys it holds
//   warps 0-3  mma.sync m16n8k16 with 16 rows each. kRowGroups = 1 (up to 16 rows): each warp a quarter of a tile's keys; 2 (up to 32): two groups
//              of rows, half of the keys each; 4 (up to 64): all of them. (tcgen05 needs 128 rows: see kernels/attn_decode.cuh.)
// Keys that no row sees, but a box holds (behind the last token of a page, before a window), may be anything: their scores are replaced
// and their values overwritten with zeros, as 0 x NaN would not vanish.
#pragma once

struct TokensArgs {
  CUtensorMap tmK, tmV;  // {d, token of a page, head, page}, boxes of {64, min(page, tile; with a window 16), 1, 1}, 128-byte swizzle
  Sequences seq;
  const void* q;
  void* o;
  long long q_row, q_head, o_row, o_head;
  float* parts;  // [2 * CTAs][rows][d], then [2 * CTAs][rows] {maximum, sum}, then [CTAs] {sequence, head, first CTA, last CTA}
  int kv_heads, group, window, sinks;
  int box_log2;  // keys of a box
  int splits;    // the cluster form: CTAs that share a (sequence, head)'s keys
  float scale_log2;
};

// Places that a CTA takes at least, where there are enough CTAs for less. (1 sequence of 4097: two 13.3 us, three 13.7, four 14.2, six 15.9.)
constexpr int kTokensMinPlaces = 2;
// Places without a tile behind each (sequence, head)'s: joining the warps' results and beginning with other rows takes as long as a tile or
// two. (48 sequences x 4 tokens with a window of 1024, three of them empty: 73 us without, as many empty ones' ends in one CTA; 55.8 with one place,
// 47.8 with two, 47.1 with three or four; 64 sequences of up to 16384 260, 260, 262.)
constexpr int kTokensPause = 2;

// How `total` places are cut into ranges: the CTAs that have one, the first place of a CTA's, the CTA that has a place.
struct Ranges {
  long long total;
  int ctas;
  __device__ __forceinline__ Ranges(long long t, int most) : total(t) {
    const long long n = t / kTokensMinPlaces;
    ctas = n < 1 ? 1 : n < most ? static_cast<int>(n) : most;
  }
  __device__ __forceinline__ long long begin(int cta) const { return total * cta / ctas; }
  __device__ __forceinline__ int owner(long long place) const { return static_cast<int>(((place + 1) * ctas - 1) / total); }
};

// kCluster: a cluster of `splits` CTAs has the keys of one (sequence, head), and joins its parts in shared memory; no second kernel.
template <int kD, bool kBf16, int kRowGroups, bool kCluster>
struct AttnTokens {
  // Keys of a tile: 32 KB of K and V. (64 keys of d = 64 left each warp one short chain of products and exponentials a tile, 0.84 us for 16 KB:
  // 16 sequences x 32 heads of 2049 keys 48 us, bound by that.)
  static constexpr int BC = kD == 128 ? 64 : 128;
  static constexpr int STAGES = 3;
  static constexpr int KEY_GROUPS = 4 / kRowGroups, WKEYS = BC / KEY_GROUPS, ROWS = 16 * kRowGroups;
  static constexpr int NUM_THREADS = 160;
  static constexpr int HALVES = kD / 64;
  static constexpr int HALF_BYTES = BC * 128;  // a tile's keys x 64 values
  static constexpr int KV_BYTES = BC * kD * 2, STAGE_BYTES = 2 * KV_BYTES, RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int JOIN_BYTES = 4 * 16 * 32 * 4;  // 32 columns of the warps' rows
  // Up to 16 rows of queries come through shared memory with the first tile of their keys, rows 16 bytes apart (no two of a fragment in one
  // bank); more are read by the warps themselves.
  static constexpr bool kQueriesAhead = kRowGroups == 1;
  static constexpr int Q_PITCH = kD * 2 + 16, Q_BYTES = kQueriesAhead ? 16 * Q_PITCH : 0;
  static constexpr int CHAINS = WKEYS <= 32 ? 2 : 1;  // accumulators per 8 keys (even and odd 16 values of d)
  static constexpr int SMEM_BYTES = RING_BYTES + JOIN_BYTES + Q_BYTES + 1024 + 1792;
  static_assert(2 * (SMEM_BYTES + 1024) <= 228 * 1024, "two CTAs an SM");
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;

  // What a stage holds, for the warps that read it.
  struct Tile {
    int b, h;      // sequence, key head
    int v0;        // first place of the tile's keys
    int keys;      // of the sequence
    int p_lo;      // position of the first row's token
    KeyList list;
    int flags;     // MASKED: some row does not see some key; FIRST, LAST of a (sequence, head)'s keys in this CTA; WHOLE: all of them; END: of all
    int slot;      // where a part goes
  };
  enum : int { MASKED = 1, FIRST = 2, LAST = 4, WHOLE = 8, END = 16 };
  struct Shared {
    uint64_t full[STAGES], empty[STAGES], q_empty;
    Tile tile[STAGES];
    float2 warp_ml[4][16];
    float2 cta_ml[ROWS];  // (the cluster form)
    long long before[5];  // places of each warp's sequences
    long long begin;      // the first place with a tile in this CTA's range
    int found[3];         // its sequence (-1: there is none), head and tile
    volatile uint32_t abort_flag;
  };
  static_assert(sizeof(Shared) <= 1792, "barrier block exceeds its shared-memory slot");

  __device__ static __forceinline__ void report(Shared* sh, uint32_t code, uint32_t d0) {
    sh->abort_flag = 1u;
    if (atomicCAS(&g_paged_status[0], 0u, code) == 0u) {
      g_paged_status[1] = blockIdx.x;
      g_paged_status[2] = d0;
      g_paged_status[3] = 0u;
    }
  }
  // Weight of a partial result with maximum and sum ml; one of no key weighs nothing. (Scores that are all NaN leave a maximum of -inf and a sum
  // of NaN, which has to reach the result.)
  __device__ static __forceinline__ float weight(float2 ml, float base) { return ml.y == 0.f ? 0.f : ex2(ml.x - base); }

  // A sequence's keys and tiles; one without a key has a tile too, in which no row sees anything.
  struct Keys {
    KeyList list;
    int keys, p_lo, count;  // of the sequence; position of the first row's token; tiles
    __device__ __forceinline__ Keys(const TokensArgs& p, int length) {
      keys = p.seq.keys(length);
      p_lo = max(length, 0) - p.seq.each;
      list = KeyList(keys, p_lo, p.window, p.sinks, 1 << p.box_log2);
      count = max(1, list.count / BC + (list.count % BC ? 1 : 0));
    }
  };

  __device__ static void run(const TokensArgs& p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* join = reinterpret_cast<float*>(smem + RING_BYTES);
    uint8_t* queries = smem + RING_BYTES + JOIN_BYTES;
    Shared* sh = reinterpret_cast<Shared*>(queries + Q_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = p.seq.each * p.group;

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&sh->full[s], 1);
        mbar_init(&sh->empty[s], 4);
      }
      mbar_init(&sh->q_empty, 4);
      sh->abort_flag = 0u;
      sh->found[0] = -1;
      fence_mbar_init();
    }
    if (threadIdx.x == 128) {
      tma_prefetch_desc(&p.tmK);
      tma_prefetch_desc(&p.tmV);
    }
    griddep_wait();

    int cta = static_cast<int>(blockIdx.x);
    long long g0 = 0, g1 = 0, total = 0;
    if constexpr (kCluster) {
      // this CTA's share of its (sequence, head)'s tiles
      if (threadIdx.x == 0) {
        const int unit = cta / p.splits, rank = static_cast<int>(cluster_cta_rank());
        const int n = Keys(p, p.seq.lengths[unit / p.kv_heads]).count;
        const int t0 = static_cast<int>(static_cast<long long>(n) * rank / p.splits), t1 = static_cast<int>(static_cast<long long>(n) * (rank + 1) / p.splits);
        if (t0 < t1) sh->found[0] = unit / p.kv_heads, sh->found[1] = unit % p.kv_heads, sh->found[2] = t0, sh->begin = t0;
        sh->before[0] = t1;
      }
      __syncthreads();
      g0 = sh->begin, g1 = sh->before[0];
    } else {
      // All sequences' places, and where this CTA's range begins: a thread counts those of its run of sequences.
      const int per = (p.seq.count + NUM_THREADS - 1) / NUM_THREADS;
      const int b0 = min(static_cast<int>(threadIdx.x) * per, p.seq.count), b1 = min(b0 + per, p.seq.count);
      long long mine = 0;
      for (int b = b0; b < b1; ++b) mine += Keys(p, p.seq.lengths[b]).count + kTokensPause;
      mine *= p.kv_heads;
      long long upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) sh->before[warp] = upto;
      __syncthreads();
      long long base = 0;
#pragma unroll
      for (int w = 0; w < 5; ++w) {
        if (w < warp) base += sh->before[w];
        total += sh->before[w];
      }
      const Ranges ranges(total, gridDim.x);
      if (cta < ranges.ctas) g0 = ranges.begin(cta), g1 = ranges.begin(cta + 1);
      base += upto - mine;
      if (g0 < g1 && g0 >= base && g0 < base + mine) {
        long long at = g0 - base;
        for (int b = b0; b < b1; ++b) {
          const int n = Keys(p, p.seq.lengths[b]).count, places = n + kTokensPause;
          if (at < static_cast<long long>(places) * p.kv_heads) {
            int h = static_cast<int>(at / places), t = static_cast<int>(at % places), to = b;
            long long begin = g0;
            if (t >= n) {  // behind the last tile: the next (sequence, head)'s first one
              begin += places - t;
              t = 0;
              if (++h == p.kv_heads) h = 0, ++to;
            }
            if (begin < g1) sh->found[0] = to, sh->found[1] = h, sh->found[2] = t, sh->begin = begin;
            break;
          }
          at -= static_cast<long long>(places) * p.kv_heads;
        }
      }
      __syncthreads();
    }
    const bool any = sh->found[0] >= 0;

    if (warp == 4) {
      // ------------------------------------------------------------------ loads
      int4 meta = make_int4(-1, 0, 0, 0);
      if (any) {
        int b = sh->found[0], h = sh->found[1], t = sh->found[2], units = 0;
        long long place = sh->begin;
        Keys seq(p, p.seq.lengths[b]);
        int next_length = b + 1 < p.seq.count ? p.seq.lengths[b + 1] : 0;
        const int boxes = BC >> p.box_log2;            // of 64 columns, in a tile of K or of V
        const int loads = boxes * HALVES * 2;          // at most 32: a lane each
        const int box = lane % boxes, half = lane / boxes % HALVES, is_v = lane / (boxes * HALVES);
        const int tok = lane / p.group;                // of this lane's row of queries
        const T* q_from = static_cast<const T*>(p.q) + tok * p.q_row + (lane - tok * p.group) * p.q_head;
        // this lane's key and page of tile t of sequence b; page -1 (zeros) where no row sees any of the box
        int key;
        auto page_of = [&]() {
          const int v = t * BC + (box << p.box_log2);
          key = seq.list.key(v);
          return lane < loads && seq.list.seen(v, 1 << p.box_log2, p.sinks) ? p.seq.page_of(b, key) : -1;
        };
        int page = page_of();
        long long unit_begin = place - t;
        bool more = true;
        for (int i = 0; more; ++i) {
          const int s = i % STAGES;
          const int v0 = t * BC;
          const int this_page = page, in_page = key & ((1 << p.seq.page_log2) - 1), this_b = b, this_h = h;
          Tile tile;
          tile.b = b, tile.h = h, tile.v0 = v0, tile.keys = seq.keys, tile.p_lo = seq.p_lo, tile.list = seq.list;
          // every row sees every key: up to the first row's position, from the last one's window on or among the sinks
          const int p_hi = seq.p_lo + p.seq.each - 1, near = p.window > 0 && p_hi >= p.window ? p_hi - p.window + 1 - seq.list.shift : 0;
          const bool all = v0 + BC <= seq.list.place(min(seq.keys, seq.p_lo + 1)) && (v0 >= near || v0 + BC <= p.sinks);
          const bool whole = kCluster ? p.splits == 1 : unit_begin >= g0 && unit_begin + seq.count <= g1;
          const bool first = i == 0 || t == 0;
          tile.flags = (all ? 0 : MASKED) | (first ? FIRST : 0) | (whole ? WHOLE : 0);
          tile.slot = 2 * cta + (unit_begin >= g0 ? 1 : 0);
          if (!kCluster && i == 0 && unit_begin < g0) {
            const Ranges ranges(total, gridDim.x);
            meta = make_int4(b, h, ranges.owner(unit_begin), ranges.owner(unit_begin + seq.count - 1));
          }
          // the next tile, and its pages while this one's stage is waited for
          ++place;
          bool last = false;
          if (++t == seq.count) {
            last = true;
            t = 0;
            place += kTokensPause;
            unit_begin = place;
            if (++h == p.kv_heads) {
              h = 0;
              if (++b < p.seq.count) {
                seq = Keys(p, next_length);
                next_length = b + 1 < p.seq.count ? p.seq.lengths[b + 1] : 0;
              }
            }
          }
          more = place < g1;
          tile.flags |= (last || !more ? LAST : 0) | (more ? 0 : END);
          if (more) page = page_of();
          bool free = mbar_wait(&sh->empty[s], ((i / STAGES) & 1u) ^ 1u, &sh->abort_flag);
          if (kQueriesAhead && first) {
            if (free) free = mbar_wait(&sh->q_empty, (units & 1u) ^ 1u, &sh->abort_flag);
            ++units;
          }
          if (!__all_sync(0xffffffffu, free)) {
            if (lane == 0) report(sh, PAGED_TIMEOUT_LOADS, static_cast<uint32_t>(i));
            break;
          }
          uint8_t* st = smem + s * STAGE_BYTES;
          if (lane == 0) {
            sh->tile[s] = tile;
            mbar_expect_tx(&sh->full[s], STAGE_BYTES + (kQueriesAhead && first ? rows * kD * 2 : 0));
          }
          __syncwarp();
          if (lane < loads)
            tma_load_4d(st + is_v * KV_BYTES + half * HALF_BYTES + (box << p.box_log2) * 128, is_v ? &p.tmV : &p.tmK, &sh->full[s], half * 64,
                        in_page, this_h, this_page);
          if (kQueriesAhead && first && lane < rows)
            bulk_load_1d(queries + lane * Q_PITCH, q_from + static_cast<long long>(this_b) * p.seq.each * p.q_row + this_h * p.group * p.q_head, kD * 2,
                         &sh->full[s]);
        }
      }
      if (!kCluster && lane == 0) {
        float* end = p.parts + 2ll * gridDim.x * rows * (kD + 2);
        reinterpret_cast<int4*>(end)[cta] = meta;
      }
      __syncwarp();
    } else if (any) {
      const int q = lane >> 2, t = lane & 3;  // row and column pair of this lane in an accumulator tile
      const int rg = warp / KEY_GROUPS, kg = warp % KEY_GROUPS;
      const int mat = lane >> 3, mrow = lane & 7;
      uint32_t qf[kD / 16][4];
      float o[kD / 8][4];
      float m[2], l[2];
      int see[2], near[2];  // places of keys below `see`, of those from `near` on (and the sinks)
      for (int i = 0;; ++i) {
        const int s = i % STAGES;
        const bool got = mbar_wait(&sh->full[s], (i / STAGES) & 1u, &sh->abort_flag);
        // (one outcome for all four: they meet again at the end of a (sequence, head))
        if (!named_bar_all(1, 128, got)) {
          if (!got && lane == 0) report(sh, PAGED_TIMEOUT_ATTENTION, static_cast<uint32_t>(i));
          break;
        }
        const Tile tile = sh->tile[s];
        if (tile.flags & FIRST) {
          const T* Q = static_cast<const T*>(p.q);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = rg * 16 + q + 8 * e, i_tok = r / p.group;
            const bool live = r < rows;
            const T* from = kQueriesAhead ? reinterpret_cast<const T*>(queries + r * Q_PITCH)
                                          : Q + (static_cast<long long>(tile.b) * p.seq.each + i_tok) * p.q_row + (tile.h * p.group + r - i_tok * p.group) * p.q_head;
#pragma unroll
            for (int ks = 0; ks < kD / 16; ++ks) {
              qf[ks][e] = live ? *reinterpret_cast<const uint32_t*>(from + ks * 16 + 2 * t) : 0u;
              qf[ks][e + 2] = live ? *reinterpret_cast<const uint32_t*>(from + ks * 16 + 2 * t + 8) : 0u;
            }
            const int position = tile.p_lo + (live ? i_tok : 0);
            see[e] = tile.list.place(min(position + 1, tile.keys));
            near[e] = p.window > 0 && position >= p.window ? position - p.window + 1 - tile.list.shift : 0;
            m[e] = -INFINITY, l[e] = 0.f;
          }
#pragma unroll
          for (int n = 0; n < kD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
          if (kQueriesAhead) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->q_empty);
          }
        }
        const uint32_t kaddr = smem_u32(smem + s * STAGE_BYTES), vaddr = kaddr + KV_BYTES;
        float c[WKEYS / 8][4], c2[CHAINS == 2 ? WKEYS / 8 : 1][4];
#pragma unroll
        for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c[n][e] = 0.f;
            if (CHAINS == 2) c2[n][e] = 0.f;
          }
#pragma unroll
        for (int ks = 0; ks < kD / 32; ++ks) {
          const int unit = ks * 4 + mat;
#pragma unroll
          for (int n = 0; n < WKEYS / 8; ++n) {
            const int key = kg * WKEYS + n * 8 + mrow;
            uint32_t b[4];
            ldmatrix_x4(b, kaddr + key * 128 + (unit >> 3) * HALF_BYTES + (((unit & 7) ^ (key & 7)) << 4));
            mma_16816<kBf16>(c[n], qf[2 * ks][0], qf[2 * ks][1], qf[2 * ks][2], qf[2 * ks][3], b[0], b[1]);
            mma_16816<kBf16>(CHAINS == 2 ? c2[n] : c[n], qf[2 * ks + 1][0], qf[2 * ks + 1][1], qf[2 * ks + 1][2], qf[2 * ks + 1][3], b[2], b[3]);
          }
        }
        if constexpr (CHAINS == 2) {
#pragma unroll
          for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[n][e] += c2[n][e];
        }
        if (tile.flags & MASKED) {
          const int first = tile.v0 + kg * WKEYS;
#pragma unroll
          for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = first + n * 8 + 2 * t + (e & 1);
              if (key >= see[e >> 1] || (key < near[e >> 1] && key >= p.sinks)) c[n][e] = -INFINITY;
            }
          // values of keys that no row sees
          bool zeroed = false;
          for (int u = lane; u < WKEYS * (kD / 8); u += 32) {
            const int k = u / (kD / 8), piece = u % (kD / 8), key = first + k, at = kg * WKEYS + k;
            if (key >= tile.list.count || (key < tile.list.lo && key >= p.sinks)) {
              *reinterpret_cast<uint4*>(smem + s * STAGE_BYTES + KV_BYTES + (piece >> 3) * HALF_BYTES + at * 128 + (((piece & 7) ^ (at & 7)) << 4)) =
                  make_uint4(0u, 0u, 0u, 0u);
              zeroed = true;
            }
          }
          if (zeroed) fence_proxy_async_smem();  // (the stage's next load comes behind these stores)
          __syncwarp();
        }
        float base_[2], alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < WKEYS / 8; ++n) mx = fmaxf(mx, fmaxf(c[n][2 * h], c[n][2 * h + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          mx = fmaxf(m[h], mx * p.scale_log2);  // (the scale is positive: checked by the host)
          base_[h] = mx == -INFINITY ? 0.f : mx;
          alpha[h] = ex2(m[h] - base_[h]);
          m[h] = mx;
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < kD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= alpha[e >> 1];
        }
        // Rows of large scores (see kLargeScores), whose products are rounded first. (The question costs 0.13 us of one sequence's 12.8; the same without
        // a branch, two products a score, 0.16.)
        float times[2] = {p.scale_log2, p.scale_log2};
        if (__builtin_expect(__any_sync(0xffffffffu, fmaxf(fabsf(base_[0]), fabsf(base_[1])) >= kLargeScores), 0)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool large = fabsf(base_[h]) >= kLargeScores;
#pragma unroll
            for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) c[n][2 * h + e] = __fmul_rn(c[n][2 * h + e], large ? p.scale_log2 : 1.f);
            times[h] = large ? 1.f : p.scale_log2;
          }
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < WKEYS / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c[n][e] = ex2(fmaf(c[n][e], times[e >> 1], -base_[e >> 1]));
            sum[e >> 1] += c[n][e];
          }
        l[0] = l[0] * alpha[0] + sum[0];
        l[1] = l[1] * alpha[1] + sum[1];
#pragma unroll
        for (int ks = 0; ks < WKEYS / 16; ++ks) {
          const uint32_t a0 = pack_pair<kBf16>(c[2 * ks][0], c[2 * ks][1]);
          const uint32_t a1 = pack_pair<kBf16>(c[2 * ks][2], c[2 * ks][3]);
          const uint32_t a2 = pack_pair<kBf16>(c[2 * ks + 1][0], c[2 * ks + 1][1]);
          const uint32_t a3 = pack_pair<kBf16>(c[2 * ks + 1][2], c[2 * ks + 1][3]);
          const int key = kg * WKEYS + ks * 16 + (mat & 1) * 8 + mrow;
          const uint32_t vrow = vaddr + key * 128;
#pragma unroll
          for (int n = 0; n < kD / 8; n += 2) {
            const int unit = n + (mat >> 1);
            uint32_t b[4];
            ldmatrix_x4_trans(b, vrow + (unit >> 3) * HALF_BYTES + (((unit & 7) ^ (key & 7)) << 4));
            mma_16816<kBf16>(o[n], a0, a1, a2, a3, b[0], b[1]);
            mma_16816<kBf16>(o[n + 1], a0, a1, a2, a3, b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->empty[s]);
        if (!(tile.flags & LAST)) continue;  // (the CTA's last tile is the last of its rows)

        // ---- the end of these rows' keys in this CTA: the warps' sums, 32 columns at a time
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
          if (t == 0) sh->warp_ml[warp][q + 8 * h] = make_float2(m[h], l[h]);
        }
        named_bar_sync(1, 128);
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < KEY_GROUPS; ++k) top = fmaxf(top, sh->warp_ml[rg * KEY_GROUPS + k][q + 8 * h].x);
          f[h] = weight(make_float2(m[h], l[h]), top);
        }
#pragma unroll
        for (int cc = 0; cc < kD / 32; ++cc) {
          float* mine_o = join + warp * 16 * 32;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            *reinterpret_cast<float2*>(mine_o + q * 32 + n * 8 + 2 * t) = make_float2(o[cc * 4 + n][0] * f[0], o[cc * 4 + n][1] * f[0]);
            *reinterpret_cast<float2*>(mine_o + (q + 8) * 32 + n * 8 + 2 * t) = make_float2(o[cc * 4 + n][2] * f[1], o[cc * 4 + n][3] * f[1]);
          }
          named_bar_sync(1, 128);
          const int row = threadIdx.x >> 3, c4 = threadIdx.x & 7;  // of a group of 16 rows
#pragma unroll
          for (int g = 0; g < kRowGroups; ++g) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, sum_l = 0.f;
#pragma unroll
            for (int k = 0; k < KEY_GROUPS; ++k) {
              const float4 x = reinterpret_cast<const float4*>(join + ((g * KEY_GROUPS + k) * 16 + row) * 32)[c4];
              a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
              top = fmaxf(top, sh->warp_ml[g * KEY_GROUPS + k][row].x);
            }
#pragma unroll
            for (int k = 0; k < KEY_GROUPS; ++k) {
              const float2 ml = sh->warp_ml[g * KEY_GROUPS + k][row];
              sum_l = fmaf(ml.y, weight(ml, top), sum_l);
            }
            const int r = g * 16 + row;
            if (r >= rows) continue;
            const int col = cc * 32 + c4 * 4;
            if (tile.flags & WHOLE) {
              const float inv = sum_l == 0.f ? 0.f : 1.f / sum_l;
              const int i_tok = r / p.group;
              T* to = static_cast<T*>(p.o) + (static_cast<long long>(tile.b) * p.seq.each + i_tok) * p.o_row + (tile.h * p.group + r - i_tok * p.group) * p.o_head + col;
              *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<kBf16>(a.x * inv, a.y * inv), pack_pair<kBf16>(a.z * inv, a.w * inv));
            } else if (kCluster) {  // (the ring is idle: the CTA's last tile has been read)
              reinterpret_cast<float4*>(smem)[r * (kD / 4) + col / 4] = a;
              if (cc == 0 && c4 == 0) sh->cta_ml[r] = make_float2(top, sum_l);
            } else {
              const long long part = static_cast<long long>(tile.slot) * rows + r;
              *reinterpret_cast<float4*>(p.parts + part * kD + col) = a;
              if (cc == 0 && c4 == 0)
                reinterpret_cast<float2*>(p.parts + 2ll * gridDim.x * rows * kD)[part] = make_float2(top, sum_l);
            }
          }
          named_bar_sync(1, 128);
        }
        if (tile.flags & END) break;
      }
    }
    if constexpr (kCluster) {
      if (p.splits > 1) {
        if (!any)
          for (int r = threadIdx.x; r < rows; r += NUM_THREADS) sh->cta_ml[r] = make_float2(-INFINITY, 0.f);
        __syncwarp();
        cluster_sync_all();
        // this CTA's share of the result, 16-byte units of fp32 rows, joined over the cluster
        constexpr int UNITS = kD / 4;
        static_assert(ROWS * kD * 4 <= RING_BYTES, "the CTA's rows fit the ring");
        const int rank = static_cast<int>(cluster_cta_rank()), unit = cta / p.splits, b = unit / p.kv_heads, h = unit % p.kv_heads;
        const int u0 = rows * UNITS * rank / p.splits, u1 = rows * UNITS * (rank + 1) / p.splits;
        const uint32_t o_addr = smem_u32(smem), ml_addr = smem_u32(&sh->cta_ml[0]);
        for (int i = u0 + threadIdx.x; i < u1; i += NUM_THREADS) {
          const int r = i / UNITS;
          float2 ml[16];
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int c = 0; c < 16; ++c) ml[c] = c < p.splits ? ld_cluster_f2(map_to_cta(ml_addr + r * 8, c)) : make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int c = 0; c < 16; ++c) top = fmaxf(top, ml[c].x);
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int c0 = 0; c0 < 16; c0 += 8) {
            float4 x[8];
#pragma unroll
            for (int c = 0; c < 8; ++c)
              if (c0 + c < p.splits) x[c] = ld_cluster_f4(map_to_cta(o_addr + i * 16, c0 + c));
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              if (ml[c0 + c].y == 0.f) continue;  // (no part, or one of no key: whatever lies there)
              const float f = weight(ml[c0 + c], top);  // (0 too: 0 x NaN is one)
              a.x = fmaf(f, x[c].x, a.x), a.y = fmaf(f, x[c].y, a.y), a.z = fmaf(f, x[c].z, a.z), a.w = fmaf(f, x[c].w, a.w);
              sum = fmaf(f, ml[c0 + c].y, sum);
            }
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int i_tok = r / p.group;
          T* to = static_cast<T*>(p.o) + (static_cast<long long>(b) * p.seq.each + i_tok) * p.o_row + (h * p.group + r - i_tok * p.group) * p.o_head + i % UNITS * 4;
          *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<kBf16>(a.x * inv, a.y * inv), pack_pair<kBf16>(a.z * inv, a.w * inv));
        }
        __syncwarp();
        cluster_sync_all();  // the other CTAs read this one's shared memory until here
      }
    }
    if (sh->abort_flag != 0u) {  // loads still in flight land before the ring is given up
      const uint64_t w0 = global_timer_ns();
      while (global_timer_ns() - w0 < 200000ull) __nanosleep(1000);
    }
    __syncthreads();
  }
};

template <int kD, bool kBf16, int kRowGroups, bool kCluster>
__global__ void __launch_bounds__(160, 2) attention_tokens_kernel(const __grid_constant__ TokensArgs p) {
  AttnTokens<kD, kBf16, kRowGroups, kCluster>::run(p);
}

// The parts of the (sequence, key head) whose keys came into CTA blockIdx.x of the kernel above from the one before. A unit of n parts has n - 1 such
// blocks, which share out its rows (one (sequence, head) of 65536 keys x 32 rows: 97 -> 22 us, in one block before; 19 in a graph); the 16 warps of a block share out a row's parts, if
// there are not as many rows, eight at a time. (Blocks of 256 threads and 40 registers, small enough to wait beside the kernel above, were slower, 18
// against 14 us for one sequence of 4097: they take what the next call's CTAs need.)
template <int kD, bool kBf16>
__global__ void __launch_bounds__(512) attention_tokens_join_kernel(const __grid_constant__ TokensArgs p, int ctas) {
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  using Vec = typename std::conditional<kD == 128, float4, float2>::type;
  constexpr int PER = kD / 32, WARPS = 16, AT_ONCE = 8;
  __shared__ float acc[WARPS][kD];
  __shared__ float2 ml_of[WARPS];
  griddep_wait();
  griddep_launch_dependents();
  const int all_rows = p.seq.each * p.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float2* ml = reinterpret_cast<const float2*>(p.parts + 2ll * ctas * all_rows * kD);
  const int4 meta = reinterpret_cast<const int4*>(p.parts + 2ll * ctas * all_rows * (kD + 2))[blockIdx.x];
  if (meta.x < 0) return;
  const int first = meta.z, n = meta.w - first + 1;  // CTAs with a part: slot 1 of the first, slot 0 of the others
  const int helper = static_cast<int>(blockIdx.x) - first - 1, helpers = n - 1;
  const int rows = (all_rows - helper + helpers - 1) / helpers;  // this block's: every helpers-th from helper on
  int shares = 1;  // warps of a row
  while (shares < WARPS && rows * shares < WARPS && n > shares) shares *= 2;
  const int rows_at_once = WARPS / shares;
  for (int r0 = 0; r0 < rows; r0 += rows_at_once) {
    const int r = helper + (r0 + warp / shares) * helpers, share = warp % shares;
    const bool live = r < all_rows;
    float top = -INFINITY, sum = 0.f, a[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) a[e] = 0.f;
    for (int i0 = share; live && i0 < n; i0 += shares * AT_ONCE) {
      float2 s[AT_ONCE];
      Vec v[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * shares;
        const long long part = (2ll * (first + i) + (i == 0 ? 1 : 0)) * all_rows + r;
        s[u] = i < n ? ml[part] : make_float2(-INFINITY, 0.f);
        if (i < n) v[u] = reinterpret_cast<const Vec*>(p.parts + part * kD)[lane];
      }
      float now = top;
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) now = fmaxf(now, s[u].x);
      const float old = sum == 0.f ? 0.f : ex2(top - now);
      top = now;
      sum *= old;
#pragma unroll
      for (int e = 0; e < PER; ++e) a[e] *= old;
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (s[u].y == 0.f) continue;  // (no key in sight: zeros, or no part)
        const float f = ex2(s[u].x - top);
        sum = fmaf(f, s[u].y, sum);
#pragma unroll
        for (int e = 0; e < PER; ++e) a[e] = fmaf(f, reinterpret_cast<const float*>(&v[u])[e], a[e]);
      }
    }
    if (shares > 1) {
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[warp][lane * PER + e] = a[e];
      if (lane == 0) ml_of[warp] = make_float2(top, sum);
      __syncthreads();
      if (live && share == 0) {
        float all = -INFINITY;
        for (int w = 0; w < shares; ++w) all = fmaxf(all, ml_of[warp + w].x);
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < PER; ++e) a[e] = 0.f;
        for (int w = 0; w < shares; ++w) {
          const float2 s = ml_of[warp + w];
          const float f = s.y == 0.f ? 0.f : ex2(s.x - all);
          sum = fmaf(f, s.y, sum);
#pragma unroll
          for (int e = 0; e < PER; ++e) a[e] = fmaf(f, acc[warp + w][lane * PER + e], a[e]);
        }
      }
      __syncthreads();
    }
    if (live && share == 0) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int i_tok = r / p.group;
      T* to = static_cast<T*>(p.o) + (static_cast<long long>(meta.x) * p.seq.each + i_tok) * p.o_row + (meta.y * p.group + r - i_tok * p.group) * p.o_head + lane * PER;
      if constexpr (PER == 4) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<kBf16>(a[0] * inv, a[1] * inv), pack_pair<kBf16>(a[2] * inv, a[3] * inv));
      } else {
        *reinterpret_cast<uint32_t*>(to) = pack_pair<kBf16>(a[0] * inv, a[1] * inv);
      }
    }
  }
}
