// Attention of prompts, or pieces of prompts, over their sequences' keys in the paged cache: causal, optionally with a sliding window and first
// tokens that stay visible. The form of the fused attention kernel (AttnFwd2 in kcg_attention.cu, where its roles, meetings and figures are
// described) over pages:
//
// A CTA takes two tiles of 128 rows at a time: the query heads that share a key head, of as many tokens as fit (32 tokens x 4 heads, say), so that
// every key tile is loaded once for all of them. It walks the keys that its rows see in tiles of 128: the sinks, then from the first row's window to
// the last row's position; a warp masks a tile only where one of its 32 rows does not see all of it.
//   warp 0    loads: both Q tiles and K tiles through a two-stage ring, a lane a box of a page; page numbers one tile ahead
//   warp 1    tcgen05.mma: S = Q K^T, O += P V with P in tensor memory
//   warp 2    waits for K and V in the issuer's place, and overwrites values that no row sees with zeros (0 x NaN would not vanish)
//   warp 3    loads V tiles in the same way; finds the next pair of tiles when the loads of this one end
//   warps 4-7 softmax of tile 0, warps 8-11 of tile 1, a row a thread
// Bound by what bounds that kernel, the chain scores - softmax - product of a tile against the other tile's (1.8 us for both tiles' steps), and, where calls
// follow one another, the power cap: 8192 tokens, 32 heads over 8 of 128 values, bf16, 525 us then, 1047 TFLOP/s of the pairs seen and 75 % of what
// a library product sustains under the cap; in short bursts, before it sets in, 451, 74 % of such a product's burst. So a quarter is the chain. A window
// makes a pair of tiles short, nine steps at a window of 1024: then what comes before the first step and behind the last one counts. So a CTA stays where
// it is and takes over a CTA that has not been launched yet (cluster launch control) as its next pair: the queries and keys of that one are loaded, and
// its first scores computed, while this one's rows are finished. 16384 tokens, a window of 1024, 4 sinks, short bursts: 408 us with a launch a pair, then 340,
// 314 with first scores ahead and fewer registers in the control warps, 283 with weights against a lagging maximum; in a row 329 (812 TFLOP/s). In what is
// left a pair has 16 us of steps and 4.5 of ends: masked steps at both of them, the results' stores, the first step's wait for its scores.
// kKeySplit: where the tiles do not fill the GPU, the CTAs of a cluster share the keys of one pair, and join their results in shared memory.
#pragma once

struct PromptArgs {
  CUtensorMap tmQ;       // {d, head, row}, boxes of {64, group, tokens of a tile}
  CUtensorMap tmK, tmV;  // {d, token of a page, head, page}, boxes of {64, min(page, 128; with a window 32), 1, 1}; 128-byte swizzle all
  Sequences seq;
  void* o;
  long long o_row, o_head;
  int kv_heads, group, tile_tokens, window, sinks;
  int box_log2;  // keys of a box
  int pairs;     // of tiles, at most
  int splits;    // CTAs that share a pair's keys
  float scale_log2;
};

template <int kD, bool kBf16, bool kKeySplit>
struct AttnPrompt {
  static constexpr int BR = 128, BC = 128, TILES = 2;
  static constexpr int K_STAGES = 2, V_STAGES = 2;
  static constexpr int NUM_THREADS = 384;
  static constexpr int HALVES = kD / 64;
  static constexpr int BOX_BYTES = 128 * 128;  // 128 rows x 64 values
  static constexpr int Q_BYTES = BR * kD * 2, KV_BYTES = BC * kD * 2;
  static constexpr int OFF_K = TILES * Q_BYTES, OFF_V = OFF_K + K_STAGES * KV_BYTES, RING_BYTES = OFF_V + V_STAGES * KV_BYTES;
  // Results leave through shared memory, 32 rows x 128 bytes of a warp at a time, as whole 128-byte lines: 3000 cycles a tile, beside the other
  // tile's products. (A row a thread, 16 bytes of 32 rows a store: 3700; 32 bytes a store cost the steps more, in registers, than it gained here: 8192
  // tokens 471 us / 482.)
  static constexpr int OUT_BYTES = 8 * 32 * 128;
  static constexpr int SMEM_BYTES = RING_BYTES + OUT_BYTES + 2048;  // 1 KB alignment slack + barriers
  static constexpr int P_PART = kD == 128 ? 96 : 64;    // keys of a step after which P V starts
  static constexpr bool kApart = kD == 64;              // tile 1 starts half a step after tile 0
  static constexpr uint32_t COL_O = TILES * BC, TMEM_COLS = 512;
  static constexpr uint32_t FMT = kBf16 ? FMT_BF16 : FMT_F16;
  static constexpr uint32_t IDESC_S = make_instr_desc(FMT, 0u, 0u, 128u, BC);
  static constexpr uint32_t IDESC_O = make_instr_desc(FMT, 0u, 1u, 128u, kD);
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;

  // A pair of tiles (and, with others, a share of its keys).
  struct Unit {
    KeyList list;
    int b, head, row0, tokens;  // sequence, key head, first row of the step, tokens (0: none)
    int p_lo, keys;             // position of the first token; keys of the sequence
    int v0, steps, tiles;       // first place of the keys, tiles of keys, tiles of rows
    int end;                    // there is no further unit, and this is none
  };
  struct Barriers {
    uint64_t q_full[TILES], q_empty[TILES];
    uint64_t k_full[K_STAGES], k_empty[K_STAGES], v_full[V_STAGES], v_empty[V_STAGES];
    uint64_t s_full[TILES];  // S_t of the current step is complete
    uint64_t o_full[TILES];  // the last P_t V of a unit has retired
    uint64_t unit_full[2], unit_empty[2];  // a unit is there, every warp has read it
    uint64_t taken;                        // the answer to a request for another CTA's work
    uint4 answer;                          // (16-byte aligned: barriers stand before it)
    Unit unit[2];
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
  };
  static_assert(sizeof(Barriers) <= 1024, "barrier block exceeds its shared-memory slot");
  static constexpr int UNIT_WARPS = 11;  // that read a unit (warp 3 makes them)

  // Named barriers: see AttnFwd2. Every meeting takes place in every step whatever else happened.
  static constexpr uint32_t BAR_PART = 1;  // + t: the first P_PART keys of P_t are in tensor memory and O_t is rescaled
  static constexpr uint32_t BAR_FULL = 3;  // + t: all of P_t is
  static constexpr uint32_t BAR_KV = 5;    // the V tile of a step and the K tile of the next are there
  static constexpr uint32_t PT_THREADS = 160, KV_THREADS = 64;

  __device__ static __forceinline__ void report(Barriers* bars, uint32_t code, uint32_t d0, uint32_t d1) {
    bars->abort_flag = 1u;
    if (atomicCAS(&g_paged_status[0], 0u, code) == 0u) {
      g_paged_status[1] = blockIdx.x;
      g_paged_status[2] = d0;
      g_paged_status[3] = d1;
    }
  }

  // The row of units, as warp 3 walks it. A sequence's pairs of tiles are counted from its last token, whose pair sees the most keys; the first may
  // have fewer tokens. Up to kOrdered sequences: pairs with the most keys come first, over all sequences, so that none of the long ones begins
  // last (6 prompts of up to 1501 tokens, 14 heads over 2 of 64 values: 37 us in the order of the sequences, 31, and 28 with the steps after it); a pair's level is the keys of its last
  // token over a pair's tokens. For a place in the row the warp bisects its level, a lane one or two
  // sequences, whose facts it has read once (read and divided for every step of it, a place took 6 us). Of more sequences that would take longer than a unit, and many short units even out by themselves:
  // the pairs of sequence b take the places from (its first row) / (tokens of a pair) + b on, of which there are enough (some have no
  // tokens), so a search over the first rows alone finds the sequence; the last ones first.
  static constexpr int kOrdered = 64;
  // Places in the row, at most.
  static long long places(const Sequences& s, int pair) {
    if (!s.starts && s.count <= kOrdered) return static_cast<long long>((s.each + pair - 1) / pair) * s.count;
    return (static_cast<long long>(s.rows) + pair - 1) / pair + s.count - 1;  // (a sequence has one pair that is not full)
  }
  struct Row {
    int first[2], rows[2], length[2];  // of sequences lane and lane + 32: first row, rows, tokens
    int pairs[2], level[2];            // pairs of tiles, level of the last one

    __device__ __forceinline__ explicit Row(const PromptArgs& p) {
      const int pair = TILES * p.tile_tokens, lane = threadIdx.x & 31;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int b = lane + 32 * i;
        first[i] = rows[i] = length[i] = pairs[i] = level[i] = 0;
        if (p.seq.count <= kOrdered && b < p.seq.count) {
          first[i] = p.seq.start(b), rows[i] = max(0, p.seq.start(b + 1) - first[i]), length[i] = p.seq.lengths[b];
          pairs[i] = (rows[i] + pair - 1) / pair;
          level[i] = (max(max(length[i], rows[i]), 1) - 1) / pair;  // (no pair's last token is before the first)
        }
      }
    }
    // Pairs of sequence lane + 32 i of at least a level.
    __device__ __forceinline__ int from(int i, int l) const { return max(0, min(pairs[i], level[i] - l + 1)); }

    __device__ __forceinline__ Unit unit(const PromptArgs& p, int index, int rank) const {
      const int pair = TILES * p.tile_tokens, lane = threadIdx.x & 31;
      int e = index / p.kv_heads;  // in the end: which of the sequence's pairs, from the last one on
      int row0, n, tokens;
      Unit x;
      x.head = index - e * p.kv_heads;
      if (p.seq.count > kOrdered) {
        const int place = p.pairs - 1 - e;
        int lo = 0, hi = p.seq.count;
        while (hi - lo > 1) {
          const int step = (hi - lo + 31) / 32, at = lo + lane * step;
          const unsigned there = __ballot_sync(0xffffffffu, at < hi && p.seq.start(at) / pair + at <= place);
          const int last = there ? 31 - __clz(there) : 0;
          lo += last * step;
          hi = min(lo + step, hi);
        }
        x.b = lo;
        row0 = p.seq.start(lo), n = max(0, p.seq.start(lo + 1) - row0), tokens = p.seq.lengths[lo];
        e = (n + pair - 1) / pair - 1 - (place - (row0 / pair + lo));
      } else {
        int lo = -1, hi = __reduce_max_sync(0xffffffffu, max(level[0], level[1])) + 1;  // all pairs are of level lo at least, none of level hi
        while (hi - lo > 1) {
          const int mid = lo + (hi - lo) / 2;
          if (__reduce_add_sync(0xffffffffu, from(0, mid) + from(1, mid)) > e) {
            lo = mid;
          } else {
            hi = mid;
          }
        }
        e -= __reduce_add_sync(0xffffffffu, from(0, hi) + from(1, hi));  // among those of level lo, one of a sequence at most
        const unsigned at0 = __ballot_sync(0xffffffffu, from(0, lo) > from(0, hi)), at1 = __ballot_sync(0xffffffffu, from(1, lo) > from(1, hi));
        const int i = e < __popc(at0) ? 0 : 1;
        unsigned at = i ? at1 : at0;
        for (int nth = e - (i ? __popc(at0) : 0); nth > 0 && at; --nth) at &= at - 1u;
        const int l = __ffs(at) - 1, from_l = max(l, 0);
        x.b = from_l + 32 * i;
        row0 = __shfl_sync(0xffffffffu, i ? first[1] : first[0], from_l);
        n = __shfl_sync(0xffffffffu, i ? rows[1] : rows[0], from_l);
        tokens = __shfl_sync(0xffffffffu, i ? length[1] : length[0], from_l);
        e = l < 0 ? -1 : __shfl_sync(0xffffffffu, i ? level[1] : level[0], from_l) - lo;
      }
      x.end = x.tokens = x.p_lo = x.keys = x.row0 = 0;
      x.tiles = 1;
      const int begin = n - (e + 1) * pair;  // (the first pair has what is left)
      if (e >= 0 && begin > -pair) {
        x.tokens = begin < 0 ? pair + begin : pair;
        x.tiles = x.tokens > p.tile_tokens ? 2 : 1;
        x.row0 = row0 + max(begin, 0);
        x.keys = p.seq.keys(tokens);
        x.p_lo = max(tokens, 0) - n + max(begin, 0);  // (a negative length: no keys)
      }
      x.list = KeyList(x.tokens > 0 ? max(0, min(x.keys, x.p_lo + x.tokens)) : 0, x.p_lo, p.window, p.sinks, 1 << p.box_log2);
      const int steps = x.list.count / BC + (x.list.count % BC ? 1 : 0);
      const int step0 = kKeySplit ? static_cast<int>(static_cast<long long>(steps) * rank / p.splits) : 0;
      x.steps = (kKeySplit ? static_cast<int>(static_cast<long long>(steps) * (rank + 1) / p.splits) : steps) - step0;
      x.v0 = step0 * BC;
      return x;
    }
  };

  // Bits below n, of 32.
  __device__ static __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

  // Takes over a CTA of this grid that has not been launched yet, if there is one; 16 bytes of answer.
  __device__ static __forceinline__ void request_cta(uint4* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 :
                 : "r"(smem_u32(answer)), "r"(smem_u32(bar))
                 : "memory");
  }
  // Its blockIdx.x, or -1: there was none (and none may be asked for again).
  __device__ static __forceinline__ int requested_cta(const uint4* answer) {
    int x;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b128 a;\n\t"
        ".reg .b32 y, z, w;\n\t"
        "ld.shared.b128 a, [%1];\n\t"
        "mov.b32 %0, -1;\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, a;\n\t"
        "}\n"
        : "=&r"(x)
        : "r"(smem_u32(answer))
        : "memory");
    return x;
  }

  __device__ static void run(const PromptArgs& p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    Barriers* bars = reinterpret_cast<Barriers*>(smem + RING_BYTES + OUT_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kKeySplit ? static_cast<int>(cluster_cta_rank()) : 0;

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
      tma_prefetch_desc(&p.tmQ);
      tma_prefetch_desc(&p.tmK);
      tma_prefetch_desc(&p.tmV);
      for (int s = 0; s < K_STAGES; ++s) mbar_init(&bars->k_full[s], 1), mbar_init(&bars->k_empty[s], 1);
      for (int s = 0; s < V_STAGES; ++s) mbar_init(&bars->v_full[s], 1), mbar_init(&bars->v_empty[s], 1);
      for (int t = 0; t < TILES; ++t) {
        mbar_init(&bars->q_full[t], 1), mbar_init(&bars->q_empty[t], 1);
        mbar_init(&bars->s_full[t], 1), mbar_init(&bars->o_full[t], 1);
      }
      for (int s = 0; s < 2; ++s) mbar_init(&bars->unit_full[s], 1), mbar_init(&bars->unit_empty[s], UNIT_WARPS);
      mbar_init(&bars->taken, 1);
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
    griddep_wait();
    const uint32_t tmem_base = bars->tmem_base;

    // The next unit, for each warp that works on it. All read the same ones, whatever went wrong (the wait does not look at the abort flag and is
    // longer than those that it follows from), so that the meetings on the way come out even.
    int taken = 0;
    auto unit_there = [&]() {
      const bool got = __all_sync(0xffffffffu, mbar_wait_for(&bars->unit_full[taken & 1], (taken >> 1) & 1u, 8 * KCG_WAIT_LIMIT_NS));
      if (!got && lane == 0) report(bars, PAGED_TIMEOUT_UNIT, static_cast<uint32_t>(taken), warp);
      return got;
    };
    auto unit_read = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->unit_empty[taken & 1]);
      ++taken;
    };
    auto next_unit = [&](Unit* x) {
      if (!unit_there()) return false;
      *x = bars->unit[taken & 1];
      unit_read();
      return x->end == 0;
    };

    // Registers: 384 threads are launched with 168 each; the control warpgroup keeps 56, the softmax warpgroups take
    // 224 (56 + 2 * 224 = 3 * 168), which a row's 128 scores need.
    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      // This lane's box of a tile of K or V: its place in the tile and in shared memory; a load of it from a page (-1: zeros).
      const int boxes = BC >> p.box_log2, loads = boxes * HALVES;  // (at most 32)
      const int box = lane % boxes, half = lane / boxes;
      const uint32_t to = half * BOX_BYTES + (box << p.box_log2) * 128;
      auto page_of = [&](const Unit& x, int j, int* key) {
        const int v = x.v0 + j * BC + (box << p.box_log2);
        *key = x.list.key(v);
        return lane < loads && x.list.seen(v, 1 << p.box_log2, p.sinks) ? p.seq.page_of(x.b, *key) : -1;
      };
      auto load = [&](uint8_t* tile, const CUtensorMap* tm, uint64_t* bar, const Unit& x, int key, int page) {
        if (lane == 0) mbar_expect_tx(bar, KV_BYTES);
        __syncwarp();
        if (lane < loads) tma_load_4d(tile + to, tm, bar, half * 64, key & ((1 << p.seq.page_log2) - 1), x.head, page);
      };
      if (warp == 0) {
        // ------------------------------------------------------------------ loads of Q and K
        uint32_t it = 0, queries[TILES] = {0, 0};  // steps and tiles of queries so far
        bool ok = true;
        // A tile of queries into its place, once the last scores of the one before are done: of tile 0 half a step earlier than of tile 1.
        auto load_queries = [&](const Unit& x, int t) {
          if (lane == 0) {
            mbar_expect_tx(&bars->q_full[t], HALVES * p.tile_tokens * p.group * 128);
#pragma unroll
            for (int b = 0; b < HALVES; ++b)
              tma_load_3d(smem + t * Q_BYTES + b * BOX_BYTES, &p.tmQ, &bars->q_full[t], b * 64, x.head * p.group, x.row0 + t * p.tile_tokens);
          }
          __syncwarp();
        };
        for (Unit x; next_unit(&x);) {
          if (x.steps == 0) continue;
          int key = 0, page = page_of(x, 0, &key), on = 0;  // on: tiles of queries under way
          if (ok && mbar_test_warp(&bars->q_empty[0], (queries[0] & 1u) ^ 1u)) load_queries(x, on++);
          for (int j = 0; j < x.steps; ++j, ++it) {
            const int ks = it % K_STAGES, this_key = key, this_page = page;
            if (ok && j + 1 < x.steps) page = page_of(x, j + 1, &key);
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty[ks], ((it / K_STAGES) & 1u) ^ 1u, &bars->abort_flag));
            if (ok) load(smem + OFF_K + ks * KV_BYTES, &p.tmK, &bars->k_full[ks], x, this_key, this_page);
            if (j == 0) {
#pragma unroll
              for (int t = 0; t < TILES; ++t) {
                if (t >= x.tiles) continue;
                if (ok && on == t) {
                  ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_empty[t], (queries[t] & 1u) ^ 1u, &bars->abort_flag));
                  if (ok) load_queries(x, on++);
                }
                ++queries[t];
              }
            }
            if (!ok && lane == 0) report(bars, PAGED_TIMEOUT_LOADS, it, 0u);
          }
        }
      } else if (warp == 1) {
        // ---------------------------------------------------------------- products
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
        const uint64_t qdesc = make_smem_desc(smem_u32(smem), 16, 1024, SWZ_128B);
        const uint64_t kdesc = make_smem_desc(smem_u32(smem + OFF_K), 16, 1024, SWZ_128B);
        const uint64_t vdesc = make_smem_desc(smem_u32(smem + OFF_V), BOX_BYTES, 1024, SWZ_128B);
        uint32_t it0 = 0, queries[TILES] = {0, 0};  // steps before the current unit's, tiles of queries before its own
        // S_t of step it0 + i, of a unit of `tiles` tiles; `last`: it is the unit's last
        auto issue_s = [&](int t, int i, int tiles, bool last) {
          const uint64_t ad = qdesc + t * (Q_BYTES >> 4), bd = kdesc + ((it0 + i) % K_STAGES) * (KV_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks) {
            const uint32_t in_row = (ks * 32) % 128, box = (ks * 32) / 128;
            umma_ss<false>(tmem + t * BC, ad + ((box * BOX_BYTES + in_row) >> 4), bd + ((box * BOX_BYTES + in_row) >> 4), IDESC_S, ks > 0 ? 1u : 0u);
          }
          umma_commit(&bars->s_full[t]);
          if (last) umma_commit(&bars->q_empty[t]);
          if (t == tiles - 1) umma_commit(&bars->k_empty[(it0 + i) % K_STAGES]);
        };
        auto issue_pv = [&](int t, int j, int ks0, int ks1) {
          const uint64_t vd = vdesc + ((it0 + j) % V_STAGES) * (KV_BYTES >> 4);
#pragma unroll
          for (int ks = 0; ks < BC / 16; ++ks)
            if (ks >= ks0 && ks < ks1)
              umma_ts<false>(tmem + COL_O + t * kD, tmem + t * BC + ks * 8, vd + ((ks * 16 * 128) >> 4), IDESC_O, (j > 0 || ks > 0) ? 1u : 0u);
        };
        int begun = 0;  // tiles of the current unit whose first scores are on their way
        for (bool known = false; known || unit_there();) {
          const int nkv = bars->unit[taken & 1].steps, tiles = bars->unit[taken & 1].tiles;
          const bool end = bars->unit[taken & 1].end != 0;
          unit_read();
          known = false;
          if (end) break;
          if (nkv == 0) continue;
          named_bar_sync(BAR_KV, KV_THREADS);  // the first K tile
          const uint32_t q_parity = (queries[0] & 1u) | (queries[1] & 1u) << 1;
          auto begin = [&](int t) {
            const bool q_there = __all_sync(0xffffffffu, mbar_wait(&bars->q_full[t], q_parity >> t & 1u, &bars->abort_flag));
            if (!q_there && lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, 0u, t);
            __syncwarp();
            tc_fence_after_sync();
            if (elect_one()) issue_s(t, 0, tiles, nkv == 1);
            __syncwarp();
          };
          const int first = kApart && begun == 0 ? 1 : tiles;  // (the second tile's follow the first one's first weights)
#pragma unroll 1
          for (int t = begun; t < first; ++t) begin(t);
          const bool second = first < tiles;
          ++queries[0];
          queries[1] += tiles - 1;
          begun = 0;  // (of the next unit, from here on)
          bool keys_there = false;
          int next_steps = 0, next_tiles = 0;
          for (int j = 0; j < nkv; ++j) {
            named_bar_sync(BAR_KV, KV_THREADS);
            const bool last = j + 1 == nkv;
#pragma unroll 1
            for (int t = 0; t < tiles; ++t) {
              named_bar_sync(BAR_PART + t, PT_THREADS);
              tc_fence_after_sync();
              if (second && j == 0 && t == 0) begin(1);
              if (elect_one()) issue_pv(t, j, 0, P_PART / 16);
              __syncwarp();
              if (last && !known && mbar_test_warp(&bars->unit_full[taken & 1], (taken >> 1) & 1u)) {  // (while the last weights are waited for)
                known = true;
                next_steps = bars->unit[taken & 1].end ? 0 : bars->unit[taken & 1].steps;
                next_tiles = bars->unit[taken & 1].tiles;
              }
              named_bar_sync(BAR_FULL + t, PT_THREADS);
              tc_fence_after_sync();
              if (elect_one()) {
                issue_pv(t, j, P_PART / 16, BC / 16);
                if (t == tiles - 1) umma_commit(&bars->v_empty[(it0 + j) % V_STAGES]);
                if (last) umma_commit(&bars->o_full[t]);
              }
              __syncwarp();
              // The next scores of this tile: of the next step, or of the next unit's first if its operands have come (the other tile has
              // still to finish then, and this one's warps their rows).
              bool ahead = false;
              if (last && next_steps > 0 && t < next_tiles && begun == t) {
                keys_there = keys_there || mbar_test_warp(&bars->k_full[(it0 + nkv) % K_STAGES], ((it0 + nkv) / K_STAGES) & 1u);
                ahead = keys_there && mbar_test_warp(&bars->q_full[t], (t ? queries[1] : queries[0]) & 1u);
                tc_fence_after_sync();
              }
              if (!last || ahead) {
                if (elect_one()) issue_s(t, j + 1, last ? next_tiles : tiles, last ? next_steps == 1 : j + 2 == nkv);
                __syncwarp();
                begun += ahead ? 1 : 0;
              }
            }
          }
          it0 += nkv;
        }
      } else if (warp == 2) {
        // ------------------------------------------- waits for K and V in the issuer's place
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t what, uint32_t i) {
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, &bars->abort_flag));
          if (!ok && lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, what, i);
        };
        uint32_t it = 0;
        for (Unit x; next_unit(&x);) {
          if (x.steps == 0) continue;
          wait(&bars->k_full[it % K_STAGES], (it / K_STAGES) & 1u, 1u, it);
          named_bar_sync(BAR_KV, KV_THREADS);
          for (int j = 0; j < x.steps; ++j, ++it) {
            wait(&bars->v_full[it % V_STAGES], (it / V_STAGES) & 1u, 2u, it);
            // values of keys that none of the rows sees: behind the last one's, and between the sinks and the first one's window
            const int v0 = x.v0 + j * BC;
            const int end = max(0, min(BC, x.list.count - v0)), gap0 = max(0, min(BC, p.sinks - v0)), gap1 = max(0, min(BC, x.list.lo - v0));
            if (end < BC || gap0 < gap1) {
              auto zero = [&](int from, int to) {  // rows of both halves, whole (their 16-byte units in any order)
                for (int u = lane; u < (to - from) * 8 * HALVES; u += 32) {
                  const int r = HALVES == 2 ? u >> 4 : u >> 3, h = HALVES == 2 ? u >> 3 & 1 : 0;
                  *reinterpret_cast<uint4*>(smem + OFF_V + (it % V_STAGES) * KV_BYTES + h * BOX_BYTES + (from + r) * 128 + (u & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
              };
              zero(end, BC);
              zero(gap0, min(gap1, end));
              fence_proxy_async_smem();
            }
            if (j + 1 < x.steps) wait(&bars->k_full[(it + 1) % K_STAGES], ((it + 1) / K_STAGES) & 1u, 1u, it + 1);
            __syncwarp();
            named_bar_sync(BAR_KV, KV_THREADS);
          }
        }
      } else {
        // ------------------------------------------------------------------ loads of V, and the units
        // Units one after the other into two slots. A slot is free once every warp has read the unit in it; what has gone wrong ends the row of units
        // with one that says so, and where a slot does not become free, with none: the warps' wait for it ends by itself.
        uint32_t it = 0, made = 0, asked = 0;
        bool ok = true;
        const Row row(p);
        auto publish = [&](Unit& x) {  // false: the row ends
          if (bars->abort_flag != 0u) x.end = 1;
          const int slot = made & 1;
          const bool free = made < 2 || mbar_wait_for(&bars->unit_empty[slot], ((made >> 1) & 1u) ^ 1u, KCG_WAIT_LIMIT_NS);
          if (!__all_sync(0xffffffffu, free)) {
            if (lane == 0) report(bars, PAGED_TIMEOUT_UNIT, made, 32u);
            return false;
          }
          if (lane == 0) {
            bars->unit[slot] = x;
            mbar_arrive(&bars->unit_full[slot]);
          }
          __syncwarp();
          ++made;
          return x.end == 0;
        };
        auto ask = [&]() {
          if (!kKeySplit && lane == 0) {
            mbar_expect_tx(&bars->taken, 16);
            request_cta(&bars->answer, &bars->taken);
          }
          __syncwarp();
        };
        // the unit behind this one, published
        auto answered = [&]() {
          int index = -1;
          if (!kKeySplit) {
            const bool there = __all_sync(0xffffffffu, mbar_wait(&bars->taken, asked & 1u, &bars->abort_flag));
            ++asked;
            if (there) index = requested_cta(&bars->answer);
            if (!there && lane == 0) report(bars, PAGED_TIMEOUT_UNIT, made, 33u);
            fence_proxy_async_smem();  // (the next answer is written behind this reading)
            __syncwarp();
          }
          Unit next = row.unit(p, index < 0 ? 0 : index, rank);
          if (index < 0) next.end = 1;
          return publish(next);
        };
        bool more;
        {
          Unit first = row.unit(p, static_cast<int>(blockIdx.x) / (kKeySplit ? p.splits : 1), rank);
          more = publish(first);
        }
        while (more) {
          const Unit x = bars->unit[(made - 1) & 1];
          if (x.steps == 0) {
            ask();
            more = answered();
            continue;
          }
          int key = 0, page = page_of(x, 0, &key);
          for (int j = 0; j < x.steps; ++j, ++it) {
            const int vs = it % V_STAGES, this_key = key, this_page = page;
            if (j + 1 < x.steps) page = page_of(x, j + 1, &key);
            if (j == max(0, x.steps - 2)) ask();
            if (ok) {
              ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_empty[vs], ((it / V_STAGES) & 1u) ^ 1u, &bars->abort_flag));
              if (ok) load(smem + OFF_V + vs * KV_BYTES, &p.tmV, &bars->v_full[vs], x, this_key, this_page);
              if (!ok && lane == 0) report(bars, PAGED_TIMEOUT_LOADS, it, 1u);
            }
          }
          more = answered();  // (behind the last V tile, which the products wait for: about a step and a half before the end)
        }
      }
      if constexpr (kKeySplit) {  // the two meetings of the cluster that join the partial results
        __syncwarp();
        cluster_sync_all();
        cluster_sync_all();
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
      // ------------------------------------------------- softmax, correction, epilogue
      const int q = warp & 3;           // TMEM lane quarter this warp may access
      const int t = (warp - 4) >> 2;    // query tile of this warp
      const int row = q * 32 + lane;    // query row of this thread inside its tile
      const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
      const uint32_t col_s = tmem_base + lane_addr + t * BC, col_o = tmem_base + lane_addr + COL_O + t * kD;
      const int in_tile = row / p.group, head_row = row - in_tile * p.group;
      const int token = row < p.tile_tokens * p.group ? t * p.tile_tokens + in_tile : 0x40000000;  // of the unit's (which has less than that)
      const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2);
      uint32_t scores = 0, results = 0;  // of this tile so far
      bool alive = true;                 // no wait of this warp has run out
      while (unit_there()) {
        const Unit& unit = bars->unit[taken & 1];
        if (unit.end) {
          unit_read();
          break;
        }
        const Unit x = unit;
        const bool live = token < x.tokens;
        // places of keys below `see`, of those from `near` on and the sinks; rows without a token (whose scores are of whatever lies there) are not masked
        const int position = x.p_lo + (live ? token : 0);
        const int see = live ? x.list.place(min(position + 1, x.keys)) : 0x7fffffff;
        const int near = live && p.window > 0 && position >= p.window ? position - p.window + 1 - x.list.shift : 0;
        // m: what the exponentials of a step are taken against, in the exp2 domain: the row's running maximum as it was when some row of the warp last
        // passed its own by 8. Weights are up to 2^8 then, which 16 bits hold as exactly as any (P's relative rounding is the same everywhere), and
        // the sums in 32 bits; what is lost is that the largest weight is no longer exactly 1. Error against 64 bits, 2048 tokens, bf16: normal scores 2.02e-3
        // -> 2.05e-3, scores of 4 times that 1.72e-3 -> 1.95e-3, of 16 times 1.44e-3 -> 1.45e-3. A window's nine steps would nearly all rescale O:
        // 16384 tokens with a window of 1024 303 -> 283 us in short bursts, 8192 without one 472 -> 451.
        float m = -INFINITY;
        uint64_t sum2[2] = {f32x2(0.f, 0.f), f32x2(0.f, 0.f)};
        const int mine = t < x.tiles ? x.steps : 0;
        int j = 0;
        for (; j < mine && alive; ++j) {
          alive = __all_sync(0xffffffffu, mbar_wait_for(&bars->s_full[t], scores & 1u, 4 * KCG_WAIT_LIMIT_NS));
          if (!alive) {
            if (lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, 3u, static_cast<uint32_t>(j));
            break;
          }
          ++scores;
          tc_fence_after_sync();
          uint32_t sr[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(col_s + c * 32, sr[c]);
          const int v0 = x.v0 + j * BC;
          const int end = see - v0, gap0 = p.sinks - v0, gap1 = near - v0;
          const bool masked = __any_sync(0xffffffffu, end < BC || (gap1 > 0 && gap0 < BC));
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) pin_32(sr[c]);
          if (masked) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // a bit a key that the row sees (a test of a bit and a select each, where 32 comparisons with three borders are five)
              const uint32_t bits = below(end - c * 32) & (below(gap0 - c * 32) | ~below(gap1 - c * 32));
              if (__any_sync(0xffffffffu, bits != 0xffffffffu)) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(bits >> i & 1u)) sr[c][i] = __float_as_uint(-INFINITY);
              }
            }
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          auto max_of = [&](int c) {
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
          };
#pragma unroll
          for (int c = 0; c < 4; ++c) max_of(c);
          // (the scale is positive: checked by the host)
          const float highest = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
          const bool moved = __any_sync(0xffffffffu, live && highest > m + 8.f);
          if (moved) {
            const float top = fmaxf(m, highest);
            if (__any_sync(0xffffffffu, live && fabsf(top) >= kLargeScores && top > -INFINITY)) break;
          }
          const float mx = moved ? fmaxf(m, highest) : m;
          // (without a finite score so far the probabilities are 0, not -inf - -inf)
          const float base = mx == -INFINITY ? 0.f : mx;
          const float alpha = ex2(m - base);
          m = mx;
          const uint64_t alpha2 = f32x2(alpha, alpha), zero2 = f32x2(0.f, 0.f), base2 = f32x2(-base, -base);
          sum2[0] = fma_f32x2(sum2[0], alpha2, zero2);
          sum2[1] = fma_f32x2(sum2[1], alpha2, zero2);
          // Exponentials and P of 32 keys: packed pairs over the S columns this thread has read.
          auto exponentials = [&](int c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 e = f32x2_split(fma_f32x2(f32x2(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), scale2, base2));
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              sum2[i & 1] = add_f32x2(sum2[i & 1], f32x2(e.x, e.y));
              w[i] = pack_pair<kBf16>(e.x, e.y);
            }
            tmem_st_32x32b_x16(col_s + c * 16, w);
          };
          // O_t <- alpha * O_t, where the warp's rows have another m (the previous P_t V has retired: the scores just read were issued
          // behind it).
          if (j > 0 && moved) {
            auto scale_store = [&](uint32_t (&o)[32], int c) {
              pin_32(o);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 v = f32x2_split(mul_f32x2(f32x2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), alpha2));
                o[i] = __float_as_uint(v.x);
                o[i + 1] = __float_as_uint(v.y);
              }
              tmem_st_32x32b_x32(col_o + c * 32, o);
            };
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(col_o + c * 32, o);
              exponentials(c);
              tmem_ld_wait();
              scale_store(o, c);
            }
            if constexpr (kD == 128) {
              static_assert(P_PART == 96, "the third piece of 32 keys comes before the publication");
              uint32_t o[2][32];
              tmem_ld_32x32b_x32(col_o + 64, o[0]);
              tmem_ld_32x32b_x32(col_o + 96, o[1]);
              exponentials(2);
              tmem_ld_wait();
              scale_store(o[0], 2);
              scale_store(o[1], 3);
            }
          } else {
            exponentials(0);
            exponentials(1);
            if constexpr (P_PART == 96) exponentials(2);
          }
          auto publish = [&](uint32_t bar) {
            tmem_st_wait();
            tc_fence_before_sync();
            named_bar_arrive(bar, PT_THREADS);
          };
          publish(BAR_PART + t);
          if constexpr (P_PART == 64) exponentials(2);
          exponentials(3);
          publish(BAR_FULL + t);
        }
        // Steps from the first one on in which a row of the warp has large scores (see kLargeScores): products rounded first, against the exact maximum.
        // (A loop of its own costs the one above nothing; as a branch in its steps this cost them 1.8 to 3.5 %, six ways.)
        for (bool there = true; j < mine && alive; ++j, there = false) {
          if (!there) {
            alive = __all_sync(0xffffffffu, mbar_wait_for(&bars->s_full[t], scores & 1u, 4 * KCG_WAIT_LIMIT_NS));
            if (!alive) {
              if (lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, 3u, static_cast<uint32_t>(j));
              break;
            }
            ++scores;
            tc_fence_after_sync();
          }
          const int v0 = x.v0 + j * BC;
          auto load = [&](int c, uint32_t (&y)[32]) {  // 32 scores times the scale
            tmem_ld_32x32b_x32(col_s + c * 32, y);
            tmem_ld_wait();
            pin_32(y);
            const uint32_t bits = below(see - v0 - c * 32) & (below(p.sinks - v0 - c * 32) | ~below(near - v0 - c * 32));
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(bits >> i & 1u ? __fmul_rn(__uint_as_float(y[i]), p.scale_log2) : -INFINITY);
          };
          float mx = m;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t y[32];
            load(c, y);
#pragma unroll
            for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(y[i]));
          }
          const float base = mx == -INFINITY ? 0.f : mx, alpha = ex2(m - base);
          m = mx;
          float sum = 0.f;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {  // (P of a piece lies where scores were that have been read)
            uint32_t y[32], w[16];
            load(c, y);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              y[i] = __float_as_uint(ex2(__uint_as_float(y[i]) - base));
              sum += __uint_as_float(y[i]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack_pair<kBf16>(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
            tmem_st_32x32b_x16(col_s + c * 16, w);
            tmem_st_wait();
          }
#pragma unroll 1
          for (int c = 0; j > 0 && c < kD / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(col_o + c * 32, o);
            tmem_ld_wait();
            pin_32(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x32(col_o + c * 32, o);
          }
          sum2[0] = fma_f32x2(sum2[0], f32x2(alpha, alpha), f32x2(sum, 0.f));
          sum2[1] = mul_f32x2(sum2[1], f32x2(alpha, alpha));
          tmem_st_wait();
          tc_fence_before_sync();
          named_bar_arrive(BAR_PART + t, PT_THREADS);
          named_bar_arrive(BAR_FULL + t, PT_THREADS);
        }
        for (; j < mine; ++j) {  // (given up)
          __syncwarp();
          named_bar_sync(BAR_PART + t, PT_THREADS);
          named_bar_sync(BAR_FULL + t, PT_THREADS);
        }
        const float2 s01 = f32x2_split(add_f32x2(sum2[0], sum2[1]));
        const float l = s01.x + s01.y;
        if (mine > 0 && alive) {
          alive = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[t], results & 1u, &bars->abort_flag));
          if (!alive && lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, 4u, 0u);
          ++results;
        }
        const bool gave_up = mine > 0 && !alive;
        if constexpr (kKeySplit) {
          // Partial results: once the products of both tiles have retired, the operand ring holds this CTA's O rows (fp32, not normalised,
          // 16-byte units XOR-swizzled by the row: a warp writes 32 rows at a time) and their {maximum, sum}; then each CTA joins an equal
          // share of the output over the cluster's shared memories.
          constexpr int UNITS = kD / 4;  // 16-byte units of a row
          constexpr int OFF_ML = TILES * BR * kD * 4;
          static_assert(OFF_ML + TILES * BR * 8 <= RING_BYTES, "the partial result must fit the ring");
          bool both = true;
          if (mine > 0 && !gave_up && x.tiles == 2) {
            both = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[t ^ 1], 0u, &bars->abort_flag));
            if (!both && lane == 0) report(bars, PAGED_TIMEOUT_ATTENTION, 5u, 0u);
          }
          if (t < x.tiles && both && !gave_up) {
            tc_fence_after_sync();
            const int r = t * BR + row;
            uint8_t* to = smem + r * kD * 4;
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) {
              uint32_t o[32];
              if (mine > 0) {
                tmem_ld_32x32b_x32(col_o + c * 32, o);
                tmem_ld_wait();
                pin_32(o);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0u;
              }
#pragma unroll
              for (int u = 0; u < 8; ++u)
                *reinterpret_cast<uint4*>(to + (((c * 8 + u) ^ (r & (UNITS - 1))) << 4)) = make_uint4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
            }
            reinterpret_cast<float2*>(smem + OFF_ML)[r] = make_float2(m, l);
          }
          __syncwarp();
          cluster_sync_all();
          {
            // This CTA's rows, as many to a warp: a lane first takes the weights of one of them, then the warp whole rows (d = 64: two), four loads of other CTAs'
            // rows in flight for each of them. (An element at a time, with its row's weights each time, was 13 us of latency for two CTAs.)
            const int all = x.tiles * BR, r0 = all * rank / p.splits, r1 = all * (rank + 1) / p.splits;
            const int per = (r1 - r0 + 7) / 8, first = r0 + (warp - 4) * per, mine_rows = max(0, min(per, r1 - first));  // (at most 16)
            const uint32_t base_addr = smem_u32(smem);
            float f[8], inv = 0.f;
            {
              const uint32_t ml_addr = base_addr + OFF_ML + (first + min(lane, max(mine_rows - 1, 0))) * 8;
              float2 ml[8];
              float top = -INFINITY, sum = 0.f;
#pragma unroll
              for (int c = 0; c < 8; ++c) ml[c] = c < p.splits && mine_rows > 0 ? ld_cluster_f2(map_to_cta(ml_addr, c)) : make_float2(-INFINITY, 0.f);
#pragma unroll
              for (int c = 0; c < 8; ++c) top = fmaxf(top, ml[c].x);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                f[c] = ml[c].y == 0.f ? 0.f : ex2(ml[c].x - top);  // (a part of no key; a sum of NaN has to reach the result)
                sum = fmaf(f[c], ml[c].y, sum);
              }
              inv = sum == 0.f ? 0.f : 1.f / sum;
            }
            constexpr int ROWS = 128 / kD, AT_ONCE = 4;  // rows a warp takes with one load, loads in flight
            const int u = lane % UNITS;
            for (int k0 = 0; k0 < mine_rows; k0 += ROWS * AT_ONCE) {
              float4 sums[AT_ONCE];
#pragma unroll
              for (int i = 0; i < AT_ONCE; ++i) sums[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                if (c >= p.splits) break;
                float4 v[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                  const int r = first + min(k0 + i * ROWS + lane / UNITS, mine_rows - 1);
                  v[i] = ld_cluster_f4(map_to_cta(base_addr + r * kD * 4 + ((u ^ (r & (UNITS - 1))) << 4), c));
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                  const float w = __shfl_sync(0xffffffffu, f[c], min(k0 + i * ROWS + lane / UNITS, mine_rows - 1));
                  if (w == 0.f) continue;  // (what a part of no key holds)
                  sums[i].x = fmaf(w, v[i].x, sums[i].x), sums[i].y = fmaf(w, v[i].y, sums[i].y);
                  sums[i].z = fmaf(w, v[i].z, sums[i].z), sums[i].w = fmaf(w, v[i].w, sums[i].w);
                }
              }
#pragma unroll
              for (int i = 0; i < AT_ONCE; ++i) {
                const int k = k0 + i * ROWS + lane / UNITS, r = first + k, in_tile = r % BR;
                const float scale = __shfl_sync(0xffffffffu, inv, min(k, mine_rows - 1));
                const int tok = r / BR * p.tile_tokens + in_tile / p.group;
                if (k >= mine_rows || in_tile >= p.tile_tokens * p.group || tok >= x.tokens) continue;
                T* out = reinterpret_cast<T*>(p.o) + static_cast<long long>(unit.row0 + tok) * p.o_row +
                         static_cast<long long>(unit.head * p.group + in_tile % p.group) * p.o_head + u * 4;
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_pair<kBf16>(sums[i].x * scale, sums[i].y * scale), pack_pair<kBf16>(sums[i].z * scale, sums[i].w * scale));
              }
            }
          }
          __syncwarp();
          cluster_sync_all();  // the other CTAs read this one's shared memory until here
        } else {
          tc_fence_after_sync();
          const float inv = mine == 0 || l == 0.f ? 0.f : 1.f / l;
          // (this thread's row, from the result's first byte on; -1: none)
          const long long at = live ? static_cast<long long>(unit.row0 + token) * p.o_row + static_cast<long long>(unit.head * p.group + head_row) * p.o_head : -1;
          uint8_t* stage = smem + RING_BYTES + (warp - 4) * (32 * 128);
          uint32_t o[kD / 32][32];
          if (mine > 0 && !gave_up) {
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) tmem_ld_32x32b_x32(col_o + c * 32, o[c]);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) pin_32(o[c]);
          } else {
#pragma unroll
            for (int i = 0; i < kD; ++i) o[i / 32][i % 32] = 0u;
          }
#pragma unroll
          for (int c2 = 0; c2 < HALVES; ++c2) {
            __syncwarp();  // (the warp has read what the last round left here)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_pair<kBf16>(__uint_as_float(o[c2 * 2 + u / 4][u % 4 * 8 + 2 * e]) * inv, __uint_as_float(o[c2 * 2 + u / 4][u % 4 * 8 + 2 * e + 1]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int r = k * 4 + lane / 8, u = lane & 7;
              v[k] = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const long long to = __shfl_sync(0xffffffffu, at, k * 4 + lane / 8);
              if (to >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + to + c2 * 64 + (lane & 7) * 8) = v[k];
            }
          }
        }
        unit_read();
      }  // (units; a cluster has one, and its meetings are in it)
    }

    // ---------------------------------------------------------------- common exit
    __syncwarp();
    if (bars->abort_flag != 0u) {  // loads and products still in flight end before their memory is given up
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

template <int kD, bool kBf16, bool kKeySplit>
__global__ void __launch_bounds__(384, 1) attention_prompt_kernel(const __grid_constant__ PromptArgs p) {
  AttnPrompt<kD, kBf16, kKeySplit>::run(p);
}
