// Attention of many query rows per sequence -- prompts and chunks of new tokens -- on the
// 5th-generation tensor cores: S = Q K^T and O += P V by tcgen05, S, P and O in TMEM.
//
// The query rows of one key/value head are packed into tiles of 128: row = token x group
// + head of the group (floor(128 / group) tokens per tile), so the heads of a group share
// every K / V tile and a chunk of few tokens still fills the tensor core's 128 lanes.
// Keys come in tiles of 128 from packed rows or from the pages of a cache (one TMA box per
// page piece and 64 columns).
//
// Three kernels:
//   tile_plan_kernel  one block turns the device-side offsets and lengths into a work list,
//                     longest items first.  An item is NT query tiles of one head.  Items
//                     that would leave CTAs idle -- those of a last, partial wave, and any
//                     longer than a CTA's fair share -- are cut along the keys.
//   tile_kernel       persistent CTAs (1 per SM) take items in turn: a TMA loader; per query
//                     tile four softmax warps (one thread per row) and two MMA-issuing warps
//                     (one at head_dim 256); and a warp that prepares V tiles; running
//                     statistics in fp32, O rescaled only when a row's maximum grew by
//                     more than 2^8.
//   tile_join_kernel  joins the pieces of cut items in the order of their keys.
//
// Hidden keys.  Scores of keys a row does not see are replaced by -inf.  Their values still
// meet P = 0 in the product, and 0 x NaN is NaN.  V rows behind the last key (stale pages, the
// next sequence) are zeroed in shared memory.  For the others the result is looked at: a row
// that is not finite may owe it to a value that it does not see, so the joining kernel searches
// its hidden values, and computes the columns in which one is not finite again, key by key.
// (Searching every V tile on the diagonal for such values took a warp 2000 cycles per tile,
// in which the tile's product waited: prompts of 128 - 256 tokens.)
//
// Every wait is bounded; a role that gives up records SRV_DEV_TIMEOUT and unwinds.
#pragma once
#include "attention_tc.cuh"
#include "serve_dev.cuh"

namespace tttj {

struct TileInfo {  // one decoded item, in shared memory
  int b, q, h, row0, n, len, tok0, part;
  int j0;     // first key tile of this piece
  int n_kv;   // key tiles of this piece; -1: no more items
  int ns[2];  // softmax steps of query tile 0 / 1 inside this piece
};
static_assert(sizeof(TileInfo) <= 64, "item info slot is 64 bytes");

// TMEM (512 columns) holds, per query tile, the scores of a step (fp32, a column per key), the
// probabilities (16 bits, half a column per key) and O (head_dim columns).  Up to head_dim 128
// a step is 64 keys, with two buffers of probabilities: nothing shares columns, S of the next step
// is computed while the softmax works on this one, and the softmax waits for no product.
// Measured at head_dim 128, prompts of 3001 and 4096 tokens, 32 / 8 heads: steps of 128 keys with P
// written over S, as in attention_tc.cuh, 286 us (the next S waits for P V); one score buffer of
// 128 keys that the tiles take in turn 250 - 258; steps of 64 with one issuing warp per tile
// 257, with one for S and one for P V 251; the wait for the P buffer moved to the issuer 227
// against 233; no exponentials on the FMA pipe 223 (a quarter: 227, 3/8: 233, 1/2: 242; issue
// slots are as scarce as the MUFU); scores read twice from TMEM in rolled loops, S double-buffered
// and P over it, 244 against 215.  At head_dim 64, 256 prompts of 128 - 256 tokens: steps of 128
// keys 150 us, of 64 keys 127.  At head_dim 256 (one query tile per item) steps of 128 keys and one
// buffer of P: 111 against 182 us, prompts of 3000 and 4096 tokens, 8 / 2 heads.
// What bounds it: with nearly all products left out the same prompts take 186 us, so the
// softmax warps do, two per scheduler; MUFU and tensor pipe are 51 % busy each.
template <int HD>
struct TileSmem : AtcSmem<HD> {  // tile sizes and stages as there
  using B = AtcSmem<HD>;
  static constexpr bool SPLIT = HD != 256;        // S and P V issued by different warps
  static constexpr int KT = HD == 256 ? 128 : 64;  // keys per step
  static constexpr int SUB = ATC_BN / KT;          // steps per loaded key tile
  static constexpr int PBUF = HD == 256 ? 1 : 2;
  // Warps: four softmax warps per query tile (their number modulo four is their TMEM
  // quadrant), the loader, the MMA issuers, the cleaner.
  static constexpr int LOADER = 4 * B::NT, ISSUER = LOADER + 1;
  static constexpr int CLEANER = ISSUER + (SPLIT ? 2 : 1) * B::NT;
  static constexpr int THREADS = 32 * (CLEANER + 1);
  __host__ __device__ static constexpr uint32_t s_col(int t) { return (uint32_t)(t * KT); }
  __host__ __device__ static constexpr uint32_t p_col(int t) { return (uint32_t)(B::NT * KT + t * PBUF * KT / 2); }
  __host__ __device__ static constexpr uint32_t o_col(int t) { return t == 0 ? B::TMEM_O0 : B::TMEM_O1; }
  static_assert(B::NT * (KT + PBUF * KT / 2) <= (int)B::TMEM_O0, "TMEM columns overlap");
  static constexpr int BARS = 4 * B::QS + 5 * B::STAGES + 8 + 4 + 4 + 4;
  static constexpr int BAR_AT = B::Q_BYTES + B::KV_BYTES;
  static constexpr int SLOT_AT = BAR_AT + BARS * 8;  // TMEM base, abort flag
  static constexpr int INFO_AT = SLOT_AT + 16;       // [side][QS] items
  static constexpr int ALL = INFO_AT + 2 * B::QS * 64 + 1024;
};

constexpr int TILE_MIN_PIECE = 4;  // key tiles (512 keys) a cut piece has at least

// Keys that the tokens [tok0, tok0 + tokens) of a sequence see (their last one's limit).
__device__ __forceinline__ int tile_kv_end(const SrvSeq& q, int causal, int tok0, int tokens) {
  if (!causal) return q.len;
  const int last = min(tok0 + tokens, q.n) - 1;
  return max(0, min(q.len, q.len - q.n + last + 1));
}
__device__ __forceinline__ int tile_kv_tiles(int kv_end) { return max(1, (kv_end + ATC_BN - 1) / ATC_BN); }

// ------------------------------------------------------------------------------ plan
constexpr int TILE_PLAN_THREADS = 1024;
constexpr int TILE_BUCKETS = 1024;

__global__ void __launch_bounds__(TILE_PLAN_THREADS) tile_plan_kernel(const TileParams p, int nt, int grid) {
  __shared__ int s_pre[SRV_MAX_BATCH + 1];  // items before each sequence
  __shared__ int s_row0[SRV_MAX_BATCH], s_n[SRV_MAX_BATCH], s_len[SRV_MAX_BATCH];
  __shared__ int s_hist[TILE_BUCKETS];
  __shared__ int s_warp[32];
  __shared__ unsigned long long s_sum[2][32];  // key tiles of all items / of those in the last wave
  __shared__ int s_joins, s_parts, s_entries;
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, batch = p.s.batch;
  const int item_tokens = nt * p.tile_tokens;
  if (tid == 0) s_joins = s_parts = s_entries = 0;
  s_hist[tid] = 0;
  // Two sequences per thread: items, then their prefix sums.
  int cnt[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * tid + i;
    if (b < batch) {
      const SrvSeq q = srv_seq(p.s, b);
      s_row0[b] = q.row0;
      s_n[b] = q.n;
      s_len[b] = q.len;
      cnt[i] = (q.n + item_tokens - 1) / item_tokens;
    }
  }
  // Sums saturate: offsets that do not rise may claim more items than there are rows for.
  constexpr int FULL_SUM = 1 << 29;
  int x = min(cnt[0], FULL_SUM / 2) + min(cnt[1], FULL_SUM / 2);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, x, d);
    if ((tid & 31) >= d) x = min(x + o, FULL_SUM);
  }
  if ((tid & 31) == 31) s_warp[tid >> 5] = x;
  __syncthreads();
  if (tid < 32) {
    int w = s_warp[tid];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, d);
      if (tid >= d) w = min(w + o, FULL_SUM);
    }
    s_warp[tid] = w;
  }
  __syncthreads();
  const bool rising = s_warp[31] <= p.s.tokens / item_tokens + batch;
  if (!rising) {
    if (tid == 0) {
      report_status(p.s.status, SRV_DEV_BAD_LENS);
      p.plan.counters[0] = p.plan.counters[1] = p.plan.counters[2] = p.plan.counters[3] = 0;
    }
    return;
  }
  const int before = (tid >= 32 ? s_warp[(tid >> 5) - 1] : 0) + x - cnt[0] - cnt[1];
  if (2 * tid <= batch) s_pre[2 * tid] = before;
  if (2 * tid + 1 <= batch) s_pre[2 * tid + 1] = before + cnt[0];
  if (tid == 0) s_pre[batch] = s_warp[31];
  __syncthreads();
  const int items = s_pre[batch];  // per key/value head
  auto locate = [&](int e, int* b) {
    int lo = 0, hi = batch - 1;  // last b with s_pre[b] <= e
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_pre[mid] <= e) lo = mid; else hi = mid - 1;
    }
    *b = lo;
    return e - s_pre[lo];
  };
  auto tiles_of = [&](int b, int q) {
    SrvSeq s;
    s.n = s_n[b];
    s.len = s_len[b];
    return tile_kv_tiles(tile_kv_end(s, p.s.causal, q * item_tokens, item_tokens));
  };
  // Item e: sequence, item of the sequence, key tiles.  A thread's first is found once.
  struct Item {
    int b, q, t;
  };
  auto find = [&](int e) {
    Item i;
    i.q = locate(e, &i.b);
    i.t = tiles_of(i.b, i.q);
    return i;
  };
  Item own{};
  if (tid < items) own = find(tid);
  auto item = [&](int e) { return e == tid ? own : find(e); };
  // Quotients in 32 bits where they fit: a 64-bit division is a few hundred cycles of latency.
  auto share = [&](unsigned long long x) {  // of all heads' x per CTA, rounded up
    x = x * p.kv_heads + grid - 1;
    return x >> 32 ? (int)(x / grid) : (int)((unsigned)x / (unsigned)grid);
  };
  // Whole waves of items stay whole; with at least four waves the last one is short
  // against the rest.  Which items are cut depends on their number alone, not on the
  // order in which threads run: results repeat exactly.
  const bool many = (long)items * p.kv_heads >= 4l * grid;
  const int whole = many ? items : items * p.kv_heads / grid * grid / p.kv_heads;
  unsigned long long sum = 0, rest = 0;
  for (int e = tid; e < items; e += TILE_PLAN_THREADS) {
    const int t = item(e).t;
    sum += t;
    if (e >= whole) rest += t;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    rest += __shfl_xor_sync(0xffffffffu, rest, d);
  }
  if ((tid & 31) == 0) {
    s_sum[0][tid >> 5] = sum;
    s_sum[1][tid >> 5] = rest;
  }
  __syncthreads();
  sum = s_sum[0][tid & 31];
  rest = s_sum[1][tid & 31];
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    rest += __shfl_xor_sync(0xffffffffu, rest, d);
  }
  const int most = max(share(sum), TILE_MIN_PIECE), most_rest = max(share(rest), TILE_MIN_PIECE);
  // Adds n to a bucket, returns what it held: lanes of one bucket share one atomic.
  auto add_to = [&](int at, int n) {
    const unsigned active = __activemask();
    const unsigned same = __match_any_sync(active, at);
    if (__all_sync(active, n == 1)) {
      const int leader = __ffs(same) - 1;
      int base = 0;
      if ((tid & 31) == leader) base = atomicAdd(&s_hist[at], __popc(same));
      return __shfl_sync(active, base, leader) + __popc(same & ((1u << (tid & 31)) - 1));
    }
    return atomicAdd(&s_hist[at], n);
  };
  auto pieces_of = [&](int e, int t) {
    const int c = e >= whole ? min(most, most_rest) : most;
    // A whole item a little above the fair share costs less than its pieces' joining.
    return t <= (e < whole ? most + most / 4 : c) ? 1 : (t + c - 1) / c;
  };
  auto bucket = [&](int len) { return TILE_BUCKETS - min(len, TILE_BUCKETS); };  // longest first
  for (int e = tid; e < items; e += TILE_PLAN_THREADS) {
    const int t = item(e).t, n = pieces_of(e, t);
    add_to(bucket(n == 1 ? t : (t + n - 1) / n), n);
  }
  __syncthreads();
  {
    const int v = s_hist[tid];
    int y = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, y, d);
      if ((tid & 31) >= d) y += o;
    }
    if ((tid & 31) == 31) s_warp[tid >> 5] = y;
    __syncthreads();
    if (tid < 32) {
      int w = s_warp[tid];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, w, d);
        if (tid >= d) w += o;
      }
      s_warp[tid] = w;
    }
    __syncthreads();
    const int base = (tid >= 32 ? s_warp[(tid >> 5) - 1] : 0) + y - v;
    s_hist[tid] = base;
    if (tid == TILE_PLAN_THREADS - 1) s_entries = base + v;
  }
  __syncthreads();
  for (int e = tid; e < items; e += TILE_PLAN_THREADS) {
    TileEntry out{};
    const Item i = item(e);
    out.b = i.b;
    out.q = i.q;
    out.row0 = s_row0[out.b];
    out.n = s_n[out.b];
    out.len = s_len[out.b];
    const int t = i.t, n = pieces_of(e, t);
    int part = -1;
    if (n > 1) {
      part = atomicAdd(&s_parts, n * p.kv_heads);
      p.plan.joins[atomicAdd(&s_joins, 1)] = TileJoin{out.b, out.q, n, part, out.row0, out.n, {0, 0}};
    }
    const int at = add_to(bucket(n == 1 ? t : (t + n - 1) / n), n);
    for (int x = 0; x < n; ++x) {
      out.j0 = n == 1 ? 0 : (int)((long)t * x / n);
      out.j1 = n == 1 ? t : (int)((long)t * (x + 1) / n);
      out.part = n > 1 ? part + x * p.kv_heads : -1;
      p.plan.entries[at + x] = out;
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.plan.counters[0] = 0;
    p.plan.counters[1] = s_entries;
    p.plan.counters[2] = s_joins;
    p.plan.counters[3] = 0;
  }
}

// -------------------------------------------------------------------------- attention
template <int HD, bool BF16>
__global__ void __launch_bounds__(TileSmem<HD>::THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const TileParams p) {
  using SM = TileSmem<HD>;
  constexpr int STAGES = SM::STAGES;
  constexpr int NT = SM::NT;
  constexpr int QBUF = SM::QBUF;
  constexpr int LOADER = SM::LOADER, ISSUER = SM::ISSUER, CLEANER = SM::CLEANER;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  const uint32_t sQ = smem_u32(smem);     // [side][QBUF]
  const uint32_t sK = sQ + SM::Q_BYTES;   // [STAGES]
  const uint32_t sV = sK + STAGES * SM::KV_TILE;
  const uint32_t bar_q_full = sQ + SM::BAR_AT;              // [side][QS]
  const uint32_t bar_q_empty = bar_q_full + 16 * SM::QS;    // [side][QS]
  const uint32_t bar_k_full = bar_q_empty + 16 * SM::QS;    // [STAGES]
  const uint32_t bar_k_empty = bar_k_full + 8 * STAGES;     // [STAGES]
  const uint32_t bar_v_full = bar_k_empty + 8 * STAGES;     // [STAGES]
  const uint32_t bar_v_ready = bar_v_full + 8 * STAGES;     // [STAGES] landed and cleaned
  const uint32_t bar_v_empty = bar_v_ready + 8 * STAGES;    // [STAGES]
  const uint32_t bar_s_full = bar_v_empty + 8 * STAGES;     // [side] ...
  const uint32_t bar_p_full = bar_s_full + 16;              // [side][2] P buffer 0 / 1 written
  const uint32_t bar_o_full = bar_p_full + 32;
  const uint32_t bar_o_free = bar_o_full + 16;
  const uint32_t bar_s_free = bar_o_free + 16;              // scores read by softmax
  const uint32_t bar_pv_done = bar_s_free + 16;             // [side][2] P V of P buffer 0 / 1 complete
  const uint32_t bar_drain = bar_pv_done + 32;              // [issuer]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::SLOT_AT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  TileInfo* info = reinterpret_cast<TileInfo*>(smem + SM::INFO_AT);  // [side][QS]

  const int warp = warp_id();
  const int lane = lane_id();
  constexpr uint64_t limit = SRV_WAIT_LIMIT_NS;
  const int TOK = p.tile_tokens;
  const bool paged = p.s.table != nullptr;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int i = 0; i < 2 * SM::QS; ++i) {
      mbar_init(bar_q_full + 8 * i, 1);
      // The issuers, the softmax warps, and for side 0 the cleaner.
      mbar_init(bar_q_empty + 8 * i, (SM::SPLIT ? 2 : 1) + 4 + (i < SM::QS ? 1 : 0));
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(bar_k_full + 8 * i, 1);
      mbar_init(bar_k_empty + 8 * i, NT);
      mbar_init(bar_v_full + 8 * i, 1);
      mbar_init(bar_v_ready + 8 * i, 1);
      mbar_init(bar_v_empty + 8 * i, NT);
    }
    for (int i = 0; i < 2; ++i) {  // softmax side: one arrival per warp
      mbar_init(bar_s_full + 8 * i, 1);
      mbar_init(bar_p_full + 16 * i, 4);
      mbar_init(bar_p_full + 16 * i + 8, 4);
      mbar_init(bar_o_full + 8 * i, 1);
      mbar_init(bar_o_free + 8 * i, 4);
      mbar_init(bar_s_free + 8 * i, 4);
      mbar_init(bar_pv_done + 16 * i, 1);
      mbar_init(bar_pv_done + 16 * i + 8, 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(bar_drain + 8 * i, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUER) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  griddep_wait();
  griddep_launch();
  const long n_items = (long)p.plan.counters[1] * p.kv_heads;

  if (warp == LOADER) {
    // ------------------------------------------------------------ TMA loader
    // The whole warp runs the loop: each lane issues the boxes of its page pieces.
    constexpr unsigned FULL = 0xffffffffu;
    const int cr = paged ? min(ATC_BN, 1 << p.s.page_shift) : ATC_BN;
    const int boxes = (ATC_BN / cr) * SM::NBOX;  // of K or of V, <= 32
    const int box_x = lane % SM::NBOX, piece = lane / SM::NBOX;
    const uint32_t box_at = (uint32_t)(box_x * SM::BOX_BYTES + piece * cr * SM::BOX_COLS * 2);
    const uint32_t q_bytes = (uint32_t)(TOK * p.group * HD * 2);
    bool ok = true;
    long kc = 0, vc = 0;  // K / V tiles issued
    int k = 0, sides = 0;  // items (including the final "no more items" marker), sides of it published
    bool v_due = false;    // the V tile of the K tile loaded last
    int v_c1 = 0, v_h = 0, v_page = 0;
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
      ok = __all_sync(FULL, srv_wait(bar, parity, abort_flag, limit));
      return ok;
    };
    auto load_v = [&]() -> bool {
      if (!v_due) return true;
      v_due = false;
      const int vs = (int)(vc % STAGES);
      if (!wait(bar_v_empty + 8 * vs, (uint32_t)((vc / STAGES) & 1) ^ 1u)) return false;
      if (lane == 0) mbar_arrive_expect_tx(bar_v_full + 8 * vs, SM::KV_TILE);
      __syncwarp();
      if (lane < boxes)
        tma_load_4d(sV + vs * SM::KV_TILE + box_at, &tmV, bar_v_full + 8 * vs, box_x * SM::BOX_COLS, v_c1, v_h, v_page);
      __syncwarp();
      ++vc;
      return true;
    };
    // The next item's number is taken two tiles before this one is loaded (early enough to
    // hide the counter's latency, late enough to go to a CTA that is free), its entry right after.
    auto take = [&] { return lane == 0 ? atomicAdd(p.plan.counters, 1) : 0; };
    auto fetch = [&](int it, int4* lo, int4* hi) {
      if (it < n_items) {
        const int4* e = reinterpret_cast<const int4*>(p.plan.entries + it / p.kv_heads);
        *lo = e[0];
        *hi = e[1];
      }
    };
    int taken = take();
    int it = __shfl_sync(FULL, taken, 0);
    int4 lo{}, hi{};
    fetch(it, &lo, &hi);
    for (;; ++k) {
      const bool stop = it >= n_items;
      TileInfo w{};
      w.n_kv = -1;
      if (!stop) {
        w.b = lo.x;
        w.q = lo.y;
        w.j0 = lo.z;
        const int j1 = lo.w;
        w.h = it % p.kv_heads;
        w.part = hi.x < 0 ? -1 : hi.x + w.h;
        w.row0 = hi.y;
        w.n = hi.z;
        w.len = hi.w;
        w.tok0 = w.q * NT * TOK;
        w.n_kv = 0;
        const SrvSeq s{w.row0, w.n, w.len};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int t0 = w.tok0 + t * TOK;
          const int steps = max(1, (tile_kv_end(s, p.s.causal, t0, TOK) + SM::KT - 1) / SM::KT);
          w.ns[t] = t0 < w.n ? max(0, min(steps, j1 * SM::SUB) - w.j0 * SM::SUB) : 0;
          w.n_kv = max(w.n_kv, (w.ns[t] + SM::SUB - 1) / SM::SUB);
        }
      }
      const int qb = k % QBUF;
      // Hand the item to a side: its query tile and the item's fields.
      auto publish = [&](int t) -> bool {
        const uint32_t full = bar_q_full + 8 * (t * SM::QS + qb);
        if (!wait(bar_q_empty + 8 * (t * SM::QS + qb), ((k / QBUF) & 1) ^ 1u)) return false;
        if (lane == 0) {
          info[t * SM::QS + qb] = w;  // published by the release of the arrive below
          const int tok0 = w.tok0 + atc_query_tile<NT>(t, k) * TOK;
          if (stop || tok0 >= w.n) {
            mbar_arrive(full);
          } else {
            mbar_arrive_expect_tx(full, q_bytes);
            for (int x = 0; x < SM::NBOX; ++x)
              tma_load_3d(sQ + (t * QBUF + qb) * SM::Q_TILE + x * SM::BOX_BYTES, &tmQ, full, x * SM::BOX_COLS,
                          w.h * p.group, w.row0 + tok0);
          }
        }
        __syncwarp();
        sides = t + 1;
        return true;
      };
      sides = 0;
      // K runs one tile ahead of V: a K stage is free as soon as its scores are computed, and
      // waiting behind a V stage would make the next scores late.
      if (!publish(0)) break;
      for (int j = 0; j < w.n_kv; ++j) {
        if (j == max(0, w.n_kv - 2)) taken = take();
        const int slot = (w.j0 + j) * ATC_BN + piece * cr;
        int page = 0, c1 = w.row0 + slot;
        if (paged) {  // fetched before the wait for the stage
          page = lane < boxes && slot < w.len ? srv_page(p.s, w.b, slot) : p.s.num_pages;
          c1 = slot & ((1 << p.s.page_shift) - 1);
        }
        const int ks = (int)(kc % STAGES);
        if (!wait(bar_k_empty + 8 * ks, (uint32_t)((kc / STAGES) & 1) ^ 1u)) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_k_full + 8 * ks, SM::KV_TILE);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(sK + ks * SM::KV_TILE + box_at, &tmK, bar_k_full + 8 * ks, box_x * SM::BOX_COLS, c1, w.h, page);
        __syncwarp();
        ++kc;
        if (!load_v()) break;  // the tile before
        v_c1 = c1;
        v_h = w.h;
        v_page = page;
        v_due = true;
        if (NT == 2 && j == 0 && !publish(1)) break;
      }
      if (!ok || !load_v()) break;
      if (stop) {
        if (NT == 2) publish(1);
        break;
      }
      it = __shfl_sync(FULL, taken, 0);
      fetch(it, &lo, &hi);
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      // Let issued loads land before the CTA can exit.
      for (long j = kc > STAGES ? kc - STAGES : 0; j < kc; ++j)
        srv_wait(bar_k_full + 8 * (int)(j % STAGES), (uint32_t)((j / STAGES) & 1), nullptr, limit);
      for (long j = vc > STAGES ? vc - STAGES : 0; j < vc; ++j)
        srv_wait(bar_v_full + 8 * (int)(j % STAGES), (uint32_t)((j / STAGES) & 1), nullptr, limit);
      for (int t = 0; t < NT; ++t) {
        const int done = k + (t < sides ? 1 : 0);  // items handed to this side
        for (int i = done > QBUF ? done - QBUF : 0; i < done; ++i)
          srv_wait(bar_q_full + 8 * (t * SM::QS + i % QBUF), (uint32_t)((i / QBUF) & 1), nullptr, limit);
      }
    }
  } else if (warp < CLEANER && warp >= ISSUER) {
    // ------------------------------------------------------------ MMA issuers
    // As in attention_tc.cuh: the whole warp runs the loop, one elected lane issues.
    constexpr unsigned FULL = 0xffffffffu;
    constexpr uint32_t idesc_s = idesc_f16_f32(ATC_BM, SM::KT, 0, 0, BF16);
    constexpr uint32_t idesc_o = idesc_f16_f32(ATC_BM, HD, 0, 1, BF16);
    constexpr uint32_t v_step = HD == 32 ? (1024u >> 4) : (2048u >> 4);  // 16 keys
    constexpr uint32_t sub_bytes = SM::KT * SM::BOX_COLS * 2;            // a step's rows of a box
    const int t = SM::SPLIT ? (warp - ISSUER) >> 1 : warp - ISSUER;
    const bool does_s = !SM::SPLIT || ((warp - ISSUER) & 1) == 0;
    const uint32_t s_col = tmem + SM::s_col(t), p_col = tmem + SM::p_col(t), o_col = tmem + SM::o_col(t);
    bool ok = true;
    bool issued = false;
    uint32_t kvc = 0;                // key tiles of all items so far
    uint32_t k_seen = 0, v_seen = 0;  // K / V tiles whose arrival this warp observed
    uint32_t pc = 0, sc = 0, oc = 0;  // steps whose P V / S this warp issued, items whose O it began
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
      if (!__all_sync(FULL, srv_wait(bar, parity, abort_flag, limit))) {
        ok = false;
        return false;
      }
      tc_fence_after();
      return true;
    };
    auto ensure_k = [&](uint32_t idx) -> bool {
      for (; k_seen <= idx; ++k_seen)
        if (!wait(bar_k_full + 8 * (k_seen % STAGES), (k_seen / STAGES) & 1)) return false;
      return true;
    };
    auto ensure_v = [&](uint32_t idx) -> bool {
      for (; v_seen <= idx; ++v_seen)
        if (!wait(bar_v_ready + 8 * (v_seen % STAGES), (v_seen / STAGES) & 1)) return false;
      return true;
    };
    // Whether step i is its key tile's last one of this side.
    auto ends_tile = [](int i, int n) { return i % SM::SUB == SM::SUB - 1 || i + 1 == n; };
    // S of step i (of n) into the side's score buffer, which the softmax has read.
    auto do_s = [&](int i, int n, int qb) -> bool {
      const uint32_t idx = kvc + i / SM::SUB;
      if (sc > 0 && !wait(bar_s_free + 8 * t, (sc - 1) & 1)) return false;
      // With two P buffers the softmax writes a step's P without a wait of its own: these scores
      // come after the P V that used the buffer last.
      if (SM::PBUF == 2 && sc >= 2 && !wait(bar_pv_done + 16 * t + 8 * (sc & 1), ((sc - 2) / 2) & 1)) return false;
      if (!ensure_k(idx)) return false;
      const uint32_t qaddr = sQ + (t * QBUF + qb) * SM::Q_TILE;
      const uint32_t kaddr = sK + (idx % STAGES) * SM::KV_TILE + (uint32_t)(i % SM::SUB) * sub_bytes;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        mma_f16_ss_warp(s_col, atc_desc_qk<HD>(qaddr, kk), atc_desc_qk<HD>(kaddr, kk), idesc_s, kk > 0 ? 1u : 0u);
      mma_commit_warp(bar_s_full + 8 * t);
      if (ends_tile(i, n)) mma_commit_warp(bar_k_empty + 8 * (idx % STAGES));
      if (i + 1 == n) mma_commit_warp(bar_q_empty + 8 * (t * SM::QS + qb));
      issued = true;
      ++sc;
      return true;
    };
    // O += P V of step i.  The first of an item overwrites O, which the softmax has read.
    auto do_pv = [&](int i, int n) -> bool {
      const uint32_t idx = kvc + i / SM::SUB;
      const uint32_t pb = pc % SM::PBUF;
      if (!wait(bar_p_full + 16 * t + 8 * pb, (pc / SM::PBUF) & 1) || !ensure_v(idx)) return false;
      if (i == 0 && !wait(bar_o_free + 8 * t, (oc++ & 1) ^ 1u)) return false;
      const uint64_t vd = atc_desc_v<HD>(sV + (idx % STAGES) * SM::KV_TILE + (uint32_t)(i % SM::SUB) * sub_bytes);
#pragma unroll
      for (int kk = 0; kk < SM::KT / 16; ++kk)
        mma_f16_ts_warp(o_col, p_col + pb * (SM::KT / 2) + (uint32_t)(kk * 8), vd + (uint64_t)(kk * v_step), idesc_o,
                        (i > 0 || kk > 0) ? 1u : 0u);
      mma_commit_warp(bar_pv_done + 16 * t + 8 * pb);
      if (i + 1 == n) mma_commit_warp(bar_o_full + 8 * t);
      if (ends_tile(i, n)) mma_commit_warp(bar_v_empty + 8 * (idx % STAGES));
      issued = true;
      ++pc;
      return true;
    };
    for (int k = 0; ok; ++k) {
      const int qb = k % QBUF;
      const uint32_t q_empty = bar_q_empty + 8 * (t * SM::QS + qb);
      if (!wait(bar_q_full + 8 * (t * SM::QS + qb), (k / QBUF) & 1)) break;
      const TileInfo& wi = info[t * SM::QS + qb];
      const int n_kv = __shfl_sync(FULL, wi.n_kv, 0);
      if (n_kv < 0) break;  // no more items
      const int n = __shfl_sync(FULL, wi.ns[atc_query_tile<NT>(t, k)], 0);
      if constexpr (SM::SPLIT) {
        __syncwarp();
        if (lane == 0 && (!does_s || n == 0)) mbar_arrive(q_empty);  // (S: with its last product)
        for (int i = 0; i < n && ok; ++i)
          if (!(does_s ? do_s(i, n, qb) : do_pv(i, n))) break;
      } else {
        if (n == 0 && lane == 0) mbar_arrive(q_empty);
        __syncwarp();
        // The next S as soon as the softmax has read this one's scores.
        if (n > 0 && !do_s(0, n, qb)) break;
        for (int i = 0; i < n && ok; ++i) {
          if (i + 1 < n && !do_s(i + 1, n, qb)) break;
          if (!do_pv(i, n)) break;
        }
      }
      // Key tiles that only the other side uses: released once they have landed.
      for (int j = (n + SM::SUB - 1) / SM::SUB; j < n_kv && ok; ++j) {
        if ((does_s && !ensure_k(kvc + j)) || ((!SM::SPLIT || !does_s) && !ensure_v(kvc + j))) break;
        if (lane == 0) {
          if (does_s) mbar_arrive(bar_k_empty + 8 * ((kvc + j) % STAGES));
          if (!SM::SPLIT || !does_s) mbar_arrive(bar_v_empty + 8 * ((kvc + j) % STAGES));
        }
        __syncwarp();
      }
      kvc += n_kv;
    }
    if (!ok) {
      if (lane == 0) *abort_flag = 1;
      if (issued) {
        mma_commit_warp(bar_drain + 8 * (warp - ISSUER));
        srv_wait(bar_drain + 8 * (warp - ISSUER), 0, nullptr, limit);
      }
    }
  } else if (warp == CLEANER) {
    // ------------------------------------------------------------ cleaner
    // Sees every V tile before the products do: rows behind the last key become zeros.
    constexpr unsigned FULL = 0xffffffffu;
    bool ok = true;
    long vc = 0;
    for (int k = 0; ok; ++k) {
      const int qb = k % QBUF;
      ok = __all_sync(FULL, srv_wait(bar_q_full + 8 * qb, (uint32_t)((k / QBUF) & 1), abort_flag, limit));
      if (!ok) break;
      const TileInfo wi = info[qb];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q_empty + 8 * qb);
      if (wi.n_kv < 0) break;  // no more items
      for (int j = 0; j < wi.n_kv; ++j, ++vc) {
        const int vs = (int)(vc % STAGES);
        ok = __all_sync(FULL, srv_wait(bar_v_full + 8 * vs, (uint32_t)((vc / STAGES) & 1), abort_flag, limit));
        if (!ok) break;
        const int keep = wi.len - (wi.j0 + j) * ATC_BN;
        if (keep < ATC_BN) {
          constexpr int CH = SM::BOX_COLS * 2 / 16;  // 16-byte chunks of a row of a box
          for (int x = 0; x < SM::NBOX; ++x) {
            const uint32_t vx = sV + vs * SM::KV_TILE + (uint32_t)(x * SM::BOX_BYTES);
            for (int i = max(0, keep) * CH + lane; i < ATC_BN * CH; i += 32)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vx + (uint32_t)(i * 16)), "r"(0u)
                           : "memory");
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_v_ready + 8 * vs);
      }
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else if (warp < 4 * NT) {
    // ------------------------------------------------------------ softmax
    constexpr int KT = SM::KT;
    const int t = warp >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;  // row inside the query tile
    const int rtok = row / p.group;    // its token inside the tile, its head in the group
    const int rhead = row - rtok * p.group;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + SM::s_col(t);
    const uint32_t p_addr0 = tmem + lane_base + SM::p_col(t);
    const uint32_t o_addr = tmem + lane_base + SM::o_col(t);
    const float scale = p.scale_log2;
    long c = 0;    // steps of all items so far
    long ofc = 0;  // items with steps so far
    bool ok = true;
    // All lanes give up together: one that left alone would leave the others waiting for it in the
    // next warp-wide instruction, without a limit.
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, srv_wait(bar, parity, abort_flag, limit));
    };
    // One arrival per warp, after every lane's reads and TMEM accesses.
    auto arrive = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // P V of step i of this side complete: phase i / PBUF of its buffer's barrier.
    auto pv_done = [&](long i) -> bool {
      const bool fine = wait(bar_pv_done + 16 * t + 8 * (uint32_t)(i % SM::PBUF), (uint32_t)((i / SM::PBUF) & 1));
      tc_fence_after();
      return fine;
    };
    for (int k = 0; ok; ++k) {
      const int qb = k % QBUF;
      if (!wait(bar_q_full + 8 * (t * SM::QS + qb), (uint32_t)((k / QBUF) & 1))) {
        ok = false;
        break;
      }
      const TileInfo& wi = info[t * SM::QS + qb];
      if (wi.n_kv < 0) break;  // no more items
      const int tq = atc_query_tile<NT>(t, k);
      const int n = tq == 0 ? wi.ns[0] : wi.ns[1];
      const int key0 = wi.j0 * ATC_BN, len = wi.len, part = wi.part, h = wi.h, b = wi.b, qi = wi.q;
      const int tok0 = wi.tok0 + tq * TOK;  // first token of the tile
      const int tokens = wi.n;
      const int token = wi.row0 + tok0 + rtok;   // packed row of this thread's token
      const int first = p.s.causal ? len - tokens + tok0 : len - 1;  // last key of the tile's first row
      arrive(bar_q_empty + 8 * (t * SM::QS + qb));  // the info slot is read
      const bool live = rtok < TOK && tok0 + rtok < tokens;
      const long prow = part < 0 ? 0 : (long)part * (NT * ATC_BM) + tq * ATC_BM + row;
      if (n == 0) {
        // No key of this piece for this tile: an empty partial result.
        if (part >= 0 && live) p.part_ml[prow] = make_float2(-INFINITY, 0.f);
        continue;
      }
      const int row_lim = p.s.causal ? min(len - 1, first + rtok) : len - 1;
      const int warp_lim_lo = __shfl_sync(0xffffffffu, row_lim, 0), warp_lim_hi = __shfl_sync(0xffffffffu, row_lim, 31);
      float m_run = -INFINITY;  // running max (log2 domain) used as the exp base
      float l_run = 0.f;
      for (int i = 0; i < n; ++i, ++c) {
        if (!wait(bar_s_full + 8 * t, (uint32_t)(c & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sv[KT];  // raw fp32 scores of this thread's row
#pragma unroll
        for (int q = 0; q < KT / 32; ++q) {
          uint32_t chunk[32];
          tmem_ld_32x32b_x32(s_addr + (uint32_t)(q * 32), chunk);
#pragma unroll
          for (int e = 0; e < 32; ++e) sv[q * 32 + e] = chunk[e];
        }
        tmem_wait_ld();
        // The scores are in registers: the buffer may take the next step's.
        tc_fence_before();
        arrive(bar_s_free + 8 * t);
        // 32 keys at a time: those that no row of the warp sees take no part (on the
        // diagonal half of them), those that some see are masked.  Column e of this step is
        // hidden when e > lim; limits rise with the rows.
        const int k0 = key0 + i * KT, lim = row_lim - k0, warp_hi = warp_lim_hi - k0, warp_lo = warp_lim_lo - k0;
        const bool partly = KT - 1 > warp_lo;  // warp-uniform
        float pm[8];
        if (!partly) {
#pragma unroll
          for (int e = 0; e < 8; ++e) pm[e] = __uint_as_float(sv[e]);
#pragma unroll
          for (int e = 8; e < KT; e += 2)
            pm[(e >> 1) & 7] = srv_max3(pm[(e >> 1) & 7], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) pm[e] = -INFINITY;
#pragma unroll
          for (int q = 0; q < KT / 32; ++q) {
            if (32 * q <= warp_hi) {
              if (32 * q + 31 > warp_lo) {
#pragma unroll
                for (int e = 32 * q; e < 32 * q + 32; ++e)
                  if (e > lim) sv[e] = __float_as_uint(-INFINITY);
              }
#pragma unroll
              for (int e = 32 * q; e < 32 * q + 32; e += 2)
                pm[(e >> 1) & 7] = srv_max3(pm[(e >> 1) & 7], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
            }
          }
        }
        const float mx =
            srv_max3(srv_max3(pm[0], pm[1], pm[2]), srv_max3(pm[3], pm[4], pm[5]), srv_max3(pm[6], pm[7], pm[7]));
        const float m_tile = mx * scale;
        float alpha = 1.f;
        bool rescale = false;
        if (i == 0) {
          m_run = m_tile;
        } else {
          // Lazy rescale: keep the old base unless the max grew by more than 2^8.  Rows
          // that no token owns do not vote.
          const bool grow = live && m_tile > m_run + 8.0f;
          if (__any_sync(0xffffffff, grow)) {
            const float m_new = fmaxf(m_run, m_tile);
            alpha = (m_run == -INFINITY) ? 0.f : ex2_approx(m_run - m_new);
            m_run = m_new;
            rescale = true;  // warp-uniform
          }
        }
        const float base = m_run == -INFINITY ? 0.f : m_run;
        const float2 sc2 = make_float2(scale, scale), nb2 = make_float2(-base, -base);
        unsigned long long ps2[2] = {0ull, 0ull};  // partial row sums, f32x2 pairs
        const uint32_t p_addr = p_addr0 + (uint32_t)(c % SM::PBUF) * (KT / 2);
        uint32_t pk[KT / 32][16];
        auto chunk = [&](int q) {  // 32 keys' probabilities
          if (32 * q > warp_hi) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[q][e] = 0u;
            return;
          }
#pragma unroll
          for (int cc = 0; cc < 16; ++cc) {
            const int e = q * 16 + cc;
            const float2 x = ffma2(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, nb2);
            const float2 y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            ps2[e & 1] = add2p(ps2[e & 1], pk2(y.x, y.y));
            pk[q][cc] = srv_pack<BF16>(y.x, y.y);
          }
        };
        // The P buffer is free once the P V that used it last is complete.  With one buffer
        // that is the previous step's, so half of the exponentials come before the wait;
        // with two the issuer waited.
        constexpr int EARLY = SM::PBUF == 1 ? KT / 64 : 0;
#pragma unroll
        for (int q = 0; q < EARLY; ++q) chunk(q);
        if (SM::PBUF == 1 && c >= 1 && !pv_done(c - 1)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int q = 0; q < KT / 32; ++q) {
          if (q >= EARLY) chunk(q);
          tmem_st_32x32b_x16(p_addr + (uint32_t)(q * 16), pk[q]);
        }
        const float2 rs2 = upk2(add2p(ps2[0], ps2[1]));
        l_run = l_run * alpha + (rs2.x + rs2.y);
        if (rescale) {
          // O holds P V of this item's steps before this one.
          if (SM::PBUF > 1 && !pv_done(c - 1)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int q = 0; q < HD / 32; ++q) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_addr + (uint32_t)(q * 32), o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x32b_x32(o_addr + (uint32_t)(q * 32), o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        // A barrier per P buffer: the softmax may be a step ahead of P V, and a barrier that
        // completed twice since it was looked at would read as not completed.
        arrive(bar_p_full + 16 * t + 8 * (uint32_t)(c % SM::PBUF));
      }
      if (!ok) break;
      if (!wait(bar_o_full + 8 * t, (uint32_t)(ofc++ & 1))) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (part >= 0) {
        // A piece: raw sums, joined later.
        float* dst = p.part_o + prow * HD;
        if (live) p.part_ml[prow] = make_float2(m_run, l_run);
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_addr + (uint32_t)(c * 32), o);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
      } else {
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        if (live && p.lse != nullptr)
          p.lse[(long)token * p.heads + h * p.group + rhead] = srv_lse(m_run, l_run);
        // Every thread stores its own row, a whole 32-byte sector at a time where rows are aligned
        // for that.  (Through shared memory, so that a warp's stores cover whole rows: 127 against
        // 123 us at 256 prompts of 128 - 256 tokens, head_dim 64.)
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (long)token * p.o_tok + (long)(h * p.group + rhead) * p.o_head;
        uint32_t odd = 0;  // two sums of result x 0: NaN once one was not finite
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_addr + (uint32_t)(c * 32), o);
          tmem_wait_ld();
          if (live) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              w[e] = srv_pack<BF16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
              odd = srv_fma_zero<BF16>(w[e], odd);
            }
            if (p.o_wide) {
              srv_st_v8(dst + c * 32, w);
              srv_st_v8(dst + c * 32 + 16, w + 8);
            } else {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<uint4*>(dst + c * 32 + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
            }
          }
        }
        if (p.s.causal && __any_sync(0xffffffffu, srv_nonfinite<BF16>(odd)) && lane == 0) {
          const int at = atomicAdd(p.plan.counters + 3, 1);
          if (at < p.plan.most_redo) p.plan.redo[at] = make_int4(b, qi, h, tq * 4 + quad);
        }
      }
      tc_fence_before();
      arrive(bar_o_free + 8 * t);
    }
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) srv_report_timeout(p.s.status, p.timeout_host);
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------- join
template <int HD, bool BF16>
__device__ __forceinline__ void tile_store_row(const TileParams& p, int token, int head,
                                               const float (&acc)[HD / 32], float inv, float top, float sum) {
  const int lane = lane_id();
  const long at = (long)token * p.o_tok + (long)head * p.o_head + lane * (HD / 32);
  if constexpr (HD == 32) {
    if constexpr (BF16)
      static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(acc[0] * inv);
    else
      static_cast<__half*>(p.out)[at] = __float2half(acc[0] * inv);
  } else {
    uint32_t* dst = static_cast<uint32_t*>(p.out) + at / 2;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) dst[i] = srv_pack<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  }
  if (p.lse != nullptr && lane == 0) p.lse[(long)token * p.heads + head] = srv_lse(top, sum);
}

constexpr int TILE_JOIN_WARPS = 8;

// This lane's HD / 32 neighbouring values of a row.
template <int HD>
__device__ __forceinline__ void tile_load_part(const float* row, float (&o)[HD / 32]) {
  const float* at = row + lane_id() * (HD / 32);
  if constexpr (HD == 32) {
    o[0] = *at;
  } else if constexpr (HD == 64) {
    const float2 v = *reinterpret_cast<const float2*>(at);
    o[0] = v.x;
    o[1] = v.y;
  } else {
#pragma unroll
    for (int x = 0; x < HD / 32; x += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + x);
      o[x] = v.x;
      o[x + 1] = v.y;
      o[x + 2] = v.z;
      o[x + 3] = v.w;
    }
  }
}

// Where key j of a head lies, in elements; false: on no page.
__device__ __forceinline__ bool tile_locate(const TileParams& p, const CacheView& c, const SrvSeq& s, int b, int kvh,
                                            int j, long* at) {
  if (p.s.table == nullptr) {
    *at = (long)(s.row0 + j) * c.slot + kvh * c.head;
    return true;
  }
  const int page = srv_page(p.s, b, j), in = j & ((1 << p.s.page_shift) - 1);
  *at = page * c.page + in * c.slot + kvh * c.head;
  return page < p.s.num_pages;
}

// The columns `need` (a bit per column of this lane) of one row key by key, hidden keys left out.
template <int HD, bool BF16>
__device__ void tile_redo_row(const TileParams& p, const SrvSeq& s, int b, int tok, int kvh, int g, unsigned need) {
  const int lane = lane_id();
  constexpr int E = HD / 32;
  const int token = s.row0 + tok, head = kvh * p.group + g;
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + (long)token * p.q_tok + (long)head * p.q_head + lane * E;
  float qv[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qv[i] = srv_to_float<BF16>(q[i]);
    acc[i] = 0.f;
  }
  const int keys = p.s.causal ? min(s.len, s.len - s.n + tok + 1) : s.len;
  for (int j = 0; j < keys; ++j) {
    if (j % 32 == 0) {  // a NaN in sight settles its column
      bool open = false;
#pragma unroll
      for (int i = 0; i < E; ++i) open |= (need >> i & 1) != 0 && acc[i] == acc[i];
      if (!__any_sync(0xffffffffu, open)) break;
    }
    long at_k, at_v;
    tile_locate(p, p.v, s, b, kvh, j, &at_v);
    const bool there = tile_locate(p, p.k, s, b, kvh, j, &at_k);
    const uint16_t* kr = static_cast<const uint16_t*>(p.k.data) + at_k + lane * E;
    const uint16_t* vr = static_cast<const uint16_t*>(p.v.data) + at_v + lane * E;
    float dot = 0.f;
    if (there)
#pragma unroll
      for (int i = 0; i < E; ++i) dot = fmaf(qv[i], srv_to_float<BF16>(kr[i]), dot);
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    const float x = dot * p.scale_log2;
    const float m_new = fmaxf(m, x);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m == m_new ? 1.f : ex2_approx(m - m_new);
    const float e = ex2_approx(x - base);
    m = m_new;
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (alpha != 1.f) acc[i] *= alpha;
      if (there) acc[i] = fmaf(e, srv_to_float<BF16>(vr[i]), acc[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = static_cast<uint16_t*>(p.out) + (long)token * p.o_tok + (long)head * p.o_head + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (need >> i & 1) out[i] = (uint16_t)srv_pack<BF16>(acc[i] * inv, 0.f);
}

// A row whose result is not finite: again in the columns in which a value that it does not see,
// among those that its tile's products read, is not finite.  (The log-sum-exp owes nothing to
// values.)
template <int HD, bool BF16>
__device__ __forceinline__ void tile_mend_row(const TileParams& p, int b, int tok0, int rtok, int kvh, int g) {
  constexpr int E = HD / 32;
  const SrvSeq s = srv_seq(p.s, b);
  const int tok = tok0 + rtok;
  if (tok >= s.n) return;
  const int end = tile_kv_tiles(tile_kv_end(s, 1, tok0, p.tile_tokens)) * ATC_BN;
  unsigned need = 0;
#pragma unroll 4
  for (int j = max(0, s.len - s.n + tok + 1); j < min(s.len, end); ++j) {
    long at;
    if (tile_locate(p, p.v, s, b, kvh, j, &at)) {
      const uint16_t* v = static_cast<const uint16_t*>(p.v.data) + at + lane_id() * E;
#pragma unroll
      for (int i = 0; i < E; ++i) need |= srv_nonfinite<BF16>(v[i]) ? 1u << i : 0u;
    }
  }
  if (__any_sync(0xffffffffu, need != 0)) tile_redo_row<HD, BF16>(p, s, b, tok, kvh, g, need);
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(32 * TILE_JOIN_WARPS) tile_join_kernel(const __grid_constant__ TileParams p) {
  constexpr int NT = AtcSmem<HD>::NT;
  constexpr int ROWS = NT * ATC_BM;
  griddep_wait();
  const int joins = p.plan.counters[2];
  const int redo = min(p.plan.counters[3], p.plan.most_redo);
  const int lane = lane_id();
  const long w0 = (long)blockIdx.x * TILE_JOIN_WARPS + warp_id(), step = (long)gridDim.x * TILE_JOIN_WARPS;
  // Four rows per warp at a time, their loads in flight together.
  constexpr int R = 4;
  for (long i = w0; i < (long)joins * p.kv_heads * (ROWS / R); i += step) {
    const int r0 = (int)(i % (ROWS / R)) * R;
    const int h = (int)(i / (ROWS / R) % p.kv_heads);
    const TileJoin e = p.plan.joins[i / (ROWS / R) / p.kv_heads];
    const int tok0 = (e.q * NT + r0 / ATC_BM) * p.tile_tokens;
    if ((r0 % ATC_BM) / p.group >= p.tile_tokens || tok0 + (r0 % ATC_BM) / p.group >= e.n) continue;
    auto at = [&](int piece) { return ((long)e.part + (long)piece * p.kv_heads + h) * ROWS + r0; };
    float top[R], sum[R], acc[R][HD / 32];
#pragma unroll
    for (int x = 0; x < R; ++x) {
      top[x] = -INFINITY;
      sum[x] = 0.f;
#pragma unroll
      for (int y = 0; y < HD / 32; ++y) acc[x][y] = 0.f;
    }
    for (int c = 0; c < e.pieces; ++c) {
#pragma unroll
      for (int x = 0; x < R; ++x) top[x] = fmaxf(top[x], p.part_ml[at(c) + x].x);
    }
    for (int c = 0; c < e.pieces; ++c) {
      float2 ml[R];
      float o[R][HD / 32];
#pragma unroll
      for (int x = 0; x < R; ++x) {
        ml[x] = p.part_ml[at(c) + x];
        tile_load_part<HD>(p.part_o + (at(c) + x) * HD, o[x]);  // (rows of empty pieces hold anything)
      }
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const float f = ml[x].x == -INFINITY ? 0.f : ex2_approx(ml[x].x - top[x]);
        sum[x] += ml[x].y * f;
        const bool none = ml[x].x == -INFINITY && ml[x].y == 0.f;
#pragma unroll
        for (int y = 0; y < HD / 32; ++y) acc[x][y] += none ? 0.f : o[x][y] * f;
      }
    }
    unsigned odd = 0;  // rows that are not finite
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const int rtok = (r0 % ATC_BM + x) / p.group, g = r0 % ATC_BM + x - rtok * p.group;
      if (rtok < p.tile_tokens && tok0 + rtok < e.n) {
        tile_store_row<HD, BF16>(p, e.row0 + tok0 + rtok, h * p.group + g, acc[x], sum[x] == 0.f ? 0.f : 1.f / sum[x],
                                 top[x], sum[x]);
#pragma unroll
        for (int y = 0; y < HD / 32; ++y) odd |= fabsf(acc[x][y]) < INFINITY ? 0u : 1u << x;
      }
    }
    odd = p.s.causal ? __reduce_or_sync(0xffffffffu, odd) : 0;
    for (; odd != 0; odd &= odd - 1) {
      const int r = r0 % ATC_BM + __ffs(odd) - 1, rtok = r / p.group;
      tile_mend_row<HD, BF16>(p, e.b, tok0, rtok, h, r - rtok * p.group);
    }
  }
  // Rows of whole items, 32 per note.
  for (long i = w0; i < (long)redo * 32; i += step) {
    const int4 e = p.plan.redo[i / 32];
    const int r = (e.w & 3) * 32 + (int)(i % 32);
    const int rtok = r / p.group;
    if (rtok < p.tile_tokens)
      tile_mend_row<HD, BF16>(p, e.x, (e.y * NT + e.w / 4) * p.tile_tokens, rtok, e.z, r - rtok * p.group);
  }
}

}  // namespace tttj
