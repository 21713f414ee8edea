// Attention mass of cached keys: for every sequence, key/value head and slot j, the sum of
// the probabilities exp(scale q k_j - lse) that the new tokens' queries gave to it.
//
// Keys stay, queries stream: S^T = K Q^T on the tensor cores with 128 keys as the rows of
// the accumulator and up to 80 query rows (token x group + head) as its columns, so a
// thread owns one key and adds its row of exponentials in registers -- no reduction across
// threads, no atomics, a fixed order.  The log-sum-exp of the attention makes every
// probability independent of the others, so one pass suffices.
//
// An item is NT key tiles of one head (two; one at head_dim 256); persistent CTAs take the items
// that have work in turn (each computes the sequences' prefix sums itself), and share the
// copying of the rest.  One warp loads K tiles (KBUF items ahead), another the query tiles with
// their log-sum-exps (one warp for both made every item wait for page numbers and then for
// log-sum-exps: 46 against 38 us at 32 sequences of 1000 - 4096 keys), one issues
// the MMAs into three accumulators per key tile in turn, and a warpgroup per accumulator adds, two keys per
// thread; their sums meet at the end of an item.
// For single tokens the bytes of K bound it; for chunks the exponentials and the products.
#pragma once
#include "attention_tc.cuh"
#include "serve_dev.cuh"

namespace tttj {

// Query rows of a tile, and accumulators per key tile: three of 80 columns cover the time
// between the reading of an accumulator and its next use (two of 128 left the adding warps
// waiting for 2000 of 4800 cycles).
constexpr int MASS_ROWS = MASS_TILE_ROWS, MASS_BUFS = 3;
constexpr int MASS_SORTED = 256;  // sequences that are ordered by their work at most
constexpr int MASS_COLS = 96;  // MASS_ROWS rounded up to the lanes of a warp

template <int HD>
struct MassSmem {
  static constexpr int NT = HD == 256 ? 1 : 2;
  static constexpr int KBUF = HD == 256 ? 1 : 2;   // items whose keys are loaded
  static constexpr int STAGES = HD == 256 ? 2 : HD == 128 ? 3 : 4;  // query tiles in flight
  static constexpr int TILE = ATC_BM * HD * 2;
  static constexpr int BOX_COLS = HD < 64 ? HD : 64;
  static constexpr int NBOX = HD / BOX_COLS;
  static constexpr int BOX_BYTES = ATC_BM * BOX_COLS * 2;
  static constexpr int K_BYTES = KBUF * NT * TILE;
  static constexpr int Q_BOX = MASS_ROWS * BOX_COLS * 2;  // 64 columns of a query tile
  static constexpr int Q_TILE = NBOX * Q_BOX;
  static constexpr int Q_BYTES = STAGES * Q_TILE;
  static constexpr int COLS = 4;                      // query tiles whose columns' data are held
  static constexpr int COL_BYTES = COLS * MASS_COLS * 8;    // (-lse, last key) of every query row
  static constexpr int NBAR = 2 * KBUF + 2 * STAGES + 2 * COLS + 2 * MASS_BUFS + 1 + 4;
  static constexpr int XCH_BYTES = 2 * (MASS_BUFS - 1) * NT * ATC_BM * 4;  // [item parity][warpgroup][key] sums
  static constexpr int FIXED = K_BYTES + Q_BYTES + COL_BYTES + XCH_BYTES + NBAR * 8 + 16 + 1024;
};
// Warps: one warpgroup per accumulator that adds (both key tiles of an item, so the columns' data
// and the bookkeeping serve two keys per thread), the key loader, the MMA issuer, the query loader.
constexpr int MASS_ADDERS = 12;
constexpr int MASS_THREADS = 32 * (MASS_ADDERS + 3);

// Of eight pairs of exponentials, those on the FMA pipe (4 chunks of 300 - 512 tokens over 2000 -
// 8192 keys, 32 / 8 heads x 128: none 106.5 us, one 104.0, two 105.9).
constexpr int MASS_FMA_PAIRS = 1;

// Position in a ring of N stages: index and phase parity, without divisions.
template <int N>
struct MassRing {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) {
      at = 0;
      parity ^= 1;
    }
  }
};

struct MassItem {
  int b, h, k0;     // first key of the item
  SrvSeq q;
  int first, steps;  // query tiles first .. first + steps - 1
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(MASS_THREADS, 1)
    mass_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const MassParams p) {
  using SM = MassSmem<HD>;
  constexpr int NT = SM::NT;
  constexpr int KEYS = MASS_ADDERS, ISSUER = KEYS + 1, QUERIES = ISSUER + 1;  // warps
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sK = smem_u32(smem);
  const uint32_t sQ = sK + SM::K_BYTES;
  float* s_lse = reinterpret_cast<float*>(smem + SM::K_BYTES + SM::Q_BYTES);         // [COLS][MASS_COLS]
  int* s_lim = reinterpret_cast<int*>(smem + SM::K_BYTES + SM::Q_BYTES) + SM::COLS * MASS_COLS;
  float* s_xch = reinterpret_cast<float*>(smem + SM::K_BYTES + SM::Q_BYTES + SM::COL_BYTES);
  const uint32_t bar0 = sQ + SM::Q_BYTES + SM::COL_BYTES + SM::XCH_BYTES;
  const uint32_t bar_k_full = bar0;                          // [KBUF]
  const uint32_t bar_k_empty = bar_k_full + 8 * SM::KBUF;    // [KBUF]
  const uint32_t bar_q_full = bar_k_empty + 8 * SM::KBUF;    // [STAGES]
  const uint32_t bar_q_empty = bar_q_full + 8 * SM::STAGES;  // [STAGES]
  const uint32_t bar_c_full = bar_q_empty + 8 * SM::STAGES;  // [COLS]
  const uint32_t bar_c_empty = bar_c_full + 8 * SM::COLS;    // [COLS]
  const uint32_t bar_s_full = bar_c_empty + 8 * SM::COLS;    // [MASS_BUFS]
  const uint32_t bar_s_free = bar_s_full + 8 * MASS_BUFS;    // [MASS_BUFS]
  const uint32_t bar_x_full = bar_s_free + 8 * MASS_BUFS;   // [item parity] the other warpgroups' sums
  const uint32_t bar_x_free = bar_x_full + 16;               // [item parity] read by the first
  const uint32_t bar_drain = bar_x_free + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::K_BYTES + SM::Q_BYTES + SM::COL_BYTES + SM::XCH_BYTES +
                                                      SM::NBAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SrvSeq* s_seq = reinterpret_cast<SrvSeq*>(tmem_slot + 4);  // [batch]
  int* s_pre = reinterpret_cast<int*>(s_seq + p.s.batch);    // [batch + 1] items of a head before each place
  int* s_order = s_pre + p.s.batch + 1;                       // [batch] sequence at each place
  const int warp = warp_id(), lane = lane_id();
  constexpr uint64_t limit = SRV_WAIT_LIMIT_NS;
  const int TOK = p.tile_tokens;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    for (int i = 0; i < SM::KBUF; ++i) {
      mbar_init(bar_k_full + 8 * i, 1);
      mbar_init(bar_k_empty + 8 * i, 1);
    }
    for (int i = 0; i < SM::STAGES; ++i) {
      mbar_init(bar_q_full + 8 * i, 1);
      mbar_init(bar_q_empty + 8 * i, 1);
    }
    for (int i = 0; i < SM::COLS; ++i) {
      mbar_init(bar_c_full + 8 * i, 1);
      mbar_init(bar_c_empty + 8 * i, 4);
    }
    for (int i = 0; i < MASS_BUFS; ++i) {
      mbar_init(bar_s_full + 8 * i, 1);
      mbar_init(bar_s_free + 8 * i, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_x_full + 8 * i, 4 * (MASS_BUFS - 1));
      mbar_init(bar_x_free + 8 * i, 4);
    }
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUER) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch();
  constexpr int ITEM_KEYS = NT * ATC_BM;
  for (int b = threadIdx.x; b < p.s.batch; b += blockDim.x) s_seq[b] = srv_seq(p.s, b);
  __syncthreads();
  // Sequences with more query tiles first; the CTAs take the items in a snake, so that the long
  // ones spread evenly (in the sequences' order the busiest CTA had 1.3 times the mean work).
  for (int b = threadIdx.x; b < p.s.batch; b += blockDim.x) {
    const SrvSeq q = s_seq[b];
    int place = b;
    if (p.s.batch <= MASS_SORTED) {
      place = 0;
      for (int o = 0; o < p.s.batch; ++o) place += s_seq[o].n > q.n || (s_seq[o].n == q.n && o < b);
    }
    s_order[place] = b;
    s_pre[place + 1] = q.n > 0 ? (q.len + ITEM_KEYS - 1) / ITEM_KEYS : 0;
  }
  __syncthreads();
  if (warp == 0) {
    int base = 0;
    for (int b0 = 0; b0 < p.s.batch; b0 += 32) {
      int v = b0 + lane < p.s.batch ? s_pre[b0 + lane + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
      }
      if (b0 + lane < p.s.batch) s_pre[b0 + lane + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) s_pre[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const long items = (long)s_pre[p.s.batch] * p.kv_heads;
  // The CTA's r-th item: round r of the snake.
  auto item_at = [&](long r) { return r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x); };
  auto decode = [&](long i) {
    MassItem w;
    // Heads inside a sequence's tile: neighbouring CTAs read the same pages.
    w.h = (int)(i % p.kv_heads);
    const int e = (int)(i / p.kv_heads);
    int lo = 0, hi = p.s.batch - 1;  // last b with s_pre[b] <= e
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_pre[mid] <= e) lo = mid; else hi = mid - 1;
    }
    w.b = s_order[lo];
    w.k0 = (e - s_pre[lo]) * ITEM_KEYS;
    w.q = s_seq[w.b];
    // The first token that sees key k0; the last one sees every key.
    w.first = max(0, w.k0 - (w.q.len - w.q.n)) / TOK;
    w.steps = (w.q.n + TOK - 1) / TOK - w.first;
    return w;
  };

  if (warp == KEYS) {
    // ------------------------------------------------------------ keys
    const int cr = min(ATC_BM, 1 << p.s.page_shift);
    const int boxes = (ATC_BM / cr) * SM::NBOX * NT;  // <= 32
    const int x = lane % SM::NBOX, key = lane / SM::NBOX * cr;  // lane -> (64-column box, page piece)
    const uint32_t dst = (uint32_t)(key / ATC_BM * SM::TILE + x * SM::BOX_BYTES + (key % ATC_BM) * SM::BOX_COLS * 2);
    bool ok = true;
    long kc = 0;
    MassRing<SM::KBUF> kr;
    // Page numbers are fetched an item ahead.
    int slot = 0, page = p.s.num_pages, head = 0;
    auto fetch = [&](long i) {
      const MassItem w = decode(i);
      slot = w.k0 + key;
      head = w.h;
      page = lane < boxes && slot < w.q.len ? srv_page(p.s, w.b, slot) : p.s.num_pages;
    };
    long i = item_at(0);
    if (i < items) fetch(i);
    for (long r = 1; i < items; ++r) {
      const int use_slot = slot, use_page = page, use_head = head;
      i = item_at(r);
      if (i < items) fetch(i);
      ok = __all_sync(0xffffffffu, srv_wait(bar_k_empty + 8 * kr.at, kr.parity ^ 1u, abort_flag, limit));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(bar_k_full + 8 * kr.at, NT * SM::TILE);
      __syncwarp();
      if (lane < boxes)
        tma_load_4d(sK + kr.at * NT * SM::TILE + dst, &tmK, bar_k_full + 8 * kr.at, x * SM::BOX_COLS,
                    use_slot & ((1 << p.s.page_shift) - 1), use_head, use_page);
      __syncwarp();
      ++kc;
      kr.next();
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      for (long j = kc > SM::KBUF ? kc - SM::KBUF : 0; j < kc; ++j)
        srv_wait(bar_k_full + 8 * (int)(j % SM::KBUF), (uint32_t)((j / SM::KBUF) & 1), nullptr, limit);
    }
  } else if (warp == QUERIES) {
    // ------------------------------------------------------------ queries
    const uint32_t q_bytes = (uint32_t)(TOK * p.group * HD * 2);
    constexpr int E = MASS_COLS / 32;
    int tk[E], g[E];  // token and head of this lane's columns
#pragma unroll
    for (int e = 0; e < E; ++e) {
      tk[e] = (lane + 32 * e) / p.group;
      g[e] = lane + 32 * e - tk[e] * p.group;
    }
    bool ok = true;
    uint32_t qc = 0;  // query tiles issued
    MassRing<SM::STAGES> qr;
    MassRing<SM::COLS> cr;
    long r = 0, i = item_at(0);
    MassItem w{};
    int t = 0;
    float nl[E];
    // The log-sum-exps of query tile t, one tile ahead of their use.
    auto fetch = [&] {
      const int tok0 = (w.first + t) * TOK;
#pragma unroll
      for (int e = 0; e < E; ++e)
        nl[e] = tk[e] < TOK && tok0 + tk[e] < w.q.n
                    ? p.lse[(long)(w.q.row0 + tok0 + tk[e]) * p.heads + w.h * p.group + g[e]]
                    : 0.f;
    };
    if (i < items) {
      w = decode(i);
      fetch();
    }
    while (i < items) {
      const int tok0 = (w.first + t) * TOK;
      const uint32_t st = qr.at, ct = cr.at;
      ok = __all_sync(0xffffffffu, srv_wait(bar_q_empty + 8 * st, qr.parity ^ 1u, abort_flag, limit));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar_q_full + 8 * st, q_bytes);
        for (int y = 0; y < SM::NBOX; ++y)
          tma_load_3d(sQ + st * SM::Q_TILE + y * SM::Q_BOX, &tmQ, bar_q_full + 8 * st, y * SM::BOX_COLS,
                      w.h * p.group, w.q.row0 + tok0);
      }
      __syncwarp();
      ++qc;
      qr.next();
      // Columns: -lse in the log2 domain and the last key that the row sees (-1: no row).  Their
      // own ring: the queries' stage is free once the products are done, these only when they are added.
      float use[E];
      int lim[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        use[e] = nl[e];
        lim[e] = tk[e] < TOK && tok0 + tk[e] < w.q.n ? w.q.len - w.q.n + tok0 + tk[e] : -1;
      }
      if (++t == w.steps) {
        t = 0;
        if ((i = item_at(++r)) < items) w = decode(i);
      }
      if (i < items) fetch();
      ok = __all_sync(0xffffffffu, srv_wait(bar_c_empty + 8 * ct, cr.parity ^ 1u, abort_flag, limit));
      if (!ok) break;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s_lse[ct * MASS_COLS + lane + 32 * e] = -1.44269504088896341f * use[e];
        s_lim[ct * MASS_COLS + lane + 32 * e] = lim[e];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_c_full + 8 * ct);
      cr.next();
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      for (uint32_t j = qc > SM::STAGES ? qc - SM::STAGES : 0; j < qc; ++j)
        srv_wait(bar_q_full + 8 * (j % SM::STAGES), (j / SM::STAGES) & 1, nullptr, limit);
    }
  } else if (warp == ISSUER) {
    // ------------------------------------------------------------ MMA issuer
    // One warp for both key tiles: with one each, the two warps' products interleave, end
    // together, and the tensor core idles while both wait for their next operands.
    constexpr unsigned FULL = 0xffffffffu;
    bool ok = true, issued = false;
    MassRing<SM::KBUF> kr;
    MassRing<SM::STAGES> qr;
    MassRing<MASS_BUFS> sr;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = __all_sync(FULL, srv_wait(bar, parity, abort_flag, limit));
      return ok;
    };
    for (long r = 0, i; (i = item_at(r)) < items && ok; ++r) {
      const MassItem w = decode(i);
      if (!wait(bar_k_full + 8 * kr.at, kr.parity)) break;
      const uint32_t kaddr = sK + kr.at * NT * SM::TILE;
      int left = (w.q.n - w.first * TOK) * p.group;  // query rows from this tile on
      for (int s = 0; s < w.steps; ++s) {
        if (!wait(bar_q_full + 8 * qr.at, qr.parity) || !wait(bar_s_free + 8 * sr.at, sr.parity ^ 1u)) break;
        tc_fence_after();
        const int rows = min(TOK * p.group, left);
        left -= TOK * p.group;
        const uint32_t idesc = idesc_f16_f32(ATC_BM, (rows + 15) / 16 * 16, 0, 0, BF16);
        const uint32_t qaddr = sQ + qr.at * SM::Q_TILE;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t qd = HD == 32 ? desc_kmajor_sw64(qaddr) + (uint64_t)(2 * kk)
                                         : desc_kmajor_sw128(qaddr + (uint32_t)((kk >> 2) * SM::Q_BOX)) + (uint64_t)(2 * (kk & 3));
            mma_f16_ss_warp(tmem + (uint32_t)((MASS_BUFS * t + (int)sr.at) * MASS_ROWS),
                            atc_desc_qk<HD>(kaddr + t * SM::TILE, kk), qd, idesc, kk > 0 ? 1u : 0u);
          }
        mma_commit_warp(bar_s_full + 8 * sr.at);
        mma_commit_warp(bar_q_empty + 8 * qr.at);
        issued = true;
        qr.next();
        sr.next();
      }
      if (!ok) break;
      mma_commit_warp(bar_k_empty + 8 * kr.at);
      kr.next();
    }
    if (!ok) {
      if (lane == 0) *abort_flag = 1;
      if (issued) {
        mma_commit_warp(bar_drain);
        srv_wait(bar_drain, 0, nullptr, limit);
      }
    }
  } else {
    // ------------------------------------------------------------ adding warps
    const uint32_t u = (uint32_t)warp >> 2;  // accumulator of this warpgroup: query tiles u, u + 3, ...
    const int row = (warp & 3) * 32 + lane;  // key of each tile
    const uint32_t s_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + u * MASS_ROWS;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    // Slots behind the items: copied while the first keys are on their way.
    if (p.out != p.mass) {
      const int rows = p.s.batch * p.kv_heads;
      for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const SrvSeq q = s_seq[r / p.kv_heads];
        const long from = q.n > 0 ? (long)(q.len + ITEM_KEYS - 1) / ITEM_KEYS * ITEM_KEYS : 0;
#pragma unroll 4
        for (long j = from + threadIdx.x; j < p.cap; j += 32 * MASS_ADDERS) p.out[r * p.cap + j] = p.mass[r * p.cap + j];
      }
    }
    bool ok = true;
    uint32_t xc = 0;  // items whose sums the warpgroups exchanged
    MassRing<SM::COLS> cr;
    MassRing<MASS_BUFS> sr;
    for (long r = 0, i; (i = item_at(r)) < items && ok; ++r) {
      const MassItem w = decode(i);
      const int key = w.k0 + row;  // and key + 128 of the second tile
      const long at = ((long)w.b * p.kv_heads + w.h) * p.cap + key;
      // One query tile: its warpgroup writes the result; more: the first does, with all sums.
      const bool alone = w.steps == 1;
      const bool writes = alone ? sr.at == u : u == 0;
      float old[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) old[t] = writes && key + t * ATC_BM < p.cap ? p.mass[at + t * ATC_BM] : 0.f;
      unsigned long long acc[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0ull;
      for (int s = 0; s < w.steps; ++s, cr.next(), sr.next()) {
        if (sr.at != u) continue;
        const int tok0 = (w.first + s) * TOK;
        const int rows = min(TOK, w.q.n - tok0) * p.group;
        // Some row of this tile does not see some key of the item.
        const bool partly = w.k0 + ITEM_KEYS - 1 > w.q.len - w.q.n + tok0;
        // All lanes give up together (the __syncwarp below has no limit).
        ok = __all_sync(0xffffffffu, srv_wait(bar_c_full + 8 * cr.at, cr.parity, abort_flag, limit) &&
                                         srv_wait(bar_s_full + 8 * u, sr.parity, abort_flag, limit));
        if (!ok) break;
        tc_fence_after();
        const float* nl = s_lse + cr.at * MASS_COLS;
        const int* lim = s_lim + cr.at * MASS_COLS;
#pragma unroll 1
        for (int c0 = 0; c0 < rows; c0 += 16) {
          uint32_t v[NT][16];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            tmem_ld_32x32b_x16(s_addr + (uint32_t)(t * MASS_BUFS * MASS_ROWS + c0), v[t]);
          float4 l4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) l4[c] = *reinterpret_cast<const float4*>(nl + c0 + 4 * c);
#pragma unroll
          for (int t = 0; t < NT; ++t) tmem_wait_ld_of(v[t]);
          float2 x[NT][8];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              x[t][2 * c] = ffma2(make_float2(__uint_as_float(v[t][4 * c]), __uint_as_float(v[t][4 * c + 1])), sc2,
                                  make_float2(l4[c].x, l4[c].y));
              x[t][2 * c + 1] = ffma2(make_float2(__uint_as_float(v[t][4 * c + 2]), __uint_as_float(v[t][4 * c + 3])),
                                      sc2, make_float2(l4[c].z, l4[c].w));
            }
          if (partly || c0 + 16 > rows) {
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
              const int4 m4 = *reinterpret_cast<const int4*>(lim + c0 + 2 * c);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const int k = key + t * ATC_BM;
                x[t][c] = make_float2(k <= m4.x ? ex2_approx(x[t][c].x) : 0.f, k <= m4.y ? ex2_approx(x[t][c].y) : 0.f);
                x[t][c + 1] = make_float2(k <= m4.z ? ex2_approx(x[t][c + 1].x) : 0.f,
                                          k <= m4.w ? ex2_approx(x[t][c + 1].y) : 0.f);
              }
            }
          } else {
            // Of every eight pairs, MASS_FMA_PAIRS take their exponentials from the FMA pipe.
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                x[t][c] = (c * MASS_FMA_PAIRS) % 8 < MASS_FMA_PAIRS ? exp2_fine2(x[t][c])
                                                                   : make_float2(ex2_approx(x[t][c].x), ex2_approx(x[t][c].y));
          }
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[t][c & 3] = add2p(acc[t][c & 3], pk2(x[t][c].x, x[t][c].y));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_s_free + 8 * u);
          mbar_arrive(bar_c_empty + 8 * cr.at);
        }
      }
      if (!ok) break;
      float sum[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 a = upk2(add2p(add2p(acc[t][0], acc[t][1]), add2p(acc[t][2], acc[t][3])));
        sum[t] = a.x + a.y;
      }
      if (!alone) {
        // The other warpgroups hand their sums to the first, through one of two buffers in turn.
        const uint32_t xb = xc & 1, turn = xc >> 1;
        float* x = s_xch + xb * (MASS_BUFS - 1) * ITEM_KEYS + row;
        if (u != 0) {
          if (turn > 0 && !srv_wait(bar_x_free + 8 * xb, (turn - 1) & 1, abort_flag, limit)) ok = false;
#pragma unroll
          for (int t = 0; t < NT; ++t) x[(u - 1) * ITEM_KEYS + t * ATC_BM] = sum[t];
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_x_full + 8 * xb);
        } else {
          if (!srv_wait(bar_x_full + 8 * xb, turn & 1, abort_flag, limit)) ok = false;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int o = 0; o < MASS_BUFS - 1; ++o) sum[t] += x[o * ITEM_KEYS + t * ATC_BM];
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_x_free + 8 * xb);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++xc;
      }
      if (writes) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int k = key + t * ATC_BM;
          if (k < p.cap) p.out[at + t * ATC_BM] = k < w.q.len ? old[t] + sum[t] : old[t];
        }
      }
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

}  // namespace tttj
