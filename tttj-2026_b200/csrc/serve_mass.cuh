// Attention mass of cached keys: for every sequence, key/value head and slot j, the sum of
// the probabilities exp(scale q k_j - lse) that the new tokens' queries gave to it.
//
// Keys stay, queries stream: S^T = K Q^T on the tensor cores with 128 keys as the rows of
// the accumulator and up to 128 query rows (token x group + head) as its columns, so a
// thread owns one key and adds its row of exponentials in registers -- no reduction across
// threads, no atomics, a fixed order.  The log-sum-exp of the attention makes every
// probability independent of the others, so one pass suffices.
//
// An item is NT key tiles of one head (two; one at head_dim 256); persistent CTAs take the items
// that have work in turn (each computes the sequences' prefix sums itself), and share the
// copying of the rest.  One warp loads K tiles (KBUF items ahead), another the query tiles with
// their log-sum-exps (one warp for both made every item wait for page numbers and then for
// log-sum-exps: 46 against 38 us at 32 sequences of 1000 - 4096 keys), one per key tile issues
// its MMAs into three accumulators in turn, and two warpgroups per key tile add every other query
// tile; their sums meet at the end of an item.
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
  static constexpr int NBAR = 2 * KBUF + 2 * STAGES + 2 * COLS + 4 * MASS_BUFS + 2 + 8;
  static constexpr int XCH_BYTES = NT * 2 * ATC_BM * 4;  // [tile][item parity][key] sums of the second warpgroup
  static constexpr int FIXED = K_BYTES + Q_BYTES + COL_BYTES + XCH_BYTES + NBAR * 8 + 16 + 1024;
};
// Warps: two warpgroups that add per key tile (each takes every other query tile, one accumulator
// each), the key loader, the MMA issuers, the query loader.
constexpr int mass_adders(int nt) { return 8 * nt; }
constexpr int mass_threads(int nt) { return 32 * (mass_adders(nt) + 2 + nt); }

#ifndef MASS_FMA_PAIRS
#define MASS_FMA_PAIRS 2
#endif

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
__global__ void __launch_bounds__(mass_threads(MassSmem<HD>::NT), 1)
    mass_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const MassParams p) {
  using SM = MassSmem<HD>;
  constexpr int NT = SM::NT;
  constexpr int KEYS = mass_adders(NT), ISSUER = KEYS + 1, QUERIES = ISSUER + NT;  // warps
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
  const uint32_t bar_s_full = bar_c_empty + 8 * SM::COLS;    // [side][MASS_BUFS]
  const uint32_t bar_s_free = bar_s_full + 16 * MASS_BUFS;   // [side][MASS_BUFS]
  const uint32_t bar_x_full = bar_s_free + 16 * MASS_BUFS;               // [side][2] second warpgroup's sums
  const uint32_t bar_x_free = bar_x_full + 32;               // [side][2] read by the first
  const uint32_t bar_drain = bar_x_free + 32;                // [side]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::K_BYTES + SM::Q_BYTES + SM::COL_BYTES + SM::XCH_BYTES +
                                                      SM::NBAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SrvSeq* s_seq = reinterpret_cast<SrvSeq*>(tmem_slot + 4);  // [batch]
  int* s_pre = reinterpret_cast<int*>(s_seq + p.s.batch);    // [batch + 1] items of a head before each place
  int* s_order = s_pre + p.s.batch + 1;                       // [batch] sequence at each place
  const int warp = warp_id(), lane = lane_id();
  const uint64_t limit = p.wait_limit_ns;
  const int TOK = p.tile_tokens;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    for (int i = 0; i < SM::KBUF; ++i) {
      mbar_init(bar_k_full + 8 * i, 1);
      mbar_init(bar_k_empty + 8 * i, NT);
    }
    for (int i = 0; i < SM::STAGES; ++i) {
      mbar_init(bar_q_full + 8 * i, 1);
      mbar_init(bar_q_empty + 8 * i, NT);
    }
    for (int i = 0; i < SM::COLS; ++i) {
      mbar_init(bar_c_full + 8 * i, 1);
      mbar_init(bar_c_empty + 8 * i, 4 * NT);
    }
    for (int i = 0; i < 2 * MASS_BUFS; ++i) {
      mbar_init(bar_s_full + 8 * i, 1);
      mbar_init(bar_s_free + 8 * i, 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar_x_full + 8 * i, 4);
      mbar_init(bar_x_free + 8 * i, 4);
    }
    mbar_init(bar_drain, 1);
    mbar_init(bar_drain + 8, 1);
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
    for (long r = 0, i; (i = item_at(r)) < items && ok; ++r) {
      const MassItem w = decode(i);
      const int slot = w.k0 + key;
      int page = p.s.num_pages;
      if (lane < boxes && slot < w.q.len) page = srv_page(p.s, w.b, slot);
      const int kb = (int)(kc % SM::KBUF);
      ok = __all_sync(0xffffffffu, srv_wait(bar_k_empty + 8 * kb, (uint32_t)((kc / SM::KBUF) & 1) ^ 1u, abort_flag, limit));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(bar_k_full + 8 * kb, NT * SM::TILE);
      __syncwarp();
      if (lane < boxes)
        tma_load_4d(sK + kb * NT * SM::TILE + dst, &tmK, bar_k_full + 8 * kb, x * SM::BOX_COLS,
                    slot & ((1 << p.s.page_shift) - 1), w.h, page);
      __syncwarp();
      ++kc;
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      report_status(p.s.status, SRV_DEV_TIMEOUT);
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
      report_status(p.s.status, SRV_DEV_TIMEOUT);
      for (uint32_t j = qc > SM::STAGES ? qc - SM::STAGES : 0; j < qc; ++j)
        srv_wait(bar_q_full + 8 * (j % SM::STAGES), (j / SM::STAGES) & 1, nullptr, limit);
    }
  } else if (warp >= ISSUER) {
    // ------------------------------------------------------------ MMA issuers
    constexpr unsigned FULL = 0xffffffffu;
    const int t = warp - ISSUER;
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
      const uint32_t kaddr = sK + (kr.at * NT + t) * SM::TILE;
      for (int s = 0; s < w.steps; ++s) {
        const uint32_t buf = MASS_BUFS * t + sr.at;
        if (!wait(bar_q_full + 8 * qr.at, qr.parity) || !wait(bar_s_free + 8 * buf, sr.parity ^ 1u)) break;
        tc_fence_after();
        const int rows = min(TOK, w.q.n - (w.first + s) * TOK) * p.group;
        const uint32_t idesc = idesc_f16_f32(ATC_BM, (rows + 15) / 16 * 16, 0, 0, BF16);
        const uint32_t qaddr = sQ + qr.at * SM::Q_TILE;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint64_t qd = HD == 32 ? desc_kmajor_sw64(qaddr) + (uint64_t)(2 * kk)
                                       : desc_kmajor_sw128(qaddr + (uint32_t)((kk >> 2) * SM::Q_BOX)) + (uint64_t)(2 * (kk & 3));
          mma_f16_ss_warp(tmem + (uint32_t)(buf * MASS_ROWS), atc_desc_qk<HD>(kaddr, kk), qd, idesc, kk > 0 ? 1u : 0u);
        }
        mma_commit_warp(bar_s_full + 8 * buf);
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
      if (lane == 0) {
        *abort_flag = 1;
        report_status(p.s.status, SRV_DEV_TIMEOUT);
      }
      if (issued) {
        mma_commit_warp(bar_drain + 8 * t);
        srv_wait(bar_drain + 8 * t, 0, nullptr, limit);
      }
    }
  } else {
    // ------------------------------------------------------------ adding warps
    const int t = warp >> 3, u = (warp >> 2) & 1;  // key tile, query tiles of one parity
    const int row = (warp & 3) * 32 + lane;
    const uint32_t s_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    // Slots behind the items: copied while the first keys are on their way.
    if (p.out != p.mass) {
      const int rows = p.s.batch * p.kv_heads;
      for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const SrvSeq q = s_seq[r / p.kv_heads];
        const long from = q.n > 0 ? (long)(q.len + ITEM_KEYS - 1) / ITEM_KEYS * ITEM_KEYS : 0;
#pragma unroll 4
        for (long j = from + threadIdx.x; j < p.cap; j += 32 * mass_adders(NT)) p.out[r * p.cap + j] = p.mass[r * p.cap + j];
      }
    }
    bool ok = true;
    uint32_t parity = 0;  // of the query tiles of earlier items
    uint32_t xc = 0;      // items whose sums the two warpgroups exchanged
    MassRing<SM::COLS> cr;
    MassRing<MASS_BUFS> sr;
    for (long r = 0, i; (i = item_at(r)) < items && ok; ++r) {
      const MassItem w = decode(i);
      const int tile0 = w.k0 + t * ATC_BM;
      const int key = tile0 + row;
      const long at = ((long)w.b * p.kv_heads + w.h) * p.cap + key;
      // One query tile: its warpgroup writes the result; more: the first does, with both sums.
      const bool alone = w.steps == 1;
      const bool writes = alone ? parity == (uint32_t)u : u == 0;
      const float old = writes && key < p.cap ? p.mass[at] : 0.f;
      unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};
      for (int s = 0; s < w.steps; ++s, cr.next(), sr.next(), parity ^= 1) {
        if (parity != (uint32_t)u) continue;
        const uint32_t ct = cr.at, buf = MASS_BUFS * t + sr.at;
        const uint32_t s_addr = s_base + buf * MASS_ROWS;
        const int tok0 = (w.first + s) * TOK;
        const int rows = min(TOK, w.q.n - tok0) * p.group;
        // Some row of this tile does not see some key of this one.
        const bool partly = tile0 + ATC_BM - 1 > w.q.len - w.q.n + tok0;
        if (!srv_wait(bar_c_full + 8 * ct, cr.parity, abort_flag, limit) ||
            !srv_wait(bar_s_full + 8 * buf, sr.parity, abort_flag, limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float* nl = s_lse + ct * MASS_COLS;
        const int* lim = s_lim + ct * MASS_COLS;
        auto add = [&](auto& v, int c0) {
          constexpr int N = sizeof(v) / 8;  // pairs
          float2 x[N];
#pragma unroll
          for (int c = 0; c < N; c += 2) {
            const float4 l4 = *reinterpret_cast<const float4*>(nl + c0 + 2 * c);
            x[c] = ffma2(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), sc2, make_float2(l4.x, l4.y));
            x[c + 1] = ffma2(make_float2(__uint_as_float(v[2 * c + 2]), __uint_as_float(v[2 * c + 3])), sc2, make_float2(l4.z, l4.w));
          }
          if (partly || c0 + 2 * N > rows) {
#pragma unroll
            for (int c = 0; c < N; c += 2) {
              const int4 m4 = *reinterpret_cast<const int4*>(lim + c0 + 2 * c);
              x[c] = make_float2(key <= m4.x ? ex2_approx(x[c].x) : 0.f, key <= m4.y ? ex2_approx(x[c].y) : 0.f);
              x[c + 1] = make_float2(key <= m4.z ? ex2_approx(x[c + 1].x) : 0.f, key <= m4.w ? ex2_approx(x[c + 1].y) : 0.f);
            }
          } else {
            // Of every eight pairs, MASS_FMA_PAIRS take their exponentials from the FMA pipe.
#pragma unroll
            for (int c = 0; c < N; ++c)
              x[c] = (c * MASS_FMA_PAIRS) % 8 < MASS_FMA_PAIRS ? exp2_fine2(x[c]) : make_float2(ex2_approx(x[c].x), ex2_approx(x[c].y));
          }
#pragma unroll
          for (int c = 0; c < N; ++c) acc[c & 3] = add2p(acc[c & 3], pk2(x[c].x, x[c].y));
        };
#pragma unroll 1
        for (int c0 = 0; c0 < min(rows, 64); c0 += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(s_addr + (uint32_t)c0, v);
          tmem_wait_ld_of(v);
          add(v, c0);
        }
        if (rows > 64) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(s_addr + 64, v);
          tmem_wait_ld_of(v);
          add(v, 64);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_s_free + 8 * buf);
          mbar_arrive(bar_c_empty + 8 * ct);
        }
      }
      if (!ok) break;
      const float2 a = upk2(add2p(add2p(acc[0], acc[1]), add2p(acc[2], acc[3])));
      float sum = a.x + a.y;
      if (!alone) {
        // The second warpgroup hands its sum over, through one of two buffers in turn.
        const uint32_t xb = 2 * t + (xc & 1), turn = xc >> 1;
        float* x = s_xch + xb * ATC_BM + row;
        if (u == 1) {
          if (turn > 0 && !srv_wait(bar_x_free + 8 * xb, (turn - 1) & 1, abort_flag, limit)) ok = false;
          *x = sum;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_x_full + 8 * xb);
        } else {
          if (!srv_wait(bar_x_full + 8 * xb, turn & 1, abort_flag, limit)) ok = false;
          sum += *x;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_x_free + 8 * xb);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++xc;
      }
      if (writes && key < p.cap) p.out[at] = key < w.q.len ? old + sum : old;
    }
    if (!ok) {
      *abort_flag = 1;
      report_status(p.s.status, SRV_DEV_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace tttj
