// Attention mass of cached keys: for every sequence, key/value head and slot j, the sum of
// the probabilities exp(scale q k_j - lse) that the new tokens' queries gave to it.
//
// Keys stay, queries stream: S^T = K Q^T on the tensor cores with 128 keys as the rows of
// the accumulator and up to 128 query rows (token x group + head) as its columns, so a
// thread owns one key and adds its row of exponentials in registers -- no reduction across
// threads, no atomics, a fixed order.  The log-sum-exp of the attention makes every
// probability independent of the others, so one pass suffices.
//
// An item is NT key tiles of one head (two; one at head_dim 256); persistent CTAs take
// items in a fixed order.  Warp 8 loads K tiles (KBUF items ahead) and query tiles with
// their log-sum-exps, warps 9 / 10 issue the MMAs of key tile 0 / 1 into two accumulators
// each, warps 0-7 add.  For single tokens the bytes of K bound it; for chunks the
// exponentials and the products.  Slots without work are copied.
#pragma once
#include "attention_tc.cuh"
#include "serve_dev.cuh"

namespace tttj {

template <int HD>
struct MassSmem {
  static constexpr int NT = HD == 256 ? 1 : 2;
  static constexpr int KBUF = HD == 256 ? 1 : 2;   // items whose keys are loaded
  static constexpr int STAGES = HD == 256 ? 2 : HD == 128 ? 2 : 4;  // query tiles in flight
  static constexpr int TILE = ATC_BM * HD * 2;
  static constexpr int BOX_COLS = HD < 64 ? HD : 64;
  static constexpr int NBOX = HD / BOX_COLS;
  static constexpr int BOX_BYTES = ATC_BM * BOX_COLS * 2;
  static constexpr int K_BYTES = KBUF * NT * TILE;
  static constexpr int Q_BYTES = STAGES * TILE;
  static constexpr int COL_BYTES = STAGES * 128 * 8;  // (-lse, last key) of every query row
  static constexpr int NBAR = 2 * KBUF + 2 * STAGES + 8 + 2;
  static constexpr int FIXED = K_BYTES + Q_BYTES + COL_BYTES + NBAR * 8 + 16 + 1024;
};
constexpr int MASS_THREADS = 352;

struct MassItem {
  int b, h, k0;     // first key of the item
  SrvSeq q;
  int first, steps;  // query tiles first .. first + steps - 1; steps = 0: nothing to add
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(MASS_THREADS, 1)
    mass_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const MassParams p) {
  using SM = MassSmem<HD>;
  constexpr int NT = SM::NT;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sK = smem_u32(smem);
  const uint32_t sQ = sK + SM::K_BYTES;
  float* s_lse = reinterpret_cast<float*>(smem + SM::K_BYTES + SM::Q_BYTES);       // [STAGES][128]
  int* s_lim = reinterpret_cast<int*>(smem + SM::K_BYTES + SM::Q_BYTES) + SM::STAGES * 128;
  const uint32_t bar0 = sQ + SM::Q_BYTES + SM::COL_BYTES;
  const uint32_t bar_k_full = bar0;                          // [KBUF]
  const uint32_t bar_k_empty = bar_k_full + 8 * SM::KBUF;    // [KBUF]
  const uint32_t bar_q_full = bar_k_empty + 8 * SM::KBUF;    // [STAGES]
  const uint32_t bar_q_empty = bar_q_full + 8 * SM::STAGES;  // [STAGES]
  const uint32_t bar_s_full = bar_q_empty + 8 * SM::STAGES;  // [side][2]
  const uint32_t bar_s_free = bar_s_full + 32;               // [side][2]
  const uint32_t bar_drain = bar_s_free + 32;                // [side]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::K_BYTES + SM::Q_BYTES + SM::COL_BYTES + SM::NBAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SrvSeq* s_seq = reinterpret_cast<SrvSeq*>(tmem_slot + 4);  // [batch]
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
      mbar_init(bar_q_empty + 8 * i, NT + 4 * NT);  // MMA warps and adding warps
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar_s_full + 8 * i, 1);
      mbar_init(bar_s_free + 8 * i, 4);
    }
    mbar_init(bar_drain, 1);
    mbar_init(bar_drain + 8, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch();
  for (int b = threadIdx.x; b < p.s.batch; b += MASS_THREADS) s_seq[b] = srv_seq(p.s, b);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  constexpr int ITEM_KEYS = NT * ATC_BM;
  const long per_head = (p.cap + ITEM_KEYS - 1) / ITEM_KEYS;
  const long items = per_head * p.s.batch * p.kv_heads;
  auto decode = [&](long i) {
    MassItem w;
    const long bh = i / per_head;
    w.k0 = (int)(i - bh * per_head) * ITEM_KEYS;
    w.b = (int)(bh / p.kv_heads);
    w.h = (int)(bh - (long)w.b * p.kv_heads);
    w.q = s_seq[w.b];
    w.first = w.steps = 0;
    if (w.k0 < w.q.len && w.q.n > 0) {
      // The first token that sees key k0; the last one sees every key.
      w.first = max(0, w.k0 - (w.q.len - w.q.n)) / TOK;
      w.steps = (w.q.n + TOK - 1) / TOK - w.first;
    }
    return w;
  };

  if (warp == 8) {
    // ------------------------------------------------------------ loader
    const int cr = min(ATC_BM, 1 << p.s.page_shift);
    const int boxes = (ATC_BM / cr) * SM::NBOX * NT;  // <= 32
    const uint32_t q_bytes = (uint32_t)(TOK * p.group * HD * 2);
    bool ok = true;
    long kc = 0, qc = 0;
    for (long i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const MassItem w = decode(i);
      if (w.steps == 0) continue;
      // lane -> (64-column box, page piece of the item's keys)
      const int x = lane % SM::NBOX, piece = lane / SM::NBOX;
      const int slot = w.k0 + piece * cr;
      int page = p.s.num_pages;
      if (lane < boxes && slot < w.q.len) page = srv_page(p.s, w.b, slot);
      const int kb = (int)(kc % SM::KBUF);
      ok = __all_sync(0xffffffffu, srv_wait(bar_k_empty + 8 * kb, (uint32_t)((kc / SM::KBUF) & 1) ^ 1u, abort_flag, limit));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(bar_k_full + 8 * kb, NT * SM::TILE);
      __syncwarp();
      if (lane < boxes) {
        const int key = piece * cr;  // inside the item
        tma_load_4d(sK + (kb * NT + key / ATC_BM) * SM::TILE + x * SM::BOX_BYTES + (key % ATC_BM) * SM::BOX_COLS * 2,
                    &tmK, bar_k_full + 8 * kb, x * SM::BOX_COLS, slot & ((1 << p.s.page_shift) - 1), w.h, page);
      }
      __syncwarp();
      ++kc;
      for (int t = 0; t < w.steps; ++t, ++qc) {
        const int tok0 = (w.first + t) * TOK;
        // Columns: -lse in the log2 domain and the last key that the row sees (-1: no row).
        float nl[4];
        int lim[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = lane + 32 * e;
          const int tk = c / p.group, g = c - tk * p.group;
          const bool live = tk < TOK && tok0 + tk < w.q.n;
          nl[e] = live ? -1.44269504088896341f *
                             p.lse[(long)(w.q.row0 + tok0 + tk) * p.heads + w.h * p.group + g]
                       : 0.f;
          lim[e] = live ? w.q.len - w.q.n + tok0 + tk : -1;
        }
        const int st = (int)(qc % SM::STAGES);
        ok = __all_sync(0xffffffffu, srv_wait(bar_q_empty + 8 * st, (uint32_t)((qc / SM::STAGES) & 1) ^ 1u, abort_flag, limit));
        if (!ok) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s_lse[st * 128 + lane + 32 * e] = nl[e];
          s_lim[st * 128 + lane + 32 * e] = lim[e];
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(bar_q_full + 8 * st, q_bytes);
          for (int y = 0; y < SM::NBOX; ++y)
            tma_load_3d(sQ + st * SM::TILE + y * SM::BOX_BYTES, &tmQ, bar_q_full + 8 * st, y * SM::BOX_COLS,
                        w.h * p.group, w.q.row0 + tok0);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      report_status(p.s.status, SRV_DEV_TIMEOUT);
      for (long j = kc > SM::KBUF ? kc - SM::KBUF : 0; j < kc; ++j)
        srv_wait(bar_k_full + 8 * (int)(j % SM::KBUF), (uint32_t)((j / SM::KBUF) & 1), nullptr, limit);
      for (long j = qc > SM::STAGES ? qc - SM::STAGES : 0; j < qc; ++j)
        srv_wait(bar_q_full + 8 * (int)(j % SM::STAGES), (uint32_t)((j / SM::STAGES) & 1), nullptr, limit);
    }
  } else if (warp == 9 || (warp == 10 && NT == 2)) {
    // ------------------------------------------------------------ MMA issuers
    constexpr unsigned FULL = 0xffffffffu;
    const int t = warp - 9;
    bool ok = true, issued = false;
    long kc = 0, qc = 0;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = __all_sync(FULL, srv_wait(bar, parity, abort_flag, limit));
      tc_fence_after();
      return ok;
    };
    for (long i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const MassItem w = decode(i);
      if (w.steps == 0) continue;
      const int kb = (int)(kc % SM::KBUF);
      if (!wait(bar_k_full + 8 * kb, (uint32_t)((kc / SM::KBUF) & 1))) break;
      const uint32_t kaddr = sK + (kb * NT + t) * SM::TILE;
      for (int s = 0; s < w.steps; ++s, ++qc) {
        const int st = (int)(qc % SM::STAGES), buf = (int)(qc & 1);
        if (!wait(bar_q_full + 8 * st, (uint32_t)((qc / SM::STAGES) & 1))) break;
        if (!wait(bar_s_free + 8 * (2 * t + buf), (uint32_t)((qc >> 1) & 1) ^ 1u)) break;
        const int rows = min(TOK, w.q.n - (w.first + s) * TOK) * p.group;
        const uint32_t idesc = idesc_f16_f32(ATC_BM, (rows + 15) / 16 * 16, 0, 0, BF16);
        const uint32_t qaddr = sQ + st * SM::TILE;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_f16_ss_warp(tmem + (uint32_t)((2 * t + buf) * 128), atc_desc_qk<HD>(kaddr, kk),
                          atc_desc_qk<HD>(qaddr, kk), idesc, kk > 0 ? 1u : 0u);
        mma_commit_warp(bar_s_full + 8 * (2 * t + buf));
        mma_commit_warp(bar_q_empty + 8 * st);
        issued = true;
      }
      if (!ok) break;
      mma_commit_warp(bar_k_empty + 8 * kb);
      ++kc;
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
  } else if (warp < 4 * NT) {
    // ------------------------------------------------------------ adding warps
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t s_base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(2 * t * 128);
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    long qc = 0;
    for (long i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const MassItem w = decode(i);
      const int tile0 = w.k0 + t * ATC_BM;
      const int key = tile0 + row;
      const long at = ((long)w.b * p.kv_heads + w.h) * p.cap + key;
      const float old = key < p.cap ? p.mass[at] : 0.f;
      unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};
      for (int s = 0; s < w.steps; ++s, ++qc) {
        const int st = (int)(qc % SM::STAGES), buf = (int)(qc & 1);
        const int tok0 = (w.first + s) * TOK;
        const int rows = min(TOK, w.q.n - tok0) * p.group;
        // Some row of this tile does not see some key of this one.
        const bool partly = tile0 + ATC_BM - 1 > w.q.len - w.q.n + tok0;
        if (!srv_wait(bar_q_full + 8 * st, (uint32_t)((qc / SM::STAGES) & 1), abort_flag, limit) ||
            !srv_wait(bar_s_full + 8 * (2 * t + buf), (uint32_t)((qc >> 1) & 1), abort_flag, limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float* nl = s_lse + st * 128;
        const int* lim = s_lim + st * 128;
        for (int c0 = 0; c0 < rows; c0 += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(s_base + (uint32_t)(buf * 128 + c0), v);
          tmem_wait_ld();
          if (partly || c0 + 32 > rows) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(nl + c0 + c);
              const int4 m4 = *reinterpret_cast<const int4*>(lim + c0 + c);
              const float x0 = fmaf(__uint_as_float(v[c]), sc2.x, l4.x), x1 = fmaf(__uint_as_float(v[c + 1]), sc2.x, l4.y);
              const float x2 = fmaf(__uint_as_float(v[c + 2]), sc2.x, l4.z), x3 = fmaf(__uint_as_float(v[c + 3]), sc2.x, l4.w);
              acc[0] = add2p(acc[0], pk2(key <= m4.x ? ex2_approx(x0) : 0.f, key <= m4.y ? ex2_approx(x1) : 0.f));
              acc[1] = add2p(acc[1], pk2(key <= m4.z ? ex2_approx(x2) : 0.f, key <= m4.w ? ex2_approx(x3) : 0.f));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(nl + c0 + c);
              const float2 a = ffma2(make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), sc2, make_float2(l4.x, l4.y));
              const float2 b = ffma2(make_float2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), sc2, make_float2(l4.z, l4.w));
              acc[(c >> 1) & 3] = add2p(acc[(c >> 1) & 3], pk2(ex2_approx(a.x), ex2_approx(a.y)));
              acc[((c >> 1) & 3) + 1] = add2p(acc[((c >> 1) & 3) + 1], pk2(ex2_approx(b.x), ex2_approx(b.y)));
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_s_free + 8 * (2 * t + buf));
          mbar_arrive(bar_q_empty + 8 * st);
        }
      }
      if (!ok) break;
      const float2 a = upk2(add2p(add2p(acc[0], acc[1]), add2p(acc[2], acc[3])));
      if (key < p.cap) p.out[at] = key < w.q.len ? old + (a.x + a.y) : old;
    }
    if (!ok) {
      *abort_flag = 1;
      report_status(p.s.status, SRV_DEV_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace tttj
