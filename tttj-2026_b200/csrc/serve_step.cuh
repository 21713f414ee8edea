// Causal attention of few query rows (single tokens, short drafts) over the many keys of a
// paged cache.
//
// For each sequence, key/value head and block of 16 query rows (row = new token x group
// + head of the group): O = softmax(scale q K^T) V over the slots a row may see.  What
// bounds it is the bytes of K and V: the rows of one group share them, and 16 rows of
// mma.m16n8k16 are far below the tensor cores' rate.  So the design is about keeping
// HBM busy and even:
//   * the call's work is one line of units, a unit = 64 keys of one (sequence, head, row
//     block); every CTA takes the same number of consecutive units, whatever the
//     sequences' lengths, computing the line's prefix sums itself (no host knowledge of
//     lengths, so the call can be captured and replayed with new ones);
//   * a producer warp streams K / V tiles by TMA into a ring of stages across the
//     boundaries of sequences; four consumer warps take 16 keys of each tile, each with
//     its own running maximum and sum, merged through shared memory at the end of a run;
//   * a run that does not cover a row block's whole key range leaves (max, sum, O) in
//     the workspace, and a second small kernel joins the runs of each row in order.
#pragma once
#include <math_constants.h>

#include "serve_dev.cuh"

namespace tttj {

template <int HD>
struct StepSmem {
  static constexpr int BOX_COLS = HD < 64 ? HD : 64;
  static constexpr int NBOX = HD / BOX_COLS;
  static constexpr int ROW_BYTES = BOX_COLS * 2;
  static constexpr int BOX_BYTES = STEP_KEYS * ROW_BYTES;
  static constexpr int TILE = STEP_KEYS * HD * 2;
  // About 96 KB in flight per CTA hides the HBM latency: 64 KB at head_dim 32, 192 KB at 256 (one CTA
  // per SM).  Two CTAs per SM fit with it, at head_dim 128 up to about 890 sequences: with more,
  // the prefix sums leave room for one at a time, and half the bytes are in flight.
  static constexpr int STAGES = HD == 256 ? 3 : HD == 128 ? 3 : HD == 64 ? 6 : 8;
  static constexpr int OSTRIDE = HD + 8;  // floats; rows 8 banks apart
  static constexpr int RING = STAGES * 2 * TILE;
  static constexpr int OBUF = STEP_ROWS * OSTRIDE * 4;
  static constexpr int ML = 4 * STEP_ROWS * 8;
  static constexpr int BARS = 2 * STAGES * 8 + 16;
  static constexpr int FIXED = RING + OBUF + ML + BARS + 1024;
};

constexpr int STEP_THREADS = 160;
// Units a CTA takes at least: shorter runs would cost more in joining than they save.
constexpr int STEP_MIN_UNITS = 2;

struct StepBlocks {  // row blocks and key tiles of a sequence
  int blocks, tiles;
};
__device__ __forceinline__ StepBlocks step_blocks(const SrvSeq& q, int group) {
  StepBlocks r;
  const long rows = (long)q.n * group;
  r.blocks = (int)((rows + STEP_ROWS - 1) / STEP_ROWS);
  r.tiles = max(1, (q.len + STEP_KEYS - 1) / STEP_KEYS);
  return r;
}
__device__ __forceinline__ long step_units(const StepParams& p, int b) {
  const SrvSeq q = srv_seq(p.s, b);
  const StepBlocks k = step_blocks(q, p.group);
  return (long)k.blocks * k.tiles * p.kv_heads;
}

// Prefix sums of the sequences' units in shared memory; returns with pre[batch] = total.
// All `threads` threads of the block call it.
__device__ __forceinline__ void step_prefix(const StepParams& p, long* pre, int threads) {
  const int batch = p.s.batch;
  for (int b = threadIdx.x; b < batch; b += threads) pre[b + 1] = step_units(p, b);
  if (threadIdx.x == 0) pre[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    long base = 0;
    for (int b0 = 0; b0 < batch; b0 += 32) {
      const int b = b0 + (int)threadIdx.x;
      long v = b < batch ? pre[b + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long o = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)threadIdx.x >= d) v += o;
      }
      if (b < batch) pre[b + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
}
__device__ __forceinline__ long step_per_cta(long total, int grid) {
  return max((total + grid - 1) / grid, (long)STEP_MIN_UNITS);
}

struct StepRun {
  int b, h, rb, t0, t1, tiles;
  SrvSeq q;
};
// The run of units that starts at unit u (and ends before u1) inside one row block.
__device__ __forceinline__ StepRun step_run(const StepParams& p, const long* pre, long u, long u1) {
  int lo = 0, hi = p.s.batch - 1;  // last b with pre[b] <= u
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= u) lo = mid; else hi = mid - 1;
  }
  StepRun r;
  r.b = lo;
  r.q = srv_seq(p.s, lo);
  const StepBlocks k = step_blocks(r.q, p.group);
  const long at = u - pre[lo];
  const long blk = at / k.tiles;
  r.tiles = k.tiles;
  r.t0 = (int)(at - blk * k.tiles);
  r.t1 = (int)min((long)k.tiles, r.t0 + (u1 - u));
  r.h = (int)(blk / k.blocks);
  r.rb = (int)(blk - (long)r.h * k.blocks);
  return r;
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(STEP_THREADS, step_ctas_per_sm(HD))
    step_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const StepParams p) {
  using SM = StepSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t ring = smem_u32(smem);
  float* obuf = reinterpret_cast<float*>(smem + SM::RING);
  float2* ml = reinterpret_cast<float2*>(smem + SM::RING + SM::OBUF);
  const uint32_t bar_full = ring + SM::RING + SM::OBUF + SM::ML;
  const uint32_t bar_empty = bar_full + 8 * SM::STAGES;
  volatile int* abort_flag =
      reinterpret_cast<volatile int*>(smem + SM::RING + SM::OBUF + SM::ML + 16 * SM::STAGES);
  long* pre = reinterpret_cast<long*>(smem + SM::RING + SM::OBUF + SM::ML + SM::BARS);
  const int warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int s = 0; s < SM::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  griddep_wait();
  griddep_launch();
  step_prefix(p, pre, STEP_THREADS);
  const long total = pre[p.s.batch];
  const long per = step_per_cta(total, gridDim.x);
  const long u0 = (long)blockIdx.x * per;
  const long u1 = min(total, u0 + per);

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    const int cr = min(STEP_KEYS, 1 << p.s.page_shift);
    const int chunks = STEP_KEYS / cr;
    const int boxes = chunks * SM::NBOX * 2;  // <= 32
    const int kv = lane & 1, box = (lane >> 1) % SM::NBOX, chunk = (lane >> 1) / SM::NBOX;
    const uint32_t dst = (uint32_t)(kv * SM::TILE + box * SM::BOX_BYTES + chunk * cr * SM::ROW_BYTES);
    long it = 0;
    bool ok = true;
    for (long u = u0; u < u1 && ok;) {
      const StepRun r = step_run(p, pre, u, u1);
      for (int t = r.t0; t < r.t1; ++t, ++it) {
        const int slot = t * STEP_KEYS + chunk * cr;
        const int page = lane < boxes && slot < r.q.len ? srv_page(p.s, r.b, slot) : p.s.num_pages;
        const int c1 = slot & ((1 << p.s.page_shift) - 1);
        const int st = (int)(it % SM::STAGES);
        ok = srv_wait(bar_empty + 8 * st, (uint32_t)((it / SM::STAGES) & 1) ^ 1u, abort_flag,
                       SRV_WAIT_LIMIT_NS);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t bar = bar_full + 8 * st;
        if (lane == 0) mbar_arrive_expect_tx(bar, 2 * SM::TILE);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(ring + st * 2 * SM::TILE + dst, kv ? &tm_v : &tm_k, bar, box * SM::BOX_COLS, c1,
                      r.h, page);
      }
      u += r.t1 - r.t0;
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      srv_report_timeout(p.s.status, p.timeout_host);
    }
    // Issued loads land before the CTA may exit.
    if (!ok)
      for (long j = it > SM::STAGES ? it - SM::STAGES : 0; j < it; ++j)
        srv_wait(bar_full + 8 * (int)(j % SM::STAGES), (uint32_t)((j / SM::STAGES) & 1), nullptr,
                  SRV_WAIT_LIMIT_NS);
    return;
  }

  // -------------------------------------------------------------- consumers
  const uint32_t* q32 = reinterpret_cast<const uint32_t*>(p.q);
  const float scale = p.scale_log2;
  long it = 0;
  bool first_run = true;
  bool ok = true;  // false for good once a wait gave up (warp-uniform)
  for (long u = u0; u < u1;) {
    const StepRun r = step_run(p, pre, u, u1);
    const int rows = r.q.n * p.group;
    // This thread's two rows of the block: their queries and the last slot each sees.
    uint32_t qf[HD / 16][4];
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = r.rb * STEP_ROWS + (lane >> 2) + 8 * e;
      const int tok = row / p.group, g = row - tok * p.group;
      const bool live = row < rows;
      lim[e] = live ? r.q.len - r.q.n + tok : -1;
      const long at = ((long)(r.q.row0 + (live ? tok : 0)) * p.q_tok +
                       (long)(r.h * p.group + (live ? g : 0)) * p.q_head) / 2 + (lane & 3);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qf[k][e] = live ? q32[at + k * 8] : 0u;
        qf[k][e + 2] = live ? q32[at + k * 8 + 4] : 0u;
      }
    }
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    // Slots from here on are hidden from some row of the block (or from all).
    const int all_see = r.q.len - r.q.n + 1;

    for (int t = r.t0; ok && t < r.t1; ++t, ++it) {
      const int st = (int)(it % SM::STAGES);
      ok = __all_sync(0xffffffffu, srv_wait(bar_full + 8 * st, (uint32_t)((it / SM::STAGES) & 1), abort_flag,
                                            SRV_WAIT_LIMIT_NS));
      if (!ok) {
        *abort_flag = 1;
        if (lane == 0) srv_report_timeout(p.s.status, p.timeout_host);
        break;
      }
      const int k0 = t * STEP_KEYS + warp * 16;  // this warp's 16 keys
      const uint32_t sk = ring + st * 2 * SM::TILE, sv = sk + SM::TILE;
      if (k0 < r.q.len) {
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        auto at = [&](uint32_t base, int key, int c16) -> uint32_t {
          if constexpr (HD == 32)
            return base + (uint32_t)(key * 64 + ((c16 ^ ((key >> 1) & 3)) << 4));
          else
            return base + (uint32_t)((c16 >> 3) * SM::BOX_BYTES + key * 128 + (((c16 & 7) ^ (key & 7)) << 4));
        };
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t b[4];
          ldsm_x4(b, at(sk, warp * 16 + ((lane >> 4) << 3) + (lane & 7), k * 2 + ((lane >> 3) & 1)));
          mma_16816<BF16>(s[0], qf[k], b[0], b[1]);
          mma_16816<BF16>(s[1], qf[k], b[2], b[3]);
        }
        bool odd = false;  // an infinite or NaN value among this warp's 16 keys
        if (k0 + 16 > all_see) {
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k0 + nb * 8 + (lane & 3) * 2 + (e & 1) > min(lim[e >> 1], r.q.len - 1)) s[nb][e] = -INFINITY;
          // Values that a row does not see must not reach it: 0 x NaN is NaN.  Rows
          // behind the last slot become zeros; an infinite or NaN element inside is
          // added to the rows that see it, then made zero for the product.
          for (int i = lane; i < 16 * (HD / 8); i += 32) {
            const int key = i / (HD / 8), c16 = i % (HD / 8);
            const uint32_t a = at(sv, warp * 16 + key, c16);
            if (k0 + key >= r.q.len) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
            } else {
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                           : "r"(a)
                           : "memory");
#pragma unroll
              for (int x = 0; x < 4; ++x) odd |= srv_nonfinite<BF16>(w[x]);
            }
          }
          __syncwarp();
          odd = __any_sync(0xffffffffu, odd);
          fence_proxy_async_smem();  // before the ring's next TMA write of these bytes
        }
        float base[2];
        bool grow = false;
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * scale;
          const float m_new = fmaxf(m[e], mx);
          alpha[e] = m_new == m[e] ? 1.f : ex2_approx(m[e] - m_new);  // m = -inf: 0
          grow |= m_new != m[e];
          m[e] = m_new;
          base[e] = m_new == -INFINITY ? 0.f : m_new;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) l[e] *= alpha[e];
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            o[i][0] *= alpha[0];
            o[i][1] *= alpha[0];
            o[i][2] *= alpha[1];
            o[i][3] *= alpha[1];
          }
        }
        if (odd) {
          for (int key = 0; key < 16; ++key) {
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
              uint32_t w;
              asm volatile("ld.shared.b32 %0, [%1];"
                           : "=r"(w)
                           : "r"(at(sv, warp * 16 + key, i) + (lane & 3) * 4)
                           : "memory");
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float v = srv_to_float<BF16>((w >> (16 * x)) & 0xffffu);
                if (!isfinite(v)) {
                  if (k0 + key <= lim[0]) o[i][x] += v;
                  if (k0 + key <= lim[1]) o[i][2 + x] += v;
                }
              }
            }
          }
          __syncwarp();
          for (int i = lane; i < 16 * (HD / 2); i += 32) {
            const uint32_t a = at(sv, warp * 16 + i / (HD / 2), (i % (HD / 2)) / 4) + (i % 4) * 4;
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(a) : "memory");
            if (srv_nonfinite<BF16>(w & 0xffffu)) w &= 0xffff0000u;
            if (srv_nonfinite<BF16>(w & 0xffff0000u)) w &= 0xffffu;
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(w) : "memory");
          }
          __syncwarp();
          fence_proxy_async_smem();
        }
        uint32_t pa[4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p0 = ex2_approx(fmaf(s[nb][2 * e], scale, -base[e]));
            const float p1 = ex2_approx(fmaf(s[nb][2 * e + 1], scale, -base[e]));
            l[e] += p0 + p1;
            pa[nb * 2 + e] = srv_pack<BF16>(p0, p1);
          }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          uint32_t b[4];
          ldsm_x4_trans(b, at(sv, warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), i * 2 + (lane >> 4)));
          mma_16816<BF16>(o[2 * i], pa, b[0], b[1]);
          mma_16816<BF16>(o[2 * i + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty + 8 * st);
    }
    if (!ok) {
      // A wait gave up, here or in a run before.  This warp waits for no tile any more (and frees no
      // stage: the producer and the other consumers see the flag, or give up in turn), but it
      // takes part in the barriers of every run that is left, with NaN for its share: no row whose
      // keys were not all read looks like a result.
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = CUDART_NAN_F;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[e] = 0.f;
        l[e] = CUDART_NAN_F;
      }
    }

    // Join the four warps: common maximum per row, then their outputs added quarter by
    // quarter (the order of the additions is fixed, so results repeat exactly).
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if ((lane & 3) == 0) ml[warp * STEP_ROWS + (lane >> 2) + 8 * e] = make_float2(m[e], l[e]);
    }
    auto sync4 = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    sync4();
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * STEP_ROWS + (lane >> 2) + 8 * e].x);
      f[e] = m[e] == -INFINITY ? 0.f : ex2_approx(m[e] - top);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        // n-block i belongs to quarter i / (HD / 32)
        if (i / (HD / 32) == ((warp + j) & 3)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2* d = reinterpret_cast<float2*>(obuf + ((lane >> 2) + 8 * e) * SM::OSTRIDE + i * 8 +
                                                  (lane & 3) * 2);
            float2 v = make_float2(o[i][2 * e] * f[e], o[i][2 * e + 1] * f[e]);
            if (j > 0) {
              const float2 w = *d;
              v.x += w.x;
              v.y += w.y;
            }
            *d = v;
          }
        }
      }
      sync4();
    }
    const int row = threadIdx.x >> 3, part = threadIdx.x & 7;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * STEP_ROWS + row].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 x = ml[w * STEP_ROWS + row];
      sum += x.y * (x.x == -INFINITY ? 0.f : ex2_approx(x.x - top));  // keeps a NaN sum
    }
    const float* src = obuf + row * SM::OSTRIDE + part * (HD / 8);
    if (r.t0 == 0 && r.t1 == r.tiles) {
      const int qrow = r.rb * STEP_ROWS + row;
      const int tok = qrow / p.group, g = qrow - tok * p.group;
      if (qrow < rows) {
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        uint32_t* dst = reinterpret_cast<uint32_t*>(p.out) +
                        ((long)(r.q.row0 + tok) * p.o_tok + (long)(r.h * p.group + g) * p.o_head +
                         part * (HD / 8)) / 2;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) dst[i] = srv_pack<BF16>(src[2 * i] * inv, src[2 * i + 1] * inv);
        if (p.lse != nullptr && part == 0)
          p.lse[(long)(r.q.row0 + tok) * p.heads + r.h * p.group + g] = srv_lse(top, sum);
      }
    } else {
      const long slot = 2 * (long)blockIdx.x + (first_run ? 0 : 1);
      float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * STEP_ROWS + row) * HD + part * (HD / 8));
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
        dst[i] = make_float4(src[4 * i], src[4 * i + 1], src[4 * i + 2], src[4 * i + 3]);
      if (part == 0) p.part_ml[slot * STEP_ROWS + row] = make_float2(top, sum);
    }
    sync4();
    first_run = false;
    u += r.t1 - r.t0;
  }
}

// Joins the runs of each row that several CTAs worked on: one warp per output row
// (token, query head), adding the runs in the order of their keys.
constexpr int STEP_JOIN_WARPS = 8;
template <int HD, bool BF16>
__global__ void __launch_bounds__(32 * STEP_JOIN_WARPS)
    step_join_kernel(const StepParams p, int step_grid) {
  extern __shared__ long pre_smem[];
  // Offsets and lengths were complete before the attention kernel began, so the prefix
  // sums are built while it runs.
  step_prefix(p, pre_smem, 32 * STEP_JOIN_WARPS);
  const int lane = lane_id();
  const long row = (long)blockIdx.x * STEP_JOIN_WARPS + warp_id();
  const long total = pre_smem[p.s.batch];
  bool work = row < (long)p.s.tokens * p.heads && total > 0;
  long c0 = 0, c1 = 0, u0 = 0;
  int tok = 0, head = 0, r_in = 0;
  const long per = step_per_cta(total, step_grid);
  if (work) {
    tok = (int)(row / p.heads);
    head = (int)(row - (long)tok * p.heads);
    int lo = 0, hi = p.s.batch - 1;  // the sequence of this token, if any
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.s.seq_off[mid] <= tok) lo = mid; else hi = mid - 1;
    }
    const SrvSeq q = srv_seq(p.s, lo);
    const StepBlocks k = step_blocks(q, p.group);
    work = tok >= q.row0 && tok < q.row0 + q.n && k.blocks > 0;
    if (work) {
      const int qrow = (tok - q.row0) * p.group + head % p.group;
      r_in = qrow % STEP_ROWS;
      u0 = pre_smem[lo] + ((long)(head / p.group) * k.blocks + qrow / STEP_ROWS) * k.tiles;
      c0 = u0 / per;
      c1 = (u0 + k.tiles - 1) / per;
      work = c1 > c0;
    }
  }
  griddep_wait();
  if (!work) return;
  auto slot_of = [&](long c) { return 2 * c + (c == c0 && u0 > c * per ? 1 : 0); };
  float top = -INFINITY;
  for (long c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.part_ml[slot_of(c) * STEP_ROWS + r_in].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float acc[HD / 32], sum = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (long c = c0; c <= c1; ++c) {
    const long at = slot_of(c) * STEP_ROWS + r_in;
    const float2 x = p.part_ml[at];
    const float f = x.x == -INFINITY ? 0.f : ex2_approx(x.x - top);
    sum += x.y * f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] += p.part_o[at * HD + lane * (HD / 32) + i] * f;
  }
  const float inv = top == -INFINITY ? 0.f : 1.f / sum;
  const long at = (long)tok * p.o_tok + (long)head * p.o_head + lane * (HD / 32);
  if constexpr (HD == 32) {
    if constexpr (BF16)
      reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(acc[0] * inv);
    else
      reinterpret_cast<__half*>(p.out)[at] = __float2half(acc[0] * inv);
  } else {
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out) + at / 2;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) dst[i] = srv_pack<BF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[(long)tok * p.heads + head] = srv_lse(top, sum);
}

}  // namespace tttj
