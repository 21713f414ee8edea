// Paged key/value cache: append of new tokens, eviction by gathered attention mass.
#include "common.cuh"
#include "launch.h"
#include "serve_dev.cuh"

namespace tttj {

namespace {

// ------------------------------------------------------------------ append
// The bytes of k, v and of the cache rows they become bound it.  A thread keeps one 16-byte
// piece of a token's k | v rows and copies it for U tokens, all loads before the first
// store, so a block has 256 x U pieces in flight; a warp's pieces are consecutive, so
// both sides move whole sectors.  The block's tokens are located (sequence, slot, page) once, by
// a binary search of the offsets per token.
constexpr int APPEND_THREADS = 256;
constexpr int APPEND_MOST_TOKENS = 256;  // of one block: U x groups, at least 8 threads a token

template <int U>
__global__ void __launch_bounds__(APPEND_THREADS, 5) append_kernel(const AppendParams p, int lanes, int per_block) {
  __shared__ int s_b[APPEND_MOST_TOKENS], s_slot[APPEND_MOST_TOKENS], s_page[APPEND_MOST_TOKENS];
  __shared__ int s_first[APPEND_MOST_TOKENS];
  griddep_wait();
  griddep_launch();
  const long t0 = (long)blockIdx.x * per_block;
  const int tokens = (int)min((long)per_block, p.s.tokens - t0);
  if ((int)threadIdx.x < tokens) {
    const int t = (int)t0 + threadIdx.x;
    int lo = 0, hi = p.s.batch - 1;  // the sequence of this token, if any
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.s.seq_off[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const SrvSeq q = srv_seq(p.s, lo);
    // The slot by the length as it was given: with the clamped one, the tokens of a sequence that
    // has outgrown its table would land on the live slots at the table's end.
    const int len = p.s.lens[lo];
    const long slot = (long)len - q.n + (t - q.row0);
    int page = p.s.num_pages;
    if (t >= q.row0 && t < q.row0 + q.n) {
      if (slot >= 0 && slot < (long)p.s.pages_per_seq << p.s.page_shift)
        page = srv_page(p.s, lo, (int)slot);
      else
        report_status(p.s.status, SRV_DEV_BAD_LENS);
    }
    s_b[threadIdx.x] = lo;
    s_slot[threadIdx.x] = (int)slot;
    s_page[threadIdx.x] = page;
    s_first[threadIdx.x] = (p.seen != nullptr ? p.seen[lo] : len) - q.n + (t - q.row0);
  }
  // Tokens look at their own sequence only: offsets that do not rise are found here.
  if (p.s.status != nullptr && blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.s.batch; b += APPEND_THREADS) srv_seq(p.s, b);
  __syncthreads();
  const int per_head = p.head_dim / 8, per_tensor = p.kv_heads * per_head;
  const int groups = APPEND_THREADS / lanes, group = threadIdx.x / lanes;
  const int page_mask = (1 << p.s.page_shift) - 1;
  for (int x = threadIdx.x - group * lanes; group < groups && x < 2 * per_tensor; x += lanes) {
    const bool is_v = x >= per_tensor;
    const int y = is_v ? x - per_tensor : x;
    const int h = y / per_head, c = y - h * per_head;
    const long tok = is_v ? p.v_tok : p.k_tok;
    const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.v : p.k) + h * (is_v ? p.v_head : p.k_head) + c * 8;
    const CacheView& to = is_v ? p.vc : p.kc;
    uint16_t* dst = static_cast<uint16_t*>(to.data) + h * to.head + c * 8;
    const long page_stride = to.page, slot_stride = to.slot;
    uint4 v[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = group + u * groups;
      there[u] = j < tokens && s_page[j] < p.s.num_pages;
      if (there[u]) v[u] = __ldg(reinterpret_cast<const uint4*>(src + (t0 + j) * tok));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = group + u * groups;
      if (there[u])
        *reinterpret_cast<uint4*>(dst + s_page[j] * page_stride + (s_slot[j] & page_mask) * slot_stride) = v[u];
    }
  }
  if (p.positions != nullptr || p.mass != nullptr) {
    const long cap = (long)p.s.pages_per_seq << p.s.page_shift;
    for (int i = threadIdx.x; i < tokens * p.kv_heads; i += APPEND_THREADS) {
      const int h = i / tokens, j = i - h * tokens;  // neighbours write neighbouring slots
      if (s_page[j] >= p.s.num_pages) continue;
      const long at = ((long)s_b[j] * p.kv_heads + h) * cap + s_slot[j];
      if (p.positions != nullptr) p.positions[at] = s_first[j];
      if (p.mass != nullptr) p.mass[at] = 0.f;
    }
  }
}

// ------------------------------------------------------------------- evict
// One cluster of 1 .. 8 blocks per (sequence, head); each warp owns a contiguous range of slots
// and holds EVICT_HELD of them per thread in registers (a longer range's rest is read again
// where it is needed).  The keep-th largest value is found two bits at a time: everyone
// counts the values above three thresholds, the warps' counts meet in every block's shared
// memory, at most 17 rounds of one barrier each, about 2000 cycles.  (A radix selection with
// histograms in shared memory: 123 against 50 us in all, 16 heads of 20000 - 32768 slots.)
// Then ballots rank the equal values, the holes (slots < keep that go) and the movers (slots >= keep that stay); the
// i-th mover goes to the i-th hole, so as few rows move as can, and since sources lie behind
// the budget and destinations in front of it, no move reads what another writes.  All counts are
// integers: the result does not depend on the order in which threads run.  Bound: for short
// caches latency, for long ones the bytes of the moved rows.
constexpr int EVICT_MAX_CLUSTER = 8;
constexpr int EVICT_MAX_THREADS = 1024;
constexpr int EVICT_HELD = 8;
constexpr int EVICT_BATCH = 2;  // moves of a thread whose rows are in flight

// Unsigned image of a mass: larger mass, larger integer; -0 as +0, NaN lowest.  Never 0.
__device__ __forceinline__ uint32_t evict_key(float mass) {
  if (mass != mass) return 0x007fffffu;  // the image of -inf
  const uint32_t u = __float_as_uint(mass + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(EVICT_MAX_THREADS) evict_kernel(const EvictParams p, int cluster) {
  // Three counts of every warp of the cluster, double-buffered.
  __shared__ int4 s_cnt[2][EVICT_MAX_CLUSTER * EVICT_MAX_THREADS / 32];
  griddep_wait();
  griddep_launch();
  constexpr unsigned FULL = 0xffffffffu;
  const int rank = cluster > 1 ? (int)cluster_ctarank() : 0;
  const int bh = blockIdx.x / cluster, b = bh / p.kv_heads;
  const int threads = blockDim.x, warps = threads >> 5, warp = warp_id(), lane = lane_id();
  const unsigned below = (1u << lane) - 1;
  const long cap = p.cap;
  int len = p.s.lens[b];
  if (len < 0 || len > cap) {
    if (threadIdx.x == 0) report_status(p.s.status, SRV_DEV_BAD_LENS);
    len = (int)min((long)max(len, 0), cap);
  }
  const float* mass = p.mass + bh * cap;
  const int* pos = p.positions + bh * cap;
  float* mass_out = p.mass_out + bh * cap;
  int* pos_out = p.positions_out + bh * cap;
  const int keep = p.keep;
  if (rank == 0 && threadIdx.x == 0 && bh % p.kv_heads == 0) p.lens_out[b] = min(len, keep);
  const int me = rank * threads + threadIdx.x, all = cluster * threads;
  // Slots behind the live ones (or the budget) are cleared by everyone.
  for (long j = min(len, keep) + me; j < cap; j += all) {
    mass_out[j] = 0.f;
    pos_out[j] = -1;
  }
  if (len <= keep) {  // uniform over the cluster
    for (int j = me; j < len; j += all) {
      mass_out[j] = mass[j];
      pos_out[j] = pos[j];
    }
    return;
  }
  // This warp's slots.
  const int all_warps = cluster * warps, my_warp = rank * warps + warp;
  const int each = ((len + all_warps - 1) / all_warps + 31) & ~31;
  const int w0 = (int)min((long)my_warp * each, (long)len), w1 = min(w0 + each, len);
  uint32_t key[EVICT_HELD];
  int ps[EVICT_HELD];
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i) {
    const int j = w0 + 32 * i + lane;
    key[i] = j < w1 ? evict_key(mass[j]) : 0u;
    ps[i] = j < w1 ? pos[j] : INT32_MIN;
  }
  const int rest = w0 + 32 * EVICT_HELD;  // slots from here on are not held
  int turn = 0;
  // Every warp's three counts, to every warp of the cluster; returns the buffer they are in.
  auto share = [&](int x, int y, int z) -> const int4* {
    int4* buf = s_cnt[turn++ & 1];
    if (cluster > 1) {
      if (lane < cluster)
        *static_cast<int4*>(__cluster_map_shared_rank(buf + my_warp, (unsigned)lane)) = make_int4(x, y, z, 0);
      cluster_sync_all();
    } else {
      if (lane == 0) buf[my_warp] = make_int4(x, y, z, 0);
      __syncthreads();
    }
    return buf;
  };
  int newest = INT32_MIN;
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i) newest = max(newest, ps[i]);
  for (int j = rest + lane; j < w1; j += 32) newest = max(newest, pos[j]);
  newest = __reduce_max_sync(FULL, newest);
  if (cluster > 1) cluster_sync_all();  // every block has started: its shared memory may be written
  {
    const int4* c = share(newest, 0, 0);
    for (int w = lane; w < all_warps; w += 32) newest = max(newest, c[w].x);
    newest = __reduce_max_sync(FULL, newest);
  }
  const long edge = (long)newest - p.recent;  // positions behind it count as +inf
  auto key_of = [&](float mass_j, int pos_j) {
    return (long)pos_j > edge ? 0xff800000u /* image of +inf */ : evict_key(mass_j);
  };
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i)
    if (key[i] != 0u && (long)ps[i] > edge) key[i] = 0xff800000u;
  // The keep-th largest value.  First whether it is zero, as where more slots than go have
  // gathered nothing (64 x 8 heads of 1025 - 1152 slots, a tenth of them zero: 26 against 34 us,
  // since no threshold separates equal values).  Masses that were gathered are hardly ever zero; the
  // round costs them nothing, since it finds the upper two bits of a positive cut (without zeros
  // 4 us more than with them).  Then two bits a round; done early once a threshold has exactly `keep`
  // values at or above it.
  constexpr uint32_t ZERO = 0x80000000u;  // the image of 0
  static_assert(32 * EVICT_HELD < 1024, "counts of a warp take ten bits");
  uint32_t cut = 0;
#pragma unroll 1
  for (int shift = 32; shift >= 0; shift -= 2) {
    const bool first = shift == 32;
    const uint32_t c1 = first ? ZERO : cut | (1u << shift), c2 = first ? ZERO + 1 : cut | (2u << shift),
                   c3 = first ? 0xc0000000u : cut | (3u << shift);
    unsigned packed = 0;  // live values at or above each threshold, ten bits each
#pragma unroll
    for (int i = 0; i < EVICT_HELD; ++i) {
      packed += key[i] >= c1 ? 1u : 0u;
      packed += key[i] >= c2 ? 1u << 10 : 0u;
      packed += key[i] >= c3 ? 1u << 20 : 0u;
    }
    packed = __reduce_add_sync(FULL, packed);
    int n1 = packed & 1023, n2 = packed >> 10 & 1023, n3 = packed >> 20;
    if (rest < w1) {
      int m1 = 0, m2 = 0, m3 = 0;
      for (int j = rest + lane; j < w1; j += 32) {
        const uint32_t x = key_of(mass[j], pos[j]);
        m1 += x >= c1;
        m2 += x >= c2;
        m3 += x >= c3;
      }
      n1 += __reduce_add_sync(FULL, m1);
      n2 += __reduce_add_sync(FULL, m2);
      n3 += __reduce_add_sync(FULL, m3);
    }
    const int4* c = share(n1, n2, n3);
    n1 = n2 = n3 = 0;
    for (int w = lane; w < all_warps; w += 32) {
      const int4 v = c[w];
      n1 += v.x;
      n2 += v.y;
      n3 += v.z;
    }
    n1 = __reduce_add_sync(FULL, n1);
    n2 = __reduce_add_sync(FULL, n2);
    n3 = __reduce_add_sync(FULL, n3);
    if (first) {
      if (n1 >= keep && n2 < keep) {
        cut = ZERO;
        break;
      }
      if (n2 >= keep) {  // the first two bits are known
        cut = n3 >= keep ? c3 : ZERO;
        shift = 30;
      }
      continue;
    }
    const int exact = n3 == keep ? 3 : n2 == keep ? 2 : n1 == keep ? 1 : 0;
    if (exact != 0) {
      cut = (cut | ((uint32_t)exact << shift)) - 1;  // all above it stay, no equal one does
      break;
    }
    cut = n3 >= keep ? c3 : n2 >= keep ? c2 : n1 >= keep ? c1 : cut;
  }
  // Kept: key > cut, and the first `need` slots with key == cut.
  int above = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i) {
    above += key[i] > cut;
    equal += key[i] == cut;
  }
  for (int j = rest + lane; j < w1; j += 32) {
    const uint32_t x = key_of(mass[j], pos[j]);
    above += x > cut;
    equal += x == cut;
  }
  int equal0 = 0;  // equal values in the warps before
  {
    const int4* c = share(__reduce_add_sync(FULL, above), __reduce_add_sync(FULL, equal), 0);
    above = 0;
    for (int w = lane; w < all_warps; w += 32) {
      above += c[w].x;
      if (w < my_warp) equal0 += c[w].y;
    }
    above = __reduce_add_sync(FULL, above);
    equal0 = __reduce_add_sync(FULL, equal0);
  }
  const int need = keep - above;
  // Which of the slots j .. j + 31 are kept, a bit per lane; `rank_eq`: equal values before them.
  auto kept_of = [&](uint32_t x, int* rank_eq) {
    const unsigned eq = __ballot_sync(FULL, x == cut);
    const bool kept = x > cut || (x == cut && *rank_eq + __popc(eq & below) < need);
    *rank_eq += __popc(eq);
    return __ballot_sync(FULL, kept);
  };
  auto span = [&](int j) {  // lanes of slots j .. that are live, and of those the ones < keep
    const int n = w1 - j, f = keep - j;
    const unsigned live = n >= 32 ? FULL : n <= 0 ? 0u : (1u << n) - 1;
    return make_uint2(live, f >= 32 ? live : f <= 0 ? 0u : live & ((1u << f) - 1));
  };
  auto key_rest = [&](int j) { return j + lane < w1 ? key_of(mass[j + lane], pos[j + lane]) : 0u; };
  int holes = 0, movers = 0, rank_eq = equal0;
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i) {
    const unsigned k = kept_of(key[i], &rank_eq);
    const uint2 sp = span(w0 + 32 * i);
    holes += __popc(~k & sp.y);
    movers += __popc(k & sp.x & ~sp.y);
  }
  for (int j = rest; j < w1; j += 32) {
    const unsigned k = kept_of(key_rest(j), &rank_eq);
    const uint2 sp = span(j);
    holes += __popc(~k & sp.y);
    movers += __popc(k & sp.x & ~sp.y);
  }
  int hole0 = 0, mover0 = 0, n_moves = 0;
  {
    const int4* c = share(holes, movers, 0);
    for (int w = lane; w < all_warps; w += 32) {
      n_moves += c[w].y;
      if (w < my_warp) {
        hole0 += c[w].x;
        mover0 += c[w].y;
      }
    }
    n_moves = __reduce_add_sync(FULL, n_moves);
    hole0 = __reduce_add_sync(FULL, hole0);
    mover0 = __reduce_add_sync(FULL, mover0);
  }
  int2* moves = p.moves + (long)bh * p.most_moves;
  // The list, and the kept slots that stay in place.
  auto list = [&](int j, uint32_t x) {
    const unsigned k = kept_of(x, &rank_eq);
    const uint2 sp = span(j);
    const unsigned hole = ~k & sp.y, mover = k & sp.x & ~sp.y, bit = 1u << lane;
    if (hole & bit) moves[hole0 + __popc(hole & below)].y = j + lane;
    if (mover & bit) moves[mover0 + __popc(mover & below)].x = j + lane;
    if (k & sp.y & bit) {
      mass_out[j + lane] = mass[j + lane];
      pos_out[j + lane] = pos[j + lane];
    }
    hole0 += __popc(hole);
    mover0 += __popc(mover);
  };
  rank_eq = equal0;
#pragma unroll
  for (int i = 0; i < EVICT_HELD; ++i) list(w0 + 32 * i, key[i]);
  for (int j = rest; j < w1; j += 32) list(j, key_rest(j));
  if (cluster > 1) cluster_sync_all(); else __syncthreads();  // the list is complete
  for (int i = me; i < n_moves; i += all) {
    const int2 mv = __ldcg(moves + i);
    mass_out[mv.y] = mass[mv.x];
    pos_out[mv.y] = pos[mv.x];
  }
  // The rows: one 16-byte piece of K and of V per thread and move, EVICT_BATCH moves' loads
  // before their stores.
  const int pieces = p.head_dim / 8;  // 4 .. 32
  const int c = threadIdx.x % pieces, h = bh - b * p.kv_heads;
  const int step = all / pieces, mask = (1 << p.s.page_shift) - 1;
  uint16_t* kbase = static_cast<uint16_t*>(p.kc.data) + h * p.kc.head + c * 8;
  uint16_t* vbase = static_cast<uint16_t*>(p.vc.data) + h * p.vc.head + c * 8;
  for (int i0 = me / pieces; i0 < n_moves; i0 += EVICT_BATCH * step) {
    int2 mv[EVICT_BATCH];
    int from[EVICT_BATCH], to[EVICT_BATCH];
    uint4 kv[EVICT_BATCH], vv[EVICT_BATCH];
#pragma unroll
    for (int u = 0; u < EVICT_BATCH; ++u)
      mv[u] = i0 + u * step < n_moves ? __ldcg(moves + i0 + u * step) : make_int2(-1, -1);
#pragma unroll
    for (int u = 0; u < EVICT_BATCH; ++u) {
      from[u] = to[u] = p.s.num_pages;
      if (mv[u].x >= 0) {
        from[u] = srv_page(p.s, b, mv[u].x);
        to[u] = srv_page(p.s, b, mv[u].y);
      }
    }
#pragma unroll
    for (int u = 0; u < EVICT_BATCH; ++u) {
      if (from[u] < p.s.num_pages && to[u] < p.s.num_pages) {
        kv[u] = *reinterpret_cast<const uint4*>(kbase + from[u] * p.kc.page + (mv[u].x & mask) * p.kc.slot);
        vv[u] = *reinterpret_cast<const uint4*>(vbase + from[u] * p.vc.page + (mv[u].x & mask) * p.vc.slot);
      }
    }
#pragma unroll
    for (int u = 0; u < EVICT_BATCH; ++u) {
      if (from[u] < p.s.num_pages && to[u] < p.s.num_pages) {
        *reinterpret_cast<uint4*>(kbase + to[u] * p.kc.page + (mv[u].y & mask) * p.kc.slot) = kv[u];
        *reinterpret_cast<uint4*>(vbase + to[u] * p.vc.page + (mv[u].y & mask) * p.vc.slot) = vv[u];
      }
    }
  }
}

// ---------------------------------------------------------------- failure detection
__global__ void serve_selftest_kernel(int* status, int* timeout_host, unsigned long long limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  mbar_init(smem_u32(&bar), 1);
  fence_barrier_init();
  if (!srv_wait(smem_u32(&bar), 0, nullptr, limit_ns)) srv_report_timeout(status, timeout_host);
}

}  // namespace

cudaError_t serve_selftest_launch(int* status, int* timeout_host, unsigned long long limit_ns, cudaStream_t stream) {
  serve_selftest_kernel<<<1, 1, 0, stream>>>(status, timeout_host, limit_ns);
  return cudaGetLastError();
}

cudaError_t append_launch(const AppendParams& p, int sms, cudaStream_t stream) {
  const long pieces = 2l * p.kv_heads * (p.head_dim / 8);
  const int lanes = (int)(pieces < APPEND_THREADS ? pieces : APPEND_THREADS);
  const int groups = APPEND_THREADS / lanes;
  // Four tokens per thread where that still gives every multiprocessor four blocks, else
  // one (a decode step: latency counts, not bytes in flight).
  const bool many = p.s.tokens / (4 * groups) >= 4 * sms;
  const int per_block = groups * (many ? 4 : 1);
  const unsigned blocks = (unsigned)((p.s.tokens + per_block - 1) / per_block);
  return launch_pdl(many ? append_kernel<4> : append_kernel<1>, dim3(blocks), dim3(APPEND_THREADS), 0, stream, p,
                    lanes, per_block);
}

cudaError_t evict_launch(const EvictParams& p, int sms, cudaStream_t stream) {
  // Blocks per head: while a block would have more than 1024 slots and two blocks per
  // multiprocessor are not reached.  Threads: one per EVICT_HELD slots, 128 at least.
  const long bh = (long)p.s.batch * p.kv_heads;
  int cluster = 1;
  while (cluster < EVICT_MAX_CLUSTER && p.cap / cluster > 1024 && bh * 2 * cluster <= 2 * sms) cluster *= 2;
  int threads = 128;
  while (threads < EVICT_MAX_THREADS && (long)threads * EVICT_HELD * cluster < p.cap) threads *= 2;
  return launch_pdl_cluster(evict_kernel, dim3((unsigned)(bh * cluster)), dim3(threads), 0, stream, cluster, p,
                            cluster);
}

}  // namespace tttj
