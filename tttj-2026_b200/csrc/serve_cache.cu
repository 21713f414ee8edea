// Paged key/value cache: append of new tokens, eviction by gathered attention mass.
#include "common.cuh"
#include "launch.h"
#include "serve.h"

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
    const int slot = q.len - q.n + (t - q.row0);
    int page = p.s.num_pages;
    if (t >= q.row0 && t < q.row0 + q.n && slot >= 0) page = srv_page(p.s, lo, slot);
    s_b[threadIdx.x] = lo;
    s_slot[threadIdx.x] = slot;
    s_page[threadIdx.x] = page;
    s_first[threadIdx.x] = (p.seen != nullptr ? p.seen[lo] : q.len) - q.n + (t - q.row0);
  }
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
// One cluster of 1 .. 8 blocks per (sequence, head); each block owns a contiguous range of
// slots, whose masses and positions it holds in shared memory.  A radix selection over
// an order-preserving integer image of the mass (digits of 11, 11 and 10 bits, counted in shared memory
// and added up across the cluster) finds the keep-th largest value.  One ordered pass
// then ranks the equal values, the holes (slots < keep that go) and the movers (slots >= keep
// that stay); the i-th mover goes to the i-th hole, so as few rows move as can, and since
// sources lie behind the budget and destinations in front of it, no move reads what
// another writes.  All counts are integers: the result does not depend on the order in
// which threads run.  Bound: for short caches latency (about twenty barriers), for long ones the bytes
// of masses, positions and moved rows.
constexpr int EVICT_MAX_CLUSTER = 8;
constexpr int EVICT_MAX_THREADS = 512;
constexpr int EVICT_BINS = 2048;
constexpr int EVICT_BATCH = 4;
constexpr int EVICT_HELD_SLOTS = 24 * 1024;  // slots of one block held in shared memory (8 bytes each)

// Unsigned image of a mass: larger mass, larger integer; -0 as +0, NaN lowest.
__device__ __forceinline__ uint32_t evict_key(float mass) {
  if (mass != mass) return 0x007fffffu;  // the image of -inf
  const uint32_t u = __float_as_uint(mass + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

struct EvictShared {
  int hist[EVICT_BINS];   // counts of one digit (read by the whole cluster)
  int total[4];           // newest position; equal, holes, movers of this block
  int warp[2][32];
  int digit, need;
};

__global__ void __launch_bounds__(EVICT_MAX_THREADS) evict_kernel(const EvictParams p, int cluster) {
  extern __shared__ __align__(16) uint8_t s_dyn[];
  __shared__ EvictShared sh;
  griddep_wait();
  griddep_launch();
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
  auto sync_all = [&] {
    if (cluster > 1) cluster_sync_all(); else __syncthreads();
  };
  auto peer = [&](int* x, int r) -> int {
    return cluster > 1 ? *static_cast<int*>(__cluster_map_shared_rank(x, (unsigned)r)) : *x;
  };
  // This block's slots, a multiple of 32 per warp.
  const int each = ((len + cluster - 1) / cluster + 31) & ~31;
  const int lo = min(rank * each, len), hi = min(lo + each, len);
  const bool held = each <= EVICT_HELD_SLOTS;
  float* s_mass = reinterpret_cast<float*>(s_dyn);
  int* s_pos = reinterpret_cast<int*>(s_dyn) + (held ? each : 0);
  int newest = INT32_MIN;
#pragma unroll 4
  for (int j = lo + (int)threadIdx.x; j < hi; j += threads) {
    const int x = pos[j];
    const float m = held ? mass[j] : 0.f;
    newest = max(newest, x);
    if (held) {
      s_mass[j - lo] = m;
      s_pos[j - lo] = x;
    }
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) sh.warp[0][warp] = newest;
  for (int i = threadIdx.x; i < EVICT_BINS; i += threads) sh.hist[i] = 0;
  __syncthreads();
  if (warp == 0) {
    newest = __reduce_max_sync(0xffffffffu, lane < warps ? sh.warp[0][lane] : INT32_MIN);
    if (lane == 0) sh.total[0] = newest;
  }
  sync_all();
  newest = INT32_MIN;
  for (int r = 0; r < cluster; ++r) newest = max(newest, peer(&sh.total[0], r));
  const long edge = (long)newest - p.recent;  // positions behind it count as +inf
  auto key_at = [&](int j) -> uint32_t {
    const int x = held ? s_pos[j - lo] : pos[j];
    return (long)x > edge ? 0xff800000u /* image of +inf */ : evict_key(held ? s_mass[j - lo] : mass[j]);
  };
  uint32_t prefix = 0;
  int need = keep;  // how many of the values that match the prefix so far are kept
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int bits = pass == 2 ? 10 : 11;
    for (int j = lo + (int)threadIdx.x; j < hi; j += threads) {
      const uint32_t key = key_at(j);
      if (pass == 0 || (key >> (shift + bits)) == (prefix >> (shift + bits)))
        atomicAdd(&sh.hist[(key >> shift) & ((1u << bits) - 1)], 1);
    }
    sync_all();
    // Largest digits first: thread t takes bins top - per t .. ; counts over the cluster.
    const int per = (1 << bits) / threads;
    const int first = (1 << bits) - 1 - per * (int)threadIdx.x;
    int c[EVICT_BINS / 128], sum = 0;  // at least 128 threads
#pragma unroll
    for (int i = 0; i < EVICT_BINS / 128; ++i) c[i] = 0;
    for (int r = 0; r < cluster; ++r) {
#pragma unroll
      for (int i = 0; i < EVICT_BINS / 128; ++i)
        if (i < per) c[i] += peer(&sh.hist[first - i], r);
    }
#pragma unroll
    for (int i = 0; i < EVICT_BINS / 128; ++i) sum += c[i];
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) sh.warp[0][warp] = inc;
    __syncthreads();
    int above = inc - sum;
    for (int w = 0; w < warp; ++w) above += sh.warp[0][w];
    if (above < need && need <= above + sum) {
#pragma unroll
      for (int i = 0; i < EVICT_BINS / 128; ++i) {
        if (i < per && above < need && need <= above + c[i]) {
          sh.digit = first - i;
          sh.need = need - above;
        }
        above += c[i];
      }
    }
    sync_all();  // digit and need are there; every block has read this one's counts
    prefix |= (uint32_t)sh.digit << shift;
    need = sh.need;
    for (int i = threadIdx.x; i < EVICT_BINS; i += threads) sh.hist[i] = 0;
    __syncthreads();
  }
  // Kept: key > prefix, and the first `need` slots with key == prefix.  Each warp owns a
  // contiguous range; ranks by ballots.
  const int per_warp = ((hi - lo + warps - 1) / warps + 31) & ~31;
  const int w0 = min(lo + warp * per_warp, hi), w1 = min(w0 + per_warp, hi);
  // Exclusive sum of one count per warp over the block (and the blocks before it).
  auto offset = [&](int mine, int which) {
    if (lane == 0) sh.warp[which & 1][warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      int t = 0;
      for (int w = 0; w < warps; ++w) t += sh.warp[which & 1][w];
      sh.total[which] = t;
    }
    int at = 0;
    for (int w = 0; w < warp; ++w) at += sh.warp[which & 1][w];
    sync_all();
    for (int r = 0; r < rank; ++r) at += peer(&sh.total[which], r);
    return at;
  };
  int equal = 0;
  for (int j = w0; j < w1; j += 32)
    equal += __popc(__ballot_sync(0xffffffffu, j + lane < w1 && key_at(j + lane) == prefix));
  const int equal0 = offset(equal, 1);
  auto kept_at = [&](int j, int* rank_eq) {  // of slots j .. j + 31, a bit per lane
    const uint32_t key = j + lane < w1 ? key_at(j + lane) : 0u;
    const bool live = j + lane < w1;
    const unsigned eq = __ballot_sync(0xffffffffu, live && key == prefix);
    const bool kept = live && (key > prefix || (key == prefix && *rank_eq + __popc(eq & below) < need));
    *rank_eq += __popc(eq);
    return __ballot_sync(0xffffffffu, kept);
  };
  auto span = [&](int j) {  // lanes of slots j .. that are live, and of those the ones < keep
    const int n = w1 - j, f = keep - j;
    const unsigned live = n >= 32 ? 0xffffffffu : (1u << n) - 1;
    return make_uint2(live, f >= 32 ? live : f <= 0 ? 0u : live & ((1u << f) - 1));
  };
  int holes = 0, movers = 0, eq_rank = equal0;
  for (int j = w0; j < w1; j += 32) {
    const unsigned kept = kept_at(j, &eq_rank);
    const uint2 sp = span(j);
    holes += __popc(~kept & sp.y);
    movers += __popc(kept & sp.x & ~sp.y);
  }
  int hole0 = offset(holes, 2);
  int mover0 = offset(movers, 3);
  int n_moves = 0;
  for (int r = 0; r < cluster; ++r) n_moves += peer(&sh.total[3], r);
  int2* moves = p.moves + (long)bh * p.most_moves;
  eq_rank = equal0;
  for (int j = w0; j < w1; j += 32) {
    const unsigned kept = kept_at(j, &eq_rank);
    const uint2 sp = span(j);
    const unsigned hole = ~kept & sp.y, mover = kept & sp.x & ~sp.y, bit = 1u << lane;
    if (hole & bit) moves[hole0 + __popc(hole & below)].y = j + lane;
    if (mover & bit) moves[mover0 + __popc(mover & below)].x = j + lane;
    if (kept & sp.y & bit) {
      mass_out[j + lane] = held ? s_mass[j + lane - lo] : mass[j + lane];
      pos_out[j + lane] = held ? s_pos[j + lane - lo] : pos[j + lane];
    }
    hole0 += __popc(hole);
    mover0 += __popc(mover);
  }
  sync_all();  // the list is complete (and no block still reads another's shared memory)
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

}  // namespace

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
  // Blocks per head: as many as keep at least 2048 slots each, while there are
  // multiprocessors for them.  Threads: one per four slots or so.
  const long bh = (long)p.s.batch * p.kv_heads;
  int cluster = 1;
  while (cluster < EVICT_MAX_CLUSTER && p.cap / (2 * cluster) >= 2048 && bh * 2 * cluster <= 2 * sms) cluster *= 2;
  const long each = ((p.cap + cluster - 1) / cluster + 31) & ~31l;
  const int threads = each <= 1024 ? 128 : each <= 2048 ? 256 : EVICT_MAX_THREADS;
  const int smem = each <= EVICT_HELD_SLOTS ? (int)each * 8 : EVICT_HELD_SLOTS * 8;
  cudaError_t e = cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl_cluster(evict_kernel, dim3((unsigned)(bh * cluster)), dim3(threads), smem, stream, cluster, p,
                            cluster);
}

}  // namespace tttj
