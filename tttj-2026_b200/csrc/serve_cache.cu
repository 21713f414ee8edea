// Paged key/value cache: append of new tokens, eviction by gathered attention mass.
#include "common.cuh"
#include "launch.h"
#include "serve.h"

namespace tttj {

namespace {

// ------------------------------------------------------------------ append
// One 16-byte piece of one head's key or value row per thread and step: the bytes of k,
// v and of the cache rows they become bound it.  A warp's pieces are consecutive, so both
// sides move whole sectors.  Blocks take APPEND_TOKENS tokens; a token's sequence is found by a
// binary search of the offsets, uniform in the block's small groups of threads.
constexpr int APPEND_THREADS = 256;
constexpr int APPEND_TOKENS = 4;

__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendParams p) {
  __shared__ int s_b[APPEND_TOKENS], s_slot[APPEND_TOKENS], s_page[APPEND_TOKENS], s_first[APPEND_TOKENS];
  griddep_wait();
  griddep_launch();
  const long t0 = (long)blockIdx.x * APPEND_TOKENS;
  const int tokens = (int)min((long)APPEND_TOKENS, p.s.tokens - t0);
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
  const int per_head = p.head_dim / 8;
  const int per_tok = 2 * p.kv_heads * per_head;
  for (int i = threadIdx.x; i < tokens * per_tok; i += APPEND_THREADS) {
    const int j = i / per_tok;
    int x = i - j * per_tok;
    const int page = s_page[j];
    if (page >= p.s.num_pages) continue;
    const bool is_v = x >= p.kv_heads * per_head;
    if (is_v) x -= p.kv_heads * per_head;
    const int h = x / per_head, c = x - h * per_head;
    const int in_page = s_slot[j] & ((1 << p.s.page_shift) - 1);
    const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.v : p.k) +
                          (t0 + j) * (is_v ? p.v_tok : p.k_tok) + h * (is_v ? p.v_head : p.k_head) + c * 8;
    const CacheView& to = is_v ? p.vc : p.kc;
    uint16_t* dst = static_cast<uint16_t*>(to.data) + page * to.page + in_page * to.slot + h * to.head + c * 8;
    *reinterpret_cast<uint4*>(dst) = __ldg(reinterpret_cast<const uint4*>(src));
  }
  if (p.positions != nullptr || p.mass != nullptr) {
    const long cap = (long)p.s.pages_per_seq << p.s.page_shift;
    for (int i = threadIdx.x; i < tokens * p.kv_heads; i += APPEND_THREADS) {
      const int j = i / p.kv_heads, h = i - j * p.kv_heads;
      if (s_page[j] >= p.s.num_pages) continue;
      const long at = ((long)s_b[j] * p.kv_heads + h) * cap + s_slot[j];
      if (p.positions != nullptr) p.positions[at] = s_first[j];
      if (p.mass != nullptr) p.mass[at] = 0.f;
    }
  }
}

// ------------------------------------------------------------------- evict
// Selection, one block per (sequence, head): a radix selection finds the keep-th largest
// value (four 8-bit digits of an order-preserving integer image of the mass, counted in
// shared memory), then one ordered pass ranks the equal values, the holes (slots < keep
// that go) and the movers (slots >= keep that stay), each thread owning a contiguous range
// of slots.  The i-th mover goes to the i-th hole, so as few rows move as can: those kept
// from behind the budget.  The integer counts make the result independent of the order in
// which threads run.
constexpr int EVICT_THREADS = 1024;
constexpr int EVICT_SMEM_SLOTS = 48 * 1024;  // values held in shared memory up to this length

// Unsigned image of a mass: larger mass, larger integer; -0 as +0, NaN lowest.
__device__ __forceinline__ uint32_t evict_key(float mass) {
  if (mass != mass) return 0x007fffffu;  // the image of -inf
  const uint32_t u = __float_as_uint(mass + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of one int per thread over the block; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = lane_id(), warp = warp_id();
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < EVICT_THREADS / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[EVICT_THREADS / 32 - 1];
  return (warp > 0 ? warp_sums[warp - 1] : 0) + x - v;
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(const EvictParams p) {
  extern __shared__ uint32_t s_key[];  // [min(len, EVICT_SMEM_SLOTS)]
  __shared__ int s_hist[256];
  __shared__ int s_warp[32];
  __shared__ int s_newest;
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  griddep_wait();
  griddep_launch();
  const int bh = blockIdx.x, b = bh / p.kv_heads;
  const long cap = p.cap;
  int len = p.s.lens[b];
  if (len < 0 || len > cap) {
    if (threadIdx.x == 0 && p.s.status != nullptr) atomicCAS(p.s.status, 0, SRV_DEV_BAD_LENS);
    len = (int)min((long)max(len, 0), cap);
  }
  const float* mass = p.mass + bh * cap;
  const int* pos = p.positions + bh * cap;
  float* mass_out = p.mass_out + bh * cap;
  int* pos_out = p.positions_out + bh * cap;
  const int keep = p.keep;
  if (threadIdx.x == 0 && bh % p.kv_heads == 0) p.lens_out[b] = min(len, keep);
  if (len <= keep) {
    if (threadIdx.x == 0) p.n_moves[bh] = 0;
    for (long j = threadIdx.x; j < cap; j += EVICT_THREADS) {
      mass_out[j] = j < len ? mass[j] : 0.f;
      pos_out[j] = j < len ? pos[j] : -1;
    }
    return;
  }
  // The newest position; slots within `recent` of it count as +inf.
  if (threadIdx.x == 0) s_newest = INT32_MIN;
  __syncthreads();
  int newest = INT32_MIN;
  for (int j = threadIdx.x; j < len; j += EVICT_THREADS) newest = max(newest, pos[j]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane_id() == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  const long edge = (long)s_newest - p.recent;
  const bool held = len <= EVICT_SMEM_SLOTS;
  auto key_at = [&](int j) -> uint32_t {
    return (long)pos[j] > edge ? 0xff800000u /* image of +inf */ : evict_key(mass[j]);
  };
  if (held)
    for (int j = threadIdx.x; j < len; j += EVICT_THREADS) s_key[j] = key_at(j);
  uint32_t prefix = 0;
  int need = keep;  // how many of the values matching the prefix so far are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) s_hist[threadIdx.x] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < len; j += EVICT_THREADS) {
      const uint32_t key = held ? s_key[j] : key_at(j);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&s_hist[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // Lane l holds digits 255 - 8 l .. 248 - 8 l: counts from the largest digit down.
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = s_hist[255 - 8 * (int)threadIdx.x - i];
      int inc = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, d);
        if ((int)threadIdx.x >= d) inc += o;
      }
      int above = inc - sum;
      if (above < need && need <= inc) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < need && need <= above + c[i]) {
            s_prefix = prefix | ((uint32_t)(255 - 8 * (int)threadIdx.x - i) << shift);
            s_need = need - above;
          }
          above += c[i];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // Kept: key > prefix, and the first `need` slots with key == prefix.
  const int each = (len + EVICT_THREADS - 1) / EVICT_THREADS;
  const int j0 = min((int)threadIdx.x * each, len), j1 = min(j0 + each, len);
  int equal = 0, total;
  for (int j = j0; j < j1; ++j) equal += (held ? s_key[j] : key_at(j)) == prefix;
  const int equal0 = block_scan(equal, s_warp, &total);
  // Both lists start at the same length, so one scan counts holes (slots < keep) for the
  // threads in front of the budget and movers for those behind it.
  int holes = 0, movers = 0, rank = equal0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = held ? s_key[j] : key_at(j);
    const bool kept = key > prefix || (key == prefix && rank++ < need);
    holes += j < keep && !kept;
    movers += j >= keep && kept;
  }
  int n_holes, n_movers;
  int hole0 = block_scan(holes, s_warp, &n_holes);
  int mover0 = block_scan(movers, s_warp, &n_movers);
  int2* moves = p.moves + (long)bh * p.most_moves;
  rank = equal0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = held ? s_key[j] : key_at(j);
    const bool kept = key > prefix || (key == prefix && rank++ < need);
    if (j < keep && !kept) moves[hole0++].y = j;
    if (j >= keep && kept) moves[mover0++].x = j;
  }
  if (threadIdx.x == 0) p.n_moves[bh] = n_movers;
  // Kept slots in place; the holes are filled below from the list.
  for (long j = threadIdx.x; j < cap; j += EVICT_THREADS) {
    mass_out[j] = j < keep ? mass[j] : 0.f;
    pos_out[j] = j < keep ? pos[j] : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_movers; i += EVICT_THREADS) {
    const int2 mv = moves[i];
    mass_out[mv.y] = mass[mv.x];
    pos_out[mv.y] = pos[mv.x];
  }
}

// Moves the listed rows of K and V: sources are slots >= keep, destinations slots < keep,
// so no move reads what another writes.  One warp per move and cache.
constexpr int EVICT_MOVE_WARPS = 8;
__global__ void __launch_bounds__(32 * EVICT_MOVE_WARPS) evict_move_kernel(const EvictParams p) {
  griddep_wait();
  griddep_launch();
  const int bh = blockIdx.x, b = bh / p.kv_heads, h = bh - b * p.kv_heads;
  const int n = p.n_moves[bh];
  const int lane = lane_id();
  const int pieces = p.head_dim / 8;  // 16-byte pieces of a row (4 .. 32)
  const int per_warp = 32 / pieces;   // rows of one warp step
  const int sub = lane / pieces, c = lane - sub * pieces;
  const int mask = (1 << p.s.page_shift) - 1;
  const long rows = 2l * n;           // move i of K is row 2 i, of V row 2 i + 1
  const long step = (long)gridDim.y * EVICT_MOVE_WARPS * per_warp;
  for (long i = ((long)blockIdx.y * EVICT_MOVE_WARPS + warp_id()) * per_warp + sub; i < rows; i += step) {
    const int2 mv = p.moves[(long)bh * p.most_moves + (i >> 1)];
    const CacheView& cv = (i & 1) ? p.vc : p.kc;
    const int from = srv_page(p.s, b, mv.x), to = srv_page(p.s, b, mv.y);
    if (from >= p.s.num_pages || to >= p.s.num_pages) continue;
    uint16_t* base = static_cast<uint16_t*>(cv.data) + h * cv.head + c * 8;
    const uint4 v = *reinterpret_cast<const uint4*>(base + from * cv.page + (mv.x & mask) * cv.slot);
    *reinterpret_cast<uint4*>(base + to * cv.page + (mv.y & mask) * cv.slot) = v;
  }
}

}  // namespace

cudaError_t append_launch(const AppendParams& p, cudaStream_t stream) {
  const int blocks = (p.s.tokens + APPEND_TOKENS - 1) / APPEND_TOKENS;
  return launch_pdl(append_kernel, dim3(blocks), dim3(APPEND_THREADS), 0, stream, p);
}

cudaError_t evict_launch(const EvictParams& p, cudaStream_t stream) {
  const int smem = (int)(p.cap < EVICT_SMEM_SLOTS ? p.cap : EVICT_SMEM_SLOTS) * 4;
  cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int bh = p.s.batch * p.kv_heads;
  e = launch_pdl(evict_select_kernel, dim3(bh), dim3(EVICT_THREADS), smem, stream, p);
  if (e != cudaSuccess || p.most_moves == 0) return e;
  // Enough blocks for the most moves a call can have, in at most about eight waves.
  const long steps = (2l * p.most_moves * (p.head_dim / 8) + 32 * EVICT_MOVE_WARPS - 1) / (32 * EVICT_MOVE_WARPS);
  long x = 148l * 8 * 8 / bh;
  x = x > steps ? steps : x;
  x = x < 1 ? 1 : x;
  return launch_pdl(evict_move_kernel, dim3((unsigned)bh, (unsigned)x), dim3(32 * EVICT_MOVE_WARPS), 0,
                    stream, p);
}

}  // namespace tttj
