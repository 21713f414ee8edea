// Parameter blocks, device helpers and launchers of the serving operators (prompt
// attention, paged-cache append / attention / gathered mass / eviction).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "params.h"

namespace tttj {

constexpr int SRV_MAX_BATCH = 1024;  // sequences of a call (prefix sums in shared memory)
constexpr int SRV_MAX_GROUP = 64;    // query heads per key / value head
// How long a device wait may take.  A constant: as a field beside timeout_host it made the
// parameters longer, and a short prompt's three launches 0.7 us slower.
constexpr unsigned long long SRV_WAIT_LIMIT_NS = TTTJ_WAIT_LIMIT_NS;
constexpr int SRV_DEV_BAD_PAGE = 0x401;   // a live page-table entry outside the cache
constexpr int SRV_DEV_BAD_LENS = 0x402;   // lengths or offsets outside the call's tensors
constexpr int SRV_DEV_TIMEOUT = 0x403;    // a bounded device wait gave up

// Where the tokens of a call live: packed new tokens, and keys / values either packed
// the same way (table == nullptr: prompts) or in the pages of a cache.
struct SrvSeqs {
  const int* seq_off;  // [batch + 1] first packed row of each sequence
  const int* lens;     // [batch] cached tokens, new ones included (nullptr: prompts)
  const int* table;    // [batch][table_stride] page numbers (nullptr: prompts)
  long table_stride;
  int pages_per_seq;
  int page_shift;      // log2 of the page size
  int num_pages;
  int batch;
  int tokens;          // rows allocated in q / out
  int causal;
  int* status;         // device status word (nullable)
};

struct SrvSeq {
  int row0, n, len;  // first packed row, new tokens, keys
};

// Offsets and lengths come from device memory and are never trusted: whatever they
// hold, rows stay inside [0, tokens) and slots inside the table.
__device__ __forceinline__ SrvSeq srv_seq(const SrvSeqs& s, int b) {
  SrvSeq r;
  const int o0 = s.seq_off[b], o1 = s.seq_off[b + 1];
  r.row0 = min(max(o0, 0), s.tokens);
  const int end = min(max(o1, r.row0), s.tokens);
  r.n = end - r.row0;
  bool bad = r.row0 != o0 || end != o1;
  if (s.lens != nullptr) {
    const int len = s.lens[b];
    const long cap = (long)s.pages_per_seq << s.page_shift;
    r.len = (int)min((long)max(len, 0), cap);
    bad |= r.len != len;
  } else {
    r.len = r.n;
  }
  if (bad && s.status != nullptr) atomicCAS(s.status, 0, SRV_DEV_BAD_LENS);
  return r;
}

// Page holding `slot` of sequence b; num_pages (a page that TMA fills with zeros and
// that plain accesses skip) for entries outside the cache.
__device__ __forceinline__ int srv_page(const SrvSeqs& s, int b, int slot) {
  const int page = s.table[(long)b * s.table_stride + (slot >> s.page_shift)];
  if (page >= 0 && page < s.num_pages) return page;
  if (s.status != nullptr) atomicCAS(s.status, 0, SRV_DEV_BAD_PAGE);
  return s.num_pages;
}

struct CacheView {
  void* data;
  long page, slot, head;  // element strides
};

// ---- attention of few query rows per sequence (serve_step.cuh) ----
struct StepParams {
  SrvSeqs s;
  const void* q;
  long q_tok, q_head;  // element strides
  void* out;
  long o_tok, o_head;
  float* lse;          // [tokens][heads] or nullptr
  int heads, kv_heads, group;
  float scale_log2;
  float* part_o;       // [2 * grid][STEP_ROWS][head_dim] partial outputs
  float2* part_ml;     // [2 * grid][STEP_ROWS] their (max, sum)
  int* timeout_host;   // the device's pinned word (serve_capi.cu)
};
constexpr int STEP_ROWS = 16;   // query rows of one mma tile
constexpr int STEP_KEYS = 64;   // keys per pipeline stage
constexpr int step_ctas_per_sm(int hd) { return hd == 256 ? 1 : 2; }
cudaError_t step_launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const StepParams& p,
                        int head_dim, int bf16, int grid, cudaStream_t stream);

// ---- attention of many query rows per sequence (serve_tile.cuh) ----
// Query rows of a key/value head: row = token x group + head of the group; a tile takes
// the rows of floor(128 / group) tokens, an item NT tiles (two; one at head_dim 256).
struct TileEntry {    // one item of every key/value head
  int b, q;           // sequence, item of the sequence
  int j0, j1;         // key tiles [j0, j1)
  int part;           // first of kv_heads partial-result slots, or -1: whole items
  int row0, n, len;   // of the sequence (SrvSeq)
};
static_assert(sizeof(TileEntry) == 32, "entries are read as two 16-byte words");
struct TileJoin {     // an entry whose keys were split
  int b, q, pieces, part;  // piece i of head h is slot part + i * kv_heads + h
  int row0, n, pad[2];     // of the sequence
};
struct TilePlan {     // in the workspace, rebuilt by every call
  int* counters;      // [4]: items taken, entries, joins, notes of rows that are not finite
  TileEntry* entries; // [most_entries]
  TileJoin* joins;    // [most_entries]
  int4* redo;         // [most_redo]: b, q, h, warp of the item (32 rows)
  int most_redo;
  int most_entries;
  int most_parts;     // partial-result slots
};
struct TileParams {
  SrvSeqs s;
  const void* q;       // for rows computed again
  long q_tok, q_head;
  CacheView k, v;      // the same (prompts: page 0)
  void* out;
  long o_tok, o_head;
  int o_wide;          // rows of out are 32-byte aligned
  float* lse;
  int heads, kv_heads, group, tile_tokens;
  float scale_log2;
  TilePlan plan;
  float* part_o;       // [most_parts][NT * 128][head_dim]
  float2* part_ml;     // [most_parts][NT * 128]
  int* timeout_host;   // the device's pinned word (serve_capi.cu)
};
constexpr int tile_nt(int hd) { return hd == 256 ? 1 : 2; }
cudaError_t tile_launch(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                        const TileParams& p, int head_dim, int bf16, int grid, cudaStream_t stream);

// ---- attention mass of cached keys (serve_mass.cuh) ----
struct MassParams {
  SrvSeqs s;
  const float* lse;   // [tokens][heads], natural
  const float* mass;  // [batch][kv_heads][cap]
  float* out;         // the same shape (may be mass)
  long cap;
  int heads, kv_heads, group, tile_tokens;
  float scale_log2;
  int* timeout_host;   // the device's pinned word (serve_capi.cu)
};
constexpr int MASS_TILE_ROWS = 80;  // query rows of a tile (MASS_ROWS)
cudaError_t mass_launch(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const MassParams& p, int head_dim,
                        int bf16, int grid, cudaStream_t stream);

// ---- cache append / evict (serve_cache.cu) ----
struct AppendParams {
  SrvSeqs s;
  const void* k;
  const void* v;
  long k_tok, k_head, v_tok, v_head;
  CacheView kc, vc;
  int kv_heads, head_dim;
  int* positions;    // [batch][kv_heads][cap] or nullptr
  float* mass;       // the same shape, or nullptr
  const int* seen;   // [batch] tokens seen by each sequence, or nullptr (= lens)
};
cudaError_t append_launch(const AppendParams& p, int sms, cudaStream_t stream);

struct EvictParams {
  SrvSeqs s;  // seq_off is unused
  CacheView kc, vc;
  int kv_heads, head_dim;
  const float* mass;
  const int* positions;
  float* mass_out;
  int* positions_out;
  int* lens_out;
  int keep, recent;
  long cap;       // slots per sequence (row length of mass / positions)
  int2* moves;    // [batch * kv_heads][most_moves] (from, to) slots
  int most_moves;
};
cudaError_t evict_launch(const EvictParams& p, int sms, cudaStream_t stream);

// One bounded wait on a barrier that nothing arrives on, reported like any other.
cudaError_t serve_selftest_launch(int* status, int* timeout_host, unsigned long long limit_ns, cudaStream_t stream);

}  // namespace tttj
