// C entry points of the serving operators (include/tttj_b200.h): argument checks,
// tensor maps and launches.  Nothing here reads device memory or synchronises.
#include <math.h>

#include <atomic>

#include "capi_util.h"
#include "serve.h"

using namespace tttj;

namespace {

constexpr size_t kAlign = 256;
inline size_t up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
inline bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int check_seqs(const char* what, const tttj_seqs* s, bool cache, bool offsets) {
  if (!s) return capi_fail(TTTJ_ERR_INVALID, "%s: null argument", what);
  if (s->dtype != TTTJ_DTYPE_F16 && s->dtype != TTTJ_DTYPE_BF16)
    return capi_fail(TTTJ_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  if (s->head_dim != 32 && s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256)
    return capi_fail(TTTJ_ERR_INVALID, "%s: head_dim=%d unsupported (32, 64, 128, 256)", what, s->head_dim);
  if (s->kv_heads <= 0 || s->heads <= 0 || s->heads % s->kv_heads || s->heads / s->kv_heads > SRV_MAX_GROUP)
    return capi_fail(TTTJ_ERR_INVALID, "%s: heads=%d must be kv_heads=%d times a group of 1 .. %d", what,
                     s->heads, s->kv_heads, SRV_MAX_GROUP);
  if (s->batch <= 0 || s->batch > SRV_MAX_BATCH)
    return capi_fail(TTTJ_ERR_INVALID, "%s: batch=%d outside 1 .. %d", what, s->batch, SRV_MAX_BATCH);
  if (s->tokens < 0 || (long)s->tokens * s->heads >= (1l << 31))
    return capi_fail(TTTJ_ERR_INVALID, "%s: tokens=%d x heads=%d out of range", what, s->tokens, s->heads);
  if (offsets && !s->seq_offsets) return capi_fail(TTTJ_ERR_INVALID, "%s: null seq_offsets", what);
  if (cache) {
    if (!s->cache_lens || !s->page_table) return capi_fail(TTTJ_ERR_INVALID, "%s: null cache_lens or page_table", what);
    const int ps = s->page_size;
    if (ps < 16 || ps > 256 || (ps & (ps - 1)))
      return capi_fail(TTTJ_ERR_INVALID, "%s: page_size=%d unsupported (16, 32, 64, 128, 256)", what, ps);
    if (s->pages_per_seq <= 0 || s->num_pages <= 0 || (long)s->pages_per_seq * ps >= (1l << 30))
      return capi_fail(TTTJ_ERR_INVALID, "%s: pages_per_seq=%d, num_pages=%d out of range", what,
                       s->pages_per_seq, s->num_pages);
    if (s->table_stride < s->pages_per_seq)
      return capi_fail(TTTJ_ERR_INVALID, "%s: page_table rows overlap", what);
  }
  return TTTJ_OK;
}

int check_rows(const char* what, const char* name, const tttj_rows* r, const tttj_seqs* s, int heads) {
  if (!r || (!r->data && s->tokens > 0)) return capi_fail(TTTJ_ERR_INVALID, "%s: null %s", what, name);
  if (misaligned(r->data)) return capi_fail(TTTJ_ERR_INVALID, "%s: %s must be 16-byte aligned", what, name);
  if ((s->tokens > 1 && r->token_stride <= 0) || r->token_stride % 8 || (heads > 1 && r->head_stride <= 0) ||
      r->head_stride % 8)
    return capi_fail(TTTJ_ERR_INVALID, "%s: %s strides must be positive multiples of 8 elements", what, name);
  return TTTJ_OK;
}

int check_pages(const char* what, const char* name, const tttj_pages* c, const tttj_seqs* s) {
  if (!c || !c->data) return capi_fail(TTTJ_ERR_INVALID, "%s: null %s", what, name);
  if (misaligned(c->data)) return capi_fail(TTTJ_ERR_INVALID, "%s: %s must be 16-byte aligned", what, name);
  if ((s->num_pages > 1 && c->page_stride <= 0) || c->page_stride % 8 || c->slot_stride <= 0 || c->slot_stride % 8 ||
      (s->kv_heads > 1 && c->head_stride <= 0) || c->head_stride % 8)
    return capi_fail(TTTJ_ERR_INVALID, "%s: %s strides must be positive multiples of 8 elements", what, name);
  return TTTJ_OK;
}

int check_scale(const char* what, float scale) {
  if (!(scale > 0.f) || !isfinite(scale))
    return capi_fail(TTTJ_ERR_INVALID, "%s: scale must be positive and finite", what);
  return TTTJ_OK;
}

#define TRY(call)             \
  do {                        \
    const int rc_ = (call);   \
    if (rc_) return rc_;      \
  } while (0)

SrvSeqs seqs_of(const tttj_seqs* s, bool cache, int causal) {
  SrvSeqs r{};
  r.seq_off = s->seq_offsets;
  r.batch = s->batch;
  r.tokens = s->tokens;
  r.causal = causal;
  r.status = s->status;
  if (cache) {
    r.lens = s->cache_lens;
    r.table = s->page_table;
    r.table_stride = s->table_stride;
    r.pages_per_seq = s->pages_per_seq;
    while ((1 << r.page_shift) < s->page_size) ++r.page_shift;
    r.num_pages = s->num_pages;
  }
  return r;
}

CacheView view_of(const tttj_pages* c) { return {c->data, c->page_stride, c->slot_stride, c->head_stride}; }

// 4-D map {head_dim, slots, heads, pages} of keys or values, moved in boxes of one
// head's `box_rows` slots x min(head_dim, 64) columns, swizzled by the box's row width.
int kv_map(CUtensorMap* m, const char* what, const tttj_seqs* s, const void* data, long page_stride,
           long slot_stride, long head_stride, int slots, int pages, int box_rows) {
  auto fn = capi_encode_fn();
  if (!fn) return capi_fail(TTTJ_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int cols = s->head_dim < 64 ? s->head_dim : 64;
  cuuint64_t dims[4] = {(cuuint64_t)s->head_dim, (cuuint64_t)slots, (cuuint64_t)s->kv_heads, (cuuint64_t)pages};
  // The stride of a dimension of size one is never used; it still has to be valid.
  const long one = s->head_dim;
  cuuint64_t strides[3] = {(cuuint64_t)(slots > 1 ? slot_stride : one) * 2,
                           (cuuint64_t)(s->kv_heads > 1 ? head_stride : one) * 2,
                           (cuuint64_t)(pages > 1 ? page_stride : one) * 2};
  cuuint32_t box[4] = {(cuuint32_t)cols, (cuuint32_t)box_rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(m, s->dtype == TTTJ_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
         const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return capi_fail(TTTJ_ERR_INVALID, "%s: strides out of range (%d)", what, (int)r);
  return TTTJ_OK;
}

// 3-D map {head_dim, heads, tokens} of queries, moved in boxes of one key/value head's
// group x `tokens` tokens x min(head_dim, 64) columns.
int q_map(CUtensorMap* m, const char* what, const tttj_seqs* s, const tttj_rows* q, int tokens) {
  auto fn = capi_encode_fn();
  if (!fn) return capi_fail(TTTJ_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int cols = s->head_dim < 64 ? s->head_dim : 64;
  const long one = s->head_dim;
  cuuint64_t dims[3] = {(cuuint64_t)s->head_dim, (cuuint64_t)s->heads, (cuuint64_t)s->tokens};
  cuuint64_t strides[2] = {(cuuint64_t)(s->heads > 1 ? q->head_stride : one) * 2,
                           (cuuint64_t)(s->tokens > 1 ? q->token_stride : one) * 2};
  cuuint32_t box[3] = {(cuuint32_t)cols, (cuuint32_t)(s->heads / s->kv_heads), (cuuint32_t)tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(m, s->dtype == TTTJ_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
         const_cast<void*>(q->data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return capi_fail(TTTJ_ERR_INVALID, "%s: strides out of range (%d)", what, (int)r);
  return TTTJ_OK;
}

// A pinned word per device, written by a kernel whose bounded wait gave up and read by the
// device's next call, without synchronising.  Allocated at the first call, which may be under
// stream capture; kept until the process ends.
constexpr int kMostDevices = 64;
std::atomic<int*> g_timeout_words[kMostDevices];

int timeout_word(int dev, int** word) {
  if (dev < 0 || dev >= kMostDevices) return capi_fail(TTTJ_ERR_CUDA, "device %d out of range", dev);
  *word = g_timeout_words[dev].load(std::memory_order_acquire);
  if (*word) return TTTJ_OK;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  CAPI_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
  void* fresh = nullptr;
  const cudaError_t e = cudaHostAlloc(&fresh, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
  if (e == cudaSuccess) {
    *static_cast<volatile int*>(fresh) = 0;
    int* first = nullptr;  // another thread's first call may have been faster: its word then
    *word = g_timeout_words[dev].compare_exchange_strong(first, static_cast<int*>(fresh), std::memory_order_acq_rel)
                ? static_cast<int*>(fresh)
                : first;
  }
  const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
  CAPI_CUDA(e);
  CAPI_CUDA(back);
  return TTTJ_OK;
}

// The current device of a call that is about to launch: its multiprocessors and its word.  An
// earlier call's wait that gave up is reported here, once.
int device_here(const char* what, int* sms, int** word) {
  int dev = 0;
  CAPI_CUDA(cudaGetDevice(&dev));
  *sms = capi_sm_count(dev);
  if (*sms <= 0) return capi_fail(TTTJ_ERR_CUDA, "no multiprocessor count");
  TRY(timeout_word(dev, word));
  if (*static_cast<volatile int*>(*word) != 0) {
    const int v = __atomic_exchange_n(*word, 0, __ATOMIC_ACQ_REL);
    if (v != 0)
      return capi_fail(TTTJ_ERR_DEVICE_TIMEOUT,
                       "%s: a device wait of an earlier serving call on this device timed out (status 0x%x); that "
                       "call's results are invalid", what, v);
  }
  return TTTJ_OK;
}

constexpr int kMostSms = 160;  // multiprocessors that a call uses at most (workspace sizes)
// Sequences of at most this many query rows per key/value head (new tokens x group) run on
// the few-row kernel, chunks of more on the tile kernel: one mma tile of rows reads the keys once,
// two read them twice.  Measured, few-row against tile kernel, bf16, us: 64 sequences of 4096 keys, 8
// key/value heads x 128: 16 rows 183 / 230-238, 24 rows 341 / 245, 64 rows 668 / 262; 64 of 2048, 4
// x 64: 16 rows 33 / 63, 32 rows 55 / 62, 48 rows 75 / 63.  Calls too small to fill the device stay
// faster on the few-row kernel beyond the limit (8 of 8192, 4 x 128: 48 rows 49 / 70, 64 rows 72 / 69;
// 4 of 1000, 4 x 64: 128 rows 15 / 23), but the host does not know the lengths.
constexpr int kStepMostRows = 16;

// Workspace of either attention kernel.
struct ServeWs {
  size_t part_o, part_ml, entries, joins, redo, counters, total;
  int most_entries, most_parts, most_redo;
};
int tile_tokens(const tttj_seqs* s) { return ATC_BM / (s->heads / s->kv_heads); }
ServeWs step_ws(const tttj_seqs* s) {
  ServeWs w{};
  const size_t parts = 2ul * kMostSms * step_ctas_per_sm(s->head_dim) * STEP_ROWS;
  w.part_o = 0;
  w.part_ml = up(parts * s->head_dim * 4);
  w.total = w.part_ml + up(parts * 8);
  return w;
}
ServeWs tile_ws(const tttj_seqs* s) {
  ServeWs w{};
  // Bounds of tile_plan_kernel: cut items leave at most 4 pieces per CTA (and one per head).
  w.most_parts = 4 * kMostSms + s->kv_heads;
  const int items = s->tokens / (tile_nt(s->head_dim) * tile_tokens(s)) + s->batch;  // of a key/value head
  w.most_entries = items + w.most_parts;
  const long notes = (long)items * s->kv_heads * 4 * tile_nt(s->head_dim);  // one per softmax warp of an item
  w.most_redo = (int)(notes < (1l << 30) ? notes : 1l << 30);
  const size_t rows = (size_t)w.most_parts * tile_nt(s->head_dim) * ATC_BM;
  w.counters = 0;
  w.entries = up(16);
  w.joins = w.entries + up((size_t)w.most_entries * sizeof(TileEntry));
  w.redo = w.joins + up((size_t)w.most_entries * sizeof(TileJoin));
  w.part_ml = w.redo + up((size_t)w.most_redo * sizeof(int4));
  w.part_o = w.part_ml + up(rows * 8);
  w.total = w.part_o + up(rows * s->head_dim * 4);
  return w;
}
bool step_runs(const tttj_seqs* s, bool cache, int max_new) {
  const long new_tokens = max_new > 0 && max_new < s->tokens ? max_new : s->tokens;
  return cache && new_tokens * (s->heads / s->kv_heads) <= kStepMostRows;
}
size_t serve_bytes(const tttj_seqs* s) {
  const size_t a = step_ws(s).total, b = tile_ws(s).total;
  return a > b ? a : b;
}

// One call of either attention: packed keys / values (cache = false; page strides unused,
// slots are tokens) or a cache.
int attention(const char* what, const tttj_seqs* s, const tttj_rows* q, const CacheView& k, const CacheView& v,
              const tttj_rows* out, float* lse, int causal, int max_new, float scale, void* workspace,
              size_t workspace_bytes, bool cache, cudaStream_t stream) {
  const size_t need = serve_bytes(s);
  if (!workspace || workspace_bytes < need)
    return capi_fail(TTTJ_ERR_INVALID, "%s: workspace too small: %zu < %zu", what, workspace ? workspace_bytes : 0,
                     need);
  if (reinterpret_cast<uintptr_t>(workspace) & (kAlign - 1))
    return capi_fail(TTTJ_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  TRY(check_scale(what, scale));
  int sms = 0, *timeout = nullptr;
  TRY(device_here(what, &sms, &timeout));
  if (sms > kMostSms) sms = kMostSms;
  const bool step = step_runs(s, cache, max_new);
  const int keys = step ? STEP_KEYS : ATC_BN;
  const int slots = cache ? s->page_size : s->tokens, pages = cache ? s->num_pages : 1;
  const int box = cache && s->page_size < keys ? s->page_size : keys;
  CUtensorMap tm_k, tm_v;
  TRY(kv_map(&tm_k, what, s, k.data, k.page, k.slot, k.head, slots, pages, box));
  TRY(kv_map(&tm_v, what, s, v.data, v.page, v.slot, v.head, slots, pages, box));
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const int bf16 = s->dtype == TTTJ_DTYPE_BF16;
  const float scale_log2 = scale * 1.44269504088896341f;
  if (step) {
    const ServeWs w = step_ws(s);
    StepParams p{};
    p.s = seqs_of(s, cache, causal);
    p.q = q->data;
    p.q_tok = q->token_stride;
    p.q_head = q->head_stride;
    p.out = const_cast<void*>(out->data);
    p.o_tok = out->token_stride;
    p.o_head = out->head_stride;
    p.lse = lse;
    p.heads = s->heads;
    p.kv_heads = s->kv_heads;
    p.group = s->heads / s->kv_heads;
    p.scale_log2 = scale_log2;
    p.part_o = reinterpret_cast<float*>(base + w.part_o);
    p.part_ml = reinterpret_cast<float2*>(base + w.part_ml);
    p.timeout_host = timeout;
    CAPI_CUDA(step_launch(tm_k, tm_v, p, s->head_dim, bf16, sms * step_ctas_per_sm(s->head_dim), stream));
    return TTTJ_OK;
  }
  const ServeWs w = tile_ws(s);
  TileParams p{};
  p.s = seqs_of(s, cache, causal);
  p.q = q->data;
  p.q_tok = q->token_stride;
  p.q_head = q->head_stride;
  p.k = k;
  p.v = v;
  p.out = const_cast<void*>(out->data);
  p.o_tok = out->token_stride;
  p.o_head = out->head_stride;
  p.o_wide = reinterpret_cast<uintptr_t>(out->data) % 32 == 0 && out->token_stride % 16 == 0 && out->head_stride % 16 == 0;
  p.lse = lse;
  p.heads = s->heads;
  p.kv_heads = s->kv_heads;
  p.group = s->heads / s->kv_heads;
  p.tile_tokens = tile_tokens(s);
  p.scale_log2 = scale_log2;
  p.plan.counters = reinterpret_cast<int*>(base + w.counters);
  p.plan.entries = reinterpret_cast<TileEntry*>(base + w.entries);
  p.plan.joins = reinterpret_cast<TileJoin*>(base + w.joins);
  p.plan.redo = reinterpret_cast<int4*>(base + w.redo);
  p.plan.most_redo = w.most_redo;
  p.plan.most_entries = w.most_entries;
  p.plan.most_parts = w.most_parts;
  p.part_o = reinterpret_cast<float*>(base + w.part_o);
  p.part_ml = reinterpret_cast<float2*>(base + w.part_ml);
  p.timeout_host = timeout;
  CUtensorMap tm_q;
  TRY(q_map(&tm_q, what, s, q, p.tile_tokens));
  CAPI_CUDA(tile_launch(tm_q, tm_k, tm_v, p, s->head_dim, bf16, sms, stream));
  return TTTJ_OK;
}

}  // namespace

extern "C" {

size_t tttj_serve_workspace_bytes(const tttj_seqs* s) {
  if (check_seqs("serve_workspace_bytes", s, false, false)) return 0;
  return serve_bytes(s);
}

int tttj_prompt_attention(const tttj_seqs* s, const tttj_rows* q, const tttj_rows* k, const tttj_rows* v,
                          const tttj_rows* out, float* lse, int causal, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
  const char* what = "prompt_attention";
  TRY(check_seqs(what, s, false, true));
  TRY(check_rows(what, "q", q, s, s->heads));
  TRY(check_rows(what, "k", k, s, s->kv_heads));
  TRY(check_rows(what, "v", v, s, s->kv_heads));
  TRY(check_rows(what, "out", out, s, s->heads));
  if (s->tokens == 0) return TTTJ_OK;
  const CacheView kv{const_cast<void*>(k->data), 0, k->token_stride, k->head_stride};
  const CacheView vv{const_cast<void*>(v->data), 0, v->token_stride, v->head_stride};
  return attention(what, s, q, kv, vv, out, lse, causal ? 1 : 0, 0, scale, workspace, workspace_bytes, false,
                   static_cast<cudaStream_t>(stream));
}

int tttj_cache_attention(const tttj_seqs* s, const tttj_rows* q, const tttj_pages* k_cache,
                         const tttj_pages* v_cache, const tttj_rows* out, float* lse, int max_new, float scale,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "cache_attention";
  TRY(check_seqs(what, s, true, true));
  TRY(check_rows(what, "q", q, s, s->heads));
  TRY(check_rows(what, "out", out, s, s->heads));
  TRY(check_pages(what, "k_cache", k_cache, s));
  TRY(check_pages(what, "v_cache", v_cache, s));
  if (max_new < 0) return capi_fail(TTTJ_ERR_INVALID, "%s: max_new=%d is negative", what, max_new);
  if (s->tokens == 0) return TTTJ_OK;
  return attention(what, s, q, view_of(k_cache), view_of(v_cache), out, lse, 1, max_new, scale, workspace,
                   workspace_bytes, true, static_cast<cudaStream_t>(stream));
}

int tttj_cache_append(const tttj_seqs* s, const tttj_rows* k, const tttj_rows* v, const tttj_pages* k_cache,
                      const tttj_pages* v_cache, int32_t* positions, float* mass, const int32_t* seen,
                      void* stream) {
  const char* what = "cache_append";
  TRY(check_seqs(what, s, true, true));
  TRY(check_rows(what, "k", k, s, s->kv_heads));
  TRY(check_rows(what, "v", v, s, s->kv_heads));
  TRY(check_pages(what, "k_cache", k_cache, s));
  TRY(check_pages(what, "v_cache", v_cache, s));
  if (s->tokens == 0) return TTTJ_OK;
  AppendParams p{};
  p.s = seqs_of(s, true, 1);
  p.k = k->data;
  p.v = v->data;
  p.k_tok = k->token_stride;
  p.k_head = k->head_stride;
  p.v_tok = v->token_stride;
  p.v_head = v->head_stride;
  p.kc = view_of(k_cache);
  p.vc = view_of(v_cache);
  p.kv_heads = s->kv_heads;
  p.head_dim = s->head_dim;
  p.positions = positions;
  p.mass = mass;
  p.seen = seen;
  int sms = 0, *timeout = nullptr;
  TRY(device_here(what, &sms, &timeout));
  CAPI_CUDA(append_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return TTTJ_OK;
}

int tttj_cache_mass(const tttj_seqs* s, const tttj_rows* q, const float* lse, const tttj_pages* k_cache,
                    const float* mass, float* mass_out, int max_new, float scale, void* stream) {
  const char* what = "cache_mass";
  TRY(check_seqs(what, s, true, true));
  TRY(check_rows(what, "q", q, s, s->heads));
  TRY(check_pages(what, "k_cache", k_cache, s));
  if (!mass || !mass_out || (!lse && s->tokens > 0)) return capi_fail(TTTJ_ERR_INVALID, "%s: null argument", what);
  TRY(check_scale(what, scale));
  if (max_new < 0) return capi_fail(TTTJ_ERR_INVALID, "%s: max_new=%d is negative", what, max_new);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long cap = (long)s->pages_per_seq * s->page_size;
  if (s->tokens == 0) {
    if (mass != mass_out)
      CAPI_CUDA(cudaMemcpyAsync(mass_out, mass, (size_t)s->batch * s->kv_heads * cap * 4, cudaMemcpyDeviceToDevice, st));
    return TTTJ_OK;
  }
  int sms = 0, *timeout = nullptr;
  TRY(device_here(what, &sms, &timeout));
  MassParams p{};
  p.s = seqs_of(s, true, 1);
  p.lse = lse;
  p.mass = mass;
  p.out = mass_out;
  p.cap = cap;
  p.heads = s->heads;
  p.kv_heads = s->kv_heads;
  p.group = s->heads / s->kv_heads;
  // Query tiles no larger than the tokens a sequence has: single tokens load one each.
  p.tile_tokens = MASS_TILE_ROWS / p.group;
  const int most = max_new > 0 && max_new < s->tokens ? max_new : s->tokens;
  if (most < p.tile_tokens) p.tile_tokens = most;
  p.scale_log2 = scale * 1.44269504088896341f;
  p.timeout_host = timeout;
  CUtensorMap tm_q, tm_k;
  TRY(q_map(&tm_q, what, s, q, p.tile_tokens));
  TRY(kv_map(&tm_k, what, s, k_cache->data, k_cache->page_stride, k_cache->slot_stride, k_cache->head_stride,
             s->page_size, s->num_pages, s->page_size < ATC_BM ? s->page_size : ATC_BM));
  CAPI_CUDA(mass_launch(tm_q, tm_k, p, s->head_dim, s->dtype == TTTJ_DTYPE_BF16, sms, st));
  return TTTJ_OK;
}

int tttj_serve_status(int* device_status) {
  if (!device_status) return capi_fail(TTTJ_ERR_INVALID, "serve_status: null argument");
  int dev = 0, *word = nullptr;
  CAPI_CUDA(cudaGetDevice(&dev));
  TRY(timeout_word(dev, &word));
  CAPI_CUDA(cudaDeviceSynchronize());
  *device_status = __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL);
  if (*device_status != 0)
    return capi_fail(TTTJ_ERR_DEVICE_TIMEOUT, "serving: a device wait timed out (status 0x%x)", *device_status);
  return TTTJ_OK;
}

int tttj_serve_selftest_timeout(int32_t* status, uint64_t limit_ns, void* stream) {
  if (limit_ns > 1000000000ull) return capi_fail(TTTJ_ERR_INVALID, "serve_selftest: limit above 1 s");
  int dev = 0, *word = nullptr;
  CAPI_CUDA(cudaGetDevice(&dev));
  TRY(timeout_word(dev, &word));
  CAPI_CUDA(serve_selftest_launch(status, word, limit_ns, static_cast<cudaStream_t>(stream)));
  return TTTJ_OK;
}

static int evict_most_moves(const tttj_seqs* s, int keep) {
  const long cap = (long)s->pages_per_seq * s->page_size;
  const long behind = cap - keep;
  return behind <= 0 ? 0 : (int)(behind < keep ? behind : keep);
}

size_t tttj_cache_evict_workspace_bytes(const tttj_seqs* s, int keep) {
  if (check_seqs("cache_evict", s, true, false) || keep <= 0) return 0;
  const size_t bh = (size_t)s->batch * s->kv_heads;
  return up(bh * evict_most_moves(s, keep) * sizeof(int2) + 1);  // never 0: that stands for an error
}

int tttj_cache_evict(const tttj_seqs* s, const tttj_pages* k_cache, const tttj_pages* v_cache, const float* mass,
                     const int32_t* positions, int keep, int recent, float* mass_out, int32_t* positions_out,
                     int32_t* lens_out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "cache_evict";
  TRY(check_seqs(what, s, true, false));
  TRY(check_pages(what, "k_cache", k_cache, s));
  TRY(check_pages(what, "v_cache", v_cache, s));
  if (!mass || !positions || !mass_out || !positions_out || !lens_out)
    return capi_fail(TTTJ_ERR_INVALID, "%s: null argument", what);
  if (mass == mass_out || positions == positions_out || s->cache_lens == lens_out)
    return capi_fail(TTTJ_ERR_INVALID, "%s: outputs may not be the inputs", what);
  if (keep <= 0) return capi_fail(TTTJ_ERR_INVALID, "%s: keep=%d must be positive", what, keep);
  if (recent < 0 || recent > keep)
    return capi_fail(TTTJ_ERR_INVALID, "%s: recent=%d outside 0 .. keep=%d", what, recent, keep);
  const size_t need = tttj_cache_evict_workspace_bytes(s, keep);
  if (!workspace || workspace_bytes < need)
    return capi_fail(TTTJ_ERR_INVALID, "%s: workspace too small: %zu < %zu", what, workspace ? workspace_bytes : 0,
                     need);
  if (reinterpret_cast<uintptr_t>(workspace) & (kAlign - 1))
    return capi_fail(TTTJ_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  EvictParams p{};
  p.s = seqs_of(s, true, 1);
  p.kc = view_of(k_cache);
  p.vc = view_of(v_cache);
  p.kv_heads = s->kv_heads;
  p.head_dim = s->head_dim;
  p.mass = mass;
  p.positions = positions;
  p.mass_out = mass_out;
  p.positions_out = positions_out;
  p.lens_out = lens_out;
  p.keep = keep;
  p.recent = recent;
  p.cap = (long)s->pages_per_seq * s->page_size;
  p.most_moves = evict_most_moves(s, keep);
  p.moves = reinterpret_cast<int2*>(workspace);
  int sms = 0, *timeout = nullptr;
  TRY(device_here(what, &sms, &timeout));
  CAPI_CUDA(evict_launch(p, sms, static_cast<cudaStream_t>(stream)));
  return TTTJ_OK;
}

}  // extern "C"
