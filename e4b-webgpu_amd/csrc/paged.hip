// paged.hip -- the C entry points of the paged key/value cache: argument
// checks and launches (kernels: k_paged*.hip).
#include <algorithm>

#include "../../include/e4b.h"
#include "paged.h"
#include "util.h"

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
bool dims_ok(int type, int kv_heads, int head_dim, int page) {
  return (type == E4B_KV_F16 || type == E4B_KV_Q4) && kv_heads >= 1 && kv_heads <= 256 &&
         (head_dim == 128 || head_dim == 256 || head_dim == 512) && page >= 16 && page <= 256 && !(page & (page - 1));
}
int shift_of(int page) { return __builtin_ctz((unsigned)page); }

int check_cache(const char* fn, const e4b_paged_kv* kv) {
  if (!kv) return e4b_fail(E4B_EINVAL, "%s: null cache", fn);
  if (!dims_ok(kv->type, kv->kv_heads, kv->head_dim, kv->page) || kv->n_pages < 1 || kv->table_stride < 1)
    return e4b_fail(E4B_EINVAL,
                    "%s: bad cache (type %d, %d KV heads, head_dim %d (128, 256 or 512), page %d (16 .. 256, a power "
                    "of two), %d pages, table_stride %d)",
                    fn, kv->type, kv->kv_heads, kv->head_dim, kv->page, kv->n_pages, kv->table_stride);
  if (!kv->k || !kv->v || !kv->table) return e4b_fail(E4B_EINVAL, "%s: null pool or table", fn);
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->table, 4))
    return e4b_fail(E4B_EINVAL, "%s: pools must be 16-byte aligned, the table 4", fn);
  return E4B_OK;
}

// the checks every call makes; *empty: there is nothing to do
int check_call(const char* fn, const e4b_paged_kv* kv, const e4b_kv_batch* b, PagedArgs* P, bool* empty) {
  int rc = check_cache(fn, kv);
  if (rc) return rc;
  if (!b) return e4b_fail(E4B_EINVAL, "%s: null batch", fn);
  // (a grid's threads are below 2^32: tokens by 256, units of attention by 512)
  if (b->n_seq < 0 || b->n_tok < 0 || b->n_seq > 65535 || b->n_tok >= (1 << 24) ||
      (int64_t)b->n_seq * kv->kv_heads > (1 << 21))
    return e4b_fail(E4B_EINVAL, "%s: %d sequences (0 .. 65535, %d KV heads: 2^21 of both), %d tokens (below 2^24)", fn,
                    b->n_seq, kv->kv_heads, b->n_tok);
  *empty = b->n_seq == 0 || b->n_tok == 0;
  if (*empty) return E4B_OK;
  if (!b->q_start || !b->kv_len || !aligned(b->q_start, 4) || !aligned(b->kv_len, 4))
    return e4b_fail(E4B_EINVAL, "%s: q_start or kv_len is null or not 4-byte aligned", fn);
  if (b->max_q < 1 || b->max_kv < 1)
    return e4b_fail(E4B_EINVAL, "%s: max_q %d and max_kv %d must be at least 1", fn, b->max_q, b->max_kv);
  *P = PagedArgs{(uint8_t*)kv->k, (uint8_t*)kv->v, kv->table, b->q_start, b->kv_len, kv->n_pages, kv->table_stride,
                 kv->kv_heads, shift_of(kv->page), b->n_seq, b->n_tok};
  return E4B_OK;
}

// rows of `heads` heads, `stride` elements apart, read 16 bytes at a time
int check_rows(const char* fn, const char* what, const void* p, int dtype, int64_t stride, int heads, int hd) {
  if (dtype != E4B_DT_F32 && dtype != E4B_DT_F16)
    return e4b_fail(E4B_EINVAL, "%s: %s dtype %d (E4B_DT_F32 or E4B_DT_F16)", fn, what, dtype);
  if (!p) return e4b_fail(E4B_EINVAL, "%s: null %s", fn, what);
  const int per16 = dtype == E4B_DT_F32 ? 4 : 8;
  if (stride < (int64_t)heads * hd || stride % per16 || !aligned(p, 16))
    return e4b_fail(E4B_EINVAL, "%s: %s must be 16-byte aligned rows of %d heads of %d (stride %lld)", fn, what, heads,
                    hd, (long long)stride);
  return E4B_OK;
}

}  // namespace

extern "C" size_t e4b_kv_page_bytes(int type, int kv_heads, int head_dim, int page) {
  if (!dims_ok(type, kv_heads, head_dim, page)) {
    e4b_fail(E4B_EINVAL, "e4b_kv_page_bytes: bad cache (type %d, %d KV heads, head_dim %d, page %d)", type, kv_heads,
             head_dim, page);
    return 0;
  }
  return (size_t)kv_heads * page * paged_row_bytes(type == E4B_KV_Q4, head_dim);
}

extern "C" int64_t e4b_kv_row(const e4b_paged_kv* kv, const uint32_t* table_row, int64_t pos) {
  if (!kv || !table_row || !dims_ok(kv->type, kv->kv_heads, kv->head_dim, kv->page) || kv->n_pages < 1 ||
      kv->table_stride < 1)
    return e4b_fail(E4B_EINVAL, "e4b_kv_row: bad cache or null table");
  const int pg = paged_page(table_row, kv->table_stride, shift_of(kv->page), kv->n_pages, pos);
  if (pg < 0) return e4b_fail(E4B_ERANGE, "e4b_kv_row: position %lld has no page", (long long)pos);
  return (int64_t)pg * kv->kv_heads * kv->page + (pos & (kv->page - 1));
}

extern "C" int e4b_k_kv_append(const e4b_paged_kv* kv, const e4b_kv_batch* batch, const e4b_head_prep* prep,
                               const void* qkv, int dtype, int64_t stride, int q_heads, void* q_out, int q_dtype,
                               int64_t q_stride, void* stream) {
  const char* fn = "e4b_k_kv_append";
  KvAppendArgs a;
  bool empty;
  int rc = check_call(fn, kv, batch, &a.P, &empty);
  if (rc) return rc;
  if (!prep) return e4b_fail(E4B_EINVAL, "%s: null head prep", fn);
  const int hd = kv->head_dim;
  if (prep->flags & ~(E4B_PREP_V_RMS | E4B_PREP_V_IS_K))
    return e4b_fail(E4B_EINVAL, "%s: unknown flags 0x%x", fn, prep->flags);
  if (prep->rope_angles < 0 || prep->rope_angles > hd / 2 || (prep->rope_angles && !prep->inv_freq))
    return e4b_fail(E4B_EINVAL, "%s: %d rotated pairs of a %d-dim head%s", fn, prep->rope_angles, hd,
                    prep->inv_freq ? "" : ", inv_freq null");
  if (!aligned(prep->q_norm, 16) || !aligned(prep->k_norm, 16) || !aligned(prep->inv_freq, 4))
    return e4b_fail(E4B_EINVAL, "%s: norm weights must be 16-byte aligned, inv_freq 4", fn);
  if (!(prep->eps >= 0.f)) return e4b_fail(E4B_EINVAL, "%s: eps %g", fn, (double)prep->eps);
  if (q_heads < 0 || q_heads > 4096) return e4b_fail(E4B_EINVAL, "%s: %d query heads", fn, q_heads);
  if (empty) return E4B_OK;
  a.v_is_k = (prep->flags & E4B_PREP_V_IS_K) != 0;
  a.v_rms = (prep->flags & E4B_PREP_V_RMS) != 0;
  if ((rc = check_rows(fn, "qkv", qkv, dtype, stride, q_heads + (a.v_is_k ? 1 : 2) * kv->kv_heads, hd))) return rc;
  if (q_out && (rc = check_rows(fn, "q_out", q_out, q_dtype, q_stride, q_heads, hd))) return rc;
  a.x = qkv;
  a.x_stride = stride;
  a.q = q_out;
  a.q_stride = q_stride;
  a.qw = prep->q_norm;
  a.kw = prep->k_norm;
  a.inv_freq = prep->inv_freq;
  a.angles = prep->rope_angles;
  a.qh = q_heads;
  a.eps = prep->eps;
  a.q16 = q_dtype == E4B_DT_F16;
  return launch_kv_append(a, hd, kv->type == E4B_KV_Q4, dtype == E4B_DT_F16, (hipStream_t)stream);
}

extern "C" int e4b_k_kv_gather(const e4b_paged_kv* kv, const e4b_kv_batch* batch, void* k_out, void* v_out,
                               void* stream) {
  const char* fn = "e4b_k_kv_gather";
  PagedArgs P;
  bool empty;
  int rc = check_call(fn, kv, batch, &P, &empty);
  if (rc) return rc;
  if (empty) return E4B_OK;
  if ((!k_out && !v_out) || !aligned(k_out, 16) || !aligned(v_out, 16))
    return e4b_fail(E4B_EINVAL, "%s: no output, or one that is not 16-byte aligned", fn);
  return launch_kv_gather(P, kv->head_dim, kv->type == E4B_KV_Q4, (uint16_t*)k_out, (uint16_t*)v_out,
                          (hipStream_t)stream);
}

// An attention call: the sequences with few query rows go to one kernel, the
// others to another.
struct AttnPlan {
  PagedAttnArgs few, chunk;
  bool use_few = false, use_chunk = false;
};
static size_t scratch_bytes(const PagedAttnArgs& a) {  // splits' outputs, then their maxima and sums
  return E4B_ALIGN256(a.part_floats * sizeof(float)) + E4B_ALIGN256(a.ml_floats * sizeof(float));
}
static size_t scratch_bytes(const AttnPlan& p) {
  return (p.use_few ? scratch_bytes(p.few) : 0) + (p.use_chunk ? scratch_bytes(p.chunk) : 0);
}
static uint8_t* give_scratch(PagedAttnArgs& a, uint8_t* ws) {
  a.part = (float*)ws;
  a.part_ml = (float*)(ws + E4B_ALIGN256(a.part_floats * sizeof(float)));
  return ws + scratch_bytes(a);
}

// the checks of an attention call; *plan is complete but for pointers and scale
static int attn_setup(const char* fn, const e4b_paged_kv* kv, const e4b_kv_batch* batch, int q_dtype, int q_heads,
                      int window, int sinks, AttnPlan* plan, bool* empty) {
  PagedAttnArgs a{};
  int rc = check_call(fn, kv, batch, &a.P, empty);
  if (rc) return rc;
  if (q_heads < 1 || q_heads > 4096 || q_heads % kv->kv_heads)
    return e4b_fail(E4B_EINVAL, "%s: %d query heads over %d KV heads", fn, q_heads, kv->kv_heads);
  if (q_dtype != E4B_DT_F32 && q_dtype != E4B_DT_F16)
    return e4b_fail(E4B_EINVAL, "%s: q dtype %d (E4B_DT_F32 or E4B_DT_F16)", fn, q_dtype);
  if (window < 0 || sinks < 0) return e4b_fail(E4B_EINVAL, "%s: window %d, sinks %d", fn, window, sinks);
  if (*empty) return E4B_OK;
  if ((int64_t)batch->n_tok * q_heads > (1 << 28))
    return e4b_fail(E4B_EINVAL, "%s: %d tokens of %d heads are more than 2^28 rows", fn, batch->n_tok, q_heads);
  a.qh = q_heads;
  a.gqa = q_heads / kv->kv_heads;
  a.window = window;
  a.sinks = window ? sinks : 0;
  a.max_q = std::min(batch->max_q, batch->n_tok);
  a.max_kv = batch->max_kv;
  plan->use_chunk = a.max_q * a.gqa > kPagedFewRows;
  // Short sequences beside long ones: where all are as long as the longest
  // there are none, and a launch is saved
  plan->use_few = !plan->use_chunk || (a.gqa <= kPagedFewRows && (int64_t)batch->n_seq * a.max_q > batch->n_tok);
  if (plan->use_few) {
    plan->few = a;
    plan->few.max_q = std::min(a.max_q, kPagedFewRows / a.gqa);
    plan_attn_paged_few(plan->few, kv->head_dim);
  }
  if (plan->use_chunk) {
    plan->chunk = a;
    plan->chunk.few_rows = plan->use_few ? kPagedFewRows : 0;
    plan_attn_paged_chunk(plan->chunk, kv->head_dim, q_dtype == E4B_DT_F16);
  }
  return E4B_OK;
}

extern "C" int e4b_attn_paged_ws_bytes(const e4b_paged_kv* kv, const e4b_kv_batch* batch, int q_dtype, int q_heads,
                                       int window, int sinks, size_t* bytes) {
  const char* fn = "e4b_attn_paged_ws_bytes";
  if (!bytes) return e4b_fail(E4B_EINVAL, "%s: null result", fn);
  AttnPlan plan;
  bool empty;
  int rc = attn_setup(fn, kv, batch, q_dtype, q_heads, window, sinks, &plan, &empty);
  if (rc) return rc;
  *bytes = scratch_bytes(plan);
  return E4B_OK;
}

extern "C" int e4b_k_attn_paged(const e4b_paged_kv* kv, const e4b_kv_batch* batch, const void* q, int q_dtype,
                                int64_t q_stride, int q_heads, float scale, int window, int sinks, void* out_f16,
                                int64_t out_stride, void* ws, size_t ws_bytes, void* stream) {
  const char* fn = "e4b_k_attn_paged";
  AttnPlan plan;
  bool empty;
  int rc = attn_setup(fn, kv, batch, q_dtype, q_heads, window, sinks, &plan, &empty);
  if (rc) return rc;
  if (!(scale - scale == 0.f)) return e4b_fail(E4B_EINVAL, "%s: scale is not finite", fn);
  if (empty) return E4B_OK;
  if ((rc = check_rows(fn, "q", q, q_dtype, q_stride, q_heads, kv->head_dim))) return rc;
  if ((rc = check_rows(fn, "out", out_f16, E4B_DT_F16, out_stride, q_heads, kv->head_dim))) return rc;
  if (const size_t need = scratch_bytes(plan)) {
    if (ws && (ws_bytes < need || !aligned(ws, 16)))
      return e4b_fail(E4B_EINVAL, "%s: %zu bytes of scratch where %zu, 16-byte aligned, are needed", fn, ws_bytes, need);
    if (!ws) {
      Workspace w;
      if ((rc = e4b_workspace(need, &w, (hipStream_t)stream))) return rc;
      ws = w.buf;
    }
  }
  uint8_t* at = (uint8_t*)ws;
  const bool q4 = kv->type == E4B_KV_Q4, q16 = q_dtype == E4B_DT_F16;
  for (PagedAttnArgs* a : {plan.use_chunk ? &plan.chunk : nullptr, plan.use_few ? &plan.few : nullptr}) {
    if (!a) continue;
    a->q = q;
    a->q_stride = q_stride;
    a->out = (uint16_t*)out_f16;
    a->out_stride = out_stride;
    a->scale = scale;
    at = give_scratch(*a, at);
  }
  hipStream_t st = (hipStream_t)stream;
  if (plan.use_chunk && plan.use_few) return launch_attn_paged_mixed(plan.chunk, plan.few, kv->head_dim, q4, q16, st);
  return plan.use_chunk ? launch_attn_paged_chunk(plan.chunk, kv->head_dim, q4, q16, st)
                        : launch_attn_paged_few(plan.few, kv->head_dim, q4, q16, st);
}
