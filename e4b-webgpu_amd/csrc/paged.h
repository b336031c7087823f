// paged.h -- the paged key/value cache: where a position's row lies, the rows'
// formats, and what its kernels take (paged.hip, k_paged*.hip).
//
// A pool (one for K, one for V) is n_pages blocks [kv_heads][page rows].  The
// rows of one page and head lie together:
//   f16    [page][hd] f16
//   4 bits [page][hd / 2] codes, then [page][hd / 32] f16 scales
// Codes: dword w of a row holds dims 8w .. 8w + 7 in the order of the q4_0
// nibble plane (common.h): dims (0,1) at bits (0,16), (2,3) at (8,24), (4,5)
// at (4,20), (6,7) at (12,28), so (w >> s) & 0x000F000F is a pair of dims.
// Value = (code - 8) d.  d has at most 8 significant bits, code - 8 at most 3
// (or is -8): the value is exact in f16, and the matrix instructions take it
// without a further rounding.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include "kernels.h"
#define E4B_HD __host__ __device__ __forceinline__
#else
#define E4B_HD static inline
#endif

// bytes of one row of one head
E4B_HD int paged_row_bytes(bool q4, int hd) { return q4 ? hd / 2 + hd / 16 : 2 * hd; }

// The page that holds position p of a sequence with table row `row`, or -1:
// before the sequence, past the table, or an entry that names no page.
template <typename Table>
E4B_HD int paged_page(Table row, int table_stride, int page_shift, int n_pages, int64_t p) {
  if (p < 0) return -1;
  const int64_t b = p >> page_shift;
  if (b >= table_stride) return -1;
  const uint32_t pg = row[b];
  return pg < (uint32_t)n_pages ? (int)pg : -1;
}

#ifdef __HIPCC__
struct PagedArgs {
  uint8_t* k;
  uint8_t* v;
  const uint32_t* table;    // [n_seq][table_stride]
  const int32_t* q_start;   // [n_seq + 1]
  const int32_t* kv_len;    // [n_seq]
  int n_pages, table_stride, kvh, page_shift, n_seq, n_tok;
};

// the new tokens of a sequence: q0 .. q0 + n - 1 at positions p0 .. p0 + n - 1
// of kv (entries that the arrays' contents put out of order or out of range
// are cut to what is there, so no kernel reads or writes past a buffer)
struct SeqSpan {
  int q0, n, p0, kv;
};
// The arrays are read with an index that is the same for all lanes and not
// written while a kernel runs: through the scalar cache.
typedef const __attribute__((address_space(4))) uint32_t* table_ptr;
typedef const __attribute__((address_space(4))) int32_t* lens_ptr;
DEV table_ptr table_row(const PagedArgs& P, int i) {
  return (table_ptr)(uintptr_t)P.table + (int64_t)i * P.table_stride;
}
DEV SeqSpan seq_span_of(const PagedArgs& P, int start, int end, int kv) {
  SeqSpan s;
  s.q0 = min(max(start, 0), P.n_tok);
  s.n = min(max(end, s.q0), P.n_tok) - s.q0;
  s.kv = max(kv, 0);
  s.p0 = s.kv - s.n;
  return s;
}
DEV SeqSpan seq_span(const PagedArgs& P, int i) {
  const lens_ptr q_start = (lens_ptr)(uintptr_t)P.q_start, kv_len = (lens_ptr)(uintptr_t)P.kv_len;
  return seq_span_of(P, q_start[i], q_start[i + 1], kv_len[i]);
}
// The sequence of token t (n_seq: behind the last one); the whole wave calls
// it.  The range that holds it is cut into 64 parts at a time: one load up to 64
// sequences, two up to 4096, three above (one token each of 2400 sequences
// appended in 12.5 us, 30.6 when all their ends were read 64 at a time).
DEV int seq_of_token(const PagedArgs& P, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = P.n_seq;
  for (;;) {
    const int part = (hi - lo + 63) / 64, from = lo + lane * part;  // the lane's: from .. from + part
    const bool before = from < hi && P.q_start[min(from + part, hi)] <= t;  // all of it ends before t
    lo = min(lo + (int)__popcll(__ballot(before)) * part, hi);
    if (part <= 1 || lo == hi) return lo;
    hi = min(lo + part, hi);
  }
}
// first byte of the rows of (page, head)
template <bool Q4, int HD>
DEV int64_t paged_block(const PagedArgs& P, int pg, int head) {
  constexpr int RB = Q4 ? HD / 2 + HD / 16 : 2 * HD;
  return (((int64_t)pg * P.kvh + head) << P.page_shift) * RB;
}

struct KvAppendArgs {
  PagedArgs P;
  const void* x;
  int64_t x_stride;         // elements
  void* q;                  // may be null
  int64_t q_stride;
  const float* qw;          // null: the q heads are not normed
  const float* kw;
  const float* inv_freq;
  int angles, qh;
  float eps;
  bool v_rms, v_is_k, q16;
};
int launch_kv_append(const KvAppendArgs& a, int hd, bool q4, bool x16, hipStream_t st);
int launch_kv_gather(const PagedArgs& P, int hd, bool q4, uint16_t* k_out, uint16_t* v_out, hipStream_t st);

constexpr int kPagedMaxSplits = 256;  // of a unit with few rows
struct PagedAttnArgs {
  PagedArgs P;
  const void* q;            // f32 or f16 rows of qh heads
  int64_t q_stride;
  uint16_t* out;
  int64_t out_stride;
  int qh, gqa, window, sinks;
  float scale;
  int max_q, max_kv;        // bounds of a sequence's tokens (<= n_tok) and positions
  // the plan: blocks of rows (tokens x heads of a group) of a sequence, splits
  // of the keys, and where the splits' results go
  int nrb, ns;
  int groups, target;       // few rows: workgroups, and how many the key tiles are cut for
  bool split;
  int second, last[2];      // first token of the second block of 8 rows, last ones of both
  int few_rows;             // chunks: sequences with no more rows than this are left out
  size_t part_floats, ml_floats;
  float* part;
  float* part_ml;
};
// a few query rows per sequence and KV head (paged_few.h)
void plan_attn_paged_few(PagedAttnArgs& a, int hd);
int launch_attn_paged_few(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st);
constexpr int kPagedFewRows = 16;  // most rows of a sequence and KV head that it takes
// any number (paged_chunk.h)
void plan_attn_paged_chunk(PagedAttnArgs& a, int hd, bool q16);
int launch_attn_paged_chunk(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st);
// both (k_paged_mixed.hip)
int launch_attn_paged_mixed(const PagedAttnArgs& chunk, const PagedAttnArgs& few, int hd, bool q4, bool q16,
                            hipStream_t st);
#endif
