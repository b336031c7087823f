// k_paged_attn.hip -- attention over the paged key/value cache (paged.h).
#include "../../include/e4b.h"
#include "paged.h"
#include "util.h"

namespace {

// One wave a (token, query head): dims E l .. of lane l, one key at a time,
// softmax with a running maximum and sum.
template <int HD, bool Q4, bool Q16>
__global__ __launch_bounds__(64) void k_attn_paged(PagedAttnArgs A) {
  constexpr int E = HD / 64;
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, g = h / A.gqa;
  const int i = __builtin_amdgcn_readfirstlane(seq_of_token(P, t));
  if (i >= P.n_seq) return;
  const SeqSpan s = seq_span(P, i);
  if (t < s.q0 || t - s.q0 >= s.n) return;
  const int pos = s.p0 + (t - s.q0);
  float q[E], o[E], m = -3.0e38f, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t at = (int64_t)t * A.q_stride + h * HD + E * lane + e;
    q[e] = (Q16 ? h2f(((const uint16_t*)A.q)[at]) : ((const float*)A.q)[at]) * A.scale;
    o[e] = 0.f;
  }
  auto row = [&](const uint8_t* pool, int64_t block, int r, float(&x)[E]) {
    const uint8_t* b = pool + block;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = E * lane + e;
      if constexpr (Q4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(b + r * (HD / 2) + (d / 8) * 4);
        const int pr = (d % 8) / 2;
        const uint32_t n = w >> (((pr & 1) << 3) + ((pr & 2) << 1) + 16 * (d & 1));
        x[e] = ((int)(n & 15) - 8) *
               h2f(*reinterpret_cast<const uint16_t*>(b + (HD / 2 << P.page_shift) + r * (HD / 16) + (d / 32) * 2));
      } else {
        x[e] = h2f(reinterpret_cast<const uint16_t*>(b)[r * HD + d]);
      }
    }
  };
  const int first = A.window > 0 ? max(0, pos - A.window + 1) : 0;
  for (int p = 0; p <= pos; ++p) {
    if (p < first && p >= A.sinks) p = first;
    const int pg = paged_page(table_row(P, i), P.table_stride, P.page_shift, P.n_pages, p);
    if (pg < 0) continue;
    const int64_t block = paged_block<Q4, HD>(P, pg, g);
    const int r = p & ((1 << P.page_shift) - 1);
    float x[E], sc = 0.f;
    row(P.k, block, r, x);
#pragma unroll
    for (int e = 0; e < E; ++e) sc = fmaf(q[e], x[e], sc);
    sc = wave_sum(sc);
    const float mn = fmaxf(m, sc), a = __expf(m - mn), w = __expf(sc - mn);
    m = mn;
    l = l * a + w;
    row(P.v, block, r, x);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * x[e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < E; ++e) A.out[(int64_t)t * A.out_stride + h * HD + E * lane + e] = f2h(o[e] * inv);
}

template <int HD>
int attn_hd(const PagedAttnArgs& a, bool q4, bool q16, hipStream_t st) {
  const dim3 grid(a.P.n_tok, a.qh);
  if (q4 && q16)
    k_attn_paged<HD, true, true><<<grid, 64, 0, st>>>(a);
  else if (q4)
    k_attn_paged<HD, true, false><<<grid, 64, 0, st>>>(a);
  else if (q16)
    k_attn_paged<HD, false, true><<<grid, 64, 0, st>>>(a);
  else
    k_attn_paged<HD, false, false><<<grid, 64, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

int launch_attn_paged(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st) {
  if (a.max_rows <= kPagedFewRows) return launch_attn_paged_few(a, hd, q4, q16, st);
  return hd == 128 ? attn_hd<128>(a, q4, q16, st) : hd == 256 ? attn_hd<256>(a, q4, q16, st) : attn_hd<512>(a, q4, q16, st);
}
