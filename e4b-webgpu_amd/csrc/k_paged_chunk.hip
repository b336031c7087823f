// k_paged_chunk.hip -- launches of the attention of many query rows per KV head
// over the paged cache (paged_chunk.h).
#include "paged_chunk.h"

namespace {

template <int HD, bool Q4, bool Q16>
__global__ __launch_bounds__(64 * kChunkWaves<HD>, 2) void k_attn_paged_chunk(PagedAttnArgs A) {
  __shared__ __align__(16) uint4 lds[kChunkLds<HD, Q4> / 16];
  attn_chunk<HD, Q4, Q16>(A, blockIdx.x, gridDim.x, lds);
}
template <int HD, bool Q16>
__global__ __launch_bounds__(256) void k_attn_chunk_merge(PagedAttnArgs A) {
  merge_chunk<HD, Q16>(A, blockIdx.x);
}

template <int HD, bool Q16>
int chunk_hd(const PagedAttnArgs& a, bool q4, hipStream_t st) {
  const unsigned grid = (unsigned)chunk_grid<HD, Q16>(a), merge = (unsigned)chunk_merge_grid<HD, Q16>(a);
  if (q4)
    k_attn_paged_chunk<HD, true, Q16><<<grid, 64 * kChunkWaves<HD>, 0, st>>>(a);
  else
    k_attn_paged_chunk<HD, false, Q16><<<grid, 64 * kChunkWaves<HD>, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  if (!merge) return E4B_OK;
  k_attn_chunk_merge<HD, Q16><<<merge, 256, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

void plan_attn_paged_chunk(PagedAttnArgs& a, int hd, bool q16) {
  const int bm = tile_rows(hd, q16);
  const int64_t units = tile_bound(a, bm) * a.P.kvh, rows = (int64_t)a.P.n_tok * a.gqa;  // units: the grid's
  // Units that have work: known where all sequences are as long as the longest,
  // else as if so many were and the others had a token each
  const int64_t longest = std::min<int64_t>(
      a.P.n_seq, std::max<int64_t>(1, (a.P.n_tok - a.P.n_seq + a.max_q - 2) / std::max(1, a.max_q - 1)));
  const int64_t work = (int64_t)a.P.n_seq * a.max_q == a.P.n_tok
                           ? a.P.n_seq * (((int64_t)a.max_q * a.gqa + bm - 1) / bm)
                           : rows / bm + longest;
  const int64_t seen = a.window ? std::min<int64_t>(a.max_kv, (int64_t)a.window + a.sinks + bm / a.gqa + 1) : a.max_kv;
  const int64_t tiles = seen / kPT + 2;
  // As many splits as run at once, two workgroups a CU (head dim 512: one); one
  // more is a second turn (6 chunks of up to 300 tokens under a window: 5 splits
  // 45 us, 6 55).  Sequences of few rows beside them take up to half of the
  // places (a prompt of 512 tokens at 2000 positions beside 60 tokens at up to
  // 4000: f16 120 us with 14 splits, 101 with 7; 4 bits 82 and 63), but not
  // so many that a workgroup has more than 64 tiles and outlasts them (2 x 1024
  // tokens at 4096 beside 120: 4 bits 268 us with 1 split, 156 with 3).
  const int64_t places = hd == 512 ? 256 : 512, units_of = std::max<int64_t>(1, work * a.P.kvh);
  const int64_t beside = a.few_rows ? std::min<int64_t>(places / 2, 4 * (a.P.n_seq - longest) * a.P.kvh) : 0;
  const int64_t fit = std::max((places - beside) / units_of, std::min((tiles + 63) / 64, places / units_of));
  const int64_t ns = std::min<int64_t>(fit, tiles / kMinTiles);
  a.ns = (int)std::max<int64_t>(1, std::min<int64_t>(ns, 64));
  a.part_floats = a.ns > 1 ? (size_t)units * a.ns * bm * hd : 0;
  a.ml_floats = a.ns > 1 ? (size_t)units * a.ns * bm * 2 : 0;
}

int launch_attn_paged_chunk(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st) {
#define CHUNK(HD) \
  if (hd == HD) return q16 ? chunk_hd<HD, true>(a, q4, st) : chunk_hd<HD, false>(a, q4, st);
  CHUNK(128)
  CHUNK(256)
  CHUNK(512)
#undef CHUNK
  return e4b_fail(E4B_EINVAL, "e4b_k_attn_paged: head_dim %d", hd);
}
