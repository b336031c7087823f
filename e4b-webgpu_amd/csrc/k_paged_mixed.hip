// k_paged_mixed.hip -- attention of a batch with chunks and with sequences of a
// few rows over the paged cache: both kinds of workgroups in one launch, both
// merges in another.  One behind the other, decoded tokens waited for the
// prompts beside them.  Head dim 256, 2 KV heads of 4 query heads, two launches
// of each kind and these: a prompt of 512 tokens and 30 tokens at up to 2000
// positions, f16 51 and 33 us, 4 bits 55 and 35; 2 chunks of 1024 tokens and 120
// tokens at up to 4000, f16 252 and 205; 6 chunks alone, 4 bits, 107 and 80.
// Head dim 128, 8 KV heads, 200 tokens and a chunk of 256, 4 bits: 164 and 160
// (the tokens' workgroups have the chunks' registers here, two on a CU).
#include "paged_chunk.h"
#include "paged_few.h"

namespace {

struct MixedArgs {
  PagedAttnArgs chunk, few;
  int n_chunk;  // workgroups of the chunks, which come first: they take the longest
};

template <int HD, bool Q4, bool Q16>
__global__ __launch_bounds__(64 * kChunkWaves<HD>, 2) void k_attn_paged_mixed(MixedArgs M) {
  __shared__ __align__(16) uint4 lds[kChunkLds<HD, Q4> / 16];
  if ((int)blockIdx.x < M.n_chunk)
    attn_chunk<HD, Q4, Q16>(M.chunk, blockIdx.x, M.n_chunk, lds);
  else
    attn_few<HD, Q4, Q16, kChunkWaves<HD>>(M.few, blockIdx.x - M.n_chunk, reinterpret_cast<float*>(lds));
}
template <int HD, bool Q16>
__global__ __launch_bounds__(256) void k_attn_mixed_merge(MixedArgs M) {
  if ((int)blockIdx.x < M.n_chunk)
    merge_chunk<HD, Q16>(M.chunk, blockIdx.x);
  else
    merge_few<HD, HD>(M.few, blockIdx.x - M.n_chunk, 0);
}

template <int HD, bool Q16>
int mixed_hd(const PagedAttnArgs& chunk, const PagedAttnArgs& few, bool q4, hipStream_t st) {
  static_assert(few_lds<HD, kChunkWaves<HD>>(kRows) <= kChunkLds<HD, false>, "a workgroup of either kind has the chunks' LDS");
  MixedArgs m{chunk, few, (int)chunk_grid<HD, Q16>(chunk)};
  const unsigned grid = (unsigned)(m.n_chunk + few.groups);
  if (q4)
    k_attn_paged_mixed<HD, true, Q16><<<grid, 64 * kChunkWaves<HD>, 0, st>>>(m);
  else
    k_attn_paged_mixed<HD, false, Q16><<<grid, 64 * kChunkWaves<HD>, 0, st>>>(m);
  E4B_HIP(hipGetLastError());
  m.n_chunk = (int)chunk_merge_grid<HD, Q16>(chunk);
  const unsigned merge = (unsigned)(m.n_chunk + (few.split ? few_units(few) * few_unit_rows(few) : 0));
  if (!merge) return E4B_OK;
  k_attn_mixed_merge<HD, Q16><<<merge, 256, 0, st>>>(m);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

int launch_attn_paged_mixed(const PagedAttnArgs& chunk, const PagedAttnArgs& few, int hd, bool q4, bool q16,
                            hipStream_t st) {
#define MIXED(HD) \
  if (hd == HD) return q16 ? mixed_hd<HD, true>(chunk, few, q4, st) : mixed_hd<HD, false>(chunk, few, q4, st);
  MIXED(128)
  MIXED(256)
  MIXED(512)
#undef MIXED
  return e4b_fail(E4B_EINVAL, "e4b_k_attn_paged: head_dim %d", hd);
}
