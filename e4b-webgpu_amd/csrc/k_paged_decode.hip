// k_paged_decode.hip -- launches of the attention of a few query rows per KV
// head over the paged cache (paged_few.h).
#include "paged_few.h"

namespace {

template <int HD, bool Q4, bool Q16, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_paged_few(PagedAttnArgs A) {
  extern __shared__ __align__(16) float lds[];
  attn_few<HD, Q4, Q16, NW>(A, blockIdx.x, lds);
}
template <int HD, int DW>
__global__ __launch_bounds__(256) void k_attn_paged_merge(PagedAttnArgs A) {
  merge_few<HD, DW>(A, blockIdx.x, blockIdx.y);
}

template <int HD, int NW>
int few_waves(const PagedAttnArgs& a, bool q4, bool q16, hipStream_t st) {
  const size_t lds = few_lds<HD, NW>(few_unit_rows(a));
  const dim3 grid((unsigned)a.groups);
  auto go = [&](auto* kernel) {
    // (more than 64 KB of LDS has to be asked for; 67 KB at most here)
    if (lds > 65536)
      E4B_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<grid, 64 * NW, lds, st>>>(a);
    E4B_HIP(hipGetLastError());
    return E4B_OK;
  };
  return q4 && q16 ? go(k_attn_paged_few<HD, true, true, NW>)
         : q4      ? go(k_attn_paged_few<HD, true, false, NW>)
         : q16     ? go(k_attn_paged_few<HD, false, true, NW>)
                   : go(k_attn_paged_few<HD, false, false, NW>);
}

template <int HD>
int few_hd(const PagedAttnArgs& a, bool q4, bool q16, hipStream_t st) {
  const int nr = few_unit_rows(a), units = few_units(a);
  // Two units a CU or more: workgroups of 4 waves, two on a CU, one's first
  // loads and merge beside the other's tiles (200 ragged sequences of up to 500
  // positions, 8 KV heads of 128: f16 67 us with 8 waves, 53 with 4; 4 bits 49
  // and 30).  Fewer units than that leave CUs with one workgroup (128 sequences
  // of up to 2000 positions, 2 KV heads of 256, f16: 70 and 78).
  const int rc = units >= 2 * kGroups ? few_waves<HD, 4>(a, q4, q16, st) : few_waves<HD, 8>(a, q4, q16, st);
  if (rc || !a.split) return rc;
  if (few_merge_wide(a))
    k_attn_paged_merge<HD, 64><<<dim3(units * nr, HD / 64), 256, 0, st>>>(a);
  else
    k_attn_paged_merge<HD, HD><<<units * nr, 256, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

void plan_attn_paged_few(PagedAttnArgs& a, int hd) {
  a.nrb = (a.max_q * a.gqa + kRows - 1) / kRows;
  const int units = a.P.n_seq * a.P.kvh * a.nrb;
  const int64_t seen = a.window ? std::min<int64_t>(a.max_kv, (int64_t)a.window + a.sinks + a.max_q) : a.max_kv;
  const int64_t tiles = seen / kPT + 2;
  // Where the units fill the CUs, splitting is for lengths that differ: from
  // 2048 keys on
  a.split = a.P.n_seq <= kSplitSeqs && (units < kGroups ? tiles > kUnsplit : tiles > 64);
  a.second = kRows / a.gqa;
  a.last[0] = (kRows - 1) / a.gqa;
  a.last[1] = (2 * kRows - 1) / a.gqa;
  a.target = std::max(units, kGroups);
  a.groups = !a.split ? units : units < kGroups ? kGroups : 2 * units;
  const int nr = std::min(a.max_q * a.gqa, kRows);
  a.part_floats = a.split ? (size_t)a.groups * nr * hd : 0;
  a.ml_floats = a.split ? (size_t)a.groups * nr * 2 : 0;
}

int launch_attn_paged_few(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st) {
  return hd == 128 ? few_hd<128>(a, q4, q16, st) : hd == 256 ? few_hd<256>(a, q4, q16, st) : few_hd<512>(a, q4, q16, st);
}
