// paged_attn.h -- what the attention kernels over the paged cache share: the
// tiles that a set of queries sees, and fragments of 4-bit rows as f16.
#pragma once
#include "paged.h"

#ifdef __HIPCC__
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

constexpr int kPT = 32;  // keys per tile: two 16-key halves, each inside one page

// a value that is the same in all lanes, in a scalar register (an integer
// division leaves it in a vector one, and what depends on it with it)
DEV int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// sums over the lanes up to this one
DEV int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: inside 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last lane of 16 to the next 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // and of 32 to the next 32
  return v;
}
DEV int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }

// Tiles of the keys that queries at positions p0 .. p1 see, in the order of
// the keys: `sink` tiles from 0 on, then the ones from `from` on.
struct TileRange {
  int sink, from, n;
  DEV int base(int t) const { return (t < sink ? t : t - sink + from) * kPT; }
};
DEV TileRange tile_range(int p0, int p1, int window, int sinks, int cap) {
  const int first = window > 0 ? max(0, max(0, p0) - window + 1) : 0;  // (p0 < 0: no key, and any window may be taken off 0)
  const int last = min(p1, cap - 1);
  TileRange r;
  r.from = first / kPT;
  r.sink = min((int)(((uint32_t)min(sinks, first) + kPT - 1) / kPT), r.from);
  r.n = last < 0 ? 0 : min(r.sink, last / kPT + 1) + max(0, last / kPT - r.from + 1);
  return r;
}
// positions that the table has entries for
DEV int paged_cap(const PagedArgs& P) {
  return (int)min((int64_t)P.table_stride << P.page_shift, (int64_t)0x7fffffff);
}
DEV bool key_seen(int key, int pos, int window, int sinks) {
  return key <= pos && (window == 0 || key > pos - window || key < sinks);
}

// Codes of a dword as f16 values: a pair of halves (code - 8), and all eight
// (code - 8) d with dims in order, d2 = (d, d).  A half 0x6400 | n is 1024 + n, one with n four bits up 1024 + 16 n: taking
// 1032 off, or 1/16 of it less 72, is exact.
DEV h2v q4_pair(uint32_t w, int i) {  // pair i = 0 .. 3, at bits 0, 8, 4, 12
  const h2v c = {(_Float16)1032.f, (_Float16)1032.f}, s = {(_Float16)0.0625f, (_Float16)0.0625f},
            e = {(_Float16)72.f, (_Float16)72.f};
  const uint32_t x = i & 1 ? w >> 8 : w;
  if (i < 2) return __builtin_bit_cast(h2v, (x & 0x000F000Fu) | 0x64006400u) - c;
  return __builtin_elementwise_fma(__builtin_bit_cast(h2v, (x & 0x00F000F0u) | 0x64006400u), s, -e);
}
DEV h2v h2_of(uint32_t w) { return __builtin_bit_cast(h2v, w); }
DEV uint32_t u_of(h2v v) { return __builtin_bit_cast(uint32_t, v); }
DEV h8v q4_frag(uint32_t w, h2v d2) {
  return __builtin_bit_cast(h8v, make_uint4(u_of(q4_pair(w, 0) * d2), u_of(q4_pair(w, 1) * d2), u_of(q4_pair(w, 2) * d2),
                                            u_of(q4_pair(w, 3) * d2)));
}
// halves 0 or 1 of two dwords side by side
DEV uint32_t lo_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
DEV uint32_t hi_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48
DEV float quad_max4(float v) {
  float t = v;
  swapx32(v, t);
  v = fmaxf(v, t);
  t = v;
  swapx16(v, t);
  return fmaxf(v, t);
}
DEV float quad_sum4(float v) { return xsum_step<16>(xsum_step<32>(v)); }
DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kNone = -3.0e38f;  // the running maximum before the first key
#endif
