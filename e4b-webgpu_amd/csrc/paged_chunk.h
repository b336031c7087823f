// paged_chunk.h -- attention of many query rows per KV head over the paged
// cache: prompts and their chunks (launches: k_paged_chunk.hip; beside
// sequences with few rows: k_paged_mixed.hip).
//
// Workgroup (tile of query rows of one sequence, KV head, split of the keys);
// a row is (token, head of the group), token major, so the heads that share
// K and V share a tile.  Key tiles of 32 are staged in LDS as f16, one tile
// ahead, in two buffers; each wave has F fragments of 16 columns, a fragment
// being 16 rows of f16 queries or 8 rows of f32 ones (high and low parts side
// by side, as in paged_few.h):
//   S^T (16 keys x 16 columns) = K . Q^T, K read row by row;
//   O^T (16 dims x 16 columns) += V^T . P^T, V^T read with the transposing
//   ds_read_b64_tr_b16, P as it lies in the registers after the softmax.
// A fragment of K or V (1 KB of LDS reads) feeds F products.
//
// What bounds it: the matrix units work for 40 % of the kernel's time and the
// waves issue for most of the rest -- the softmax's exponentials and
// conversions are 16 values a lane and tile beside 32 products, and 256
// registers a wave leave two waves a SIMD to hide them behind each other.  At
// head dim 256, 4 query heads a KV head, f16 queries: 8 sequences of 1024
// tokens at 4096 positions 257 us (0.94 PFLOP/s), 16 of them 504; 4 sequences
// with f32 queries 277 (each product twice); 4 bits 8 sequences 367 (a tile is
// turned into f16 by each workgroup that reads it).  Wider and narrower tiles
// (F 1 with 8 waves, F 1 with 4) were 1.1 to 1.4 times slower: fewer products
// for each fragment that LDS delivers.
#pragma once
#include <algorithm>

#include "../../include/e4b.h"
#include "paged_attn.h"
#include "util.h"

namespace {

typedef __fp16 tr4 __attribute__((__vector_size__(8)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) tr4 lds_tr4;

// head dim 512: one fragment (its output alone is 128 registers) and 8 waves,
// as LDS holds one workgroup's tiles
template <int HD>
constexpr int kFrags = HD == 512 ? 1 : 2;
template <int HD>
constexpr int kChunkWaves = HD == 512 ? 8 : 4;
template <int HD, bool Q16>
constexpr int kTileRows = kChunkWaves<HD> * kFrags<HD> * (Q16 ? 16 : 8);

// The sequence and its tile that tile number `at` of the whole batch is; the
// sequences that paged_few.h takes have none.  Later tiles first: they
// see the most keys.
struct TileAt {
  int seq, tile;
  SeqSpan s;
};
DEV TileAt find_tile(const PagedAttnArgs& A, int rows_per, int at) {
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x & 63;
  int ahead[3];
  auto load = [&](int b) {  // (all at once, and one round ahead: each is a trip to memory)
    const int i = min(b + lane, P.n_seq - 1);
    ahead[0] = P.q_start[i];
    ahead[1] = P.q_start[i + 1];
    ahead[2] = P.kv_len[i];
  };
  load(0);
  for (int b = 0; b < P.n_seq; b += 64) {
    const int start = ahead[0], end = ahead[1], kv = ahead[2];
    if (b + 64 < P.n_seq) load(b + 64);
    const int rows = seq_span_of(P, start, end, kv).n * A.gqa;
    const int n = b + lane >= P.n_seq || rows <= A.few_rows ? 0 : (rows + rows_per - 1) / rows_per;
    const int upto = wave_scan(n);
    const uint64_t past = __ballot(at < upto);
    if (past) {
      const int f = __builtin_ctzll(past);
      return {b + f, __builtin_amdgcn_readlane(upto, f) - 1 - at,
              seq_span_of(P, __builtin_amdgcn_readlane(start, f), __builtin_amdgcn_readlane(end, f),
                          __builtin_amdgcn_readlane(kv, f))};
    }
    at -= last_lane(upto);
  }
  return {-1, 0, {}};
}

// key tiles of a split at least (6 tokens at 4096 positions 24.6 us with 8, 21.1
// with 4, 20.3 with 3; 100 at 600 28.1, 20.8, 21.1; 300 at 4096 the same)
constexpr int kMinTiles = 4;
DEV int chunk_per(int n, int ns) { return max(kMinTiles, uni((n + ns - 1) / ns)); }

// what the wave's lanes wrote to LDS is there for all of them
DEV void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// whether one of two f16 values is not finite
DEV bool not_finite(uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; }
// dim d of a row
template <int HD, bool Q4>
DEV float cache_value(const uint8_t* block, int row, int d, int page_shift) {
  if constexpr (Q4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(block + row * (HD / 2) + d / 8 * 4);
    const int pr = d % 8 / 2;
    const int n = (int)(w >> (((pr & 1) << 3) + ((pr & 2) << 1) + 16 * (d & 1)) & 15) - 8;
    return n * h2f(*reinterpret_cast<const uint16_t*>(block + (HD / 2 << page_shift) + row * (HD / 16) + d / 32 * 2));
  } else {
    return h2f(reinterpret_cast<const uint16_t*>(block)[row * HD + d]);
  }
}

// 16-byte piece `p` of row r (of 16) of a tile in LDS.  Rows are whole rounds of
// the banks apart, so the pieces are moved by the row: the 16 rows of a K
// fragment to 16 places, and of a V fragment (two pieces side by side of each
// row, 8 rows at a time) to 8 pairs of places.
DEV int piece(int r, int p) { return p ^ ((r & 7) << 1 | (r >> 3 & 1)); }

// Query fragments that LDS keeps for a wave: 256 registers do not hold all of
// them beside the output, and the reload of one that the compiler has moved to
// scratch memory waits for the loads of the next tile before it (8 sequences
// of 1024 tokens at 4096 positions, f16: none 290 us, 2 275; 4 bits, whose
// tile's codes wait in registers too: none 376, 2 357, 3 355, and a ragged batch of
// chunks under a window 55.6, 51.7, 51.0).  More would not leave room for two
// workgroups on a CU.
template <int HD, bool Q4>
constexpr int kQLds = HD == 128 ? 0 : Q4 ? 3 : 2;
// bytes of LDS of a workgroup: two buffers of a K and a V tile, a mark, queries
template <int HD, bool Q4>
constexpr int kChunkLds = (4 * kPT * (HD / 8) + 1 + kChunkWaves<HD> * kQLds<HD, Q4> * 64) * 16;

// Workgroup `block` of `grid`, kChunkWaves<HD> waves
template <int HD, bool Q4, bool Q16>
DEV void attn_chunk(const PagedAttnArgs& A, int block, int grid, uint4* lds) {
  constexpr int F = kFrags<HD>, NW = kChunkWaves<HD>, BM = kTileRows<HD, Q16>, RF = Q16 ? 16 : 8;
  // fragments of K and V that are read ahead of their products; 4-bit tiles need
  // the registers on their way (f32 queries of f16 310 us with 2, 301 with 3;
  // 8 sequences of 4 bits 380 and 390)
  constexpr int kAhead = Q4 ? 2 : 3, kAheadV = Q4 ? 2 : 3;
  constexpr int QS = HD / 32, DT = HD / 16, KP = HD / 8, TP = kPT * KP;  // TP: 16-byte pieces of a K or V tile
  // lds: two buffers of a K and a V tile, and the mark of a broken cache.  One
  // array: beside a second LDS variable the compiler drops what it knows of the two
  // buffers (below) and waits for the copies into one at each read of the other.
  auto buf_of = [&](int n) { return lds + (n & 1) * 2 * TP; };
  uint32_t* mark = reinterpret_cast<uint32_t*>(lds + 4 * TP);
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g4 = lane >> 4;
  // Workgroups n and n + 256 share a CU while the first 512 start, and tiles go
  // from the most keys to the fewest along a sequence: the second 256 in
  // reverse put long beside short (8 x 1024 tokens at 4096 positions: 267 us
  // without, 257 with; 8 ragged prompts of up to 2048 tokens: 126 and 132).
  int unit = block;
  if (unit >> 8 == 1) unit = 256 + min(512, grid) - 1 - unit;
  const int sp = unit % A.ns, g = unit / A.ns % P.kvh, at = unit / A.ns / P.kvh;
  const TileAt ta = find_tile(A, BM, at);
  const int i = __builtin_amdgcn_readfirstlane(ta.seq), qt = __builtin_amdgcn_readfirstlane(ta.tile);
  if (i < 0) return;
  const SeqSpan s = ta.s;
  const int rows = s.n * A.gqa;
  const int t0 = qt * BM, t1 = min(t0 + BM, rows);  // rows of the tile
  const int cap = paged_cap(P);
  // their positions (the first that there can be: a window is taken off it)
  const int pa = max(0, s.p0 + uni(t0 / A.gqa)), pb = s.p0 + uni((t1 - 1) / A.gqa);
  const TileRange R = tile_range(pa, pb, A.window, A.sinks, cap);
  const int per = chunk_per(R.n, A.ns), live = uni((R.n + per - 1) / per);  // tiles of a split, splits that have any
  const int n_tiles = max(0, min(per, R.n - sp * per)), first = sp * per;
  if (n_tiles == 0 && !(sp == 0 && R.n == 0)) return;

  // this wave's rows, and this lane's column of each fragment
  const int w0 = t0 + wave * F * RF, w1 = min(w0 + F * RF, t1);
  const bool any = w0 < t1;
  const int wp0 = max(0, s.p0 + uni(min(w0, rows - 1) / A.gqa)), wp1 = s.p0 + uni((max(w1, 1) - 1) / A.gqa);
  int tok[F];
#pragma unroll
  for (int f = 0; f < F; ++f) tok[f] = min(w0 + f * RF + (c & (RF - 1)), rows - 1) / A.gqa;
  // the column's row: whether there is one, and its head
  auto row_of = [&](int f, bool& have) {
    const int r = w0 + f * RF + (c & (RF - 1)), rc = min(r, rows - 1);
    have = r < t1;
    return g * A.gqa + rc - rc / A.gqa * A.gqa;
  };

  // ---- staging ----
  struct Half {  // 16 keys: their page's blocks and the first row there
    const uint8_t *k, *v;
    int row;
    bool there;
  };
  // The table's entries for a tile are asked for two tiles ahead, with vector
  // loads that come back in order with the rows': no wait of their own.
  const uint32_t* tab = P.table + (int64_t)i * P.table_stride;
  auto ask = [&](int n, uint32_t(&pg)[2]) __attribute__((always_inline)) {
    const int kb = R.base(first + min(n, n_tiles - 1));
#pragma unroll
    for (int u = 0; u < 2; ++u) pg[u] = tab[min((kb + 16 * u) >> P.page_shift, P.table_stride - 1)];
  };
  auto half_of = [&](int kb, int u, uint32_t entry) __attribute__((always_inline)) {
    const int p = kb + 16 * u;
    const uint32_t pg = uni(entry);
    const bool there = (p >> P.page_shift) < P.table_stride && pg < (uint32_t)P.n_pages;
    const int64_t blk = paged_block<Q4, HD>(P, there ? (int)pg : 0, g);
    return Half{P.k + blk, P.v + blk, p & ((1 << P.page_shift) - 1), there};
  };
  auto second_half = [&](Half h, int kb, uint32_t entry) __attribute__((always_inline)) {
    if (P.page_shift < 5) return half_of(kb, 1, entry);
    h.row += 16;  // both halves of a tile are in one page
    return h;
  };
  // f16: rows go straight into LDS, 1 KB a wave at a time
  constexpr int RI = 1024 / (2 * HD);             // rows of a copy
  constexpr int HC = 16 / RI / NW;                // copies of a wave for a half of K or V
  static_assert(HC * NW * RI == 16, "the waves share a half evenly");
  int from[HC];
#pragma unroll
  for (int j = 0; j < HC; ++j) {
    const int r = (j * NW + wave) * RI + lane / KP, p = lane % KP;
    from[j] = r * (2 * HD) + piece(r, p) * 16;
  }
  auto copy16 = [](const uint8_t* base, uint4* dst, int lane_off, int off) __attribute__((always_inline)) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0xffffffffu, 0x00020000), (lds_void*)dst, 16, lane_off, off, 0, 0);
  };
  constexpr int NC = 4 * HC;  // copies of a wave for a tile
  auto copy = [&](uint4* buf, Half H0, Half H1, int n) __attribute__((always_inline)) {  // number n of them
    const int u = n / HC % 2, j = n % HC;
    const Half H = u ? H1 : H0;
    uint4* dst = buf + u * 16 * KP + (j * NW + wave) * 64;
    if (n < 2 * HC)
      copy16(H.k, dst, from[j], H.row * (2 * HD));
    else
      copy16(H.v, dst + TP, from[j], H.row * (2 * HD));
  };
  // 4 bits: a thread takes 32 dims of a row (16 bytes of codes and their
  // scale) into registers one tile ahead and writes them to LDS as f16
  constexpr int ST = 2 * kPT * (HD / 32) / (64 * NW);  // blocks of a thread: K's first, then V's
  uint4 codes[ST];
  uint32_t scales[ST];
  auto fetch = [&](Half H0, Half H1) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < ST; ++j) {
      const int n = j * 64 * NW + threadIdx.x, r = n / (HD / 32) % kPT, b = n % (HD / 32);
      const bool isv = n >= kPT * (HD / 32);
      const uint8_t* base = r < 16 ? (isv ? H0.v : H0.k) : (isv ? H1.v : H1.k);
      const uint32_t row = (r < 16 ? H0.row : H1.row) + (r & 15);
      codes[j] = *reinterpret_cast<const uint4*>(base + (row * (HD / 2) + b * 16));
      scales[j] = *reinterpret_cast<const uint16_t*>(base + ((HD / 2 << P.page_shift) + row * (HD / 16) + b * 2));
    }
  };
  auto unpack = [&](uint4* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < ST; ++j) {
      const int n = j * 64 * NW + threadIdx.x, r = n / (HD / 32) % kPT, b = n % (HD / 32);
      const bool isv = n >= kPT * (HD / 32);
      const h2v d2 = h2_of(scales[j] | scales[j] << 16);
      const uint32_t w[4] = {codes[j].x, codes[j].y, codes[j].z, codes[j].w};
      uint4* row = buf + (isv ? TP : 0) + r * KP;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = 4 * b + k;
        row[piece(r & 15, p)] = __builtin_bit_cast(uint4, q4_frag(w[k], d2));
      }
    }
  };

  if (threadIdx.x == 0) *mark = 0;  // (a barrier comes before its first use)
  uint32_t entry[2];  // of the tile behind the one that is staged
  uint32_t there = 0, there_next = 0;
  if (n_tiles > 0) {
    ask(0, entry);
    const Half H0 = half_of(R.base(first), 0, entry[0]), H1 = second_half(H0, R.base(first), entry[1]);
    there_next = (H0.there ? 1u : 0u) | (H1.there ? 2u : 0u);
    if constexpr (Q4) {
      fetch(H0, H1);
    } else {
#pragma unroll
      for (int n = 0; n < NC; ++n) copy(buf_of(0), H0, H1, n);
    }
    ask(1, entry);
  }
  // Q^T: dims 32 k + 8 g4 .. + 7
  // step by step (number k F + f): 0 .. QL - 1 in LDS, the others in registers
  constexpr int QL = kQLds<HD, Q4>;
  h8v q[F * QS - QL];
  uint4* q_lds = lds + 4 * TP + 1 + wave * (QL * 64) + lane;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    bool have;
    const int64_t q_at = (int64_t)(s.q0 + tok[f]) * A.q_stride + row_of(f, have) * HD;
#pragma unroll
    for (int k = 0; k < QS; ++k) {
      const int64_t a = q_at + k * 32 + g4 * 8;
      h8v x;
      if constexpr (Q16) {
        x = *reinterpret_cast<const h8v*>((const uint16_t*)A.q + a);
        if (A.scale < 0.f) x = -x;
      } else {
        const float4 v0 = *reinterpret_cast<const float4*>((const float*)A.q + a);
        const float4 v1 = *reinterpret_cast<const float4*>((const float*)A.q + a + 4);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float y = A.scale < 0.f ? -v[t] : v[t];
          const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
          x[t] = c < 8 ? hi : lo;
        }
      }
      if (k * F + f < QL)
        q_lds[(k * F + f) * 64] = __builtin_bit_cast(uint4, x);
      else
        q[k * F + f - QL] = x;
    }
  }
  f4v o[F][DT];
  float m[F], l[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    m[f] = kNone;
    l[f] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[f][d] = f4v{0.f, 0.f, 0.f, 0.f};
  }
  // scores are taken in powers of 2; the sign of a negative scale is the
  // queries', and a scale of 0 is next to it (a masked score times it is -inf)
  const float scale2 = fmaxf(fabsf(A.scale) * 1.44269504088896341f, 1e-37f);
  // Byte offsets in a tile of this lane's part of K row c, dims 8 g4, and of V
  // row 4 g4 + c / 4, dims 4 (c % 4); other dims are an xor away.  Kept from the
  // compiler's view in the loop: the 24 sums would be held in registers.
  const int vrow = 4 * g4 + (c >> 2);
  int kx = (c * KP + piece(c, g4)) * 16, vx = (vrow * KP + piece(vrow, (c & 3) >> 1)) * 16 + (c & 1) * 8;

  // scores of this wave's columns with the keys of a tile
  // (`beside`: what else is issued in its steps, one call a step)
  auto scores = [&](const uint4* buf, uint4* ahead, const h8v(&q0)[QL + 1], f4v(&sc)[F][2], auto beside) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < F; ++f) sc[f][0] = sc[f][1] = f4v{0.f, 0.f, 0.f, 0.f};
    h8v ka[kAhead + 1];  // fragments in flight: step k, half u is number 2 k + u
    auto ld_k = [&](int n) __attribute__((always_inline)) {
      ka[n % (kAhead + 1)] = *reinterpret_cast<const h8v*>(
          reinterpret_cast<const char*>(buf + 16 * (n & 1) * KP) + (kx ^ (64 * (n >> 1))));
    };
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ld_k(n);
#pragma unroll
    for (int n = 0; n < 2 * QS; ++n) {
      if (n + kAhead < 2 * QS) ld_k(n + kAhead);
      if (n & 1) beside(ahead, n >> 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < F; ++f)
        sc[f][n & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[n % (kAhead + 1)], (n >> 1) * F + f < QL ? q0[(n >> 1) * F + f] : q[(n >> 1) * F + f - QL], sc[f][n & 1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = sc[f][j >> 2][j & 3];
        if constexpr (!Q16) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));
        sc[f][j >> 2][j & 3] = x;
      }
  };
  auto mask_scores = [&](int kb, uint32_t there, f4v(&sc)[F][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 16 * (j >> 2) + 4 * g4 + (j & 3);
        const bool on = (there >> (j >> 2) & 1) && key < cap && key_seen(key, s.p0 + tok[f], A.window, A.sinks);
        sc[f][j >> 2][j & 3] = on ? sc[f][j >> 2][j & 3] : -__builtin_inff();
      }
  };
  // weights exp2(score - m) as the B operand
  auto weight = [&](int f, int j, float e, h8v& pf) __attribute__((always_inline)) {
    const _Float16 hi = (_Float16)e;
    if constexpr (Q16) {
      pf[j] = hi;
    } else {
      const _Float16 lo = (_Float16)(e - (float)hi);
      pf[j] = c < 8 ? hi : lo;
    }
  };
  // V^T rows 16 d + c, keys 4 g4 .. + 3 of both halves
  auto ld_v = [&](const uint4* buf, int d) __attribute__((always_inline)) {
    u2v x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      x[u] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4*)(
                                         reinterpret_cast<const char*>(buf + TP + 16 * u * KP) + (vx ^ (32 * d)))));
    return __builtin_bit_cast(h8v, make_uint4(x[0].x, x[0].y, x[1].x, x[1].y));
  };
  auto tile = [&](const uint4* buf, uint4* ahead, const h8v(&q0)[QL + 1], int kb, bool whole, uint32_t there, auto beside) __attribute__((always_inline)) {
    f4v sc[F][2];
    scores(buf, ahead, q0, sc, beside);
    if (!whole) mask_scores(kb, there, sc);
    h8v vf[kAheadV + 1];
#pragma unroll
    for (int d = 0; d < kAheadV; ++d) vf[d] = ld_v(buf, d);
    h8v pf[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      float top = kNone;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[f][j >> 2][j & 3]);
      top = quad_max4(top) * scale2;
      if (__any(top > m[f] + 8.f)) {
        const float mn = fmaxf(m[f], top), a = exp2_(m[f] - mn);
        m[f] = mn;
        l[f] *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[f][d] *= a;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = exp2_(fmaf(sc[f][j >> 2][j & 3], scale2, -m[f]));
        l[f] += e;
        weight(f, j, e, pf[f]);
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (d + kAheadV < DT) vf[(d + kAheadV) % (kAheadV + 1)] = ld_v(buf, d + kAheadV);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < F; ++f)
        o[f][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d % (kAheadV + 1)], pf[f], o[f][d], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // every row of p0 .. p1 sees the whole tile
  auto all_see = [&](int kb, uint32_t there, int p0, int p1) {
    return there == 3 && kb + kPT - 1 <= p0 && (A.window == 0 || kb > p1 - A.window || kb + kPT <= A.sinks);
  };
  // A row of V that a query does not see must not reach its output even as
  // 0 x infinity.  In a tile that some query does not see all of, rows that none
  // of them sees become zeros; true where another one holds a value that is not
  // finite, in this tile or one before.  The whole workgroup calls it.
  auto clean = [&](uint4* buf, int kb, uint32_t there) {
    bool found = false;
#pragma unroll 1
    for (int j = threadIdx.x; j < TP; j += 64 * NW) {
      const int r = j / KP, key = kb + r;
      const bool used = (there >> (r >> 4) & 1) && key < cap && key <= pb &&
                        (A.window == 0 || key > pa - A.window || key < A.sinks);
      const uint4 x = buf[TP + j];
      if (!used)
        buf[TP + j] = make_uint4(0, 0, 0, 0);
      else
        found = found || not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
    }
    if (found) *mark = 1;
    lds_sync();
    return uni(*mark) != 0;
  };
  bool odd = false;
  for (int n = 0; n < n_tiles; ++n) {
    const int kb = R.base(first + n);
    uint4* buf = buf_of(n);
    asm volatile("" : "+v"(kx), "+v"(vx));
    h8v q0[QL + 1];  // (read before the wait for the tile)
#pragma unroll
    for (int k = 0; k < QL; ++k) q0[k] = __builtin_bit_cast(h8v, q_lds[k * 64]);
    there = there_next;
    const bool more = n + 1 < n_tiles;
    const int kb1 = R.base(first + n + (more ? 1 : 0));
    if constexpr (Q4) {
      unpack(buf);
    } else {
      // every wave's copies of this tile have landed, and every wave is done
      // with the buffer that the next ones overwrite
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      lds_sync();
    }
    const Half H0 = half_of(kb1, 0, entry[0]), H1 = second_half(H0, kb1, entry[1]);
    there_next = (H0.there ? 1u : 0u) | (H1.there ? 2u : 0u);
    if constexpr (Q4) {
      if (more) {
        fetch(H0, H1);
        ask(n + 2, entry);
      }
      lds_sync();
    }
    // what the workgroup's rows, and what this wave's, see of it
    if (!all_see(kb, there, pa, pb)) odd = clean(buf, kb, there);
    const bool past = kb > wp1, before = A.window > 0 && kb + kPT - 1 <= wp0 - A.window && kb >= A.sinks;
    // the next tile's copies go out between the products (one behind the other
    // they hold up the wave for 500 clocks); the last tile's are its own again
    auto beside = [&](uint4* ahead, int k) __attribute__((always_inline)) {
      if constexpr (!Q4) {
#pragma unroll
        for (int j = k * NC / QS; j < (k + 1) * NC / QS; ++j) copy(ahead, H0, H1, j);
        if (k == QS - 1) ask(n + 2, entry);
      }
    };
    // (no alias between the two buffers: a copy into one needs no wait before the reads of the other)
    auto step = [&](const uint4* __restrict__ cur, uint4* __restrict__ ahead) __attribute__((always_inline)) {
      int sees = uni(any && !past && !before);
      if (!sees) {
#pragma unroll
        for (int k = 0; k < QS; ++k) beside(ahead, k);
      }
      asm volatile("" : "+v"(sees));  // (joined with the branch above, it keeps two copies of the outputs)
      if (uni(sees)) tile(cur, ahead, q0, kb, all_see(kb, there, wp0, wp1), there, beside);
    };
    step(buf, buf_of(n + 1));
  }
  if (odd) {
    // (a broken cache) Row by row and key by key, a wave a row, from memory
    for (int r = t0 + wave; r < t1; r += NW) {
      const int t = r / A.gqa, h = g * A.gqa + r % A.gqa, pos = s.p0 + t;
      constexpr int E = HD / 64;
      float x[E], y[E], m1 = kNone, l1 = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t qa = (int64_t)(s.q0 + t) * A.q_stride + h * HD + E * lane + e;
        x[e] = Q16 ? h2f(((const uint16_t*)A.q)[qa]) : ((const float*)A.q)[qa];
        y[e] = 0.f;
      }
      for (int n = 0; n < n_tiles; ++n)
        for (int key = R.base(first + n), end = key + kPT; key < end; ++key) {
          const Half H = half_of(key & ~15, 0, tab[min(key >> P.page_shift, P.table_stride - 1)]);
          if (!H.there || key >= cap || !key_seen(key, pos, A.window, A.sinks)) continue;
          float sc = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) sc = fmaf(x[e], cache_value<HD, Q4>(H.k, H.row + (key & 15), E * lane + e, P.page_shift), sc);
          sc = wave_sum(sc) * A.scale * 1.44269504088896341f;
          const float mn = fmaxf(m1, sc), f = exp2_(m1 - mn), w = exp2_(sc - mn);
          m1 = mn;
          l1 = l1 * f + w;
#pragma unroll
          for (int e = 0; e < E; ++e) y[e] = y[e] * f + w * cache_value<HD, Q4>(H.v, H.row + (key & 15), E * lane + e, P.page_shift);
        }
      const int64_t row = ((int64_t)(at * P.kvh + g) * A.ns + sp) * BM + (r - t0);
      const float inv = l1 == 0.f ? 0.f : 1.f / l1;
      if (live > 1 && lane == 0) *reinterpret_cast<float2*>(A.part_ml + row * 2) = make_float2(m1, l1);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (live > 1)
          A.part[row * HD + E * lane + e] = y[e];
        else
          A.out[(int64_t)(s.q0 + t) * A.out_stride + h * HD + E * lane + e] = f2h(y[e] * inv);
      }
    }
    return;
  }

  // ---- results ----
  // A register's columns are 16 rows: stored from there, each store would touch
  // 16 of them, 32 or 64 bytes each.  Through LDS (DC dims of a fragment in the
  // wave's part of the tiles' buffers) whole rows are stored, 1 KB at a time.
  constexpr int DC = HD < 256 ? HD : 256, RP = DC / 4;  // RP: 16-byte pieces of a row
  static_assert(NW * 16 * RP == 4 * TP, "the waves' parts are the buffers");
  if constexpr (!Q4) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the copies behind the last tile have landed
  lds_sync();
  f4v* mine = reinterpret_cast<f4v*>(lds) + wave * 16 * RP;
  const bool direct = live <= 1;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const float L = quad_sum4(l[f]);
    bool have;
    const int head = row_of(f, have);
    const float inv = !direct ? 1.f : L == 0.f ? 0.f : 1.f / L;
    const int r0 = w0 + f * RF;  // rows of the fragment that there are: r0 .. r0 + n - 1
    const int n = min(RF, t1 - r0);
    const int64_t out_at = (int64_t)(s.q0 + tok[f]) * A.out_stride + head * HD;  // of this lane's column
    const int64_t part_row = ((int64_t)(at * P.kvh + g) * A.ns + sp) * BM + r0 - t0;
    if (!direct && have && lane < RF) *reinterpret_cast<float2*>(A.part_ml + (part_row + lane) * 2) = make_float2(m[f], L);
#pragma unroll
    for (int h = 0; h < HD / DC; ++h) {
#pragma unroll
      for (int d = 0; d < DC / 16; ++d) {
        f4v x = o[f][h * (DC / 16) + d];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (!Q16) x[r] += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x[r]), 0x128, 0xf, 0xf, true));
          x[r] *= inv;
        }
        if (c < RF) mine[c * RP + ((4 * d + g4) ^ c)] = x;
      }
      wave_fence();
      if (direct) {
        constexpr int PL = RP / 2, RI2 = 64 / PL;  // lanes of a row (8 dims each), rows at a time
#pragma unroll
        for (int k = 0; k < RF; k += RI2) {
          const int r = k + lane / PL, e = lane % PL;
          const int64_t to = (int64_t)__shfl((int)(out_at >> 32), r, 64) << 32 | (uint32_t)__shfl((int)out_at, r, 64);
          const f4v x = mine[r * RP + ((2 * e) ^ r)], y = mine[r * RP + ((2 * e + 1) ^ r)];
          if (r < n)
            *reinterpret_cast<uint4*>(A.out + to + h * DC + 8 * e) =
                make_uint4((uint32_t)f2h(x[0]) | (uint32_t)f2h(x[1]) << 16, (uint32_t)f2h(x[2]) | (uint32_t)f2h(x[3]) << 16,
                           (uint32_t)f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, (uint32_t)f2h(y[2]) | (uint32_t)f2h(y[3]) << 16);
        }
      } else {
        constexpr int RI2 = 64 / RP;
#pragma unroll
        for (int k = 0; k < RF; k += RI2) {
          const int r = k + lane / RP, e = lane % RP;
          if (r < n) *reinterpret_cast<f4v*>(A.part + (part_row + r) * HD + h * DC + 4 * e) = mine[r * RP + (e ^ r)];
        }
      }
      wave_fence();
    }
  }
}

// Merge of the splits: workgroup of 256 threads, HD / 4 of them a row
template <int HD, bool Q16>
DEV void merge_chunk(const PagedAttnArgs& A, int block) {
  constexpr int BM = kTileRows<HD, Q16>, T = HD / 4, RW = 256 / T;
  const PagedArgs& P = A.P;
  const int part = block % (BM / RW), g = block / (BM / RW) % P.kvh, at = block / (BM / RW) / P.kvh;
  const TileAt ta = find_tile(A, BM, at);
  const int i = __builtin_amdgcn_readfirstlane(ta.seq), qt = __builtin_amdgcn_readfirstlane(ta.tile);
  if (i < 0) return;
  const SeqSpan s = ta.s;
  const int rows = s.n * A.gqa, t0 = qt * BM, t1 = min(t0 + BM, rows);
  const TileRange R = tile_range(s.p0 + t0 / A.gqa, s.p0 + (t1 - 1) / A.gqa, A.window, A.sinks, paged_cap(P));
  const int per = chunk_per(R.n, A.ns), live = uni((R.n + per - 1) / per);
  const int r = part * RW + threadIdx.x / T, d = threadIdx.x % T * 4;
  if (live <= 1 || t0 + r >= t1) return;
  const int64_t row = (int64_t)(at * P.kvh + g) * A.ns * BM + r;  // + sp * BM
  // 4 splits at a time, the next ones' loads before these are added up
  float M = kNone, L = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y[4];
  float2 st[4];
  auto load = [&](int sp) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t p = row + (int64_t)min(sp + k, live - 1) * BM;
      st[k] = *reinterpret_cast<const float2*>(A.part_ml + p * 2);
      y[k] = *reinterpret_cast<const float4*>(A.part + p * HD + d);
    }
  };
  load(0);
  for (int sp = 0; sp < live; sp += 4) {
    float2 s4[4];
    float4 z[4];
    float top = M;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s4[k] = st[k];
      z[k] = y[k];
      top = fmaxf(top, st[k].x);  // (the last split again behind the last one)
    }
    if (sp + 4 < live) load(sp + 4);
    const float a = exp2_(M - top);
    M = top;
    L *= a;
    x.x *= a;
    x.y *= a;
    x.z *= a;
    x.w *= a;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = sp + k < live ? exp2_(s4[k].x - M) : 0.f;
      if (sp + k >= live) z[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      L += w * (sp + k < live ? s4[k].y : 0.f);
      x.x += w * z[k].x;
      x.y += w * z[k].y;
      x.z += w * z[k].z;
      x.w += w * z[k].w;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int rr = t0 + r, t = rr / A.gqa, h = g * A.gqa + rr % A.gqa;
  *reinterpret_cast<uint2*>(A.out + (int64_t)(s.q0 + t) * A.out_stride + h * HD + d) =
      make_uint2((uint32_t)f2h(x.x * inv) | (uint32_t)f2h(x.y * inv) << 16,
                 (uint32_t)f2h(x.z * inv) | (uint32_t)f2h(x.w * inv) << 16);
}

inline int tile_rows(int hd, bool q16) {
  return hd == 512 ? (q16 ? kTileRows<512, true> : kTileRows<512, false>)
                   : (q16 ? kTileRows<256, true> : kTileRows<256, false>);
}
// at most this many tiles: each sequence's last may be part full, and there
// are no more sequences than rows allow
inline int64_t tile_bound(const PagedAttnArgs& a, int bm) {
  const int64_t rows = (int64_t)a.P.n_tok * a.gqa;
  return rows / bm + std::min({(int64_t)a.P.n_seq, (int64_t)a.P.n_tok, rows / (a.few_rows + 1)});
}
// workgroups: of the attention, and of the merge (0: no split)
template <int HD, bool Q16>
int64_t chunk_grid(const PagedAttnArgs& a) {
  return tile_bound(a, kTileRows<HD, Q16>) * a.P.kvh * a.ns;
}
template <int HD, bool Q16>
int64_t chunk_merge_grid(const PagedAttnArgs& a) {
  constexpr int BM = kTileRows<HD, Q16>;
  return a.ns == 1 ? 0 : tile_bound(a, BM) * a.P.kvh * (BM / (1024 / HD));
}

}  // namespace
