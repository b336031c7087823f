// paged_few.h -- attention of a few query rows per KV head over the paged
// cache: decoded tokens (launches: k_paged_decode.hip; beside chunks:
// k_paged_mixed.hip).
//
// Unit (sequence, KV head, 8 query rows: tokens x heads of the group); its key
// tiles are cut into ns runs, one workgroup each, and inside it over the
// waves, every wave with a running maximum and sum of its own; the waves are
// merged in LDS, the runs by merge_few.
//
// v_mfma_f32_16x16x32_f16 (lane l, c = l % 16, g = l / 16: A[c][8g + t],
// B[8g + t][c], D[4g + r][c]):
//   S^T (16 keys x 16 columns) = K . Q^T; a lane loads its part of key row c
//   as it lies in memory.  8 rows fill half of the 16 columns, so every row
//   has two: an f32 query as f16 hi (column c) and lo (column c + 8), whose
//   scores are added, and the weights P the same way, whose outputs are added
//   at the end.  Both products are then as exact as f32 ones (2^-22) at no
//   cost in matrix instructions.
//   Each lane then holds the weights of its column for keys 4g + r of both
//   16-key halves: a B operand of the 32-key product O^T = V^T . P^T, when A
//   takes V in the same key order.  A lane loads 8 keys' rows 4g + r, 8 dims
//   of each, and turns them over in registers (one v_perm a pair): dims become
//   rows of A without a pass through LDS.
// What bounds it: in f16 the cache's bytes (64 tokens at 8192 positions, 2 KV
// heads of 256: 1.07 GB in 186 us, 5.8 TB/s; a tile of 32 keys is 32 KB in
// flight per wave); in 4 bits the unpacking (48 tokens at up to 4096, head dim
// 512: 130 MB in 47 us, VALU 55 % of the issue slots); few tokens latency (one
// at 300 positions 11.7 us).
#pragma once
#include <algorithm>

#include "../../include/e4b.h"
#include "paged_attn.h"
#include "util.h"

namespace {

constexpr int kRows = 8;
// Waves that share a tile.  Head dim 512 has no room for all of the output
// (128 registers) beside the rows in flight: two waves take half of the dims
// each, add up their halves of the scores through LDS, and keep half of V's.
template <int HD>
constexpr int kParts = HD / 256 > 1 ? 2 : 1;

// Splits.  A workgroup of 8 waves fills a CU, so there are about as many as CUs
// (one token at 32767 positions in 4 bits 15.7 us with 256 workgroups, 21.2
// with 512), dealt out by the sequences' lengths.  A split is a launch more (about
// 4 us), and what it saves is the time in which one CU takes in its share: none
// up to 7 tiles (one token at 128 positions 7.2 us in one workgroup, 9.0 in
// two), shares of 4 tiles above (at 300 positions 10.6 us, 12.9 in one
// workgroup; shares of 2 10.7 us).
constexpr int kMinShare = 4, kUnsplit = 7, kGroups = 256;
constexpr int kSplitSeqs = 256;  // sequences whose lengths a workgroup looks through

// rows and key tiles of block rb of sequence i (any i: by lanes)
struct Block {
  SeqSpan s;
  int rows, t_first, t_last;  // its tokens
  TileRange R;
};
DEV Block block_of(const PagedAttnArgs& A, const SeqSpan& s, int rb, int cap) {
  Block b;
  b.s = s;
  b.rows = (int64_t)s.n * A.gqa > kPagedFewRows ? 0  // paged_chunk.h's
                                                : max(0, min(min(s.n, A.max_q) * A.gqa - kRows * rb, kRows));
  b.t_first = rb ? A.second : 0;
  b.t_last = max(b.t_first, min(s.n - 1, rb ? A.last[1] : A.last[0]));
  b.R = tile_range(s.p0 + b.t_first, s.p0 + b.t_last, A.window, A.sinks, cap);
  return b;
}

// A unit (sequence, block of rows, KV head), and of its `live` splits number
// sp, the workgroup `first` + sp
struct Slot {
  int seq, rb, head, sp, live, first;
  SeqSpan s;
};
// Without splits workgroup and unit are the same.  Else a unit has a split for
// each `per` tiles (and takes even shares of its tiles), per being as small as
// leaves no more than A.groups workgroups in all, from the lengths of all
// sequences (a lane a sequence, 64 at a time; 131072 units at most).  The slot
// of workgroup `at`, or (by unit) of the unit `at` with sp = 0; seq < 0: there
// is none.
DEV int quotient(int a, int b) {  // a / b for a < 2^21: the error of (a + 1/2) / b in f32 is below 1 / (2 b)
  return uni((int)(((float)a + 0.5f) / (float)b));
}
DEV Slot find_slot(const PagedAttnArgs& A, int at, bool by_unit) {
  const PagedArgs& P = A.P;
  if (!A.split) {
    const int u = uni(at / A.nrb), i = uni(u / P.kvh);
    return {i, at - u * A.nrb, u - i * P.kvh, 0, 1, at, seq_span(P, i)};
  }
  constexpr int NC = kSplitSeqs / 64, NB = (kPagedFewRows + kRows - 1) / kRows;
  const int lane = threadIdx.x & 63, cap = paged_cap(P);
  int tiles[NC][NB];  // -1: no such block
  int start[NC], end[NC], kv[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int b = 0; b < NB; ++b) tiles[c][b] = -1;
  int sum = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (64 * c < P.n_seq) {
      const int i = min(64 * c + lane, P.n_seq - 1);
      start[c] = P.q_start[i];
      end[c] = P.q_start[i + 1];
      kv[c] = P.kv_len[i];
      const SeqSpan s = seq_span_of(P, start[c], end[c], kv[c]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const Block k = block_of(A, s, b, cap);
        if (64 * c + lane < P.n_seq && k.rows > 0) tiles[c][b] = k.R.n;
        sum += max(tiles[c][b], 0);
      }
    }
  // (t / per rounded up, or one more or less: every workgroup finds the same)
  auto splits = [&](int t, float by) {
    return t < 0 ? 0 : t <= kUnsplit ? 1 : max(1, min((int)((float)t * by + 0.999f), kPagedMaxSplits));
  };
  auto all = [&](float by) {
    int n = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (64 * c < P.n_seq)
#pragma unroll
        for (int b = 0; b < NB; ++b) n += splits(tiles[c][b], by);
    return last_lane(wave_scan(n)) * P.kvh;
  };
  const float share = (float)last_lane(wave_scan(min(sum, 1 << 24))) * (float)P.kvh / (float)A.target;
  float by = 1.f / fmaxf((float)kMinShare, share);  // splits a tile
#pragma unroll 1
  for (int k = 0; k < 4; ++k) {
    const int n = all(by);
    if (n <= A.groups) break;
    by = k == 3 ? 0.f : by * 0.99f * (float)A.groups / (float)n;
  }
  int before = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (64 * c < P.n_seq) {
      int n = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) n += splits(tiles[c][b], by);
      const int upto = before + wave_scan(n) * P.kvh;
      int f;
      if (by_unit) {
        const int i = quotient(at, A.nrb * P.kvh);
        if (i >= 64 * (c + 1)) {
          before = last_lane(upto);
          continue;
        }
        f = i - 64 * c;
      } else {
        const uint64_t past = __ballot(at < upto);
        if (!past) {
          before = last_lane(upto);
          continue;
        }
        f = __builtin_ctzll(past);
      }
      Slot r{64 * c + f, 0, 0, 0, 0, __builtin_amdgcn_readlane(upto - n * P.kvh, f),
             seq_span_of(P, __builtin_amdgcn_readlane(start[c], f), __builtin_amdgcn_readlane(end[c], f),
                         __builtin_amdgcn_readlane(kv[c], f))};
      const int i = by_unit ? at - r.seq * A.nrb * P.kvh : 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int live = __builtin_amdgcn_readlane(splits(tiles[c][b], by), f);
        r.rb = b;
        r.live = live;
        if (by_unit) {
          if ((A.nrb == 2 ? i & 1 : 0) == b) {
            r.head = A.nrb == 2 ? i >> 1 : i;
            r.first += r.head * live;
            return r;
          }
        } else if (at < r.first + live * P.kvh) {
          r.head = quotient(at - r.first, live);
          r.first += r.head * live;
          r.sp = at - r.first;
          return r;
        }
        r.first += live * P.kvh;
      }
    }
  return {-1, 0, 0, 0, 0, 0, {}};
}

// row r of a unit: token and head
struct RowOf {
  int tok, head;
};
DEV RowOf row_of(const PagedAttnArgs& A, int g, int r) { return {r / A.gqa, g * A.gqa + r % A.gqa}; }

// what a page that is not there is read as (never written): codes of a page
// and 16 rows' scales, or 16 rows, whichever is more
__device__ uint4 zeros[(512 / 2 * 256 + 16 * 32) / 16];

template <int N>
DEV void ld_dwords(const uint8_t* p, uint32_t* x) {
  if constexpr (N == 1) {
    x[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = v.x;
    x[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
  }
}

// Workgroup `block`, NW waves.  lds: few_lds() bytes.
template <int HD, bool Q4, bool Q16, int NW>
DEV void attn_few(const PagedAttnArgs& A, int block, float* lds) {
  constexpr int VP = kParts<HD>, W = NW / VP, HW = HD / VP, NH = HW / 128, QS = HW / 32;  // HW: dims of a wave
  constexpr int LD = HD + 4;  // floats between rows in LDS
  // lds: queries; later [W][rows][LD] outputs, [W][8][2] maxima and sums
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g4 = lane >> 4;
  const Slot slot = find_slot(A, block, false);
  const int i = uni(slot.seq), g = uni(slot.head), rb = uni(slot.rb), sp = uni(slot.sp), live = uni(slot.live);
  if (i < 0) return;
  const int cap = paged_cap(P);
  const Block blk = block_of(A, slot.s, rb, cap);
  const SeqSpan& s = blk.s;
  const int rows = blk.rows, r0 = kRows * rb, t_first = uni(blk.t_first), t_last = uni(blk.t_last);
  if (rows <= 0) return;
  const int p_first = s.p0 + t_first, p_last = s.p0 + t_last;
  const TileRange R = tile_range(p_first, p_last, A.window, A.sinks, cap);
  const bool whole_unit = live <= 1;
  const int per = uni((R.n + max(live, 1) - 1) / max(live, 1));
  const int sha = min(sp * per, R.n), shb = min((sp + 1) * per, R.n);
  const RowOf ro = row_of(A, g, r0 + min(c & 7, rows - 1));
  const int pos = s.p0 + ro.tok;  // of this lane's column
  const table_ptr trow = table_row(P, i);


  // This stream's tiles: first those that every row sees all of, then the
  // others (a loop with both kinds kept two copies of the output registers)
  const int stream = wave / VP, part = wave % VP;  // part: the wave's dims are HW part ..
  const int wa = R.sink - R.from + (A.window > 0 ? max(0, p_last - A.window + kPT) / kPT : 0);
  const int wb = R.sink - R.from + max(0, min(p_first, cap - 1) + 1) / kPT;
  const int a0 = min(max(sha, wa), shb), n_whole = max(0, min(shb, wb) - a0), n_all = shb - sha;
  auto base_of = [&](int v) {
    const int before = a0 - sha, e = v - n_whole;
    return R.base(v < n_whole ? a0 + v : e < before ? sha + e : v + sha);
  };
  // A tile's halves: their pages' blocks and the first rows there.  A half
  // without a page is read from zeros.
  struct Where {
    const uint8_t *k[2], *v[2];
    int row[2], kb;
    uint32_t there;
  };
  auto locate = [&](int kb) __attribute__((always_inline)) {
    Where w;
    w.kb = kb;
    w.there = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int p = kb + 16 * u, b = p >> P.page_shift;
      const uint32_t pg = trow[min(b, P.table_stride - 1)];
      const bool is = b < P.table_stride && pg < (uint32_t)P.n_pages;
      const int64_t blk = paged_block<Q4, HD>(P, is ? (int)pg : 0, g);
      w.k[u] = is ? P.k + blk : (const uint8_t*)zeros;
      w.v[u] = is ? P.v + blk : (const uint8_t*)zeros;
      w.row[u] = is ? p & ((1 << P.page_shift) - 1) : 0;
      w.there |= is ? 1u << u : 0u;
    }
    return w;
  };
  // K: row 16 u + c; kd: the scales of this lane's blocks, two a dword
  uint32_t kw[2][Q4 ? QS : 4 * QS], kd[2];
  auto load_k = [&](const Where& w, int u) __attribute__((always_inline)) {
    if constexpr (Q4) {
      const uint32_t at = (w.row[u] + c) * (HD / 2) + part * (HW / 2) + g4 * (HW / 8);
#pragma unroll
      for (int k = 0; k < QS; k += 4) ld_dwords<4>(w.k[u] + (at + k * 4), kw[u] + k);
      const uint8_t* ks = w.k[u] + (uint32_t)((HD / 2 << P.page_shift) + (w.row[u] + c) * (HD / 16) + part * (HW / 16) + g4 * (HW / 64));
      if constexpr (HW == 128)
        kd[u] = *reinterpret_cast<const uint16_t*>(ks);
      else
        kd[u] = *reinterpret_cast<const uint32_t*>(ks);
    } else {
      const uint32_t at = ((w.row[u] + c) * HD + part * HW + g4 * 8) * 2;
#pragma unroll
      for (int k = 0; k < QS; ++k) ld_dwords<4>(w.k[u] + (at + k * 64), kw[u] + 4 * k);
    }
  };
  // V: this lane's 8 keys 16 u + 4 g4 + r, some dims of each, and their scales
  uint32_t v[8][Q4 ? NH : 4 * NH];
  uint16_t vd[8];
  auto load_v = [&](const Where& w) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int u = k >> 2, row = w.row[u] + 4 * g4 + (k & 3);
      if constexpr (Q4) {
        ld_dwords<NH>(w.v[u] + (uint32_t)(row * (HD / 2) + part * (HW / 2) + c * 4 * NH), v[k]);
        vd[k] = *reinterpret_cast<const uint16_t*>(
            w.v[u] + (uint32_t)((HD / 2 << P.page_shift) + row * (HD / 16) + part * (HW / 16) + (c * NH / 4) * 2));
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h)
          ld_dwords<4>(w.v[u] + (uint32_t)((row * HD + part * HW + c * 8 + h * 128) * 2), v[k] + 4 * h);
      }
    }
  };
  constexpr bool kBoth = Q4 || HW <= 128;  // registers for both halves of K of the next tile beside V and the output

  // Q^T fragments, dims in the order that K's rows are read, through LDS: in
  // registers they would cost every wave HD / 8 of them.  Their loads go out
  // first, then the first tile's.
  h8v* qf = reinterpret_cast<h8v*>(lds);
  constexpr int QF = HD / 32, QN = (QF + NW - 1) / NW;  // fragments, and of a wave
  uint32_t qraw[QN][Q16 ? 4 : 8];
  const int64_t q_at = (int64_t)(s.q0 + ro.tok) * A.q_stride + ro.head * HD;
#pragma unroll
  for (int j = 0; j < QN; ++j) {
    const int f = min(j * NW + wave, QF - 1), k = f % QS, d = f / QS * HW + (Q4 ? (g4 * QS + k) * 8 : k * 32 + g4 * 8);
    const uint8_t* p = (const uint8_t*)A.q + (q_at + d) * (Q16 ? 2 : 4);
    ld_dwords<4>(p, qraw[j]);
    if constexpr (!Q16) ld_dwords<4>(p + 16, qraw[j] + 4);
  }
  __builtin_amdgcn_sched_barrier(0);
  int at = stream;  // of this stream's tiles
  Where next{};
  if (at < n_all) {
    next = locate(base_of(at));
    load_k(next, 0);
    if constexpr (kBoth) load_k(next, 1);
    load_v(next);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < QN; ++j) {
    const int k = j * NW + wave;
    h8v q;
    if constexpr (Q16) {
      q = __builtin_bit_cast(h8v, make_uint4(qraw[j][0], qraw[j][1], qraw[j][2], qraw[j][3]));
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float x = __uint_as_float(qraw[j][t]);
        const _Float16 hi = (_Float16)x, lo = (_Float16)(x - (float)hi);
        q[t] = c < 8 ? hi : lo;
      }
    }
    if (k < QF) qf[k * 64 + lane] = q;
  }
  lds_sync();
  f4v o[NH][8];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int t = 0; t < 8; ++t) o[h][t] = f4v{0.f, 0.f, 0.f, 0.f};
  float m = kNone, l = 0.f;  // of this lane's column; l over this lane's keys alone
  const float scale2 = A.scale * 1.44269504088896341f;
  int qat = lane;
  [[maybe_unused]] int round = 0;

  auto tile = [&](auto whole_tag) __attribute__((always_inline)) {
    constexpr bool whole = decltype(whole_tag)::value;
    asm volatile("" : "+v"(qat));  // the query fragments stay in LDS
    const Where cur = next;
    const int kb = cur.kb;
    const bool more = at + W < n_all;
    if (more) next = locate(base_of(at + W));
    // keys that this lane weighs: bit 4 u + r is key kb + 16 u + 4 g4 + r
    uint32_t seen = (cur.there & 1 ? 0xfu : 0u) | (cur.there & 2 ? 0xf0u : 0u);
    if constexpr (!whole) {
      uint32_t by = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int key = kb + 16 * (k >> 2) + 4 * g4 + (k & 3);
        if (key < cap && key_seen(key, pos, A.window, A.sinks)) by |= 1u << k;
      }
      seen &= by;
    }
    f4v sc[2] = {f4v{0.f, 0.f, 0.f, 0.f}, f4v{0.f, 0.f, 0.f, 0.f}};
    auto scores = [&](int u) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < QS; ++k) {
        h8v a;
        if constexpr (Q4) {
          const uint32_t x = kd[u];
          a = q4_frag(kw[u][k], h2_of(k / 4 ? hi_halves(x, x) : lo_halves(x, x)));
        } else {
          a = __builtin_bit_cast(h8v, make_uint4(kw[u][4 * k], kw[u][4 * k + 1], kw[u][4 * k + 2], kw[u][4 * k + 3]));
        }
        sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[qat + (part * QS + k) * 64], sc[u], 0, 0, 0);
      }
    };
    if constexpr (!kBoth) load_k(cur, 1);
    scores(0);
    scores(1);
    if constexpr (VP == 2) {
      f4v* xs = reinterpret_cast<f4v*>(lds + HD * 8) + round * (NW * 128);
#pragma unroll
      for (int u = 0; u < 2; ++u) xs[wave * 128 + u * 64 + lane] = sc[u];
      lds_sync();
#pragma unroll
      for (int u = 0; u < 2; ++u) sc[u] += xs[(wave ^ 1) * 128 + u * 64 + lane];
      round ^= 1;
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) {  // K's registers are free: the next tile's rows
      load_k(next, 0);
      if constexpr (kBoth) load_k(next, 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    // weights
    float p[8], top = kNone;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = sc[u][r];
        if constexpr (!Q16)  // hi and lo parts of the query
          x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));
        x *= scale2;
        p[4 * u + r] = x;
      }
    if (!whole || cur.there != 3) {
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = (seen >> k & 1) ? p[k] : -__builtin_inff();
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, p[k]);
    top = quad_max4(top);
    // The maximum is moved where it grows by more than 2^8: until then the
    // weights stay below 2^8 and nothing has to be scaled
    if (__any(top > m + 8.f)) {
      const float mn = fmaxf(m, top), a = exp2_(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int k = 0; k < 8; ++k) o[h][k] *= a;
    }
    h8v pf;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float e = exp2_(p[k] - m);
      l += e;
      const _Float16 hi = (_Float16)e, lo = (_Float16)(e - (float)hi);
      pf[k] = c < 8 ? hi : lo;
    }
    // Two A operands, of the dim tiles (h, 2 t) and (h, 2 t + 1): dims 128 h + 8 c + .. (f16), 8 NH c + 8 h + ..
    // (4 bits) of this wave's part; the keys whose bit of `mask` is clear count as zeros
    auto frags = [&](int h, int t, uint32_t mask, h8v(&f)[2]) __attribute__((always_inline)) {
      uint32_t x[2][4];
#pragma unroll
      for (int kp = 0; kp < 4; ++kp) {
        const bool on0 = mask >> (2 * kp) & 1, on1 = mask >> (2 * kp + 1) & 1;
        if constexpr (Q4) {
          const h2v d2 = h2_of((on0 ? (uint32_t)vd[2 * kp] : 0u) | (on1 ? (uint32_t)vd[2 * kp + 1] << 16 : 0u));
          // a half of a dword has dims 0, 4, 2, 6 (1, 5, 3, 7) from bit 0 up
          x[0][kp] = u_of(q4_pair(lo_halves(v[2 * kp][h], v[2 * kp + 1][h]), t) * d2);
          x[1][kp] = u_of(q4_pair(hi_halves(v[2 * kp][h], v[2 * kp + 1][h]), t) * d2);
        } else {
          const uint32_t a = on0 ? v[2 * kp][4 * h + t] : 0u, b = on1 ? v[2 * kp + 1][4 * h + t] : 0u;
          x[0][kp] = lo_halves(a, b);
          x[1][kp] = hi_halves(a, b);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) f[e] = __builtin_bit_cast(h8v, make_uint4(x[e][0], x[e][1], x[e][2], x[e][3]));
    };
    if constexpr (whole) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          h8v f[2];
          frags(h, t, 0xffu, f);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            o[h][2 * t + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[e], pf, o[h][2 * t + e], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
    } else {
      // A row that a token does not see must not reach its output even as 0 x
      // infinity: token by token, with the rows it does not see as zeros
      for (int tok = t_first; tok <= t_last; ++tok) {
        const int pt = s.p0 + tok;
        uint32_t mask = 0;
        if constexpr (Q4) {  // (what can be unpacked before the loop does not fit in registers)
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int h = 0; h < NH; ++h) asm volatile("" : "+v"(v[k][h]));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int key = kb + 16 * (k >> 2) + 4 * g4 + (k & 3);
          if (key < cap && key_seen(key, pt, A.window, A.sinks)) mask |= 1u << k;
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            h8v f[2];
            frags(h, t, mask, f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const f4v x = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[e], pf, f4v{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) o[h][2 * t + e][r] += ro.tok == tok ? x[r] : 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      }
    }
    if (more) load_v(next);
    at += W;
  };
  while (at < n_whole) tile(std::true_type());
  while (at < n_all) tile(std::false_type());
  if constexpr (VP == 2) {  // the streams keep step: as many barriers as the longest one's
    for (; at - stream < n_all; at += W) lds_sync();
  }

  // the column's sum over the lane groups, the two columns of a row, the waves
  l = quad_sum4(l);
  lds_sync();  // every wave is done with the queries
  const int nr = min(A.max_q * A.gqa, kRows);  // rows that LDS has room for
  float* ml = lds + W * nr * LD;
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[8];
#pragma unroll
      for (int t = 0; t < 8; ++t)
        x[t] = o[h][t][r] + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(o[h][t][r]), 0x128, 0xf, 0xf, true));
      const int dim = 4 * g4 + r, d = part * HW + (Q4 ? dim * 8 * NH + h * 8 : h * 128 + dim * 8);
      if (c < rows) {
        float* dst = lds + (stream * nr + c) * LD + d;
        *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  if (part == 0 && lane < rows) *reinterpret_cast<float2*>(ml + (stream * kRows + lane) * 2) = make_float2(m, l);
  lds_sync();
  for (int e = threadIdx.x; e < rows * (HD / 4); e += 64 * NW) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
    float2 st[W];
    float M = kNone, L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      st[w] = *reinterpret_cast<const float2*>(ml + (w * kRows + r) * 2);
      M = fmaxf(M, st[w].x);
    }
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2_(st[w].x - M);
      const float4 y = *reinterpret_cast<const float4*>(lds + (w * nr + r) * LD + d);
      L += f * st[w].y;
      x.x += f * y.x;
      x.y += f * y.y;
      x.z += f * y.z;
      x.w += f * y.w;
    }
    if (whole_unit) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const RowOf to = row_of(A, g, r0 + r);
      uint16_t* out = A.out + (int64_t)(s.q0 + to.tok) * A.out_stride + to.head * HD + d;
      *reinterpret_cast<uint2*>(out) = make_uint2((uint32_t)f2h(x.x * inv) | (uint32_t)f2h(x.y * inv) << 16,
                                                  (uint32_t)f2h(x.z * inv) | (uint32_t)f2h(x.w * inv) << 16);
    } else {
      const int64_t at = (int64_t)block * nr + r;
      *reinterpret_cast<float4*>(A.part + at * HD + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(A.part_ml + at * 2) = make_float2(M, L);
    }
  }
}

// Merge of a row's splits: workgroup (unit and row `block`, part `part` of DW
// dims) of 256 threads, DW / 4 threads a split
template <int HD, int DW>
DEV void merge_few(const PagedAttnArgs& A, int block, int part) {
  constexpr int T = DW / 4, NG = 256 / T;
  __shared__ float wt[kPagedMaxSplits];
  __shared__ float red[4];
  __shared__ __align__(16) float sum[NG][DW + 4];
  const PagedArgs& P = A.P;
  const int nr = min(A.max_q * A.gqa, kRows);
  const int unit = uni(block / nr), r = block - unit * nr;
  const Slot slot = find_slot(A, unit, true);
  const int i = uni(slot.seq), g = uni(slot.head), rb = uni(slot.rb), live = uni(slot.live);
  if (i < 0 || live <= 1) return;  // written by its workgroup
  const SeqSpan s = slot.s;
  const int r0 = kRows * rb;
  if (r >= block_of(A, s, rb, paged_cap(P)).rows) return;
  const int t = threadIdx.x, grp = t / T, d = part * DW + t % T * 4;
  const int64_t at = (int64_t)slot.first * nr + r;  // + sp * nr
  float4 y[4];  // the first rounds' loads beside the statistics'
#pragma unroll
  for (int k = 0; k < 4; ++k)
    y[k] = *reinterpret_cast<const float4*>(A.part + (at + (int64_t)min(grp + k * NG, live - 1) * nr) * HD + d);
  float2 st = make_float2(kNone, 0.f);
  if (t < live) st = *reinterpret_cast<const float2*>(A.part_ml + (at + (int64_t)t * nr) * 2);  // (live <= kGroups)
  const float M = block_max(st.x, red);
  const float f = exp2_(st.x - M);
  if (t < live) wt[t] = f;
  const float L = block_sum(t < live ? f * st.y : 0.f, red);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = grp; s0 < live; s0 += 4 * NG) {
    float4 z[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = y[k];
    if (s0 + 4 * NG < live) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        y[k] = *reinterpret_cast<const float4*>(A.part + (at + (int64_t)min(s0 + (k + 4) * NG, live - 1) * nr) * HD + d);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int sp = s0 + k * NG;
      if (sp < live) {
        const float w = wt[sp];
        x.x += w * z[k].x;
        x.y += w * z[k].y;
        x.z += w * z[k].z;
        x.w += w * z[k].w;
      }
    }
  }
  *reinterpret_cast<float4*>(&sum[grp][t % T * 4]) = x;
  lds_sync();
  const RowOf to = row_of(A, g, r0 + r);
  uint16_t* out = A.out + (int64_t)(s.q0 + to.tok) * A.out_stride + to.head * HD + part * DW;
#pragma unroll
  for (int j = t; j < DW; j += 256) {
    float e = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) e += sum[k][j];
    out[j] = f2h(L == 0.f ? 0.f : e / L);
  }
}

inline int few_units(const PagedAttnArgs& a) { return a.P.n_seq * a.P.kvh * a.nrb; }
inline int few_unit_rows(const PagedAttnArgs& a) { return std::min(a.max_q * a.gqa, kRows); }
// bytes of LDS of a workgroup of NW waves, nr rows a unit
template <int HD, int NW>
constexpr size_t few_lds(int nr) {
  const int parts = kParts<HD>, W = NW / parts;
  return std::max((size_t)W * nr * (HD + 4) * 4 + W * kRows * 8, (size_t)HD * 32 + (parts == 2 ? 2 * NW * 128 * 16 : 0));
}
// a few rows: more workgroups a row in the merge, each with fewer splits to add up in turn
inline bool few_merge_wide(const PagedAttnArgs& a) { return few_units(a) * few_unit_rows(a) < 128; }

}  // namespace
