// k_paged_decode.hip -- attention of a few query rows per KV head over the
// paged cache: decoded tokens (paged.h; chunks: k_paged_chunk.hip).
//
// Unit (sequence, KV head, 8 query rows: tokens x heads of the group); its key
// tiles are cut into ns runs, one workgroup each, and inside it over the
// waves, every wave with a running maximum and sum of its own; the waves are
// merged in LDS, the runs by k_attn_paged_merge.
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
// What bounds it: the cache's bytes.  A tile of 32 keys is 32 KB (head dim
// 256, f16) in flight per wave, a few microseconds of a CU's share of HBM.
#include <algorithm>

#include "../../include/e4b.h"
#include "paged_attn.h"
#include "util.h"

namespace {

constexpr int kRows = 8;
constexpr int kWaves = 8;
// waves that share a tile, each with 256 of V's dims at most (a wave's output
// is HD / 4 registers else); both compute the scores
template <int HD>
constexpr int kParts = HD == 512 ? 2 : 1;
template <int HD>
constexpr int kStreams = kWaves / kParts<HD>;  // tiles at a time in a workgroup

// row c of a unit: token and head
struct RowOf {
  int tok, head;
};
DEV RowOf row_of(const PagedAttnArgs& A, int g, int r) { return {r / A.gqa, g * A.gqa + r % A.gqa}; }

// the share of split sp: tiles a .. b - 1
struct Share {
  int a, b, live;  // live: splits that have any
};
DEV Share share_of(const TileRange& R, int ns, int sp, int waves) {
  const int per = max(waves, uni((R.n + ns - 1) / ns));
  return {min(sp * per, R.n), min((sp + 1) * per, R.n), uni((R.n + per - 1) / per)};
}

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

template <int HD, bool Q4, bool Q16>
__global__ __launch_bounds__(64 * kWaves, 2) void k_attn_paged_few(PagedAttnArgs A) {
  constexpr int W = kStreams<HD>, VP = kParts<HD>, NH = HD / 128 / VP, QS = HD / 32;
  constexpr int LD = HD + 4;  // floats between rows in LDS
  extern __shared__ __align__(16) float lds[];  // queries; later [W][rows][LD] outputs, [W][8][2] maxima and sums
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g4 = lane >> 4;
  const int unit = uni(blockIdx.x / A.ns), sp = blockIdx.x - unit * A.ns;
  const int head = uni(unit / A.nrb), rb = unit - head * A.nrb, i = uni(head / P.kvh), g = head - i * P.kvh;
  const SeqSpan s = seq_span(P, i);
  if ((int64_t)s.n * A.gqa > kPagedFewRows) return;  // k_paged_chunk.hip's
  const int rows = min(min(s.n, A.max_q) * A.gqa - kRows * rb, kRows);
  if (rows <= 0) return;
  const int cap = paged_cap(P);
  const int r0 = kRows * rb, t_first = uni(r0 / A.gqa), t_last = uni((r0 + rows - 1) / A.gqa);
  const int p_first = s.p0 + t_first, p_last = s.p0 + t_last;
  const TileRange R = tile_range(p_first, p_last, A.window, A.sinks, cap);
  const Share sh = share_of(R, A.ns, sp, W);
  if (sh.a >= sh.b && !(sp == 0 && R.n == 0)) return;
  const RowOf ro = row_of(A, g, r0 + min(c & 7, rows - 1));
  const int pos = s.p0 + ro.tok;  // of this lane's column
  const table_ptr trow = table_row(P, i);

  // Q^T fragments, dims in the order that K's rows are read, through LDS: in
  // registers they would cost every wave HD / 8 of them
  h8v* qf = reinterpret_cast<h8v*>(lds);
  {
    const int64_t at = (int64_t)(s.q0 + ro.tok) * A.q_stride + ro.head * HD;
#pragma unroll
    for (int k0 = 0; k0 < QS; k0 += kWaves) {
      const int k = k0 + wave;
      if (k < QS) {
        const int d = Q4 ? (g4 * QS + k) * 8 : k * 32 + g4 * 8;
        h8v q;
        if constexpr (Q16) {
          q = *reinterpret_cast<const h8v*>((const uint16_t*)A.q + at + d);
        } else {
          const float4 a = *reinterpret_cast<const float4*>((const float*)A.q + at + d);
          const float4 b = *reinterpret_cast<const float4*>((const float*)A.q + at + d + 4);
          const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const _Float16 hi = (_Float16)v[t], lo = (_Float16)(v[t] - (float)hi);
            q[t] = c < 8 ? hi : lo;
          }
        }
        qf[k * 64 + lane] = q;
      }
    }
  }
  lds_sync();
  f4v o[NH][8];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int t = 0; t < 8; ++t) o[h][t] = f4v{0.f, 0.f, 0.f, 0.f};
  float m = kNone, l = 0.f;  // of this lane's column; l over this lane's keys alone
  const float scale2 = A.scale * 1.44269504088896341f;

  const int stream = wave / VP, part = wave % VP;  // part: V's dims 256 part .. of head dim 512
  int qat = lane;
  auto tile = [&](int kb, auto whole_tag) __attribute__((always_inline)) {
    constexpr bool whole = decltype(whole_tag)::value;
    asm volatile("" : "+v"(qat));  // the query fragments stay in LDS
    // where the two halves lie
    const uint8_t *kh[2], *vh[2];
    [[maybe_unused]] bool there[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int pg = paged_page(trow, P.table_stride, P.page_shift, P.n_pages, kb + 16 * u);
      there[u] = pg >= 0;
      const int64_t blk = paged_block<Q4, HD>(P, max(pg, 0), g);
      kh[u] = P.k + blk;
      vh[u] = P.v + blk;
    }
    const int r16 = kb & ((1 << P.page_shift) - 1) & ~15;
    const int row0[2] = {r16, (r16 + 16) & ((1 << P.page_shift) - 1)};
    // keys that this lane weighs: bit 4 u + r is key kb + 16 u + 4 g4 + r
    uint32_t seen = 0xff;
    if constexpr (!whole) {
      seen = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = kb + 16 * u + 4 * g4 + r;
          if (there[u] && key < cap && key_seen(key, pos, A.window, A.sinks)) seen |= 1u << (4 * u + r);
        }
    }
    // K: row 16 u + c
    uint32_t kw[2][Q4 ? QS : 4 * QS], kd[2][HD == 128 ? 1 : HD / 256];  // kd: scales of this lane's blocks, two a dword
    auto load_k = [&](int u) __attribute__((always_inline)) {
      if constexpr (Q4) {
        const uint32_t at = (row0[u] + c) * (HD / 2) + g4 * (HD / 8);
#pragma unroll
        for (int k = 0; k < QS; k += 4) ld_dwords<4>(kh[u] + (at + k * 4), kw[u] + k);
        const uint8_t* ks = kh[u] + (uint32_t)((HD / 2 << P.page_shift) + (row0[u] + c) * (HD / 16) + g4 * (HD / 64));
        if constexpr (HD == 128)
          kd[u][0] = *reinterpret_cast<const uint16_t*>(ks);
        else
          ld_dwords<HD / 256>(ks, kd[u]);
      } else {
        const uint32_t at = ((row0[u] + c) * HD + g4 * 8) * 2;
#pragma unroll
        for (int k = 0; k < QS; ++k) ld_dwords<4>(kh[u] + (at + k * 64), kw[u] + 4 * k);
      }
    };
    f4v sc[2] = {f4v{0.f, 0.f, 0.f, 0.f}, f4v{0.f, 0.f, 0.f, 0.f}};
    auto scores = [&](int u) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < QS; ++k) {
        h8v a;
        if constexpr (Q4) {
          const uint32_t x = kd[u][k / 8];
          a = q4_frag(kw[u][k], h2_of((k / 4) & 1 ? hi_halves(x, x) : lo_halves(x, x)));
        } else {
          a = __builtin_bit_cast(h8v, make_uint4(kw[u][4 * k], kw[u][4 * k + 1], kw[u][4 * k + 2], kw[u][4 * k + 3]));
        }
        sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[qat + k * 64], sc[u], 0, 0, 0);
      }
    };
    constexpr bool kBoth = Q4 || HD <= 256;  // both halves of K beside V in registers
    load_k(0);
    if constexpr (kBoth) load_k(1);
    // V: this lane's 8 keys 16 u + 4 g4 + r, some dims of each
    uint32_t v[8][Q4 ? NH : 4 * NH], dp[4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int u = k >> 2, row = row0[u] + 4 * g4 + (k & 3);
      if constexpr (Q4) {
        ld_dwords<NH>(vh[u] + (uint32_t)(row * (HD / 2) + part * 128 + c * 4 * NH), v[k]);
        const uint32_t d = *reinterpret_cast<const uint16_t*>(
            vh[u] + (uint32_t)((HD / 2 << P.page_shift) + row * (HD / 16) + (part * 8 + c * NH / 4) * 2));
        dp[k >> 1] = (k & 1) ? dp[k >> 1] | d << 16 : d;
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          uint32_t x[4];
          ld_dwords<4>(vh[u] + (uint32_t)((row * HD + part * 256 + c * 8 + h * 128) * 2), x);
#pragma unroll
          for (int t = 0; t < 4; ++t) v[k][4 * h + t] = x[t];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    scores(0);
    if constexpr (!kBoth) load_k(1);
    scores(1);
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
        if constexpr (!whole) x = (seen >> (4 * u + r) & 1) ? x : -__builtin_inff();
        p[4 * u + r] = x;
        top = fmaxf(top, x);
      }
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
    // A operands of the dim tiles (h, 0..7): dims 128 h + 8 c + t (f16), 8 NH c + 8 h + t (4 bits) of this
    // wave's part; the keys whose bit of `mask` is clear count as zeros
    auto frags = [&](int h, uint32_t mask, h8v(&f)[8]) __attribute__((always_inline)) {
      uint32_t x[8][4];
#pragma unroll
      for (int kp = 0; kp < 4; ++kp) {
        const bool on0 = mask >> (2 * kp) & 1, on1 = mask >> (2 * kp + 1) & 1;
        if constexpr (Q4) {
          const h2v d2 = h2_of(dp[kp] & ((on0 ? 0xffffu : 0u) | (on1 ? 0xffff0000u : 0u)));
          h2v e[4], od[4];
          q4_pairs(lo_halves(v[2 * kp][h], v[2 * kp + 1][h]), e);   // dims 0, 4, 2, 6 of the dword, from bit 0 up
          q4_pairs(hi_halves(v[2 * kp][h], v[2 * kp + 1][h]), od);  // dims 1, 5, 3, 7
          constexpr int at[4] = {0, 2, 4, 6};                       // q4_pairs' order: bits 0, 8, 4, 12
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            x[at[t]][kp] = u_of(e[t] * d2);
            x[at[t] + 1][kp] = u_of(od[t] * d2);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t a = on0 ? v[2 * kp][4 * h + t] : 0u, b = on1 ? v[2 * kp + 1][4 * h + t] : 0u;
            x[2 * t][kp] = lo_halves(a, b);
            x[2 * t + 1][kp] = hi_halves(a, b);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) f[t] = __builtin_bit_cast(h8v, make_uint4(x[t][0], x[t][1], x[t][2], x[t][3]));
    };
    if constexpr (whole) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        h8v f[8];
        frags(h, 0xffu, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[h][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[k], pf, o[h][k], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // A row that a token does not see must not reach its output even as 0 x
      // infinity: token by token, with the rows it does not see as zeros
      for (int tok = t_first; tok <= t_last; ++tok) {
        const int pt = s.p0 + tok;
        uint32_t mask = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int key = kb + 16 * (k >> 2) + 4 * g4 + (k & 3);
          if (there[k >> 2] && key < cap && key_seen(key, pt, A.window, A.sinks)) mask |= 1u << k;
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          h8v f[8];
          frags(h, mask, f);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const f4v x = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[k], pf, f4v{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[h][k][r] += ro.tok == tok ? x[r] : 0.f;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // Whole tiles, which every row sees all of, then the others: a loop that has
  // both kept two copies of the output registers
  auto whole = [&](int kb) {
    return kb + kPT - 1 <= p_first && (A.window == 0 || kb > p_last - A.window || kb + kPT <= A.sinks) &&
           paged_page(trow, P.table_stride, P.page_shift, P.n_pages, kb) >= 0 &&
           paged_page(trow, P.table_stride, P.page_shift, P.n_pages, kb + 16) >= 0;
  };
  for (int t = sh.a + stream; t < sh.b; t += W)
    if (whole(R.base(t))) tile(R.base(t), std::true_type());
  for (int t = sh.a + stream; t < sh.b; t += W)
    if (!whole(R.base(t))) tile(R.base(t), std::false_type());

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
      const int dim = 4 * g4 + r, d = part * 256 + (Q4 ? dim * 8 * NH + h * 8 : h * 128 + dim * 8);
      if (c < rows) {
        float* dst = lds + (stream * nr + c) * LD + d;
        *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  if (part == 0 && lane < rows) *reinterpret_cast<float2*>(ml + (stream * kRows + lane) * 2) = make_float2(m, l);
  lds_sync();
  for (int e = threadIdx.x; e < rows * (HD / 4); e += 64 * kWaves) {
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
    if (sh.live <= 1) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const RowOf to = row_of(A, g, r0 + r);
      uint16_t* out = A.out + (int64_t)(s.q0 + to.tok) * A.out_stride + to.head * HD + d;
      *reinterpret_cast<uint2*>(out) = make_uint2((uint32_t)f2h(x.x * inv) | (uint32_t)f2h(x.y * inv) << 16,
                                                  (uint32_t)f2h(x.z * inv) | (uint32_t)f2h(x.w * inv) << 16);
    } else {
      const int64_t at = ((int64_t)unit * A.ns + sp) * nr + r;
      *reinterpret_cast<float4*>(A.part + at * HD + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(A.part_ml + at * 2) = make_float2(M, L);
    }
  }
}

// Merge of a row's splits: workgroup (unit, row), HD / 4 threads a split.
template <int HD>
__global__ __launch_bounds__(256) void k_attn_paged_merge(PagedAttnArgs A) {
  constexpr int T = HD / 4, NG = 256 / T;
  __shared__ float wt[kPagedMaxSplits];
  __shared__ float red[4];
  __shared__ __align__(16) float sum[NG][HD];
  const PagedArgs& P = A.P;
  const int nr = min(A.max_q * A.gqa, kRows);
  const int r = blockIdx.x % nr, unit = blockIdx.x / nr;
  const int rb = unit % A.nrb, g = unit / A.nrb % P.kvh, i = unit / A.nrb / P.kvh;
  const SeqSpan s = seq_span(P, i);
  if ((int64_t)s.n * A.gqa > kPagedFewRows) return;
  const int rows = min(min(s.n, A.max_q) * A.gqa - kRows * rb, kRows);
  if (r >= rows) return;
  const int r0 = kRows * rb;
  const TileRange R = tile_range(s.p0 + r0 / A.gqa, s.p0 + (r0 + rows - 1) / A.gqa, A.window, A.sinks, paged_cap(P));
  const int live = share_of(R, A.ns, 0, kStreams<HD>).live;
  if (live <= 1) return;  // written by its workgroup
  const int t = threadIdx.x, grp = t / T, d = t % T * 4;
  const int64_t at = (int64_t)unit * A.ns * nr + r;  // + sp * nr
  float2 st = make_float2(kNone, 0.f);
  if (t < live) st = *reinterpret_cast<const float2*>(A.part_ml + (at + (int64_t)t * nr) * 2);
  const float M = block_max(st.x, red);
  const float f = exp2_(st.x - M);
  if (t < live) wt[t] = f;
  const float L = block_sum(t < live ? f * st.y : 0.f, red);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int sp = grp; sp < live; sp += NG) {
    const float4 y = *reinterpret_cast<const float4*>(A.part + (at + (int64_t)sp * nr) * HD + d);
    const float w = wt[sp];
    x.x += w * y.x;
    x.y += w * y.y;
    x.z += w * y.z;
    x.w += w * y.w;
  }
  *reinterpret_cast<float4*>(&sum[grp][d]) = x;
  lds_sync();
  if (grp) return;
#pragma unroll
  for (int k = 1; k < NG; ++k) {
    const float4 y = *reinterpret_cast<const float4*>(&sum[k][d]);
    x.x += y.x;
    x.y += y.y;
    x.z += y.z;
    x.w += y.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const RowOf to = row_of(A, g, r0 + r);
  uint16_t* out = A.out + (int64_t)(s.q0 + to.tok) * A.out_stride + to.head * HD + d;
  *reinterpret_cast<uint2*>(out) = make_uint2((uint32_t)f2h(x.x * inv) | (uint32_t)f2h(x.y * inv) << 16,
                                              (uint32_t)f2h(x.z * inv) | (uint32_t)f2h(x.w * inv) << 16);
}

template <int HD>
int few_hd(const PagedAttnArgs& a, bool q4, bool q16, hipStream_t st) {
  constexpr int W = kStreams<HD>;
  const int nr = std::min(a.max_q * a.gqa, kRows), units = a.P.n_seq * a.P.kvh * a.nrb;
  const size_t lds = std::max((size_t)W * nr * (HD + 4) * 4 + W * kRows * 8, (size_t)HD * 32);
  const dim3 grid((unsigned)(units * a.ns));
  auto go = [&](auto* kernel) {
    // (more than 64 KB of LDS has to be asked for; 68.1 KB at most here)
    if (lds > 65536)
      E4B_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<grid, 64 * kWaves, lds, st>>>(a);
    E4B_HIP(hipGetLastError());
    return E4B_OK;
  };
  int rc = q4 && q16 ? go(k_attn_paged_few<HD, true, true>)
           : q4      ? go(k_attn_paged_few<HD, true, false>)
           : q16     ? go(k_attn_paged_few<HD, false, true>)
                     : go(k_attn_paged_few<HD, false, false>);
  if (rc || a.ns == 1) return rc;
  k_attn_paged_merge<HD><<<units * nr, 256, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

void plan_attn_paged_few(PagedAttnArgs& a, int hd) {
  const int W = hd == 512 ? kStreams<512> : kStreams<256>;
  a.nrb = (a.max_q * a.gqa + kRows - 1) / kRows;
  const int64_t units = (int64_t)a.P.n_seq * a.P.kvh * a.nrb;
  const int64_t seen = a.window ? std::min<int64_t>(a.max_kv, (int64_t)a.window + a.sinks + a.max_q) : a.max_kv;
  const int64_t tiles = seen / kPT + 2;
  int64_t ns = std::min<int64_t>((512 + units - 1) / units, tiles / W);
  if (tiles <= 2 * W) ns = 1;
  a.ns = (int)std::max<int64_t>(1, std::min<int64_t>(ns, kPagedMaxSplits));
  const int nr = std::min(a.max_q * a.gqa, kRows);
  a.part_floats = a.ns > 1 ? (size_t)units * a.ns * nr * hd : 0;
  a.ml_floats = a.ns > 1 ? (size_t)units * a.ns * nr * 2 : 0;
}

int launch_attn_paged_few(const PagedAttnArgs& a, int hd, bool q4, bool q16, hipStream_t st) {
  return hd == 128 ? few_hd<128>(a, q4, q16, st) : hd == 256 ? few_hd<256>(a, q4, q16, st) : few_hd<512>(a, q4, q16, st);
}
