// k_paged.hip -- what writes and reads the rows of the paged key/value cache
// (paged.h): the append of a batch's new tokens and the read-back of its rows.
#include "../../include/e4b.h"
#include "paged.h"
#include "util.h"

namespace {

// E contiguous elements as floats
template <int E>
DEV void ld_f32(const float* p, float (&v)[E]) {
  if constexpr (E == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x;
    v[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = t.x;
      v[4 * i + 1] = t.y;
      v[4 * i + 2] = t.z;
      v[4 * i + 3] = t.w;
    }
  }
}
template <int E>
DEV void ld_words(const void* p, uint32_t (&w)[E / 2]) {
  if constexpr (E == 2) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (E == 4) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    w[0] = t.x;
    w[1] = t.y;
  } else {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    w[0] = t.x;
    w[1] = t.y;
    w[2] = t.z;
    w[3] = t.w;
  }
}
template <int E>
DEV void st_words(void* p, const uint32_t (&w)[E / 2]) {
  if constexpr (E == 2) {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  } else if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <int E, typename T>
DEV void st_f16(void* p, const T (&x)[E]) {
  uint32_t w[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) w[i] = (uint32_t)f2h((float)x[2 * i]) | ((uint32_t)f2h((float)x[2 * i + 1]) << 16);
  st_words<E>(p, w);
}

DEV float wsum(float v) { return wave_sum(v); }
DEV double wsum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
DEV float rsq(float m) { return 1.0f / sqrtf(m); }
DEV double rsq(double m) { return 1.0 / sqrt(m); }
DEV void sin_cos(double r, float& s, float& c) { sincosf((float)r, &s, &c); }
DEV void sin_cos(double r, double& s, double& c) { sincos(r, &s, &c); }

// x / rms(x), times w
template <int E, typename T>
DEV void head_rms(T (&x)[E], const float* w, float eps) {
  T ss = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) ss += x[i] * x[i];
  const T inv = rsq(wsum(ss) / (T)(64 * E) + (T)eps);
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] *= inv;
  if (!w) return;
  float wv[E];
  ld_f32<E>(w + E * (threadIdx.x & 63), wv);
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] *= (T)wv[i];
}

// Pairs (d, d + hd / 2), d < angles: lane l < 32 holds dims E l .. and lane
// l + 32 their partners.  turns: (cos, sin) of the token's pairs.
template <int E, typename T, typename T2>
DEV void rotate(T (&x)[E], const T2* turns, int angles) {
  const int lane = threadIdx.x & 63, d0 = E * (lane & 31);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const T other = __shfl_xor(x[i], 32, 64);
    if (d0 + i < angles) {
      const T2 t = turns[d0 + i];
      x[i] = lane < 32 ? x[i] * (T)t.x - other * (T)t.y : x[i] * (T)t.x + other * (T)t.y;
    }
  }
}

// One row in 4 bits, codes at `codes`, scales at `scales`: of each 32 dims the
// value a of largest magnitude (the first of several) is -8 steps, the step d
// is a / -8 rounded to 8 significant bits (and at most 8160 = 65280 / 8, the
// largest that keeps 8 d finite in f16), the code rint(x / d) + 8 cut to 0..15.
// A block that holds a value that is not finite gets a NaN scale: it reads as
// NaN.  In 64 bits: a value beside the border of two codes gets the code of
// the exact one.
template <int E>
DEV void st_q4(uint8_t* codes, uint8_t* scales, const double (&x)[E]) {
  constexpr int LB = 32 / E;  // lanes of a block
  const int lane = threadIdx.x & 63;
  double a = x[0];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    odd = odd || !(fabs(x[i]) <= 3.4e38);
    if (fabs(x[i]) > fabs(a)) a = x[i];
  }
#pragma unroll
  for (int m = 1; m < LB; m <<= 1) {
    const double b = __shfl_xor(a, m, 64);
    if (fabs(b) > fabs(a) || (fabs(b) == fabs(a) && (lane & m))) a = b;
  }
  const uint64_t group = ((1ull << LB) - 1) << (lane & ~(LB - 1));
  odd = (__ballot(odd) & group) != 0;
  uint64_t u = __builtin_bit_cast(uint64_t, a * -0.125);
  u += ((u >> 45) & 1) + (1ull << 44) - 1;
  double d = __builtin_bit_cast(double, u >> 45 << 45);
  d = fmin(fmax(d, -8160.0), 8160.0);
  const _Float16 dh = odd ? (_Float16)__builtin_nanf("") : (_Float16)(float)d;
  const bool none = odd || dh == (_Float16)0.f;
  const double by = none ? 1.0 : (double)dh;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    constexpr uint32_t at[8] = {0, 16, 8, 24, 4, 20, 12, 28};
    const double s = none ? 0.0 : fmin(fmax(rint(x[i] / by), -8.0), 7.0);
    const uint32_t c = (uint32_t)((int)s + 8);
    if constexpr (E == 8)
      w |= c << at[i];
    else if constexpr (E == 4)
      w |= c << ((lane & 1) ? at[4 + i] : at[i]);
    else
      w |= c << (at[i] + ((lane & 1) ? 8 : 0) + ((lane & 2) ? 4 : 0));
  }
#pragma unroll
  for (int m = 1; m < 8 / E; m <<= 1) w |= __shfl_xor(w, m, 64);
  if ((lane & (8 / E - 1)) == 0) *reinterpret_cast<uint32_t*>(codes + (E * lane / 8) * 4) = w;
  if ((lane & (LB - 1)) == 0)
    *reinterpret_cast<uint16_t*>(scales + (lane / LB) * 2) = __builtin_bit_cast(uint16_t, dh);
}

// Append: workgroup (token, part of the heads), a wave takes every
// (4 gridDim.y)-th head row of [q heads | k heads | v heads], E = HD / 64 dims
// a lane, the next row requested before one is worked on.  K and V of a 4-bit
// cache are prepared in 64 bits (st_q4), all else in 32.
// The angle pos * inv_freq[d] is made and reduced in 64 bits: at position
// 30000 a 32-bit product is off by up to 2^-10 of a radian, several roundings
// of an f16 result.  Its sine and cosine are taken once a token, one pair a
// thread (every head's wave for itself: 57 us for 2600 tokens of 32 heads).
// What bounds it: latency (a load of the row, the sequence's entries and the
// table's, the store); bytes once there are thousands of tokens.
template <int HD, bool Q4, bool X16>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs A) {
  constexpr int E = HD / 64;
  using T = std::conditional_t<Q4, double, float>;
  using T2 = std::conditional_t<Q4, double2, float2>;
  __shared__ T2 turns[HD / 2];
  const PagedArgs& P = A.P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, step = 4 * gridDim.y;
  const int heads = A.qh + (A.v_is_k ? 1 : 2) * P.kvh;
  int h = blockIdx.y * 4 + wave;
  if (!A.q && h < A.qh) h += (A.qh - h + step - 1) / step * step;  // the first row that is wanted
  auto load = [&](int h, float(&x)[E]) __attribute__((always_inline)) {
    const int64_t at = (int64_t)t * A.x_stride + h * HD + E * lane;
    if constexpr (X16) {
      uint32_t w[E / 2];
      ld_words<E>((const uint16_t*)A.x + at, w);
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = h2f((uint16_t)(w[j / 2] >> (16 * (j & 1))));
    } else {
      ld_f32<E>((const float*)A.x + at, x);
    }
  };
  float x[E], ahead[E];
  if (h < heads) load(h, ahead);
  const int i = __builtin_amdgcn_readfirstlane(seq_of_token(P, t));
  if (i >= P.n_seq) return;  // behind the last sequence
  const SeqSpan s = seq_span(P, i);
  const int pos = s.p0 + (t - s.q0);
  if (pos < 0 || t < s.q0 || t - s.q0 >= s.n) return;
  if ((int)threadIdx.x < A.angles) {
    const double a = (double)pos * (double)A.inv_freq[threadIdx.x], turn = 6.283185307179586476925;
    T sn, cs;
    sin_cos(fma(-rint(a * (1.0 / turn)), turn, a), sn, cs);
    turns[threadIdx.x] = T2{cs, sn};
  }
  lds_sync();
  const int pg = paged_page(table_row(P, i), P.table_stride, P.page_shift, P.n_pages, pos);
  const int row = pos & ((1 << P.page_shift) - 1);
  auto put = [&](uint8_t* pool, int g, const T(&x)[E]) {
    if (pg < 0) return;
    uint8_t* b = pool + paged_block<Q4, HD>(P, pg, g);
    if constexpr (Q4)
      st_q4<E>(b + row * (HD / 2), b + (HD / 2 << P.page_shift) + row * (HD / 16), x);
    else
      st_f16<E>(b + (row * HD + E * lane) * 2, x);
  };
  for (; h < heads; h += step) {
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = ahead[j];
    if (h + step < heads) load(h + step, ahead);
    if (h < A.qh) {
      if (A.qw) head_rms<E>(x, A.qw, A.eps);
      rotate<E>(x, turns, A.angles);
      const int64_t o = (int64_t)t * A.q_stride + h * HD + E * lane;
      if (A.q16) {
        st_f16<E>((uint16_t*)A.q + o, x);
      } else {
        float* q = (float*)A.q + o;
        if constexpr (E == 2) {
          *reinterpret_cast<float2*>(q) = make_float2(x[0], x[1]);
        } else {
#pragma unroll
          for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(q + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        }
      }
      continue;
    }
    const int g = h < A.qh + P.kvh ? h - A.qh : h - A.qh - P.kvh;
    const bool isk = h < A.qh + P.kvh;
    T y[E];
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = (T)x[j];
    if (isk) {
      if (A.kw) head_rms<E>(y, A.kw, A.eps);
      rotate<E>(y, turns, A.angles);
      put(P.k, g, y);
      if (!A.v_is_k) continue;
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = (T)x[j];
    }
    if (A.v_rms) head_rms<E>(y, (const float*)nullptr, A.eps);
    put(P.v, g, y);
  }
}

// Read-back: workgroup = one token, wave w takes the KV heads w, w + 4, ...
template <int HD, bool Q4>
__global__ __launch_bounds__(256) void k_kv_gather(PagedArgs P, uint16_t* __restrict__ ko, uint16_t* __restrict__ vo) {
  constexpr int E = HD / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x;
  const int i = __builtin_amdgcn_readfirstlane(seq_of_token(P, t));
  if (i >= P.n_seq) return;
  const SeqSpan s = seq_span(P, i);
  if (t < s.q0 || t - s.q0 >= s.n) return;
  const int pos = s.p0 + (t - s.q0);
  const int pg = paged_page(table_row(P, i), P.table_stride, P.page_shift, P.n_pages, pos);
  const int row = pos & ((1 << P.page_shift) - 1);
  for (int j = blockIdx.y * 4 + wave; j < 2 * P.kvh; j += 4 * gridDim.y) {
    const int g = j >> 1;
    uint16_t* out = (j & 1) ? vo : ko;
    if (!out) continue;
    uint32_t w[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) w[e] = 0;
    if (pg >= 0) {
      const uint8_t* b = ((j & 1) ? P.v : P.k) + paged_block<Q4, HD>(P, pg, g);
      if constexpr (Q4) {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(b + row * (HD / 2) + (E * lane / 8) * 4);
        const float d = h2f(*reinterpret_cast<const uint16_t*>(b + (HD / 2 << P.page_shift) + row * (HD / 16) + (E * lane / 32) * 2));
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const int pr = (E * lane % 8) / 2 + e;  // pair 0..3 of the dword at bits 0, 8, 4, 12
          const uint32_t n = c >> (((pr & 1) << 3) + ((pr & 2) << 1));
          const uint16_t lo = f2h(((int)(n & 15) - 8) * d), hi = f2h(((int)((n >> 16) & 15) - 8) * d);
          w[e] = (uint32_t)lo | ((uint32_t)hi << 16);
        }
      } else {
        ld_words<E>(b + (row * HD + E * lane) * 2, w);
      }
    }
    st_words<E>(out + ((int64_t)t * P.kvh + g) * HD + E * lane, w);
  }
}

// heads of a token over workgroups of 4 waves: all waves apart while there
// are few tokens, one workgroup a token from two a CU on (the sequence is
// looked up once)
int head_parts(int n_tok, int rows) { return n_tok < 512 ? (rows + 3) / 4 : 1; }

template <int HD>
int append_hd(const KvAppendArgs& a, bool q4, bool x16, dim3 grid, hipStream_t st) {
  if (q4 && x16)
    k_kv_append<HD, true, true><<<grid, 256, 0, st>>>(a);
  else if (q4)
    k_kv_append<HD, true, false><<<grid, 256, 0, st>>>(a);
  else if (x16)
    k_kv_append<HD, false, true><<<grid, 256, 0, st>>>(a);
  else
    k_kv_append<HD, false, false><<<grid, 256, 0, st>>>(a);
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, int hd, bool q4, bool x16, hipStream_t st) {
  const int rows = a.qh + (a.v_is_k ? 1 : 2) * a.P.kvh;
  const dim3 grid(a.P.n_tok, head_parts(a.P.n_tok, rows));
  return hd == 128 ? append_hd<128>(a, q4, x16, grid, st)
         : hd == 256 ? append_hd<256>(a, q4, x16, grid, st)
                     : append_hd<512>(a, q4, x16, grid, st);
}

int launch_kv_gather(const PagedArgs& P, int hd, bool q4, uint16_t* ko, uint16_t* vo, hipStream_t st) {
  const dim3 grid(P.n_tok, head_parts(P.n_tok, 2 * P.kvh));
#define GATHER(HD)                                                   \
  if (hd == HD) {                                                    \
    if (q4)                                                          \
      k_kv_gather<HD, true><<<grid, 256, 0, st>>>(P, ko, vo);        \
    else                                                             \
      k_kv_gather<HD, false><<<grid, 256, 0, st>>>(P, ko, vo);       \
  }
  GATHER(128)
  GATHER(256)
  GATHER(512)
#undef GATHER
  E4B_HIP(hipGetLastError());
  return E4B_OK;
}
