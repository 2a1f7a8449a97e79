// row.cuh -- one row of logits: the running maximum and sum of its softmax, and
// the gradient of its elements.
#pragma once

#include <cfloat>
#include <cmath>

#include "common.cuh"
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

constexpr int kRowUnroll = 4;  // 16-byte loads in flight per thread

// log2(e) / T as the sum of two floats.  One float's rounding (up to 2^-25 of every
// exponent) would have the same sign for a whole row: at differences of -10 to -20 it
// shifted each log-probability by 1.5e-7, which does not average out over a
// sequence (measured on 2000-token sums).
__device__ __forceinline__ float exp_scaled(float d, Scale2 c) {
  return exp2_fast(fmaf(d, c.hi, d * c.lo));
}

// The difference z - m, in logit units, from which on exp((z - m) / T) is 0 for sure
// (exp2_fast flushes under 2^-126, from -87.4 T on).  Where the exponential
// is multiplied by its own argument, the difference is held at it: 0 times an infinite
// difference, or one that 1 / T or an outer gradient makes infinite, is NaN.  (A bound
// without T in it, -1e30, was infinite once it had been scaled: T under 3e-9, or 0.01
// under a loss scale of 2^17.)
__host__ __device__ inline float exp_low(float inv_temp) { return -128.0f / inv_temp; }

// Running (max, sum of exp(z - max), sum of exp(z - max) (z - max)); differences
// in logit units, exponents in base 2.
struct Online {
  float m = -FLT_MAX, s = 0.0f, w = 0.0f;
};

// (a factor's error stays in the sum, and a term meets about ten of them on its
// way: expf here, where exp2_fast's mean error would add up)
template <bool kEnt>
__device__ __forceinline__ void rebase(Online& o, float m2, Scale2 c) {
  const float d = o.m - m2;  // <= 0
  const float a = expf(fmaf(d, c.inv, d * c.inv_lo));
  if (kEnt) o.w = a > 0.0f ? (o.w + o.s * d) * a : 0.0f;  // d may be -inf, or near it, where a is 0
  o.s *= a;
  o.m = m2;
}

// Adds the elements of U vectors, none of them above o.m.  Two elements for each
// instruction but the exponential: five instructions an element otherwise kept the
// pass from the memory's rate.
template <typename T, bool kEnt, int U>
__device__ __forceinline__ void absorb(Online& o, const uint4 (&u)[U], Scale2 c) {
  constexpr int N = Vec16<T>::N;
  const f32x2 nm = pair(-o.m, -o.m), hi = pair(c.hi, c.hi), lo = pair(c.lo, c.lo);
  f32x2 s = pair(0.0f, 0.0f), w = s;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float f[N];
    unpack(u[k], f, (const T*)nullptr);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const f32x2 d = add2(pair(f[i], f[i + 1]), nm);
      const float2 x = parts(fma2(d, hi, mul2(d, lo)));
      const f32x2 e = pair(exp2_fast(x.x), exp2_fast(x.y));
      s = add2(s, e);
      if (kEnt) {  // exp(-inf) * -inf counts as 0
        const float2 t = parts(d);
        w = fma2(e, pair(fmaxf(t.x, c.low), fmaxf(t.y, c.low)), w);
      }
    }
  }
  const float2 a = parts(s);
  o.s += a.x + a.y;
  if (kEnt) {
    const float2 b = parts(w);
    o.w += b.x + b.y;
  }
}

// The largest value over the warp (NaNs count as nothing).
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The lanes' pairs as one, on every lane.
template <bool kEnt>
__device__ __forceinline__ void join_warp(Online& o, Scale2 c) {
  rebase<kEnt>(o, warp_max(o.m), c);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    o.s += __shfl_xor_sync(0xffffffffu, o.s, d);
    if (kEnt) o.w += __shfl_xor_sync(0xffffffffu, o.w, d);
  }
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t r) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[r]
                    : (int64_t) static_cast<const int32_t*>(tokens)[r];
}

// ln s in fp64: logf's error has a mean of its own, 1e-7 of a log-probability
// (measured), which a sequence's sum would keep.  So has the sum's: it comes out low
// by 2.0e-8 to 4.0e-8 of its value, the largest term, 1, apart (64 to 262144 normal
// logits of spread 0.3 and 2, uniform ones over 20, in the three types; exp2_fast is low
// by 5e-8 on average in every octave but the first).  With the correction 2e-8 or less
// is left.  Where all terms are exact (equal logits) the correction is the error, under
// half a step of the float32 result; where most terms vanish beside the largest (spread
// 6, 262144 float32 logits) the additions' own 1e-7 remains.
__device__ __forceinline__ double log_sum(float s) {
  return log((double)s) + 2.7e-8 * (1.0 - 1.0 / (double)s);
}
__device__ __forceinline__ float token_logp_of(const Online& o, float at_tok, bool inside,
                                               double inv_temp) {
  if (!inside) return __int_as_float(0x7fc00000);
  if (o.s == 0.0f) return -INFINITY;
  return (float)((double)(at_tok - o.m) * inv_temp - log_sum(o.s));
}
template <typename T>
__device__ __forceinline__ float token_logp(const Online& o, const T* p, int64_t vocab,
                                            int64_t tok, double inv_temp) {
  const bool inside = tok >= 0 && tok < vocab;
  return token_logp_of(o, inside ? to_f32(p[tok]) : 0.0f, inside, inv_temp);
}

// Reads this CTA's share of a row (`rank` of `split`) into `o`, as thread `tid` of
// `threads` (whole warps): rounds of kRowUnroll vectors for each thread, and the
// elements around the row's vectors.  A warp sums against its own maximum, raised
// where a round brings a larger one: all its lanes leave with the same o.m.
template <typename T, bool kEnt>
__device__ __forceinline__ void read_row(Online& o, const T* __restrict__ p, int64_t vocab,
                                         int tid, int threads, int rank, int split, Scale2 c) {
  constexpr int N = Vec16<T>::N;
  const RowSpan sp = row_span(p, vocab);
  const int body = (int)sp.body, share = (body + split - 1) / split;
  const int v0 = min(body, share * rank), v1 = min(body, v0 + share);
  const uint4* at = reinterpret_cast<const uint4*>(p + sp.head) + v0 + tid;
  const int round = kRowUnroll * threads;
  int left = v1 - v0;
  for (; left >= round; left -= round, at += round) {
    uint4 u[kRowUnroll];
#pragma unroll
    for (int k = 0; k < kRowUnroll; ++k) u[k] = __ldg(at + k * threads);
    float mx = max_of(u[0], (const T*)nullptr);
#pragma unroll
    for (int k = 1; k < kRowUnroll; ++k) mx = fmaxf(mx, max_of(u[k], (const T*)nullptr));
    mx = warp_max(mx);
    if (mx > o.m) rebase<kEnt>(o, mx, c);
    absorb<T, kEnt>(o, u, c);
  }
  // what is left of a round, and the row's ends (fewer than two vectors' elements)
  const int64_t tail0 = sp.head + sp.body * N;
  const int edge = rank == 0 ? (int)(sp.head + (vocab - tail0)) : 0;
  if (left > 0 || edge > 0) {
    uint4 u[kRowUnroll];
    float mx = -FLT_MAX, f = 0.0f;
#pragma unroll
    for (int k = 0; k < kRowUnroll; ++k)
      if (tid + k * threads < left) {
        u[k] = __ldg(at + k * threads);
        mx = fmaxf(mx, max_of(u[k], (const T*)nullptr));
      }
    if (tid < edge) {
      f = to_f32(p[tid < sp.head ? tid : tail0 + tid - sp.head]);
      mx = fmaxf(mx, f);
    }
    mx = warp_max(mx);
    if (mx > o.m) rebase<kEnt>(o, mx, c);
#pragma unroll
    for (int k = 0; k < kRowUnroll; ++k)
      if (tid + k * threads < left) {
        const uint4 one[1] = {u[k]};
        absorb<T, kEnt>(o, one, c);
      }
    if (tid < edge) {
      const float d = f - o.m, x = exp_scaled(d, c);
      o.s += x;
      if (kEnt) o.w = fmaf(x, fmaxf(d, c.low), o.w);
    }
  }
}

struct RowCoef {
  float m, c;       // exponent: (z - m) * c
  float cp, ce, k;  // d = e * (cp + ce * ((z - m) * inv_temp + k))
  float inv_temp;
  float low;  // what z - m counts as where it is less (exp_low)
  float hit;  // added at the token
};

template <bool kEnt>
__device__ __forceinline__ float grad_at(float z, const RowCoef& q) {
  const float d = z - q.m;
  const float e = exp2_fast(d * q.c);
  if (!kEnt) return e * q.cp;
  return e * fmaf(q.ce, fmaf(fmaxf(d, q.low), q.inv_temp, q.k), q.cp);
}

template <typename T, bool kEnt>
__device__ __forceinline__ uint4 grad_vec(const uint4& u, const RowCoef& q) {
  constexpr int N = Vec16<T>::N;
  float f[N];
  unpack(u, f, (const T*)nullptr);
  const f32x2 nm = pair(-q.m, -q.m), c = pair(q.c, q.c), cp = pair(q.cp, q.cp);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 d = add2(pair(f[i], f[i + 1]), nm);
    const float2 x = parts(mul2(d, c));
    const f32x2 e = pair(exp2_fast(x.x), exp2_fast(x.y));
    float2 r;
    if (!kEnt) {
      r = parts(mul2(e, cp));
    } else {
      const float2 t = parts(d);
      const f32x2 l = fma2(pair(fmaxf(t.x, q.low), fmaxf(t.y, q.low)),
                           pair(q.inv_temp, q.inv_temp), pair(q.k, q.k));
      r = parts(mul2(e, fma2(pair(q.ce, q.ce), l, cp)));
    }
    f[i] = r.x;
    f[i + 1] = r.y;
  }
  return pack(f, (const T*)nullptr);
}

// Writes the gradient of vectors [v0, v1) of a row (cut by the output's 16-byte
// boundaries) and, where `edges`, of the elements around its vectors.
// same: the logits' row lies on the output's phase.
template <typename T, bool kEnt>
__device__ __forceinline__ void write_grad(const T* __restrict__ p, T* __restrict__ out,
                                           int64_t vocab, int v0, int v1, bool edges, bool same,
                                           int lane, int lanes, int64_t tok, const RowCoef& q) {
  constexpr int N = Vec16<T>::N;
  const RowSpan sp = row_span(out, vocab);
  uint4* ob = reinterpret_cast<uint4*>(out + sp.head) + v0 + lane;
  const T* first = p + sp.head + ((int64_t)v0 + lane) * N;
  int left = v1 - v0 - lane;
  if (same) {
    const uint4* ib = reinterpret_cast<const uint4*>(first);
    for (; left > (kRowUnroll - 1) * lanes;
         left -= kRowUnroll * lanes, ib += kRowUnroll * lanes, ob += kRowUnroll * lanes) {
      uint4 u[kRowUnroll];
#pragma unroll
      for (int k = 0; k < kRowUnroll; ++k) u[k] = __ldg(ib + k * lanes);
#pragma unroll
      for (int k = 0; k < kRowUnroll; ++k) __stcs(ob + k * lanes, grad_vec<T, kEnt>(u[k], q));
    }
    for (; left > 0; left -= lanes, ib += lanes, ob += lanes)
      __stcs(ob, grad_vec<T, kEnt>(__ldg(ib), q));
  } else {
    for (; left > 0; left -= lanes, first += (int64_t)lanes * N, ob += lanes) {
      T t[N];
#pragma unroll
      for (int j = 0; j < N; ++j) t[j] = first[j];
      uint4 u;
      memcpy(&u, t, 16);
      *ob = grad_vec<T, kEnt>(u, q);
    }
  }
  const int64_t tail0 = sp.head + sp.body * N;
  if (edges) {
    const int edge = (int)(sp.head + (vocab - tail0));
    for (int e = lane; e < edge; e += lanes) {
      const int64_t at = e < sp.head ? e : tail0 + e - sp.head;
      out[at] = from_f32<T>(grad_at<kEnt>(to_f32(p[at]), q) + (at == tok ? q.hit : 0.0f));
    }
  }
  // the token's own element, by the thread that wrote its vector
  if (tok >= sp.head && tok < tail0) {
    const int64_t tv = (tok - sp.head) / N;
    if (tv >= v0 && tv < v1 && (tv - v0) % lanes == lane)
      out[tok] = from_f32<T>(grad_at<kEnt>(to_f32(p[tok]), q) + q.hit);
  }
}

template <typename T>
__device__ __forceinline__ void write_zeros(T* __restrict__ out, int64_t vocab, int v0, int v1,
                                            bool edges, int lane, int lanes) {
  const RowSpan sp = row_span(out, vocab);
  uint4* ob = reinterpret_cast<uint4*>(out + sp.head);
  for (int i = v0 + lane; i < v1; i += lanes) __stcs(ob + i, make_uint4(0, 0, 0, 0));
  if (!edges) return;
  const int64_t tail0 = sp.head + sp.body * Vec16<T>::N;
  const int edge = (int)(sp.head + (vocab - tail0));
  for (int e = lane; e < edge; e += lanes)
    out[e < sp.head ? e : tail0 + e - sp.head] = from_f32<T>(0.0f);
}

// 1 / s, 0 for a row of nothing but -inf (no gradient), NaN for NaN.
__device__ __forceinline__ float inverse_sum(float s) {
  return s > 0.0f ? 1.0f / s : (s == 0.0f ? 0.0f : s);
}

// hi is below v, and v - hi is lo > 0: -inf times either is -inf.
inline void halves(double v, float& hi, float& lo) {
  hi = (float)v;
  if ((double)hi >= v) hi = std::nextafterf(hi, 0.0f);
  lo = (float)(v - (double)hi);
}
inline Scale2 scale2(double inv_temp) {
  Scale2 c;
  halves(inv_temp * 1.4426950408889634, c.hi, c.lo);
  halves(inv_temp, c.inv, c.inv_lo);
  c.low = exp_low(c.inv);
  return c;
}

}  // namespace sinkslot
