// logprobs.cu -- log-probabilities (and entropies) of chosen tokens under rows
// of logits, and the logits' gradient.
//
//   z = logits / T,  m = max_v z_v,  s = sum_v exp(z_v - m)
//   logp = z_tok - m - ln s,   H = ln s - sum_v exp(z_v - m) (z_v - m) / s
//   dlogits_v = [g (1[v = tok] - p_v) - gH p_v (z_v - m - ln s + H)] / T
//
// Forward: one pass over the row with the running maximum and sum of a softmax,
// each thread's own pair rescaled once for every 64 bytes that it reads; the
// pairs are joined by block (and by cluster, where there are few rows) in a
// fixed order.  (m, s) are kept for the backward pass, in the logits' own scale:
// differences from m are taken before they are scaled, so rows at the type's
// lowest value or far from zero lose nothing.
#include <cfloat>
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;  // 16-byte loads in flight per thread
constexpr int kMaxSplit = 8;   // CTAs of a cluster that share a row

// log2(e) / T as the sum of two floats.  One float's rounding (up to 2^-25 of every
// exponent) would have the same sign for a whole row: at differences of -10 to -20 it
// shifted each log-probability by 1.5e-7, which does not average out over a
// sequence (measured on 2000-token sums).
// hi is the next float below the value, so that lo > 0 and -inf times either is -inf.
__device__ __forceinline__ float exp_scaled(float d, Scale2 c) {
  return exp2_fast(fmaf(d, c.hi, d * c.lo));
}

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
  const float a = expf(d * c.inv);
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
        w = fma2(e, pair(fmaxf(t.x, -1e30f), fmaxf(t.y, -1e30f)), w);
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

template <bool kEnt>
__device__ __forceinline__ void join(Online& a, const Online& b, Scale2 c) {
  const float m = fmaxf(a.m, b.m);
  Online t = b;
  rebase<kEnt>(a, m, c);
  rebase<kEnt>(t, m, c);
  a.s += t.s;
  if (kEnt) a.w += t.w;
}

template <bool kEnt>
__device__ __forceinline__ void join_warp(Online& o, Scale2 c) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    Online t;
    t.m = __shfl_xor_sync(0xffffffffu, o.m, d);
    t.s = __shfl_xor_sync(0xffffffffu, o.s, d);
    if (kEnt) t.w = __shfl_xor_sync(0xffffffffu, o.w, d);
    join<kEnt>(o, t, c);
  }
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t r) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[r]
                    : (int64_t) static_cast<const int32_t*>(tokens)[r];
}

// Reads this CTA's share of a row (`rank` of `split`) into `o`, as thread `lane` of
// `lanes`: rounds of kRowUnroll vectors, then vector by vector, then the elements
// before the first boundary and behind the last.
template <typename T, bool kEnt>
__device__ __forceinline__ void read_row(Online& o, const T* __restrict__ p, int64_t vocab,
                                         int lane, int lanes, int rank, int split, Scale2 c) {
  constexpr int N = Vec16<T>::N;
  const RowSpan sp = row_span(p, vocab);
  const int body = (int)sp.body, share = (body + split - 1) / split;
  const int v0 = min(body, share * rank), v1 = min(body, v0 + share);
  const uint4* at = reinterpret_cast<const uint4*>(p + sp.head) + v0 + lane;
  int left = v1 - v0 - lane;  // vectors from `at` on, of which every lanes-th is this thread's
  for (; left > (kRowUnroll - 1) * lanes; left -= kRowUnroll * lanes, at += kRowUnroll * lanes) {
    uint4 u[kRowUnroll];
#pragma unroll
    for (int k = 0; k < kRowUnroll; ++k) u[k] = __ldg(at + k * lanes);
    float mx = max_of(u[0], (const T*)nullptr);
#pragma unroll
    for (int k = 1; k < kRowUnroll; ++k) mx = fmaxf(mx, max_of(u[k], (const T*)nullptr));
    rebase<kEnt>(o, fmaxf(o.m, mx), c);
    absorb<T, kEnt>(o, u, c);
  }
  for (; left > 0; left -= lanes, at += lanes) {
    const uint4 u[1] = {__ldg(at)};
    rebase<kEnt>(o, fmaxf(o.m, max_of(u[0], (const T*)nullptr)), c);
    absorb<T, kEnt>(o, u, c);
  }
  if (rank == 0) {
    const int64_t tail0 = sp.head + sp.body * N;
    const int edge = (int)(sp.head + (vocab - tail0));
    for (int e = lane; e < edge; e += lanes) {
      const float f = to_f32(p[e < sp.head ? e : tail0 + e - sp.head]);
      rebase<kEnt>(o, fmaxf(o.m, f), c);
      const float d = f - o.m, x = exp_scaled(d, c);
      o.s += x;
      if (kEnt) o.w = fmaf(x, fmaxf(d, -1e30f), o.w);
    }
  }
}

template <typename T, bool kEnt>
__device__ __forceinline__ void write_row(const Online& o, const T* p, int64_t vocab, int64_t row,
                                          int64_t tok, double inv_temp, float* logp, float* entropy,
                                          float2* stats) {
  // in fp64 until the result is rounded: logf's error has a mean of its own, 1e-7
  // of a log-probability (measured), which a sequence's sum would keep
  const double ls = log((double)o.s);
  float v;
  if (tok < 0 || tok >= vocab) {
    v = __int_as_float(0x7fc00000);
  } else {
    v = o.s == 0.0f ? -INFINITY : (float)((double)(to_f32(p[tok]) - o.m) * inv_temp - ls);
  }
  logp[row] = v;
  if (kEnt) entropy[row] = o.s == 0.0f ? 0.0f : (float)(ls - inv_temp * (double)(o.w / o.s));
  stats[row] = make_float2(o.m, o.s);
}

// A warp for each row: rows of a few KB.
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kRowThreads) logprob_warp_kernel(LogitRows r,
                                                                   float* __restrict__ logp,
                                                                   float* __restrict__ entropy,
                                                                   float2* __restrict__ stats) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  if (row >= r.rows) return;
  const int64_t tok = token_at(r.tokens, r.token_bytes, row);
  if (tok == r.ignore || (r.mask && !r.mask[row])) {
    if (lane == 0) {
      logp[row] = 0.0f;
      if (kEnt) entropy[row] = 0.0f;
      stats[row] = make_float2(0.0f, 0.0f);
    }
    return;
  }
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  const Scale2 c = r.scale;
  Online o;
  read_row<T, kEnt>(o, p, r.vocab, lane, 32, 0, 1, c);
  join_warp<kEnt>(o, c);
  if (lane == 0) write_row<T, kEnt>(o, p, r.vocab, row, tok, r.inv_temp, logp, entropy, stats);
}

// A cluster of `split` CTAs for each row.
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kRowThreads) logprob_row_kernel(LogitRows r, int split,
                                                                  float* __restrict__ logp,
                                                                  float* __restrict__ entropy,
                                                                  float2* __restrict__ stats) {
  __shared__ Online warp_part[kRowThreads / 32];
  __shared__ Online cta_part[kMaxSplit];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / (unsigned)split;
  const int rank = (int)(blockIdx.x % (unsigned)split);
  const int64_t tok = token_at(r.tokens, r.token_bytes, row);
  if (tok == r.ignore || (r.mask && !r.mask[row])) {  // the whole cluster leaves
    if (rank == 0 && threadIdx.x == 0) {
      logp[row] = 0.0f;
      if (kEnt) entropy[row] = 0.0f;
      stats[row] = make_float2(0.0f, 0.0f);
    }
    return;
  }
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  const Scale2 c = r.scale;
  Online o;
  read_row<T, kEnt>(o, p, r.vocab, threadIdx.x, kRowThreads, rank, split, c);
  join_warp<kEnt>(o, c);
  if (lane == 0) warp_part[warp] = o;
  __syncthreads();
  if (warp == 0) {
    o = warp_part[lane & (kRowThreads / 32 - 1)];
    if (lane >= kRowThreads / 32) o = Online();
    join_warp<kEnt>(o, c);
    if (split > 1 && lane == 0) {
      Online* to = cg::this_cluster().map_shared_rank(cta_part, 0);
      to[rank] = o;
    }
  }
  if (split > 1) {
    cg::this_cluster().sync();
    if (rank != 0) return;
    if (warp == 0) {
      o = lane < split ? cta_part[lane] : Online();
      join_warp<kEnt>(o, c);
    }
  }
  if (threadIdx.x == 0)
    write_row<T, kEnt>(o, p, r.vocab, row, tok, r.inv_temp, logp, entropy, stats);
}

// Rows of at most this many bytes go to a warp each.
constexpr int64_t kWarpRowBytes = 4096;

static Scale2 scale2(double inv_temp) {
  const double c = inv_temp * 1.4426950408889634;
  float hi = (float)c;
  if ((double)hi >= c) hi = std::nextafterf(hi, 0.0f);
  return {hi, (float)(c - (double)hi), (float)inv_temp};
}

static int check_rows(const LogitRows& r) {
  SINKSLOT_REQUIRE(dtype_ok(r.dtype), "token_logprobs: dtype must be 0, 1 or 2");
  SINKSLOT_REQUIRE(r.rows >= 0 && r.vocab >= 1 && r.stride >= 0, "token_logprobs: bad sizes");
  SINKSLOT_REQUIRE(r.vocab <= int64_t(1) << 30, "token_logprobs: more than 2^30 tokens to choose");
  SINKSLOT_REQUIRE(r.token_bytes == 4 || r.token_bytes == 8,
                   "token_logprobs: tokens must be int32 or int64");
  SINKSLOT_REQUIRE(r.inv_temp >= 0.99e-30 && r.inv_temp <= 1.01e30,
                   "token_logprobs: temperature must be in [1e-30, 1e30]");
  SINKSLOT_REQUIRE(r.rows <= (int64_t(1) << 27), "token_logprobs: more than 2^27 rows");
  SINKSLOT_REQUIRE(r.rows == 0 || (r.z && r.tokens), "token_logprobs: null argument");
  return kOk;
}

// CTAs for each row: one while the rows fill the GPU twice over, else as many
// (up to a cluster of 8) as leave each CTA 8 KB.
static int row_split(const LogitRows& r) {
  int split = 1;
  const int64_t bytes = r.vocab * dtype_bytes(r.dtype);
  while (split < kMaxSplit && r.rows * split < 2 * num_sms() && bytes / (2 * split) >= 8192)
    split *= 2;
  return split;
}

template <typename T, bool kEnt>
static int launch_logprob(const LogitRows& r, float* logp, float* entropy, float2* stats,
                          cudaStream_t st) {
  if (r.vocab * (int64_t)sizeof(T) <= kWarpRowBytes) {
    const int64_t grid = ceil_div64(r.rows, kRowThreads / 32);
    logprob_warp_kernel<T, kEnt><<<(unsigned)grid, kRowThreads, 0, st>>>(r, logp, entropy, stats);
    SINKSLOT_CHECK_LAUNCH();
    return kOk;
  }
  const int split = row_split(r);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(r.rows * split));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  SINKSLOT_CUDA_TRY(
      cudaLaunchKernelEx(&cfg, logprob_row_kernel<T, kEnt>, r, split, logp, entropy, stats));
  return kOk;
}

int token_logprobs(const LogitRows& rows, float* logp, float* entropy, float2* stats,
                   cudaStream_t st) {
  LogitRows r = rows;
  SINKSLOT_TRY(check_rows(r));
  if (r.rows == 0) return kOk;
  r.scale = scale2(r.inv_temp);
  SINKSLOT_REQUIRE(logp && stats, "token_logprobs: null argument");
#define GO(T)                                                         \
  return entropy ? launch_logprob<T, true>(r, logp, entropy, stats, st) \
                 : launch_logprob<T, false>(r, logp, nullptr, stats, st)
  if (r.dtype == kF32) GO(float);
  if (r.dtype == kF16) GO(__half);
  GO(__nv_bfloat16);
#undef GO
}

// --------------------------------------------------------------------------
// Gradient: elementwise once (m, s, H) are known; a row's CTAs need nothing of
// one another.  Rows left out are filled with zeros and not read.
// --------------------------------------------------------------------------
struct RowCoef {
  float m, c;       // exponent: (z - m) * c
  float cp, ce, k;  // d = e * (cp + ce * ((z - m) * inv_temp + k))
  float inv_temp;
  float hit;  // added at the token
};

template <bool kEnt>
__device__ __forceinline__ float grad_at(float z, const RowCoef& q) {
  const float d = z - q.m;
  const float e = exp2_fast(d * q.c);
  if (!kEnt) return e * q.cp;
  return e * fmaf(q.ce, fmaf(fmaxf(d, -1e30f), q.inv_temp, q.k), q.cp);
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
      const f32x2 l = fma2(pair(fmaxf(t.x, -1e30f), fmaxf(t.y, -1e30f)),
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

template <typename T, bool kEnt>
__global__ void __launch_bounds__(kRowThreads) logprob_grad_kernel(LogitRows r, LogitGrad g,
                                                                   int share) {
  const int64_t row = blockIdx.x;
  const int64_t tok = token_at(r.tokens, r.token_bytes, row);
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  T* out = static_cast<T*>(g.dz) + row * g.dz_stride;
  const int body = (int)row_span(out, r.vocab).body;
  const int v0 = min(body, share * (int)blockIdx.y), v1 = min(body, v0 + share);
  const bool edges = blockIdx.y == 0;
  if (tok == r.ignore || (r.mask && !r.mask[row])) {
    write_zeros(out, r.vocab, v0, v1, edges, threadIdx.x, kRowThreads);
    return;
  }
  RowCoef q;
  const float2 ms = g.stats[row];
  q.inv_temp = (float)r.inv_temp;
  float f = q.inv_temp * g.scale;
  if (g.scale_dev) f *= g.scale_dev[0];
  const float gp = g.g ? g.g[row * g.g_stride] * f : 0.0f;
  const float rs = inverse_sum(ms.y);
  q.m = ms.x;
  q.c = (float)(r.inv_temp * 1.4426950408889634);
  q.cp = -gp * rs;
  q.ce = q.k = 0.0f;
  if (kEnt) {
    const float ge = g.g_entropy ? g.g_entropy[row * g.g_entropy_stride] * f : 0.0f;
    q.ce = -ge * rs;
    q.k = ms.y > 0.0f ? g.entropy[row] - logf(ms.y) : 0.0f;
  }
  q.hit = ms.y == 0.0f ? 0.0f : gp;
  const bool same = !((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(out)) & 15);
  write_grad<T, kEnt>(p, out, r.vocab, v0, v1, edges, same, threadIdx.x, kRowThreads, tok, q);
}

template <typename T>
static int launch_grad(const LogitRows& r, const LogitGrad& g, cudaStream_t st) {
  const int64_t body = ceil_div64(r.vocab, Vec16<T>::N);
  // pieces of a row: whole rows while they fill the GPU four times over, else
  // down to one round of loads for each CTA
  const int64_t least = (int64_t)kRowThreads * kRowUnroll;
  int64_t pieces = ceil_div64(4 * num_sms(), r.rows);
  if (pieces > ceil_div64(body, least)) pieces = ceil_div64(body, least);
  if (pieces < 1) pieces = 1;
  if (pieces > 65535) pieces = 65535;
  const int share = (int)ceil_div64(body, pieces);
  const dim3 grid((unsigned)r.rows, (unsigned)pieces);
  if (g.g_entropy)
    logprob_grad_kernel<T, true><<<grid, kRowThreads, 0, st>>>(r, g, share);
  else
    logprob_grad_kernel<T, false><<<grid, kRowThreads, 0, st>>>(r, g, share);
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

int token_logprobs_grad(const LogitRows& r, const LogitGrad& g, cudaStream_t st) {
  SINKSLOT_TRY(check_rows(r));
  if (r.rows == 0) return kOk;
  SINKSLOT_REQUIRE(g.dz && g.stats && (g.g || g.g_entropy) && (!g.g_entropy || g.entropy),
                   "token_logprobs_grad: null argument");
  SINKSLOT_REQUIRE(g.dz_stride >= r.vocab || r.rows == 1, "token_logprobs_grad: rows overlap");
  if (r.dtype == kF32) return launch_grad<float>(r, g, st);
  if (r.dtype == kF16) return launch_grad<__half>(r, g, st);
  return launch_grad<__nv_bfloat16>(r, g, st);
}

// --------------------------------------------------------------------------
// In-place scaling of a finished gradient by g / grad_scale (read on the device:
// usually 1, and then nothing is touched).
// --------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kRowThreads) scale_rows_kernel(T* dz, int64_t stride,
                                                                 int64_t rows, int64_t vocab,
                                                                 const float* __restrict__ g,
                                                                 float grad_scale) {
  const float f = g[0] / grad_scale;
  if (f == 1.0f) return;
  constexpr int N = Vec16<T>::N;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    T* p = dz + row * stride;
    const RowSpan sp = row_span(p, vocab);
    uint4* b = reinterpret_cast<uint4*>(p + sp.head);
    for (int64_t i = threadIdx.x; i < sp.body; i += kRowThreads) {
      float v[N];
      unpack(b[i], v, (const T*)nullptr);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] *= f;
      b[i] = pack(v, (const T*)nullptr);
    }
    const int64_t tail0 = sp.head + sp.body * N;
    const int64_t edge = sp.head + (vocab - tail0);
    for (int64_t e = threadIdx.x; e < edge; e += kRowThreads) {
      T* q = p + (e < sp.head ? e : tail0 + e - sp.head);
      *q = from_f32<T>(to_f32(*q) * f);
    }
  }
}

int scale_rows(void* dz, int dtype, int64_t stride, int64_t rows, int64_t vocab, const float* g,
               float grad_scale, cudaStream_t st) {
  SINKSLOT_REQUIRE(dtype_ok(dtype) && rows >= 0 && vocab >= 1 && g, "scale_rows: bad args");
  if (rows == 0) return kOk;
  const int64_t cap = (int64_t)num_sms() * 8;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
  if (dtype == kF32)
    scale_rows_kernel<float><<<grid, kRowThreads, 0, st>>>((float*)dz, stride, rows, vocab, g,
                                                           grad_scale);
  else if (dtype == kF16)
    scale_rows_kernel<__half><<<grid, kRowThreads, 0, st>>>((__half*)dz, stride, rows, vocab, g,
                                                            grad_scale);
  else
    scale_rows_kernel<__nv_bfloat16><<<grid, kRowThreads, 0, st>>>(
        (__nv_bfloat16*)dz, stride, rows, vocab, g, grad_scale);
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

}  // namespace sinkslot
