// logprobs.cu -- log-probabilities (and entropies) of chosen tokens under rows
// of logits, and the logits' gradient.
//
//   z = logits / T,  m = max_v z_v,  s = sum_v exp(z_v - m)
//   logp = z_tok - m - ln s,   H = ln s - sum_v exp(z_v - m) (z_v - m) / s
//   dlogits_v = [g (1[v = tok] - p_v) - gH p_v (z_v - m - ln s + H)] / T
//
// Forward: one pass over the row with the running maximum and sum of a softmax, each
// warp against its own maximum; the warps' pairs are joined by block (and by cluster,
// where there are few rows) in a fixed order.  (m, s) are kept for the backward pass,
// in the logits' own scale: differences from m are taken before they are scaled, so
// rows at the type's lowest value or far from zero lose nothing.
//
// Memory bounds it, once the instructions are few enough: 8192 x 131072 bf16 forward
// 316 us (6.8 TB/s; 380 us with an instruction for each element's step), gradient
// 656 us (6.5 TB/s); 4096 x 32768 fp32 82 and 164 us.  With the entropy of fp16 rows
// instructions still show: 1537 of 2049 x 50021 34 us (4.5 TB/s), gradient 59 us.
#include <cfloat>
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "row.cuh"
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 256;
constexpr int kMaxSplit = 8;  // CTAs of a cluster that share a row

template <typename T, bool kEnt>
__device__ __forceinline__ void write_row(const Online& o, const T* p, int64_t vocab, int64_t row,
                                          int64_t tok, double inv_temp, float* logp,
                                          float* entropy, float2* stats) {
  logp[row] = token_logp(o, p, vocab, tok, inv_temp);
  if (kEnt)
    entropy[row] =
        o.s == 0.0f ? 0.0f : (float)(log_sum(o.s) - inv_temp * (double)(o.w / o.s));
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
  if (split > 1) cluster_started();
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  const Scale2 c = r.scale;
  Online o;
  read_row<T, kEnt>(o, p, r.vocab, threadIdx.x, kRowThreads, rank, split, c);
  join_warp<kEnt>(o, c);
  if (lane == 0) warp_part[warp] = o;
  __syncthreads();
  if (split > 1) cluster_wait_started();
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

int check_rows(const LogitRows& r) {
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
// (up to a cluster of 8) as leave each CTA 8 KB.  Split for balance, with more rows,
// they lose more by joining than they gain (1537 rows of 100 KB: 34.5 us by one CTA
// each, 37.3 by two).
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
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kRowThreads) logprob_grad_kernel(LogitRows r, LogitGrad g,
                                                                   int share) {
  // from the last row on: the forward pass left the end of the logits in L2
  const int64_t row = r.rows - 1 - (int64_t)blockIdx.x;
  const int64_t tok = token_at(r.tokens, r.token_bytes, row);
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  T* out = static_cast<T*>(g.dz) + row * g.dz_stride;
  const int body = (int)row_span(out, r.vocab).body;
  const int v0 = min(body, share * (int)blockIdx.y), v1 = min(body, v0 + share);
  const bool edges = blockIdx.y == 0;
  RowCoef q;
  const float2 ms = g.stats[row];
  q.inv_temp = (float)r.inv_temp;
  float f = q.inv_temp * g.scale;
  if (g.scale_dev) f *= g.scale_dev[0];
  const float gp = g.g ? g.g[row * g.g_stride] * f : 0.0f;
  const float ge = kEnt && g.g_entropy ? g.g_entropy[row * g.g_entropy_stride] * f : 0.0f;
  // no gradient: zeros, whatever the row holds (0 * NaN is not taken)
  if (tok == r.ignore || (r.mask && !r.mask[row]) || (gp == 0.0f && ge == 0.0f)) {
    write_zeros(out, r.vocab, v0, v1, edges, threadIdx.x, kRowThreads);
    return;
  }
  const float rs = inverse_sum(ms.y);
  q.m = ms.x;
  q.c = (float)(r.inv_temp * 1.4426950408889634);
  q.cp = -gp * rs;
  q.ce = q.k = q.low = 0.0f;
  if (kEnt) {
    q.ce = -ge * rs;
    q.low = exp_low(q.inv_temp);
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
// usually 1, and then nothing is touched: 7 us, the launch among them).  Otherwise it
// reads and writes everything: 8192 x 131072 bf16 729 us (5.9 TB/s), 2049 x 50021 fp16
// 74 us, 4096 x 32768 fp32 200 us, in bursts at 1.97 GHz.
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
