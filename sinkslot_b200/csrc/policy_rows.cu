// policy_rows.cu -- the policy loss from logits larger than L2: one pass over the
// rows gives each token's log-probability and its row's gradient, and the logits
// are read from memory once.
//
// A cluster of CTAs takes a row, 64 KB of it for each CTA: it sums its slice, swaps
// sums with the cluster through distributed shared memory, works out the token's
// coefficient and turns its slice into the gradient, reading it again from L2, where
// the slices under way (47 MB at 5 CTAs on each SM) stay: 314 MB came from memory
// for 310 MB of logits.  Stores are marked to leave L2 first.
//
// Each CTA spends its time in turn on loads, on the swap and on stores, so several fill
// the memory's time best, as long as L2 holds them.  Threads x CTAs on an SM x KB, us
// for 8192 x 131072 bf16, 8192 x 50021 fp16, 4096 x 65536 fp32:
//   256 x 5 x 64  777 335 386     256 x 4 x 64  815 363 404     256 x 6 x 64  845 316 434
//   128 x 10 x 32 802 372 379     128 x 8 x 64  925 344 479     512 x 2 x 128 826 371 412
//   1024 x 1, whole rows          917 572 446
//   log-probabilities and gradient by their own kernels, three passes: 988 391 495
// What bounds it: exponentials (two for each element) hold their unit for 66% of the
// time, and memory runs at 5.5 of 6.5 TB/s.
//
// A persistent form with the rows in shared memory (bulk copies in and out, warps by
// role, sums exchanged a row ahead) was measured at 1013 us: a row's exchange took
// longer than a row, and clusters of SMs left 11% of the GPU idle.
#include <cooperative_groups.h>

#include "common.cuh"
#include "policy.cuh"
#include "row.cuh"
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

namespace cg = cooperative_groups;

constexpr int kSweepThreads = 256;
constexpr int kSweepCtas = 5;              // on each SM
constexpr int64_t kSweepBytes = 64 << 10;  // of a row, for each CTA
constexpr int kMaxCluster = 8;

template <typename T>
__global__ void __launch_bounds__(kSweepThreads, kSweepCtas) policy_rows_kernel(
    LogitRows r, PolicyTerms t, PolicyEdges e, PolicyRows w, int split, float grad_scale,
    float* __restrict__ logp, T* __restrict__ dz, int64_t dz_stride) {
  constexpr int kWarps = kSweepThreads / 32;
  __shared__ Online warp_part[kWarps];
  __shared__ Online cta_part[kMaxCluster];
  __shared__ RowCoef coef;
  __shared__ bool idle;
  const int64_t row = blockIdx.x / (unsigned)split;
  const int rank = (int)(blockIdx.x % (unsigned)split);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* p = static_cast<const T*>(r.z) + row * r.stride;
  T* out = dz + row * dz_stride;
  const int body = (int)row_span(p, r.vocab).body;  // (the output's row is on the same phase)
  const int share = (body + split - 1) / split;
  const int v0 = min(body, share * rank), v1 = min(body, v0 + share);
  if (r.mask && !r.mask[row]) {  // the whole cluster leaves
    if (rank == 0 && threadIdx.x == 0) logp[row] = 0.0f;
    write_zeros(out, r.vocab, v0, v1, rank == 0, threadIdx.x, kSweepThreads);
    return;
  }
  if (split > 1) cluster_started();
  const int64_t tok = token_at(r.tokens, r.token_bytes, row);
  const bool inside = tok >= 0 && tok < r.vocab;
  // what the coefficient needs besides the sums, on its way while the row is read
  float zt = 0.0f, old_logp = 0.0f, ref_logp = 0.0f, adv = 0.0f, weight = 0.0f;
  if (threadIdx.x == 0) {
    const int seq = w.owner[row];
    if (inside) zt = to_f32(p[tok]);
    old_logp = t.old_logp[row];
    if (t.ref_logp) ref_logp = t.ref_logp[row];
    if (seq >= 0) {  // (a token outside the sequences is not counted)
      adv = t.adv[t.adv_per_token ? row : seq];
      weight = w.norm[0];
      if (t.sequence_average) weight = weight / (float)w.counts[seq];
    }
  }
  Online o;
  read_row<T, false>(o, p, r.vocab, threadIdx.x, kSweepThreads, rank, split, r.scale);
  join_warp<false>(o, r.scale);
  if (lane == 0) warp_part[warp] = o;
  __syncthreads();
  if (split > 1) cluster_wait_started();
  if (warp == 0) {
    o = lane < kWarps ? warp_part[lane] : Online();
    join_warp<false>(o, r.scale);
    if (split > 1 && lane < split)
      cg::this_cluster().map_shared_rank(cta_part, lane)[rank] = o;
  }
  if (split > 1) {
    cg::this_cluster().sync();
    if (warp == 0) {
      o = lane < split ? cta_part[lane] : Online();
      join_warp<false>(o, r.scale);
    }
  }
  if (threadIdx.x == 0) {
    const float lp = token_logp_of(o, zt, inside, r.inv_temp);
    if (rank == 0) logp[row] = lp;
    const float g = weight == 0.0f ? 0.0f
                                   : policy_term(t, e, lp, old_logp, ref_logp, adv).coef *
                                         weight * grad_scale * (float)r.inv_temp;
    RowCoef q = {};
    q.m = o.m;
    q.c = (float)(r.inv_temp * 1.4426950408889634);
    q.cp = -g * inverse_sum(o.s);
    q.hit = o.s == 0.0f ? 0.0f : g;
    coef = q;
    idle = g == 0.0f;
  }
  __syncthreads();
  if (idle) {  // no gradient (outside the sequences, or clipped): zeros, whatever the row holds
    write_zeros(out, r.vocab, v0, v1, rank == 0, threadIdx.x, kSweepThreads);
    return;
  }
  const RowCoef q = coef;
  write_grad<T, false>(p, out, r.vocab, v0, v1, rank == 0, true, threadIdx.x, kSweepThreads, tok,
                       q);
}

// CTAs for each row, 0 where a cluster does not hold one.
static int rows_split(const LogitRows& r) {
  const int64_t row = r.vocab * dtype_bytes(r.dtype);
  for (int split = 1; split <= kMaxCluster; split *= 2)
    if (row <= split * kSweepBytes) return split;
  return 0;
}

// From 24 KB a row on: 16384 rows of 32 KB 213 us (257 in three passes), of 16 KB 142
// (129).
bool policy_rows_fit(const LogitRows& r, const void* dz, int64_t dz_stride) {
  const int64_t size = dtype_bytes(r.dtype), row = r.vocab * size;
  const bool same = ((reinterpret_cast<uintptr_t>(r.z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0 &&
                    (r.stride - dz_stride) * size % 16 == 0;
  return same && row >= (24 << 10) && r.rows * row >= (128 << 20) && rows_split(r) > 0;
}

template <typename T>
static int launch_rows(const LogitRows& r, const PolicyTerms& t, const PolicyRows& w,
                       float grad_scale, float* logp, void* dz, int64_t dz_stride,
                       cudaStream_t st) {
  const int split = rows_split(r);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(r.rows * split));
  cfg.blockDim = dim3(kSweepThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  SINKSLOT_CUDA_TRY(cudaLaunchKernelEx(&cfg, policy_rows_kernel<T>, r, t, policy_edges(t), w,
                                       split, grad_scale, logp, (T*)dz, dz_stride));
  return kOk;
}

int policy_rows(const LogitRows& rows, const PolicyTerms& t, const PolicyRows& w, float grad_scale,
                float* logp, void* dz, int64_t dz_stride, cudaStream_t st) {
  LogitRows r = rows;
  r.scale = scale2(r.inv_temp);
#define GO(T) return launch_rows<T>(r, t, w, grad_scale, logp, dz, dz_stride, st)
  if (r.dtype == kF32) GO(float);
  if (r.dtype == kF16) GO(__half);
  GO(__nv_bfloat16);
#undef GO
}

}  // namespace sinkslot
