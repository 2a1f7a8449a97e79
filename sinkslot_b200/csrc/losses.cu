// losses.cu -- losses over the log-probabilities of packed sequences, with the
// gradient of each token.
//
//   policy      r = exp(logp - old), L = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta KL,
//               averaged over the counted tokens, or over the sequences' means;
//               KL from d = ref - logp: k1 -d, k2 d^2 / 2, k3 e^d - d - 1
//   preference  R_i = sum_t (logp - ref) (or its mean), h = beta (R_chosen - R_rejected),
//               -(1 - ls) log sigma(h) - ls log sigma(-h), max(0, 1 - h), or
//               (h / beta - 1 / (2 beta))^2, averaged over the pairs
//
// Both read a few bytes for each token: launch latency bounds the ordinary
// sizes.  A cluster of CTAs takes a sequence (8 of them where there are few),
// its sums are joined in a fixed order in fp64, and one CTA, launched so that it
// starts while the first kernel ends, joins the sequences.  512 sequences, 393216
// tokens: 7.4 + 3.9 us; 32 sequences, 16384 tokens, clipped with a KL term: 10.9 +
// 3.6 us.  Up to 8 sequences go in one launch (8 of 250 tokens: 6.1 us).
#include <cmath>
#include <cooperative_groups.h>

#include "common.cuh"
#include "policy.cuh"
#include "training.h"

namespace sinkslot {

namespace cg = cooperative_groups;

constexpr int kLossThreads = 512;
constexpr int kLossWarps = kLossThreads / 32;
constexpr int kLossSplit = 8;
constexpr int kAtOnce = 4;  // tokens that a thread loads together

struct Sums {
  double a, b, c;
};

// Sums over the CTA's threads and the cluster's CTAs, in a fixed order; every
// thread of the cluster gets them.  `turn` alternates between consecutive calls.
struct ClusterSum {
  Sums warp[kLossWarps];
  Sums cta[2][kLossSplit];
};

__device__ __forceinline__ Sums warp_sums(Sums v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    v.a += __shfl_xor_sync(0xffffffffu, v.a, o);
    v.b += __shfl_xor_sync(0xffffffffu, v.b, o);
    v.c += __shfl_xor_sync(0xffffffffu, v.c, o);
  }
  return v;
}

// (`first`: the kernel's first call; it began with cluster_started() where split > 1)
__device__ __forceinline__ Sums cluster_sums(Sums v, ClusterSum& sh, int turn, int rank,
                                             int split, bool first = false) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_sums(v);
  __syncthreads();
  if (lane == 0) sh.warp[warp] = v;
  __syncthreads();
  if (first && split > 1) cluster_wait_started();
  if (warp == 0) {
    const Sums zero = {0.0, 0.0, 0.0};
    v = warp_sums(lane < kLossWarps ? sh.warp[lane] : zero);
    if (lane < split) {
      if (split > 1)
        cg::this_cluster().map_shared_rank(&sh.cta[turn][0], lane)[rank] = v;
      else
        sh.cta[turn][0] = v;
    }
  }
  if (split > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  Sums t = {0.0, 0.0, 0.0};
  for (int k = 0; k < split; ++k) {
    t.a += sh.cta[turn][k].a;
    t.b += sh.cta[turn][k].b;
    t.c += sh.cta[turn][k].c;
  }
  return t;
}

// Bounds of sequence i, kept within the tokens whatever the offsets hold.
__device__ __forceinline__ int64_t offset_at(const Packed& p, int64_t i) {
  int64_t v = p.offset_bytes == 8 ? static_cast<const int64_t*>(p.offsets)[i]
                                  : (int64_t) static_cast<const int32_t*>(p.offsets)[i];
  v = v < 0 ? 0 : v;
  return v > p.tokens ? p.tokens : v;
}
__device__ __forceinline__ void bounds(const Packed& p, int64_t i, int64_t& lo, int64_t& hi) {
  lo = p.offsets ? offset_at(p, i) : 0;
  hi = p.offsets ? offset_at(p, i + 1) : p.tokens;
  if (hi < lo) hi = lo;
}

// Zeros for the tokens before the first sequence and behind the last.
__device__ __forceinline__ void zero_outside(const Packed& p, int64_t seq, int64_t at, int64_t step,
                                             float* out) {
  if (!p.offsets || !out) return;
  if (seq == 0)
    for (int64_t t = at, e = offset_at(p, 0); t < e; t += step) out[t] = 0.0f;
  if (seq == p.count - 1)
    for (int64_t t = offset_at(p, p.count) + at; t < p.tokens; t += step) out[t] = 0.0f;
}

// One sequence, by `split` CTAs of a cluster: part = {loss, kl, clipped, counted}.
__device__ __forceinline__ void policy_seq(const Packed& p, const PolicyTerms& t,
                                           const PolicyEdges& e, int64_t seq, int rank, int split,
                                           ClusterSum& sh, double4* part,
                                           float* __restrict__ coef) {
  const int64_t at = (int64_t)rank * kLossThreads + threadIdx.x;
  const int64_t step = (int64_t)split * kLossThreads;
  int64_t lo, hi;
  bounds(p, seq, lo, hi);
  double inv = 1.0;
  if (t.sequence_average) {
    double n = (double)(hi - lo);
    if (p.mask) {
      int64_t k = 0;
#pragma unroll 4
      for (int64_t i = lo + at; i < hi; i += step) k += p.mask[i] != 0;
      n = cluster_sums({(double)k, 0.0, 0.0}, sh, 0, rank, split, true).a;
    }
    inv = n > 0.0 ? 1.0 / n : 0.0;
  }
  const float finv = (float)inv;
  Sums s = {0.0, 0.0, 0.0};
  int64_t n = 0;
  const float seq_adv = t.adv_per_token || lo >= hi ? 0.0f : t.adv[seq];
  for (int64_t i = lo + at; i < hi; i += kAtOnce * step) {
    // what the tokens need is loaded for all of them at once, masked ones too (their
    // values are not looked at)
    bool on[kAtOnce];
    float logp[kAtOnce], old_logp[kAtOnce], ref_logp[kAtOnce], adv[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t j = i + k * step;
      on[k] = j < hi;
      logp[k] = old_logp[k] = ref_logp[k] = 0.0f;
      adv[k] = seq_adv;
      if (j < hi) {
        if (p.mask) on[k] = p.mask[j] != 0;
        logp[k] = t.logp[j];
        old_logp[k] = t.old_logp[j];
        if (t.ref_logp) ref_logp[k] = t.ref_logp[j];
        if (t.adv_per_token) adv[k] = t.adv[j];
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t j = i + k * step;
      if (j >= hi) break;
      float cf = 0.0f;
      if (on[k]) {
        const TokenTerm o = policy_term(t, e, logp[k], old_logp[k], ref_logp[k], adv[k]);
        s.a += (double)o.loss;
        s.b += (double)o.kl;
        n += 1 + ((int64_t)o.clipped << 32);
        cf = o.coef * finv;
      }
      if (coef) coef[j] = cf;
    }
  }
  zero_outside(p, seq, at, step, coef);
  // counts of counted and of clipped tokens, both under 2^32, apart in fp64
  s.c = (double)(n & 0xffffffff);
  const Sums f = cluster_sums(s, sh, 1, rank, split, !(t.sequence_average && p.mask));
  const Sums k = cluster_sums({(double)(n >> 32), 0.0, 0.0}, sh, 0, rank, split);
  if (rank == 0 && threadIdx.x == 0) part[seq] = make_double4(f.a * inv, f.b * inv, k.a, f.c);
}

__global__ void __launch_bounds__(kLossThreads) policy_seq_kernel(Packed p, PolicyTerms t,
                                                                  PolicyEdges e, int split,
                                                                  double4* __restrict__ part,
                                                                  float* __restrict__ coef) {
  __shared__ ClusterSum sh;
  if (split > 1) cluster_started();
  policy_seq(p, t, e, blockIdx.x / (unsigned)split, (int)(blockIdx.x % (unsigned)split), split, sh,
             part, coef);
  chain_release();
}

// Sums over one CTA of kLossThreads (no cluster).
__device__ __forceinline__ Sums cta_sums(Sums v, ClusterSum& sh, int turn) {
  return cluster_sums(v, sh, turn, 0, 1);
}

// All sequences, by one CTA.
__device__ __forceinline__ void policy_end(const double4* part, int64_t count, int by_sequence,
                                           ClusterSum& sh, float* __restrict__ values) {
  Sums s = {0.0, 0.0, 0.0}, k = {0.0, 0.0, 0.0};
  for (int64_t i = threadIdx.x; i < count; i += kLossThreads) {
    const double4 v = part[i];
    s.a += v.x;
    s.b += v.y;
    s.c += v.z;
    k.a += v.w;
    k.b += v.w > 0.0 ? 1.0 : 0.0;
  }
  s = cta_sums(s, sh, 0);
  k = cta_sums(k, sh, 1);
  if (threadIdx.x == 0) {
    const double over = by_sequence ? k.b : k.a;
    const double norm = over > 0.0 ? 1.0 / over : 0.0;
    values[0] = (float)(s.a * norm);
    values[1] = (float)(s.b * norm);
    values[2] = k.a > 0.0 ? (float)(s.c / k.a) : 0.0f;
    values[3] = (float)norm;
  }
}

__global__ void __launch_bounds__(kLossThreads) policy_end_kernel(const double4* __restrict__ part,
                                                                  int64_t count, int by_sequence,
                                                                  float* __restrict__ values) {
  __shared__ ClusterSum sh;
  chain_enter();
  policy_end(part, count, by_sequence, sh, values);
}

// Both in one launch, for few tokens: one cluster, its CTAs taking sequences in turn.
__global__ void __launch_bounds__(kLossThreads) policy_small_kernel(Packed p, PolicyTerms t,
                                                                    PolicyEdges e, double4* part,
                                                                    float* __restrict__ coef,
                                                                    float* __restrict__ values) {
  __shared__ ClusterSum sh;
  for (int64_t seq = blockIdx.x; seq < p.count; seq += gridDim.x)
    policy_seq(p, t, e, seq, 0, 1, sh, part, coef);
  cg::this_cluster().sync();
  if (blockIdx.x == 0) policy_end(part, p.count, t.sequence_average, sh, values);
}

// One launch where that costs no time on the GPU, a sequence for each CTA: the host's
// is what small calls wait for (a launch is 3 of 70 us, forward and backward).
static bool small_loss(const Packed& p) { return p.tokens <= 16384 && p.count <= kLossSplit; }
static int small_ctas(const Packed& p) {
  int ctas = 1;
  while (ctas < kLossSplit && ctas < p.count) ctas *= 2;
  return ctas;
}

// CTAs for each sequence: a cluster of 8 while the sequences do not fill the
// GPU, each with 1024 tokens of an average sequence or more.
static int loss_split(const Packed& p) {
  int split = 1;
  while (split < kLossSplit && p.count * split * 2 <= 2 * num_sms() &&
         p.tokens / p.count >= (int64_t)split * 2 * 1024)
    split *= 2;
  return split;
}

template <typename... Params, typename... Args>
static cudaError_t launch_cluster(void (*kernel)(Params...), int64_t count, int split, int threads,
                                  cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(count * split));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

static int check_packed(const Packed& p) {
  SINKSLOT_REQUIRE(p.tokens >= 0 && p.count >= 1 && p.count <= (int64_t(1) << 27),
                   "loss: bad sizes");
  SINKSLOT_REQUIRE(p.tokens < (int64_t(1) << 32), "loss: 2^32 tokens or more");
  SINKSLOT_REQUIRE(p.offsets || p.count == 1, "loss: offsets are required");
  SINKSLOT_REQUIRE(p.offset_bytes == 4 || p.offset_bytes == 8, "loss: offsets int32 or int64");
  return kOk;
}

size_t loss_workspace_bytes(int64_t count) {
  return align_up((size_t)(count > 0 ? count : 1) * sizeof(double4));
}

int policy_loss(const Packed& p, const PolicyTerms& t, float* values, float* coef, void* ws,
                size_t ws_bytes, cudaStream_t st) {
  SINKSLOT_TRY(check_packed(p));
  SINKSLOT_REQUIRE(values && ws, "policy_loss: null argument");
  SINKSLOT_REQUIRE(p.tokens == 0 || (t.logp && t.old_logp && t.adv), "policy_loss: null argument");
  SINKSLOT_REQUIRE(t.clip_low >= 0.0 && t.clip_high >= 0.0, "policy_loss: clip must be >= 0");
  SINKSLOT_REQUIRE(t.kl_kind >= 1 && t.kl_kind <= 3, "policy_loss: kl must be 1, 2 or 3");
  if (ws_bytes < loss_workspace_bytes(p.count)) {
    set_error("policy_loss: workspace too small");
    return kWorkspaceTooSmall;
  }
  double4* part = static_cast<double4*>(ws);
  if (small_loss(p)) {
    const int ctas = small_ctas(p);
    SINKSLOT_CUDA_TRY(launch_cluster(policy_small_kernel, 1, ctas, kLossThreads, st, p, t,
                                     policy_edges(t), part, coef, values));
    return kOk;
  }
  const int split = loss_split(p);
  SINKSLOT_CUDA_TRY(launch_cluster(policy_seq_kernel, p.count, split, kLossThreads, st, p, t,
                                   policy_edges(t), split, part, coef));
  SINKSLOT_CUDA_TRY(launch_chained(policy_end_kernel, dim3(1), dim3(kLossThreads), 0, st,
                                   (const double4*)part, p.count, t.sequence_average, values));
  return kOk;
}

// --------------------------------------------------------------------------
// Preference loss
// --------------------------------------------------------------------------
__device__ __forceinline__ void preference_seq(const Packed& p, const float* __restrict__ logp,
                                               const float* __restrict__ ref, int64_t seq,
                                               int rank, int split, ClusterSum& sh,
                                               double2* part) {
  int64_t lo, hi;
  bounds(p, seq, lo, hi);
  Sums s = {0.0, 0.0, 0.0};
  int64_t n = 0;
  const int64_t step = (int64_t)split * kLossThreads;
  for (int64_t i = lo + (int64_t)rank * kLossThreads + threadIdx.x; i < hi; i += kAtOnce * step) {
    bool on[kAtOnce];
    float a[kAtOnce], b[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t j = i + k * step;
      on[k] = j < hi;
      a[k] = b[k] = 0.0f;
      if (j < hi) {
        if (p.mask) on[k] = p.mask[j] != 0;
        a[k] = logp[j];
        if (ref) b[k] = ref[j];
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (on[k]) {
        s.a += (double)a[k] - (double)b[k];
        ++n;
      }
  }
  s.b = (double)n;
  const Sums f = cluster_sums(s, sh, 0, rank, split, true);
  if (rank == 0 && threadIdx.x == 0) part[seq] = make_double2(f.a, f.b);
}

__global__ void __launch_bounds__(kLossThreads) preference_seq_kernel(
    Packed p, const float* __restrict__ logp, const float* __restrict__ ref, int split,
    double2* __restrict__ part) {
  __shared__ ClusterSum sh;
  if (split > 1) cluster_started();
  preference_seq(p, logp, ref, blockIdx.x / (unsigned)split, (int)(blockIdx.x % (unsigned)split),
                 split, sh, part);
  chain_release();
}

__device__ __forceinline__ void preference_end(const double2* part, int64_t pairs, double beta,
                                               double smoothing, int kind, int normalize,
                                               ClusterSum& sh, float* __restrict__ loss,
                                               float* __restrict__ rewards,
                                               float* __restrict__ slope) {
  Sums s = {0.0, 0.0, 0.0};
  for (int64_t i = threadIdx.x; i < pairs; i += kLossThreads) {
    const double2 c = part[i], r = part[pairs + i];
    const double wc = normalize && c.y > 0.0 ? 1.0 / c.y : 1.0;
    const double wr = normalize && r.y > 0.0 ? 1.0 / r.y : 1.0;
    const double rc = beta * c.x * wc, rr = beta * r.x * wr;
    const double h = rc - rr;
    double each, d;  // the pair's loss and its derivative by h
    if (kind == 0) {
      const double u = exp(-fabs(h));           // sigma(-|h|) = u / (1 + u)
      const double soft = log1p(u);
      const double neg = (h > 0.0 ? u : 1.0) / (1.0 + u), pos = (h > 0.0 ? 1.0 : u) / (1.0 + u);
      each = (1.0 - smoothing) * (soft + (h < 0.0 ? -h : 0.0));
      // (without smoothing its term is nothing, also where h is inf)
      if (smoothing > 0.0) each += smoothing * (soft + (h > 0.0 ? h : 0.0));
      if (h != h) each = h;
      d = smoothing * pos - (1.0 - smoothing) * neg;
    } else if (kind == 1) {
      each = h < 1.0 ? 1.0 - h : 0.0;
      if (h != h) each = h;
      d = h < 1.0 ? -1.0 : 0.0;
    } else {
      const double x = h / beta - 0.5 / beta;
      each = x * x;
      d = 2.0 * x / beta;
    }
    s.a += each;
    d *= beta / (double)pairs;
    rewards[i] = (float)rc;
    rewards[pairs + i] = (float)rr;
    slope[i] = (float)(d * wc);
    slope[pairs + i] = (float)(-d * wr);
  }
  s = cta_sums(s, sh, 0);
  if (threadIdx.x == 0) loss[0] = (float)(s.a / (double)pairs);
}

__global__ void __launch_bounds__(kLossThreads) preference_end_kernel(
    const double2* __restrict__ part, int64_t pairs, double beta, double smoothing, int kind,
    int normalize, float* __restrict__ loss, float* __restrict__ rewards,
    float* __restrict__ slope) {
  __shared__ ClusterSum sh;
  chain_enter();
  preference_end(part, pairs, beta, smoothing, kind, normalize, sh, loss, rewards, slope);
}

__global__ void __launch_bounds__(kLossThreads) preference_small_kernel(
    Packed p, PreferenceTerms t, double2* part, float* __restrict__ loss,
    float* __restrict__ rewards, float* __restrict__ slope) {
  __shared__ ClusterSum sh;
  for (int64_t seq = blockIdx.x; seq < p.count; seq += gridDim.x)
    preference_seq(p, t.logp, t.ref_logp, seq, 0, 1, sh, part);
  cg::this_cluster().sync();
  if (blockIdx.x == 0)
    preference_end(part, p.count / 2, t.beta, t.smoothing, t.kind, t.normalize, sh, loss, rewards,
                   slope);
}

int preference_loss(const Packed& p, const PreferenceTerms& t, float* loss, float* rewards,
                    float* slope, void* ws, size_t ws_bytes, cudaStream_t st) {
  SINKSLOT_TRY(check_packed(p));
  SINKSLOT_REQUIRE(p.offsets && p.count % 2 == 0, "preference_loss: sequences come in pairs");
  SINKSLOT_REQUIRE(loss && rewards && slope && ws && (p.tokens == 0 || t.logp),
                   "preference_loss: null argument");
  SINKSLOT_REQUIRE(t.kind >= 0 && t.kind <= 2 && t.beta > 0.0, "preference_loss: bad args");
  if (ws_bytes < loss_workspace_bytes(p.count)) {
    set_error("preference_loss: workspace too small");
    return kWorkspaceTooSmall;
  }
  double2* part = static_cast<double2*>(ws);
  if (small_loss(p)) {
    const int ctas = small_ctas(p);
    SINKSLOT_CUDA_TRY(launch_cluster(preference_small_kernel, 1, ctas, kLossThreads, st, p, t,
                                     part, loss, rewards, slope));
    return kOk;
  }
  const int split = loss_split(p);
  SINKSLOT_CUDA_TRY(launch_cluster(preference_seq_kernel, p.count, split, kLossThreads, st, p,
                                   t.logp, t.ref_logp, split, part));
  SINKSLOT_CUDA_TRY(launch_chained(preference_end_kernel, dim3(1), dim3(kLossThreads), 0, st,
                                   (const double2*)part, p.count / 2, t.beta, t.smoothing, t.kind,
                                   t.normalize, loss, rewards, slope));
  return kOk;
}

__global__ void __launch_bounds__(kLossThreads) preference_grad_kernel(
    Packed p, const float* __restrict__ slope, const float* __restrict__ g, int split,
    float* __restrict__ out) {
  const int64_t seq = blockIdx.x / (unsigned)split;
  const int64_t at = (int64_t)(blockIdx.x % (unsigned)split) * kLossThreads + threadIdx.x;
  const int64_t step = (int64_t)split * kLossThreads;
  int64_t lo, hi;
  bounds(p, seq, lo, hi);
  const float v = slope[seq] * g[0];
#pragma unroll 4
  for (int64_t i = lo + at; i < hi; i += step) out[i] = !p.mask || p.mask[i] ? v : 0.0f;
  zero_outside(p, seq, at, step, out);
}

int preference_grad(const Packed& p, const float* slope, const float* g, float* out,
                    cudaStream_t st) {
  SINKSLOT_TRY(check_packed(p));
  if (p.tokens == 0) return kOk;
  SINKSLOT_REQUIRE(slope && g && out, "preference_grad: null argument");
  const int split = loss_split(p);
  preference_grad_kernel<<<(unsigned)(p.count * split), kLossThreads, 0, st>>>(p, slope, g, split,
                                                                              out);
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

__global__ void __launch_bounds__(256) scale_tokens_kernel(const float* __restrict__ coef,
                                                           int64_t tokens,
                                                           const float* __restrict__ norm,
                                                           const float* __restrict__ g,
                                                           float* __restrict__ out) {
  const float f = norm[0] * g[0];
  const int64_t i0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i0 + 4 <= tokens) {
    float4 v = reinterpret_cast<const float4*>(coef)[i0 / 4];
    v.x *= f; v.y *= f; v.z *= f; v.w *= f;
    reinterpret_cast<float4*>(out)[i0 / 4] = v;
  } else {
    for (int64_t i = i0; i < tokens; ++i) out[i] = coef[i] * f;
  }
}

int scale_tokens(const float* coef, int64_t tokens, const float* norm, const float* g, float* out,
                 cudaStream_t st) {
  SINKSLOT_REQUIRE(tokens >= 0, "scale_tokens: bad sizes");
  if (tokens == 0) return kOk;
  SINKSLOT_REQUIRE(coef && norm && g && out, "scale_tokens: null argument");
  SINKSLOT_REQUIRE(((reinterpret_cast<uintptr_t>(coef) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                   "scale_tokens: 16-byte alignment is required");
  scale_tokens_kernel<<<(unsigned)ceil_div64(tokens, 1024), 256, 0, st>>>(coef, tokens, norm, g,
                                                                         out);
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

// --------------------------------------------------------------------------
// Policy loss from the logits.  Where they are larger than L2, one pass over the
// rows gives log-probabilities and gradient (policy_rows.cu: the logits are read
// from memory once); it needs the counts of the whole batch first.  Others go
// through the log-probabilities' own kernels.
// --------------------------------------------------------------------------

// Counts, and the sequence of each token (-1: none).
__global__ void __launch_bounds__(kLossThreads) policy_count_kernel(Packed p, int split,
                                                                    int64_t* __restrict__ counts,
                                                                    int* __restrict__ owner) {
  __shared__ ClusterSum sh;
  if (split > 1) cluster_started();
  const int64_t seq = blockIdx.x / (unsigned)split;
  const int rank = (int)(blockIdx.x % (unsigned)split);
  const int64_t at = (int64_t)rank * kLossThreads + threadIdx.x;
  const int64_t step = (int64_t)split * kLossThreads;
  int64_t lo, hi, n = 0;
  bounds(p, seq, lo, hi);
  for (int64_t i = lo + at; i < hi; i += step) {
    n += !p.mask || p.mask[i];
    owner[i] = (int)seq;
  }
  if (p.offsets && seq == 0)
    for (int64_t i = at, e = offset_at(p, 0); i < e; i += step) owner[i] = -1;
  if (p.offsets && seq == p.count - 1)
    for (int64_t i = offset_at(p, p.count) + at; i < p.tokens; i += step) owner[i] = -1;
  const Sums f = cluster_sums({(double)n, 0.0, 0.0}, sh, 0, rank, split, true);
  if (rank == 0 && threadIdx.x == 0) counts[seq] = (int64_t)f.a;
  chain_release();
}

__global__ void __launch_bounds__(kLossThreads) policy_norm_kernel(
    const int64_t* __restrict__ counts, int64_t count, int by_sequence, float* __restrict__ norm) {
  __shared__ ClusterSum sh;
  chain_enter();
  Sums k = {0.0, 0.0, 0.0};
  for (int64_t i = threadIdx.x; i < count; i += kLossThreads)
    k.a += by_sequence ? (counts[i] > 0 ? 1.0 : 0.0) : (double)counts[i];
  k = cta_sums(k, sh, 0);
  if (threadIdx.x == 0) norm[0] = k.a > 0.0 ? (float)(1.0 / k.a) : 0.0f;
}

size_t policy_logits_workspace_bytes(int64_t rows, int64_t count) {
  const size_t r = (size_t)(rows > 0 ? rows : 1);
  return loss_workspace_bytes(count) + align_up(r * sizeof(float2)) + align_up(r * sizeof(float)) +
         align_up((size_t)count * sizeof(int64_t)) + align_up(sizeof(float));
}

int policy_loss_logits(const LogitRows& r, const Packed& p, const PolicyTerms& t, float grad_scale,
                       float* values, float* logp, void* dz, int64_t dz_stride, void* ws,
                       size_t ws_bytes, cudaStream_t st) {
  SINKSLOT_REQUIRE(p.tokens == r.rows, "policy_loss_from_logits: bad sizes");
  SINKSLOT_TRY(check_rows(r));
  SINKSLOT_TRY(check_packed(p));
  SINKSLOT_REQUIRE(values && (r.rows == 0 || (logp && t.old_logp && t.adv)),
                   "policy_loss_from_logits: null argument");
  SINKSLOT_REQUIRE(!dz || dz_stride >= r.vocab || r.rows <= 1,
                   "policy_loss_from_logits: rows of the gradient overlap");
  Carver cv(ws, ws_bytes);
  float2* stats = cv.take<float2>((size_t)(r.rows > 0 ? r.rows : 1));
  float* coef = cv.take<float>((size_t)(r.rows > 0 ? r.rows : 1));
  char* part = cv.take<char>(loss_workspace_bytes(p.count));
  int64_t* counts = cv.take<int64_t>((size_t)p.count);
  float* norm = cv.take<float>(1);
  if (!cv.ok) {
    set_error("policy_loss_from_logits: workspace too small");
    return kWorkspaceTooSmall;
  }
  PolicyTerms u = t;
  u.logp = logp;
  if (dz && r.rows > 0 && policy_rows_fit(r, dz, dz_stride)) {
    const int split = loss_split(p);
    int* owner = reinterpret_cast<int*>(coef);
    SINKSLOT_CUDA_TRY(launch_cluster(policy_count_kernel, p.count, split, kLossThreads, st, p,
                                     split, counts, owner));
    SINKSLOT_CUDA_TRY(launch_chained(policy_norm_kernel, dim3(1), dim3(kLossThreads), 0, st,
                                     (const int64_t*)counts, p.count, t.sequence_average, norm));
    PolicyRows w;
    w.owner = owner;
    w.counts = counts;
    w.norm = norm;
    SINKSLOT_TRY(policy_rows(r, u, w, grad_scale, logp, dz, dz_stride, st));
    return policy_loss(p, u, values, nullptr, part, loss_workspace_bytes(p.count), st);
  }
  SINKSLOT_TRY(token_logprobs(r, logp, nullptr, stats, st));
  SINKSLOT_TRY(policy_loss(p, u, values, dz ? coef : nullptr, part, loss_workspace_bytes(p.count),
                           st));
  if (!dz || r.rows == 0) return kOk;
  LogitGrad g;
  g.g = coef;
  g.g_stride = 1;
  g.scale_dev = values + 3;
  g.scale = grad_scale;
  g.stats = stats;
  g.dz = dz;
  g.dz_stride = dz_stride;
  return token_logprobs_grad(r, g, st);
}

}  // namespace sinkslot
