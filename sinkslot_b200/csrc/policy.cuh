// policy.cuh -- one token's terms of the clipped policy loss.
#pragma once

#include <cmath>
#include <cuda_runtime.h>

#include "training.h"

namespace sinkslot {

// e^d - d - 1.  Near 0 its terms cancel; there it is summed as its series
// d^2/2! + d^3/3! + ... + d^11/11! (the rest is under 2^-30 of it for |d| <= 1/2).
__device__ __forceinline__ float exp_gap(float d) {
  if (d >= 1e4f) return INFINITY;
  if (!(fabsf(d) <= 0.5f)) return expm1f(d) - d;
  float t = 1.0f;
#pragma unroll
  for (int k = 11; k >= 3; --k) t = fmaf(t, d * (1.0f / (float)k), 1.0f);
  return 0.5f * d * d * t;
}

struct PolicyEdges {
  double under, over;  // log(1 - lo), log(1 + hi)
  float rlo, rhi, kl_coef;
};

struct TokenTerm {
  float loss, kl, coef;
  bool clipped;
};

// One token's loss, KL estimate and d loss / d logp.  The clip is decided on the
// difference of the log-probabilities in fp64, which is exact.  The ratio, the KL term
// and the coefficient are float32 (as the log-probabilities and the result are; a
// token's loss is good to a few steps, and the sums over tokens are fp64): over 16384
// tokens the outputs are 7e-8 of their size off where fp64 terms, rounded once, are 3e-8.
__device__ __forceinline__ TokenTerm policy_term(const PolicyTerms& t, const PolicyEdges& e,
                                                 float logp, float old_logp, float ref_logp,
                                                 float adv) {
  TokenTerm o;
  const double d = (double)logp - (double)old_logp;
  const bool over = d > e.over, under = d < e.under;
  const float r = expf((float)d);
  const float rc = over ? e.rhi : (under ? e.rlo : r);
  // min(r A, clip(r) A) is the clipped one where r is outside on A's side
  o.clipped = adv > 0.0f ? over : (adv < 0.0f ? under : false);
  const float ra = adv == 0.0f && d < INFINITY ? 0.0f : r * adv;  // r may be past float32
  o.loss = o.clipped ? -rc * adv : -ra;
  o.coef = o.clipped ? 0.0f : -ra;
  o.kl = 0.0f;
  if (t.ref_logp) {
    const float g = (float)((double)ref_logp - (double)logp);
    float slope;
    if (t.kl_kind == 1) {
      o.kl = -g;
      slope = 1.0f;
    } else if (t.kl_kind == 2) {
      o.kl = 0.5f * g * g;
      slope = -g;
    } else {
      o.kl = exp_gap(g);
      slope = -expm1f(g);
    }
    if (e.kl_coef != 0.0f) {
      o.loss = fmaf(e.kl_coef, o.kl, o.loss);
      o.coef = fmaf(e.kl_coef, slope, o.coef);
    }
  }
  return o;
}

inline PolicyEdges policy_edges(const PolicyTerms& t) {
  PolicyEdges e;
  e.under = t.clip_low >= 1.0 ? -INFINITY : log1p(-t.clip_low);
  e.over = log1p(t.clip_high);
  e.rlo = t.clip_low >= 1.0 ? 0.0f : (float)(1.0 - t.clip_low);
  e.rhi = (float)(1.0 + t.clip_high);
  e.kl_coef = (float)t.kl_coef;
  return e;
}

}  // namespace sinkslot
