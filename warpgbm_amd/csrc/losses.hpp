// Losses of class scores [n rows, K classes]: types and arithmetic shared by
// their kernels (losses*.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"

namespace wgbm {

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

// scores (or a gradient of them): element (i, k) at data[i * rs + k * ks] of
// its type; one of the two strides is 1
struct ScoresView {
  void* data;
  int32_t dtype;
  int64_t n;
  int32_t K;
  int64_t rs, ks;
  // rows next to each other (class-major), else classes (row-major)
  bool class_major() const { return rs == 1 && ks != 1; }
};

// per-row inputs and outputs of the policy loss (null: not given / not wanted)
struct PolicyRows {
  const int32_t* action;
  const float* old_log_prob;
  const float* advantage;
  const float* weight;
  const float* ref_log_prob;
  double clip_lo, clip_hi;  // the ratio's borders, 1 - low and 1 + high
  float log_lo, log_hi;     // their logarithms
  float kl_coef;
  float* loss;
  float* log_prob;
  float* kl;
};

// what a row's gradient is made of: with d = s - m, p_k = exp(d_k) * iz,
//   g_k = p_k * (c1 * (d_k - (r_k - mr)) + c0),  and at the label g_a = gl
// (c1 and mr only with reference scores).  live = 0: the row's gradient is 0.
struct RowCoef {
  float m, iz, c0, c1, mr, gl;
  int32_t label;
  int32_t live;
};

// ---------------------------------------------------------------------------
// element types: arithmetic in float32, one rounding (to nearest even) when a
// gradient is stored
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;
}

// e^x for x <= 0 (-inf gives 0, NaN stays): v_exp_f32 of x log2(e).  The
// product's rounding costs |x| 2^-24 of the value, that is at most 2^-25 of the
// row's largest exponential (|x| e^x has its maximum 1/e): what a softmax's sums
// and gradients are rounded by anyway.  Taking the rounding error along would
// cost six instructions more, as much again as the exponential (the balance
// loss's first pass over 1M x 100 classes is bound by instructions then).
__device__ __forceinline__ float loss_expf(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
}

// running maximum and sums of a set of a row's classes, all in float32:
//   m = max s_k, z = sum of e^(s_k - m) over the classes but the label,
//   za = the label's e^(s_a - m) (0 when it is in another set); with
//   reference scores r: mr = max r_k, zr = sum of e^(r_k - mr),
//   u = sum of e^(s_k - m) ((s_k - m) - (r_k - mr))
// The label is summed apart so that 1 - p_a = z / (z + za) keeps its digits
// for a row that is sure of its label.
struct RowStats {
  float m, z, za, mr, zr, u;
};

__device__ __forceinline__ RowStats empty_stats() {
  return {-__builtin_inff(), 0.0f, 0.0f, -__builtin_inff(), 0.0f, 0.0f};
}

// a maximum that can be subtracted: a row without a class (every score -inf)
// takes 0, so that its exponentials are 0 rather than NaN
__device__ __forceinline__ float safe_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// the same statistics relative to the larger maxima m and mr
template <bool REF>
__device__ __forceinline__ void rebase_stats(RowStats& a, float m, float mr) {
  const float ms = safe_max(m), f = loss_expf(a.m - ms);  // 0 for an empty set
  if (REF) {
    const float mrs = safe_max(mr), t = a.z + a.za;
    // an empty set has no difference to move (its maxima are -inf)
    if (t != 0.0f) a.u = f * (a.u + ((a.m - ms) - (safe_max(a.mr) - mrs)) * t);
    a.zr *= loss_expf(a.mr - mrs);
    a.mr = mr;
  }
  a.z *= f;
  a.za *= f;
  a.m = m;
}

// one more class: e is e^(s - m), d = s - m, dr = r - mr, er = e^(r - mr)
template <bool REF>
__device__ __forceinline__ void add_class(RowStats& a, float d, float dr, bool is_label) {
  const float e = loss_expf(d);
  if (is_label)
    a.za += e;
  else
    a.z += e;
  if (REF) {
    a.zr += loss_expf(dr);
    // a class of probability 0 takes no part in the divergence, whatever the
    // reference says of it (both are -inf at classes that a row may not take)
    a.u += e == 0.0f ? 0.0f : e * (d - dr);
  }
}

template <bool REF>
__device__ __forceinline__ RowStats join_stats(RowStats a, RowStats b) {
  const float m = fmaxf(a.m, b.m), mr = REF ? fmaxf(a.mr, b.mr) : 0.0f;
  rebase_stats<REF>(a, m, mr);
  rebase_stats<REF>(b, m, mr);
  a.z += b.z;
  a.za += b.za;
  if (REF) {
    a.zr += b.zr;
    a.u += b.u;
  }
  return a;
}

// ---------------------------------------------------------------------------
// what follows from a row's statistics
// ---------------------------------------------------------------------------
// (float64 from the row's sum on: the logarithm of many classes' sum, some
// ten, would lose a digit in float32 that the ratio and the divergence of a
// policy near its reference need)
struct LogProb {
  double logp, l;  // l = log of the sum of e^(s - m)
  float m;
  bool live;  // the row has a class
};

// sa: the label's score
__device__ __forceinline__ LogProb row_log_prob(const RowStats& a, float sa) {
  const float z = a.z + a.za;
  LogProb o;
  o.live = !(z == 0.0f);  // (NaN is live: it shows in the results)
  o.m = safe_max(a.m);
  o.l = log((double)z);
  o.logp = ((double)sa - (double)o.m) - o.l;
  return o;
}

// The policy loss of one row and its gradient's coefficients.
//   ratio = e^(logp - old), value = -min(ratio A, clip(ratio) A) + c KL,
//   KL = e^x - x - 1 with x = ref - logp (sampled), or
//        sum_k p_k (log p_k - log q_k) (reference scores)
// The gradient through the ratio is -A ratio where the unclipped product is
// the smaller one, else 0: a step.  When logp - old is so near the border's
// logarithm that float32 cannot tell (`near`), the caller passes the log-prob
// in float64 (exact_logp) and calls again.
struct PolicyRow {
  float loss, logp, kl;
  RowCoef c;
  bool near;
};

template <bool REF>
__device__ __forceinline__ PolicyRow policy_row(const RowStats& st, float sa, float ra, float A,
                                                float old, float w, const PolicyRows& g, int64_t i,
                                                int32_t label, const double* exact_logp) {
  PolicyRow o;
  const LogProb lp = row_log_prob(st, sa);
  const float z = st.z + st.za;
  o.c.m = lp.m;
  o.c.iz = 1.0f / z;
  o.c.label = label;
  o.c.live = lp.live;
  o.near = false;
  if (!lp.live) {
    o.loss = o.logp = o.kl = 0.0f;
    o.c.c0 = o.c.c1 = o.c.mr = o.c.gl = o.c.iz = 0.0f;
    return o;
  }
  o.logp = (float)lp.logp;
  const float x = (float)(lp.logp - (double)old);
  const float ratio = expf(x);
  // positive advantages stop above the upper border, negative ones below the
  // lower
  const bool up = A > 0.0f;
  bool stop = false;
  if (A != 0.0f) {
    if (exact_logp) {
      const double r = exp(*exact_logp - (double)old);
      stop = up ? r > g.clip_hi : r < g.clip_lo;
    } else {
      const float edge = up ? g.log_hi : g.log_lo;
      stop = up ? x > edge : x < edge;
      // the sum's error is 2^-24 for each class that one thread adds to it
      // (256 of them are within this bound), that of x and edge 2^-24 of theirs
      o.near = fabsf(x - edge) < 2e-5f * (1.0f + fabsf(edge));
    }
  }
  float value = stop ? -A * (float)(up ? g.clip_hi : g.clip_lo) : -A * ratio;
  if (A == 0.0f) value = 0.0f;  // (also where the ratio overflows)
  float c = stop || A == 0.0f ? 0.0f : -A * ratio;
  o.kl = 0.0f;
  float wk = 0.0f, base = 0.0f;
  if (REF) {
    const double lr = log((double)st.zr) - lp.l;
    const double kl = (double)st.u / (double)z + lr;
    o.kl = (float)kl;
    base = (float)(lr - kl);  // log p_k - log q_k - KL = (d_k - dr_k) + base
    value += g.kl_coef * o.kl;
    wk = w * g.kl_coef;
  } else if (g.ref_log_prob) {
    const float d = (float)((double)g.ref_log_prob[i] - lp.logp);
    const float e = expm1f(d);
    o.kl = e - d;
    // near 0 the difference loses what the series keeps
    if (fabsf(d) < 0.03125f)
      o.kl = d * d * fmaf(d, fmaf(d, fmaf(d, 1.0f / 120.0f, 1.0f / 24.0f), 1.0f / 6.0f), 0.5f);
    value += g.kl_coef * o.kl;
    c -= g.kl_coef * e;
  }
  c *= w;
  o.loss = w * value;
  const float pa = st.za / z;
  o.c.c0 = wk * base - c;
  o.c.c1 = wk;
  o.c.mr = REF ? safe_max(st.mr) : 0.0f;
  o.c.gl = c * (st.z / z);
  if (REF && pa != 0.0f) o.c.gl += pa * wk * (((sa - lp.m) - (ra - o.c.mr)) + base);
  return o;
}

// gradient at a class that is not the label
template <bool REF>
__device__ __forceinline__ float coef_grad(const RowCoef& c, float s, float r) {
  const float d = s - c.m, e = loss_expf(d);
  float t = c.c0;
  if (REF) t = e == 0.0f ? 0.0f : fmaf(c.c1, d - (r - c.mr), t);
  return e * c.iz * t;
}

}  // namespace wgbm
