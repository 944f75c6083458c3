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

// what a row's gradient is made of: with x = s - m of the scores and y = r - mr
// of the reference's (m, mr: the maxima)
//   g_k = e^x (c1 (x - y) + c0),  and at the label g_a = gl
// (c1 and mr only with reference scores).  live = 0: the row's gradient is 0.
struct RowCoef {
  float m, mr;
  float c0, c1, gl;
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

// Exponentials: e^x, x = s - m, by v_exp_f32 of x log2(e).  The difference comes
// first: it is exact for the scores that count (s within a factor of two of m, or
// both small), 0 at the maximum whatever its size, and -inf at worst.  (One fused
// multiply-add, s log2(e) - fl(m log2(e)), would save an instruction a class but
// leaves m log2(e)'s rounding in the power: 10^-3 at a maximum of 10^5, a factor
// of 2^440 at 10^10.  Both forms take the same time where memory bounds them, 8191 x
// 16001 bfloat16 110 us, 1M x 10 float32 against a reference 37; long rows against a
// reference lose 3 to 7%.)  The difference's, the product's and log2(e)'s roundings
// cost 2.3 |x| 2^-24 of the value, that is less than 2^-24 of the row's largest
// exponential (|x| e^-|x| has its maximum 1/e): what a softmax's sums and gradients are
// rounded by anyway.
constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.693147180559945309417;
__device__ __forceinline__ float exp2_f32(float h) { return __builtin_amdgcn_exp2f(h); }
__device__ __forceinline__ float exp_diff(float x) { return exp2_f32(x * kLog2e); }

// running maximum and sums of a set of a row's classes, all in float32:
//   m = max s_k, z = sum of e^x_k over the classes but the label (x = s - m),
//   za = the label's e^x_a (0 when it is in another set); with reference scores
//   r: mr = max r_k, zr = sum of e^y_k (y = r - mr), u = sum of e^x_k (x_k - y_k)
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
  const float b = safe_max(m) - safe_max(a.m);
  const float f = a.m == -__builtin_inff() ? 0.0f : exp_diff(-b);  // 0 for an empty set
  if (REF) {
    const float br = safe_max(mr) - safe_max(a.mr), t = a.z + a.za;
    // a set that counts for nothing has no difference to move
    a.u = t != 0.0f && f != 0.0f ? f * (a.u + (br - b) * t) : 0.0f;
    a.zr *= a.mr == -__builtin_inff() ? 0.0f : exp_diff(-br);
    a.mr = mr;
  }
  a.z *= f;
  a.za *= f;
  a.m = m;
}

// one more class of differences x and y
template <bool REF>
__device__ __forceinline__ void add_class(RowStats& a, float x, float y, bool is_label) {
  const float e = exp_diff(x);
  if (is_label)
    a.za += e;
  else
    a.z += e;
  if (REF) {
    a.zr += exp_diff(y);
    // a class of probability 0 takes no part in the divergence, whatever the
    // reference says of it (both are -inf at classes that a row may not take)
    a.u += e == 0.0f ? 0.0f : e * (x - y);
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
// Logarithms of float32 sums to some 10^-8, with the exponent's part in float64:
// log2(z) = k + log2(f), f in [0.7, 1.41), where a float32 logarithm's absolute
// error is 2^-25.  (A float32 logarithm of many classes' sum, some ten, would
// lose a digit that the ratio and the divergence of a policy near its reference
// need; a float64 one costs as much as ten classes.)
struct Split {
  float k, f;
};
__device__ __forceinline__ Split split_f32(float z) {
  Split o{(float)__builtin_amdgcn_frexp_expf(z), __builtin_amdgcn_frexp_mantf(z)};
  if (o.f < 0.70710678f) {
    o.f *= 2.0f;
    o.k -= 1.0f;
  }
  return o;
}
// (v_log_f32: the logarithm to base 2 of a normal number)
__device__ __forceinline__ float log2_f32(float f) { return __builtin_amdgcn_logf(f); }
__device__ __forceinline__ double log_of(float z) {
  const Split s = split_f32(z);
  return ((double)s.k + (double)log2_f32(s.f)) * kLn2;
}
// log(a / b)
__device__ __forceinline__ double log_ratio(float a, float b) {
  const Split x = split_f32(a), y = split_f32(b);
  return ((double)(x.k - y.k) + (double)(log2_f32(x.f) - log2_f32(y.f))) * kLn2;
}
// log(1 + q) for q in [0, 1]: the logarithm of the rounded sum, and what the
// rounding left out
__device__ __forceinline__ float log1p_of(float q) {
  const float w = 1.0f + q;
  return fmaf(log2_f32(w), (float)kLn2, (q - (w - 1.0f)) * __builtin_amdgcn_rcpf(w));
}
// e^x within 2 ulp: the product's rounding taken along, and log2(e)'s own (1.3 10^-8
// |x| of the value, 10 ulp at 80)
__device__ __forceinline__ float exp_of(float x) {
  constexpr float kLow = (float)(1.44269504088896340736 - (double)kLog2e);
  const float h = x * kLog2e, lo = fmaf(x, kLow, fmaf(x, kLog2e, -h)), e = exp2_f32(h);
  return fabsf(h) < 200.0f ? fmaf(e, lo * (float)kLn2, e) : e;  // (no inf * 0)
}

__device__ __forceinline__ bool row_live(const RowStats& a) {
  return !(a.z + a.za == 0.0f);  // the row has a class (NaN: it shows in the results)
}
// log-probability of the label, whose score is sa.  A label of at least half:
// from the others' share, which keeps the digits of a row that is sure of its
// label (and the sign).
__device__ __forceinline__ double row_log_prob(const RowStats& a, float sa) {
  if (a.za >= a.z) return -(double)log1p_of(a.z / a.za);
  return ((double)sa - (double)safe_max(a.m)) - log_of(a.z + a.za);
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
  const float z = st.z + st.za, iz = __builtin_amdgcn_rcpf(z);
  o.c.m = safe_max(st.m);
  o.c.mr = REF ? safe_max(st.mr) : 0.0f;
  o.c.label = label;
  o.c.live = row_live(st);
  o.near = false;
  if (!o.c.live) {
    o.loss = o.logp = o.kl = 0.0f;
    o.c.c0 = o.c.c1 = o.c.gl = 0.0f;
    return o;
  }
  const double logp = row_log_prob(st, sa);
  o.logp = (float)logp;
  // (the ratio's and the divergence's terms are float32, of a float64 difference: its
  // rounding costs 2^-24 |x| of the ratio, beside the sums' roundings)
  const float x = (float)(logp - (double)old);
  const float ratio = exp_of(x);
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
    // log p_k - log q_k = (x_k - y_k) + lr, lr = log of the sums' quotient
    // (a reference without a class: u is infinite, and so is the divergence)
    const double lr = st.zr == 0.0f ? 0.0 : log_ratio(st.zr, z);
    const double kl = (double)(st.u / z) + lr;
    o.kl = (float)kl;
    base = (float)(lr - kl);  // (log p_k - log q_k - KL) - (x_k - y_k)
    // (a divergence that does not count may be infinite)
    if (g.kl_coef != 0.0f)
      value += g.kl_coef * o.kl;
    else
      base = 0.0f;
    wk = w * g.kl_coef;
  } else if (g.ref_log_prob) {
    const float d = (float)((double)g.ref_log_prob[i] - logp);
    const float e = expm1f(d);
    o.kl = d > 88.0f ? e : e - d;  // (no inf - inf)
    // near 0 the difference loses what the series keeps
    if (fabsf(d) < 0.03125f)
      o.kl = d * d * fmaf(d, fmaf(d, fmaf(d, 1.0f / 120.0f, 1.0f / 24.0f), 1.0f / 6.0f), 0.5f);
    if (g.kl_coef != 0.0f) {
      value += g.kl_coef * o.kl;
      c -= g.kl_coef * e;
    }
  }
  c *= w;
  o.loss = w * value;
  o.c.c0 = (wk * base - c) * iz;
  o.c.c1 = wk * iz;
  o.c.gl = c * (st.z * iz);
  if (REF && wk != 0.0f && st.za != 0.0f)
    o.c.gl += st.za * iz * wk * (((sa - o.c.m) - (ra - o.c.mr)) + base);
  return o;
}

// gradient at a class that is not the label
template <bool REF>
__device__ __forceinline__ float coef_grad(const RowCoef& c, float s, float r) {
  const float x = s - c.m, e = exp_diff(x);
  if (!REF || c.c1 == 0.0f) return e * c.c0;
  return e == 0.0f ? 0.0f : e * fmaf(c.c1, x - (r - c.mr), c.c0);
}

}  // namespace wgbm
