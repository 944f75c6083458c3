// Divergence of a row's scores from a teacher's listed classes, and its gradient.
// With x = s / tau, p = softmax(x), the teacher's shares q_j of the listed classes
// and Q of all the others together (P: the scores' own), scaled to sum 1 over
// those that the row may take,
//   loss = w tau^2 (sum q_j log(q_j / p_j) + Q log(Q / P))
//   ds_k = w tau (p_k - q_k) at a listed class, w tau p_k (1 - Q / P) at others
// q_j = e^(l_j / tau - log norm), Q = 1 - sum q_j; without log norms q = softmax(l /
// tau) over the list and Q = 0.
//
// As both sides sum to 1 the loss is also a sum of terms >= 0,
//   p - q - q x = q (e^x - 1 - x) with x = log(p / q),
// in which the rounding of log sum e^x, common to all, cancels to first order;
// the gradient is q (e^x - 1).  Logarithms are differences in float64 of float32
// sums.  The listed classes' sum leaves out its largest term, 1, so that a row sure of
// one of them keeps what is left.  The others' sum has its own in: log sum e^x of a row
// sure of one of the others is off by 2^-24, a rounding of each listed p, and P itself
// comes from the quotient of the two sums.
//
// The listed classes are taken out of the rows as they sit in registers (a bit a
// slot): what is left is the others' maximum and sum, and their gradient
// needs one exponential a class.  The list's own terms are worked out an entry a
// thread.
//
// 1M x 10 float32 class-major, four listed: 32 us (124 MB, 3.8 TB/s).  1M x 100, 16
// listed, at a temperature of 2: 219 us (940 MB, 4.3 TB/s; vector instructions in three
// fifths of the cycles); at 1: 181 us with one listed, 228 with 16, 313 with 32.  8191 x
// 16001 bfloat16, 64 listed: 127 us (529 MB, 4.1 TB/s, two exponentials a class), 123 with
// one.  256 x 1000 float32: 7 us, latency.
#pragma once
#include "losses_lists.hpp"

namespace wgbm {

// a rest smaller than this is the rounding of the list's numbers: 0
constexpr float kLeastRest = 9.5367431640625e-07f;  // 2^-20

// sums over a row, relative to maxima: m of all its scores, mr of those not
// listed, lm of the listed classes' logits that count
struct DistillSums {
  float zr;                // others: sum of e^(s - mr)
  float zl, zl_ties;       // listed: of e^(s - m) below m, and scores equal to m
  float q, q_ties;         // counting: of e^(l - lm) below lm, and logits equal to lm
  float out;               // not counting: of their shares (with log norms)
};

struct DistillRow {
  bool live;
  float m, lm;         // (0 where there is none)
  float to_p, to_q;    // p = to_p e^(s - m), q = to_q e^(l - lm)
  // log(p / q) = ((s - m) - (l - lm)) / tau - apart: scores and logits of any size count by
  // their differences
  double apart;
  float others;        // gradient of another class: others * e^(s - mr)
  float rest_term;     // the others' term
  float scale;         // w tau
};

// a bucket's term, times tau / 4, and what its gradient is made of, log_ratio = log(p / q).
// (The logarithm of a class masked by the lowest finite score passes float32's range at a
// tau below 1; tau times it is a difference of scores, and a sum of such by shares that
// round to more than 1 fits by the 4.)
constexpr float kTermUnit = 0.25f;
struct Bucket {
  float term, slope;
};
__device__ __forceinline__ Bucket bucket(float p, float q, double log_ratio, float tau) {
  const float x = (float)log_ratio, unit = kTermUnit * tau;
  if (fabsf(x) <= 1.0f) {
    const float f = phi_small(x);
    return {unit * q * f, q * (x + f)};
  }
  if (q == 0.0f) return {unit * p, p};
  return {unit * (p - q) - q * (float)(log_ratio * (double)unit), p - q};
}

__device__ __forceinline__ float power_of(float v, float from, const DistillRows& g) {
  return exp2_f32((v - from) * g.scale);
}

// e^x in float64 for x up to some 1, to some 10^-14: x = n ln 2 + r, and e^r - 1 from the
// first terms of its series at r / 1024, doubled ten times, q -> q (q + 2).  (Seldom
// called; a longer series' coefficients would take the registers of a wave in five.)
__device__ __forceinline__ double exp_wide(double x) {
  const double n = rint(x * 1.44269504088896340736);
  const double r = fma(n, -0.693147180559945286227, x) * 0x1p-10;
  double q = fma(fma(fma(r, 1.0 / 24.0, 1.0 / 6.0), r, 0.5), r * r, r);
#pragma unroll 1
  for (int d = 0; d < 10; ++d) q = fma(q, q, q + q);
  return x < -700.0 ? 0.0 : ldexp(1.0 + q, (int)n);
}

// the logarithm of the teacher's sum over all classes (0 where it does not count)
__device__ __forceinline__ double row_norm(const DistillRows& g, int64_t i) {
  if (!g.rest) return 0.0;
  return g.log_norm ? (double)g.log_norm[i] : g.log_norm_all;
}

// logit(j): the logits of the row's entries j < k (-infinity: not used)
template <typename Logit>
__device__ __forceinline__ DistillRow distill_row(const DistillSums& a, const DistillRows& g,
                                                  int64_t i, float m, float mr, float lm, float w,
                                                  int k, Logit logit) {
  DistillRow o{};
  o.m = safe_max(m);
  o.lm = safe_max(lm);
  o.scale = w * g.tau;
  const bool has_rest = mr > -__builtin_inff() || a.zr != a.zr;
  // shares: `one` of the largest logit, C of the other counting ones; top its logarithm
  const bool counts = lm > -__builtin_inff() || a.q != a.q;
  const float more = a.q + (a.q_ties - 1.0f);  // relative to the largest
  double top_q = 0.0, log_Q = 0.0;             // logs of the largest q, of the others' share
  bool rest = false, odd = false;
  o.live = true;
  if (g.rest) {
    const double top = (double)o.lm * g.inv_tau - row_norm(g, i);
    odd = top != top || (has_rest && a.out != a.out);
    const float one = counts ? exp_of((float)top) : 0.0f, C = counts ? more * one : 0.0f;
    const float held = one + C;
    float left = counts ? one_less_exp((float)top) - C - a.out : 1.0f - a.out;
    // next to the border whether a rest is one is decided in float64 (the roundings above
    // come to less than 100 * 2^-24); so is what is left of a list that the row may
    // mostly not take, whose roundings the scaling to sum 1 would enlarge (shares of 2 and
    // more, of a log norm too small, leave none)
    if (has_rest && (fabsf(left - kLeastRest) < 1e-5f || (a.out > 0.5f && left > -1.0f))) {
      const double norm = row_norm(g, i);
      double sum = 0.0;
#pragma unroll 1
      for (int j = 0; j < k; ++j) sum += exp_wide((double)logit(j) * g.inv_tau - norm);
      left = (float)(1.0 - sum);
    }
    rest = left >= kLeastRest && has_rest;
    if (rest) {
      // what is left, scaled to sum 1 (of a small list: 1 - listed would round its digits
      // away)
      double log_mass = (double)log1p_of(-a.out);
      if (!(a.out < 0.5f)) log_mass = log_of(held + left);
      const float listed = held + a.out;
      log_Q = (listed < 0.5f ? (double)log1p_of(-listed) : log_of(left)) - log_mass;
      if (counts) top_q = top - log_mass;
    }
  }
  // without a rest the counting shares sum to 1 whatever they were, also past float32's
  // range (NaN of what the rest is made of shows in the results)
  if (!rest) {
    o.live = counts;
    top_q = counts ? -log_1p(more) : 0.0;
    if (odd) top_q = __builtin_nan("");
  }
  // scores: listed A, others B, relative to m
  const double drop = has_rest ? ((double)mr - (double)o.m) * g.inv_tau : 0.0;
  const float B = has_rest ? exp_of((float)drop) * a.zr : 0.0f;
  const float A = a.zl + a.zl_ties;
  o.live = o.live && w != 0.0f && !(A + B == 0.0f);
  // without the largest term, 1, where it is among the listed; among the others it is
  // part of their sum
  const double lse = log_1p(a.zl_ties > 0.0f ? a.zl + (a.zl_ties - 1.0f) + B : A + (B - 1.0f));
  o.to_p = exp_of((float)-lse);
  o.to_q = exp_of((float)top_q);
  o.apart = lse + top_q;
  // the others
  if (has_rest) {
    double log_P = -log_1p(A / B);
    if (!(B > 1e-30f * A)) log_P = drop + log_of(a.zr) - lse;
    const float P = exp_of((float)log_P);
    Bucket b{kTermUnit * g.tau * P, P};
    if (rest) b = bucket(P, exp_of((float)log_Q), log_P - log_Q, g.tau);
    o.rest_term = b.term;
    if (o.live) o.others = o.scale * b.slope / a.zr;
  }
  return o;
}
// a listed class that counts (score above -infinity)
__device__ __forceinline__ Bucket distill_entry(const DistillRow& r, const DistillRows& g, float s,
                                                float l) {
  return bucket(r.to_p * power_of(s, r.m, g), r.to_q * power_of(l, r.lm, g),
                (((double)s - (double)r.m) - ((double)l - (double)r.lm)) * g.inv_tau - r.apart,
                g.tau);
}
// a listed class that does not count: the row may not take it
__device__ __forceinline__ bool closed(float s) { return s == -__builtin_inff(); }

// ---------------------------------------------------------------------------
// a thread a row.  A list names classes by number, and registers have none: the
// row's scores also lie in LDS, a column a thread, beside the listed classes' logits,
// and their gradients go back through it.
// ---------------------------------------------------------------------------
template <typename F>
__global__ __launch_bounds__(F::kMax) void distill_lane_kernel(ScoresView s, DistillRows g,
                                                               ScoresView out, bool accumulate) {
  constexpr int N = F::N;
  __shared__ float score[N][256], logit[N][256];
  const F f(s);
  const int t = threadIdx.x;
  const int64_t i = F::row(blockIdx.x);
  if (i >= s.n) return;
  const int32_t* const classes = g.classes + i * g.class_stride;
  const float* const logits = g.logits + i * g.logit_stride;
  using Batch = EntryBatch<float>;
  Batch b;
  b.load(classes, g.class_step, logits, g.logit_step, 0, 1, g.k);
  const float w = g.weight ? g.weight[i] : 1.0f;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  f.trim(v);
  // (left out: no class; rows that count and rows that do not go the same way)
  if (w == 0.0f) f.drop(v);
#pragma unroll
  for (int j = 0; j < N; ++j) score[j][t] = F::value(v, j);
  uint32_t listed = 0;
  float m = -__builtin_inff(), lm = m;
  const int k = w != 0.0f ? g.k : 0;
  for (int first = 0; first < k; first += Batch::kSize) {
    if (first) b.load(classes, g.class_step, logits, g.logit_step, first, 1, k);
#pragma unroll
    for (int q = 0; q < Batch::kSize; ++q) {
      const int32_t c = b.cls[q];
      // (the first of the entries that name a class counts)
      if (first + q >= k || (uint32_t)c >= (uint32_t)s.K || (listed >> c & 1)) continue;
      listed |= 1u << c;
      logit[c][t] = b.value[q];
      const float sc = score[c][t];
      m = fmaxf(m, sc);
      lm = closed(sc) ? lm : fmaxf(lm, b.value[q]);
    }
  }
  float mr = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < N; ++j) mr = listed >> j & 1 ? mr : fmaxf(mr, F::value(v, j));
  m = fmaxf(m, mr);
  const float ms = safe_max(m), mrs = safe_max(mr), lms = safe_max(lm);
  DistillSums a{};
  float e[N];  // exponentials of the others
#pragma unroll
  for (int j = 0; j < N; ++j) {
    e[j] = listed >> j & 1 ? 0.0f : power_of(F::value(v, j), mrs, g);
    a.zr += e[j];
  }
  const double norm = row_norm(g, i);
  for (uint32_t left = listed; left; left &= left - 1) {
    const int c = __ffs(left) - 1;
    const float sc = score[c][t], l = logit[c][t];
    if (closed(sc)) {
      if (g.rest) a.out += exp_of((float)((double)l * g.inv_tau - norm));
      continue;
    }
    const float es = power_of(sc, ms, g), el = power_of(l, lms, g);
    a.zl += sc == m ? 0.0f : es;
    a.zl_ties += sc == m ? 1.0f : 0.0f;
    a.q += l == lm ? 0.0f : el;
    a.q_ties += l == lm ? 1.0f : 0.0f;
  }
  const DistillRow r = distill_row(a, g, i, m, mr, lm, w, N, [&](int j) {
    return listed >> j & 1 ? logit[j][t] : -__builtin_inff();
  });
  float loss = r.rest_term;
  for (uint32_t left = listed; left; left &= left - 1) {
    const int c = __ffs(left) - 1;
    const float sc = score[c][t];
    float grad = 0.0f;
    if (!closed(sc)) {
      const Bucket u = distill_entry(r, g, sc, logit[c][t]);
      loss += u.term;
      grad = r.scale * u.slope;
    }
    score[c][t] = grad;
  }
  g.loss[i] = r.live ? r.scale / kTermUnit * loss : 0.0f;
  if (!out.data || (!r.live && accumulate)) return;
  f.store(out, blockIdx.x, accumulate, [&](int j) {
    const float x = listed >> j & 1 ? score[j][t] : r.others * e[j];
    return r.live ? x : 0.0f;
  });
}

// a listed class's part of the sums x[1] .. x[5]
__device__ __forceinline__ void add_entry(const DistillRows& g, double norm, float sc, float l,
                                          float m, float ms, float lm, float lms,
                                          float (&x)[6]) {
  if (closed(sc)) {
    if (g.rest) x[5] += exp_of((float)((double)l * g.inv_tau - norm));
    return;
  }
  const float es = power_of(sc, ms, g), el = power_of(l, lms, g);
  x[1] += sc == m ? 0.0f : es;
  x[2] += sc == m ? 1.0f : 0.0f;
  x[3] += l == lm ? 0.0f : el;
  x[4] += l == lm ? 1.0f : 0.0f;
}

// ---------------------------------------------------------------------------
// class-major rows in slices (SliceMap)
// ---------------------------------------------------------------------------
template <typename F>
static size_t distill_slices_lds(int32_t k, int threads) {
  return ((size_t)SliceMap<F>::kWords * threads + 2 * 64 * (size_t)k + 10 * (size_t)threads) * 4;
}

template <typename F>
__global__ __launch_bounds__(F::kMax) void distill_slices_kernel(ScoresView s, DistillRows g,
                                                                 ScoresView out, bool accumulate) {
  using Map = SliceMap<F>;
  extern __shared__ uint32_t lds[];
  __shared__ DistillRow share[64];
  const int k = g.k, lane = threadIdx.x & 63;
  const Map map{lds};
  // logits of the lists, and their scores, later gradients
  float* const logit = (float*)(lds + Map::kWords * blockDim.x) + lane;
  float* const score = logit + 64 * k;
  float* const buf = (float*)(lds + Map::kWords * blockDim.x) + 128 * k;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  const int64_t i = in ? row : s.n - 1;
  const int32_t* const classes = g.classes + i * g.class_stride;
  const float* const logits = g.logits + i * g.logit_stride;
  using Batch = EntryBatch<float>;
  Batch b;
  b.load(classes, g.class_step, logits, g.logit_step, f.w, f.S, k);
  const float w = !in ? 0.0f : g.weight ? g.weight[i] : 1.0f;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  map.clear();
  __syncthreads();
  // (entries that are not used have score and logit -infinity)
  bool twice = false;
  for (int first = f.w; first < k; first += Batch::kSize * f.S) {
    if (first != f.w) b.load(classes, g.class_step, logits, g.logit_step, first, f.S, k);
#pragma unroll
    for (int q = 0; q < Batch::kSize; ++q) {
      const int j = first + q * f.S;
      if (j >= k) break;
      const bool used = w != 0.0f && (uint32_t)b.cls[q] < (uint32_t)s.K;
      logit[64 * j] = used ? b.value[q] : -__builtin_inff();
      score[64 * j] = -__builtin_inff();
      if (used) twice |= map.put(f, b.cls[q], j);
    }
  }
  if (__syncthreads_or(twice)) {
    // the first of the entries that name a class takes its place
    for (int j = f.w; j < k; j += f.S) {
      const int32_t c = classes[j * g.class_step];
      bool first = w != 0.0f && (uint32_t)c < (uint32_t)s.K;
      for (int o = 0; o < j; ++o) first &= classes[o * g.class_step] != c;
      if (first)
        map.set(f, c, j);
      else
        logit[64 * j] = -__builtin_inff();
    }
    __syncthreads();
  }
  uint32_t mine[Map::kWords];
  map.mine(mine);
  f.trim(v);
  if (w == 0.0f) f.drop(v);
  float x[3];
  x[0] = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < F::N; ++j) {
    const int e = Map::entry(mine, j);
    if (e) score[64 * (e - 1)] = F::value(v, j);
    f.take_out(v, j, e != 0);
    x[0] = fmaxf(x[0], F::value(v, j));
  }
  __syncthreads();
  x[1] = x[2] = -__builtin_inff();
  for (int j = f.w; j < k; j += f.S) {
    const float sc = score[64 * j], l = logit[64 * j];
    x[1] = fmaxf(x[1], sc);
    x[2] = closed(sc) ? x[2] : fmaxf(x[2], l);
  }
  f.reduce_all(x, MaxF(), buf);
  const float mr = x[0], m = fmaxf(x[0], x[1]), lm = x[2];
  const float ms = safe_max(m), mrs = safe_max(mr), lms = safe_max(lm);
  float z[2] = {0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < F::N; ++j) z[j % 2] += power_of(F::value(v, j), mrs, g);
  float y[6] = {z[0] + z[1], 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  const double norm = row_norm(g, i);
  for (int j = f.w; j < k; j += f.S)
    add_entry(g, norm, score[64 * j], logit[64 * j], m, ms, lm, lms, y);
  f.put_all(y, AddF(), buf + 3 * blockDim.x);
  __syncthreads();
  // what follows from the row as a whole costs as much as some 20 classes: the first wave
  // works it out for all
  DistillRow r;
  if (f.w == 0) {
    f.join_all(y, AddF(), buf + 3 * blockDim.x);
    r = distill_row(DistillSums{y[0], y[1], y[2], y[3], y[4], y[5]}, g, i, m, mr, lm, w, k,
                    [&](int j) { return logit[64 * j]; });
    share[lane] = r;
  }
  __syncthreads();
  if (f.w != 0) r = share[lane];
  float loss[1] = {0.0f};
  for (int j = f.w; j < k; j += f.S) {
    const float sc = score[64 * j];
    Bucket u{0.0f, 0.0f};
    if (!closed(sc)) u = distill_entry(r, g, sc, logit[64 * j]);
    loss[0] += u.term;
    score[64 * j] = r.scale * u.slope;
  }
  f.put_all(loss, AddF(), buf + 9 * blockDim.x);
  __syncthreads();
  if (f.w == 0) {
    f.join_all(loss, AddF(), buf + 9 * blockDim.x);
    if (in) g.loss[i] = r.live ? r.scale / kTermUnit * (loss[0] + r.rest_term) : 0.0f;
  }
  // (one store for rows that count and rows left out: lanes of a wave may hold both)
  if (!in || !out.data || (!r.live && accumulate)) return;
  f.store(out, blockIdx.x, accumulate, [&](int j) {
    const int e = Map::entry(mine, j);
    float y = r.others * power_of(F::value(v, j), mrs, g);
    if (e) y = score[64 * (e - 1)];
    return r.live ? y : 0.0f;
  });
}

// ---------------------------------------------------------------------------
// rows that threads share
// ---------------------------------------------------------------------------
// a workgroup's lists in LDS: classes, logits, scores of these (an entry that is not used
// has class -1, and logit and score -infinity)
struct ListTable {
  int32_t* cls;
  float* logit;
  float* score;
  uint32_t* bits;  // of the threads' slots
  float* buf;      // of the reductions, six values at most
};
template <typename F>
__device__ __forceinline__ ListTable list_table(uint32_t* lds, int k) {
  ListTable t;
  t.cls = (int32_t*)lds;
  t.logit = (float*)(t.cls + F::kListRows * k);
  t.score = t.logit + F::kListRows * k;
  t.bits = (uint32_t*)(t.score + F::kListRows * k);
  t.buf = (float*)(t.bits + F::kMaskWords * blockDim.x);
  return t;
}

// entries that name a class again no longer count
template <typename F>
__device__ __forceinline__ void drop_repeated(const F& f, const ListTable& t, int k) {
  uint32_t again = 0;
  int n = 0;
  for (int j = f.entry(); j < k; j += f.entry_step(), ++n) {
    const int32_t c = t.cls[f.entry_at(j, k)];
    if (c >= 0 && listed_before(f, t.cls, j, k, c)) again |= 1u << n;
  }
  __syncthreads();
  n = 0;
  for (int j = f.entry(); j < k; j += f.entry_step(), ++n)
    if (again >> n & 1) {
      t.cls[f.entry_at(j, k)] = -1;
      t.logit[f.entry_at(j, k)] = t.score[f.entry_at(j, k)] = -__builtin_inff();
    }
}

// the list's part of the maxima: x[1] of listed scores, x[2] of counting logits
template <typename F>
__device__ __forceinline__ void list_maxima(const F& f, const ListTable& t, int k, float (&x)[3]) {
  x[1] = x[2] = -__builtin_inff();
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    const int at = f.entry_at(j, k);
    const float sc = t.score[at], l = t.logit[at];
    x[1] = fmaxf(x[1], sc);
    x[2] = closed(sc) ? x[2] : fmaxf(x[2], l);
  }
}
// the list's part of the sums: x[1] .. x[5]
template <typename F>
__device__ __forceinline__ void list_sums(const F& f, const ListTable& t, const DistillRows& g,
                                          int64_t i, float m, float lm, float (&x)[6]) {
  const int k = g.k;
  const float ms = safe_max(m), lms = safe_max(lm);
  const double norm = row_norm(g, i);
  x[1] = x[2] = x[3] = x[4] = x[5] = 0.0f;
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    const int at = f.entry_at(j, k);
    add_entry(g, norm, t.score[at], t.logit[at], m, ms, lm, lms, x);
  }
}

// (registers for eight waves where that takes two from the seldom loop of distill_row: 15000
// x 3900 float32 97 us, 100 in 66 registers)
template <typename F>
__global__ __launch_bounds__(F::kMax, F::G == 256 && F::NC == 4 ? 8 : 1) void distill_frame_kernel(
    ScoresView s, DistillRows g, ScoresView out, bool accumulate) {
  using T = typename F::T;
  extern __shared__ uint32_t lds[];
  __shared__ DistillRow share;
  const int k = g.k;
  const ListTable tab = list_table<F>(lds, k);
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  const int64_t i = in ? row : s.n - 1;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  const float w = !in ? 0.0f : g.weight ? g.weight[i] : 1.0f;
#pragma unroll
  for (int b = 0; b < F::kMaskWords; ++b) tab.bits[b * blockDim.x + threadIdx.x] = 0;
  __syncthreads();
  bool twice = false;
  const int32_t* const classes = g.classes + i * g.class_stride;
  const float* const logits = g.logits + i * g.logit_stride;
  const T* const scores = (const T*)s.data + i * s.rs;
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    int32_t c = w != 0.0f ? classes[j * g.class_step] : -1;
    float l = logits[j * g.logit_step], sc = -__builtin_inff();
    if (c < 0 || c >= s.K) c = -1;
    if (c >= 0) {
      int word;
      uint32_t bit;
      f.locate(c, word, bit);
      twice |= (atomicOr(&tab.bits[word], bit) & bit) != 0;
      sc = to_f32(scores[c * s.ks]);
    }
    const int at = f.entry_at(j, k);
    tab.cls[at] = c;
    tab.logit[at] = c >= 0 ? l : -__builtin_inff();
    tab.score[at] = sc;
  }
  if (__syncthreads_or(twice)) drop_repeated(f, tab, k);
  f.trim(v);
  uint32_t mine[F::kMaskWords];
#pragma unroll
  for (int b = 0; b < F::kMaskWords; ++b) mine[b] = tab.bits[b * blockDim.x + threadIdx.x];
  f.take_out(v, mine);
  if (w == 0.0f) f.drop(v);
  float x[3];
  x[0] = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < F::N; ++j) x[0] = fmaxf(x[0], F::value(v, j));
  list_maxima(f, tab, k, x);
  f.reduce_all(x, MaxF(), tab.buf);
  const float mr = x[0], m = fmaxf(x[0], x[1]), lm = x[2], mrs = safe_max(mr);
  if (F::N >= 32) f.hide(v);
  float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < F::N; ++j) z[j % 4] += exp2_f32((F::value(v, j) - mrs) * g.scale);
  float y[6];
  y[0] = (z[0] + z[1]) + (z[2] + z[3]);
  list_sums(f, tab, g, i, m, lm, y);
  if (F::kBarrier) __syncthreads();  // the maxima have been read
  f.put_all(y, AddF(), tab.buf);
  // what follows from the row as a whole costs as much as some 20 classes: where waves
  // share rows, the first one works it out for all
  const bool owner = !F::kBarrier || threadIdx.x < 64;
  if (F::kBarrier) __syncthreads();
  DistillRow r;
  if (owner) {
    f.join_all(y, AddF(), tab.buf);
    r = distill_row(DistillSums{y[0], y[1], y[2], y[3], y[4], y[5]}, g, i, m, mr, lm, w, k,
                    [&](int j) { return tab.logit[f.entry_at(j, k)]; });
    if (F::kBarrier && threadIdx.x == 0) share = r;
  }
  if (F::kBarrier) {
    __syncthreads();
    if (!owner) r = share;
  }
  if (F::N >= 32) f.hide(v);
  // (one store for rows that count and rows left out, whose others' gradient is 0 times
  // an exponential of -infinity: a wave may hold both)
  if (!r.live) f.drop(v);
  if (in && out.data && (r.live || !accumulate))
    f.store(out, blockIdx.x, accumulate, [&](int j) {
      return r.others * exp2_f32((F::value(v, j) - mrs) * g.scale);
    });
  __syncthreads();  // the others' gradients are written before the list's
  T* const grads = (T*)out.data + i * out.rs;
  float loss[1] = {0.0f};
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    const int at = f.entry_at(j, k);
    const float sc = tab.score[at];
    if (closed(sc)) continue;
    const Bucket b = distill_entry(r, g, sc, tab.logit[at]);
    loss[0] += b.term;
    if (in && r.live && out.data) {
      float d = r.scale * b.slope;
      T* q = grads + tab.cls[at] * out.ks;
      if (accumulate) d += to_f32(*q);
      *q = from_f32<T>(d);
    }
  }
  // (rows of several waves have their list in the first one)
  if (owner) loss[0] = lanes_reduce<(F::kListLanes)>(loss[0], AddF());
  if (in && f.first_lane()) g.loss[i] = r.live ? r.scale / kTermUnit * (loss[0] + r.rest_term) : 0.0f;
}

// ---------------------------------------------------------------------------
// rows longer than a workgroup's registers: a workgroup a row, its tiles one after
// the other, twice (maximum and sum of each thread's classes as they come, then the
// gradient)
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(1024) void distill_long_kernel(ScoresView s, DistillRows g,
                                                            ScoresView out, bool accumulate,
                                                            int32_t span, int32_t tiles) {
  using F = RowFrame<T, 1024, 4>;
  extern __shared__ uint32_t lds[];
  __shared__ float buf[6 * F::kBuf];
  const int k = g.k;
  const ListTable tab = list_table<F>(lds, k);
  const F whole(s);
  const int64_t i = blockIdx.x;
  const float w = g.weight ? g.weight[i] : 1.0f;
  // the list: an entry a thread; repeated classes by comparison (a tile's bits say
  // nothing of the others)
  for (int j = threadIdx.x; j < k; j += 1024) {
    int32_t c = w != 0.0f ? g.classes[i * g.class_stride + j * g.class_step] : -1;
    if (c < 0 || c >= s.K) c = -1;
    tab.cls[j] = c;
    tab.logit[j] =
        c >= 0 ? g.logits[i * g.logit_stride + j * g.logit_step] : -__builtin_inff();
    tab.score[j] = c >= 0 ? score_at<T>(s, i, c) : -__builtin_inff();
  }
  __syncthreads();
  drop_repeated(whole, tab, k);
  __syncthreads();
  // this thread's bits of tile t
  const auto bits_of = [&](const F& f, int32_t t, uint32_t (&b)[F::kMaskWords]) {
    tab.bits[threadIdx.x] = 0;
    __syncthreads();
    if ((int)threadIdx.x < k) {
      const int32_t c = tab.cls[threadIdx.x] - t * span;
      if (tab.cls[threadIdx.x] >= 0 && c >= 0 && c < f.K) {
        int word;
        uint32_t bit;
        f.locate(c, word, bit);
        atomicOr(&tab.bits[word], bit);
      }
    }
    __syncthreads();
    b[0] = tab.bits[threadIdx.x];
  };
  static_assert(F::kMaskWords == 1, "a word a thread");
  float most = -__builtin_inff();
  double sum = 0.0;
  if (w != 0.0f) {
    for (int32_t t = 0; t < tiles; ++t) {
      const ScoresView p = tile_of(s, span, t);
      const F f(p);
      typename F::Regs v;
      f.load(v, p, i);
      uint32_t b[F::kMaskWords];
      bits_of(f, t, b);
      f.trim(v);
      f.take_out(v, b);
      float m = most;
#pragma unroll
      for (int j = 0; j < F::N; ++j) m = fmaxf(m, F::value(v, j));
      const float ms = safe_max(m);
      float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < F::N; ++j) z[j % 4] += exp2_f32((F::value(v, j) - ms) * g.scale);
      if (most > -__builtin_inff()) sum *= (double)exp2_f32((most - ms) * g.scale);
      sum += (double)((z[0] + z[1]) + (z[2] + z[3]));
      most = m;
    }
  }
  float x[3] = {most, 0.0f, 0.0f};
  list_maxima(whole, tab, k, x);
  whole.reduce_all(x, MaxF(), buf);
  const float mr = x[0], m = fmaxf(x[0], x[1]), lm = x[2], mrs = safe_max(mr);
  float y[6];
  // (a thread without a class has sum 0, or NaN)
  y[0] = (float)sum * (most > -__builtin_inff() ? exp2_f32((most - mrs) * g.scale) : 1.0f);
  list_sums(whole, tab, g, i, m, lm, y);
  __syncthreads();
  whole.reduce_all(y, AddF(), buf);
  const DistillRow r =
      distill_row(DistillSums{y[0], y[1], y[2], y[3], y[4], y[5]}, g, i, m, mr, lm, w, k,
                  [&](int j) { return tab.logit[j]; });
  if (out.data && (r.live || !accumulate)) {
    for (int32_t t = 0; t < tiles; ++t) {
      const ScoresView p = tile_of(s, span, t), o = tile_of(out, span, t);
      const F f(p);
      if (!r.live) {
        f.store_zero(o, i);
        continue;
      }
      typename F::Regs v;
      f.load(v, p, i);
      uint32_t b[F::kMaskWords];
      bits_of(f, t, b);
      f.trim(v);
      f.take_out(v, b);
      f.store(o, i, accumulate, [&](int j) {
        return r.others * exp2_f32((F::value(v, j) - mrs) * g.scale);
      });
    }
  }
  __syncthreads();
  float loss[1] = {0.0f};
  for (int j = threadIdx.x; j < k; j += 1024) {
    const float sc = tab.score[j];
    if (closed(sc)) continue;
    const Bucket b = distill_entry(r, g, sc, tab.logit[j]);
    loss[0] += b.term;
    if (r.live && out.data) {
      float d = r.scale * b.slope;
      T* q = (T*)out.data + i * out.rs + tab.cls[j];
      if (accumulate) d += to_f32(*q);
      *q = from_f32<T>(d);
    }
  }
  whole.reduce_all(loss, AddF(), buf);
  if (threadIdx.x == 0) g.loss[i] = r.live ? r.scale / kTermUnit * (loss[0] + r.rest_term) : 0.0f;
}

template <typename T>
static int distill_frames(const ScoresView& s, const DistillRows& g, const ScoresView& out,
                          bool accumulate, hipStream_t st) {
  if (!rows_fit(s, false)) {
    using F = RowFrame<T, 1024, 4>;
    static_assert(F::N * 1024 == kTileChunks * F::VE, "a tile");
    int32_t span;
    const int32_t tiles = row_tiles(s, false, &span);
    hipLaunchKernelGGL((distill_long_kernel<T>), dim3((unsigned)s.n), dim3(1024),
                       (size_t)g.k * 12 + 1024 * 4, st, s, g, out, accumulate, span, tiles);
    WGBM_LAUNCH_CHECK();
    return 0;
  }
  const auto launch = [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    if constexpr (F::kLaneRows && !F::kSlices) {
      hipLaunchKernelGGL((distill_lane_kernel<F>), dim3((unsigned)blocks), dim3(threads), 0, st, s,
                         g, out, accumulate);
    } else if constexpr (F::kSlices) {
      hipLaunchKernelGGL((distill_slices_kernel<F>), dim3((unsigned)blocks), dim3(threads),
                         distill_slices_lds<F>(g.k, threads), st, s, g, out, accumulate);
    } else {
      const size_t lds = (size_t)F::kListRows * g.k * 12 + (size_t)F::kMaskWords * threads * 4 +
                         6 * F::kBuf * 4;
      hipLaunchKernelGGL((distill_frame_kernel<F>), dim3((unsigned)blocks), dim3(threads), lds, st,
                         s, g, out, accumulate);
    }
  };
  const int64_t chunks = (s.K + Chunk<T>::VE - 1) / Chunk<T>::VE;
  if (thread_rows(s))
    pick_thread_rows<T>(s, launch);
  else if (s.class_major())
    pick_list_slices<T>(s, launch);
  else if (chunks <= 32)
    pick_few_threads<T>(s, chunks, launch);
  else if (chunks <= 64)  // (200470 x 257 float16 83 us, with 32 threads of two chunks 112)
    launch(FrameTag<RowFrame<T, 16, 4>>(), (s.n + 15) / 16, 256);
  else
    pick_row_frame<T, false, true>(s, launch);
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
