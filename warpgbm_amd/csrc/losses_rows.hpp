// Log-probabilities and the policy loss of rows held in registers: one launch
// that reads the scores once and writes the gradient (losses_rows_*.hip).  Bound
// by memory where rows have few classes a thread or are read once without sums,
// by memory and vector instructions alike for 16-bit scores.
#pragma once
#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

// a row's statistics from its registers, all but the label's own term za; buf:
// five reductions' words (null where a row is one wave's)
template <typename F, bool REF>
__device__ __forceinline__ RowStats frame_stats(const F& f, typename F::Regs& s,
                                                typename F::Regs& r, int32_t label,
                                                float (*buf)[F::kBuf]) {
  RowStats a = empty_stats();
#pragma unroll
  for (int j = 0; j < F::N; ++j) a.m = fmaxf(a.m, F::value(s, j));
  a.m = f.reduce(a.m, MaxF(), buf[0]);
  const float m = safe_max(a.m);
  float mr = m;
  if (REF) {
#pragma unroll
    for (int j = 0; j < F::N; ++j) a.mr = fmaxf(a.mr, F::value(r, j));
    a.mr = f.reduce(a.mr, MaxF(), buf[1]);
    mr = safe_max(a.mr);
  }
  if (F::kHide) f.hide(s);
  if (REF && F::kHide) f.hide(r);
  // four sums a thread: shorter chains of additions, and fewer roundings
  float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  // Float16 scores that are converted anew for this pass: s log2(e) - m2 takes them as
  // they are (v_fma_mix_f32).  m2 is m log2(e) rounded, off by 2^-8 at most, as m is at
  // most 65504; the sum, 2^(m log2(e) - m2) times too large, is set right below.
  // Log-probabilities of 30000 x 3300 43 us, 47 with the difference first.
  constexpr bool kScaled = !REF && F::kHide && __is_same(typename F::T, _Float16);
  const float m2 = m * kLog2e;
#pragma unroll
  for (int j = 0; j < F::N; ++j) {
    const float x = F::value(s, j) - m;
    const float e = kScaled ? exp2_f32(fmaf(F::value(s, j), kLog2e, -m2)) : exp_diff(x);
    z[j % 4] += f.cls(j) == label ? 0.0f : e;
    if (REF) {
      const float y = F::value(r, j) - mr;
      a.zr += exp_diff(y);
      a.u += e == 0.0f ? 0.0f : e * (x - y);
    }
  }
  // (the sums of 32 and more classes now, not when the reductions want them: their
  // terms would stay in registers until then, some in memory.  8000 x 12000 bfloat16
  // against a reference 139 us, 312 without; 200000 x 300 float32 class-major 386 and
  // 463; but 8000 x 12000 float32, 16 classes a thread, 285 and 273.)
  if (REF && F::N >= 32) asm volatile("" : "+v"(a.zr), "+v"(a.u));
  if (F::kHide) f.hide(s);
  if (REF && F::kHide) f.hide(r);
  a.z = f.reduce((z[0] + z[1]) + (z[2] + z[3]), AddF(), buf[2]);
  if (kScaled) a.z *= exp2_f32(-fmaf(m, kLog2e, -m2));
  if (REF) {
    a.zr = f.reduce(a.zr, AddF(), buf[3]);
    a.u = f.reduce(a.u, AddF(), buf[4]);
  }
  return a;
}

// log p_a = s_a - log sum_k e^(s_k), and the row's norm.  1M x 10 float32
// class-major 12 us (56 MB, 4.8 TB/s); one row of 50001 float32 6.8 us, a
// workgroup's latency (two reductions between 1024 threads).
template <typename F>
__global__ __launch_bounds__(F::kMax) void log_probs_frame_kernel(
    ScoresView s, const int32_t* __restrict__ label, float* __restrict__ log_prob,
    float2* __restrict__ norm) {
  __shared__ float buf[3][F::kBuf];
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  if (!F::kBarrier && !in) return;
  const int64_t i = in ? row : s.n - 1;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  const int32_t lab = row_label(label, i, s.K);
  const float sa = lab >= 0 ? score_at<typename F::T>(s, i, lab) : 0.0f;
  f.trim(v);
  RowStats a = frame_stats<F, false>(f, v, v, lab, buf);
  if (lab >= 0) a.za = exp_diff(sa - safe_max(a.m));
  if (!in || !f.first_lane()) return;
  write_log_prob(a, sa, lab, i, log_prob, norm);
}

// its gradient, g (1[k = a] - p_k): no reduction, the norm is given.  4099 x 32000
// bfloat16 95 us (525 MB, 5.5 TB/s); 20047 x 257 float16 8, bound by latency: rows
// are short and wait for their label and norm; 500000 x 32 float32 class-major 32.
template <typename F>
__global__ __launch_bounds__(F::kMax) void log_probs_grad_frame_kernel(
    ScoresView s, LogProbGrad<typename F::T> g, ScoresView out) {
  const F f(s);
  const int64_t i = F::row(blockIdx.x);
  if (i >= s.n) return;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  const RowCoef c = g.row(s, i);
  if (!c.live) return f.store_zero(out, blockIdx.x);
  f.store_row(out, blockIdx.x, false, c.label, c.gl,
              [&](int j) { return g.at(c, F::value(v, j), 0.0f); });
}

// the clipped policy loss and its gradient (policy_row).  8191 x 16001 bfloat16
// 110 us (524 MB, 4.75 TB/s, vector instructions in 75% of the cycles); 1M x 10
// float32 class-major against a reference's scores 37 (4 TB/s).
template <typename F, bool REF>
__global__ __launch_bounds__(F::kMax) void policy_frame_kernel(ScoresView s, ScoresView ref,
                                                               PolicyRows g, ScoresView out,
                                                               bool accumulate) {
  using T = typename F::T;
  __shared__ float buf[5][F::kBuf];
  __shared__ double wide[F::kBuf];
  __shared__ RowCoef share[F::kShared];
  __shared__ int share_near;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  if (!F::kBarrier && !in) return;
  const int64_t i = in ? row : s.n - 1;
  const float w = !in ? 0.0f : g.weight ? g.weight[i] : 1.0f;
  const int32_t lab = row_label(g.action, i, s.K);
  const bool live = w != 0.0f && lab >= 0;
  // (a workgroup whose waves share rows goes on: other lanes' rows may be live)
  if (!F::kSlices && !live) {
    if (f.first_lane()) {
      g.loss[i] = g.log_prob[i] = 0.0f;
      if (g.kl) g.kl[i] = 0.0f;
    }
    if (out.data && !accumulate) f.store_zero(out, blockIdx.x);
    return;
  }
  typename F::Regs v, r;
  f.load(v, s, blockIdx.x);
  if (REF) f.load(r, ref, blockIdx.x);
  const int32_t a = lab >= 0 ? lab : 0;
  const float sa = score_at<T>(s, i, a);
  const float ra = REF ? score_at<T>(ref, i, a) : 0.0f;
  const float A = g.advantage[i], old = g.old_log_prob[i];
  f.trim(v);
  if (REF) f.trim(r);
  RowStats st = frame_stats<F, REF>(f, v, r, lab, buf);
  if (lab >= 0) st.za = exp_diff(sa - safe_max(st.m));
  // what follows from the row as a whole costs as much as some ten classes:
  // where waves share rows, the first one works it out for all
  const bool owner = !F::kBarrier || threadIdx.x < 64;
  const int slot = F::kSlices ? threadIdx.x & 63 : 0;
  PolicyRow o{};
  if (owner) o = policy_row<REF>(st, sa, ra, A, old, w, g, i, lab, nullptr);
  bool near = o.near && live;
  if (F::kBarrier) {
    const bool any = __any(near);
    if (threadIdx.x == 0) share_near = any;
    __syncthreads();
    near = share_near;
  }
  if (near) {
    // next to a border: the row's sum again, in float64
    const float m = safe_max(st.m);
    const double z = f.wide_sum(s, i, m, wide);
    const double logp = ((double)sa - (double)m) - log(z);
    if (o.near) o = policy_row<REF>(st, sa, ra, A, old, w, g, i, lab, &logp);
  }
  if (F::kSlices && !live) o = PolicyRow{};
  if (in && owner && f.first_lane()) {
    g.loss[i] = o.loss;
    g.log_prob[i] = o.logp;
    if (g.kl) g.kl[i] = o.kl;
  }
  if (F::kBarrier) {
    if (owner && (F::kSlices || threadIdx.x == 0)) share[slot] = o.c;
    __syncthreads();
    o.c = share[slot];
  }
  if (!in || !out.data) return;
  if (!o.c.live) {
    if (!accumulate) f.store_zero(out, blockIdx.x);
    return;
  }
  f.store_row(out, blockIdx.x, accumulate, lab, o.c.gl, [&](int j) {
    return coef_grad<REF>(o.c, F::value(v, j), REF ? F::value(r, j) : 0.0f);
  });
}

// ---------------------------------------------------------------------------
// Log-probabilities of many rows of up to 64 threads each: a workgroup takes B
// rows a thread group, all loads in flight at once, and a thread a row works out
// what follows from the row as a whole.  A row at a time and several: 300000 x
// 100 float32 30 and 22 us, 100000 x 500 bfloat16 28 and 24, 60000 x 1000 28 and
// 25, 1M x 10 float32 19 and 13.  (The policy loss, whose registers hold the row
// until its gradient is written, gains nothing: 300000 x 100 float32 44 either
// way, x 30 21 a row at a time and 23.)
// ---------------------------------------------------------------------------
template <typename F, int B>
__global__ __launch_bounds__(256) void log_probs_batch_kernel(ScoresView s,
                                                              const int32_t* __restrict__ label,
                                                              float* __restrict__ log_prob,
                                                              float2* __restrict__ norm) {
  constexpr int R = F::kRows * B;
  static_assert(R <= 256, "a thread a row");
  __shared__ int32_t s_label[R];
  __shared__ RowStats s_stats[R];
  const F f(s);
  const int64_t i = (int64_t)blockIdx.x * R + threadIdx.x;
  const bool mine = (int)threadIdx.x < R && i < s.n;
  typename F::Regs v[B];
#pragma unroll
  for (int b = 0; b < B; ++b) f.load(v[b], s, (int64_t)blockIdx.x * B + b);
  const int32_t lab = mine ? row_label(label, i, s.K) : -1;
  const float sa = lab >= 0 ? score_at<typename F::T>(s, i, lab) : 0.0f;
  if ((int)threadIdx.x < R) s_label[threadIdx.x] = lab;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < B; ++b) {
    const int r = b * F::kRows + threadIdx.x / F::G;
    f.trim(v[b]);
    const RowStats a = frame_stats<F, false>(f, v[b], v[b], s_label[r], nullptr);
    if (f.first_lane()) s_stats[r] = a;
  }
  __syncthreads();
  if (!mine) return;
  RowStats a = s_stats[threadIdx.x];
  if (lab >= 0) a.za = exp_diff(sa - safe_max(a.m));
  write_log_prob(a, sa, lab, i, log_prob, norm);
}

// rows of a thread group in the kernel above (1: a row at a time): four chunks of
// a thread's registers, or two rows of four
template <typename F>
constexpr int batch_rows() {
  if constexpr (F::kLaneRows) {
    return 1;
  } else {
    if (F::G > 64 || F::NC > 4) return 1;
    return F::NC == 4 ? 2 : 4 / F::NC;
  }
}
// from 4 workgroups a CU on; with fewer the rows of a group would wait for one
// another while CUs are idle
template <typename F, int B>
static bool batch_pays(const ScoresView& s) {
  return s.n >= (int64_t)1024 * F::kRows * B;
}

// ---------------------------------------------------------------------------
// which frame a call takes: fn(frame tag, workgroups, threads) for the smallest
// one that holds the rows (rows_fit).  Row-major rows take two to eight chunks a
// thread rather than one, so that a wave has more loads in flight and spends
// what a row costs as a whole on more rows: with one chunk a thread the policy
// loss of 300000 x 100 float32 takes 57 us instead of 43, of 100000 x 500
// bfloat16 57 and 40, the log-probabilities' gradient 59 and 44, 47 and 38; 30000 x
// 3000 bfloat16, eight chunks of a wave's threads instead of two of a
// workgroup's, whose waves wait for one another: 95 and 65 (not the gradient
// without sums: 66 and 68).  Up to eight chunks a thread each: log-probabilities'
// gradient of 300000 x 30 float32 19 us, 20 with two.
// ---------------------------------------------------------------------------
template <typename T, bool REF, bool SUMS, typename Fn>
static void pick_row_frame(const ScoresView& s, Fn fn) {
  constexpr int VE = Chunk<T>::VE;
  const int64_t chunks = (s.K + VE - 1) / VE;
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 8) return go(FrameTag<RowFrame<T, 8, 1>>());
  if (chunks <= 16) return go(FrameTag<RowFrame<T, 8, 2>>());
  if (chunks <= 32) return go(FrameTag<RowFrame<T, 16, 2>>());
  if (chunks <= 64) return go(FrameTag<RowFrame<T, 32, 2>>());
  if (chunks <= 128) return go(FrameTag<RowFrame<T, 32, 4>>());
  if (chunks <= 256) return go(FrameTag<RowFrame<T, 32, 8>>());
  if constexpr (!SUMS) {
    if (chunks <= 512) return go(FrameTag<RowFrame<T, 256, 2>>());
  }
  if (chunks <= 512) return go(FrameTag<RowFrame<T, 64, 8>>());
  if (chunks <= 1024) return go(FrameTag<RowFrame<T, 256, 4>>());
  if (chunks <= 2048) return go(FrameTag<RowFrame<T, 256, 8>>());
  if (REF || chunks <= 4096) return go(FrameTag<RowFrame<T, 1024, 4>>());
  if constexpr (!REF) {
    if (chunks <= 8192) return go(FrameTag<RowFrame<T, 1024, 8>>());
    go(FrameTag<RowFrame<T, 1024, 16>>());
  }
}

template <typename T, typename Fn>
static void pick_class_frame(const ScoresView& s, Fn fn) {
  const int64_t blocks = (s.n + 255) / 256;
  if (!s.class_major()) {  // rows shorter than a chunk
    if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, false>>(), blocks, 256);
    return fn(FrameTag<ClassFrame<T, 8, false, false>>(), blocks, 256);
  }
  if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, true>>(), blocks, 256);
  if (s.K <= 8) return fn(FrameTag<ClassFrame<T, 8, false, true>>(), blocks, 256);
  if (s.K <= 12) return fn(FrameTag<ClassFrame<T, 12, false, true>>(), blocks, 256);
  if (s.K <= 16) return fn(FrameTag<ClassFrame<T, 16, false, true>>(), blocks, 256);
  pick_slices<T>(s, fn);
}

template <typename T, bool REF, bool SUMS, typename Fn>
static void pick_frame(const ScoresView& s, Fn fn) {
  if (s.class_major() || s.K < Chunk<T>::VE)
    pick_class_frame<T>(s, fn);
  else
    pick_row_frame<T, REF, SUMS>(s, fn);
}

template <typename T>
static int log_probs_frames(const ScoresView& s, const int32_t* label, float* log_prob,
                            float* norm, hipStream_t st) {
  pick_frame<T, false, true>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    constexpr int B = batch_rows<F>();
    if constexpr (B > 1) {
      if (batch_pays<F, B>(s)) {
        hipLaunchKernelGGL((log_probs_batch_kernel<F, B>), dim3((unsigned)((blocks + B - 1) / B)),
                           dim3(threads), 0, st, s, label, log_prob, (float2*)norm);
        return;
      }
    }
    hipLaunchKernelGGL((log_probs_frame_kernel<F>), dim3((unsigned)blocks), dim3(threads), 0, st, s,
                       label, log_prob, (float2*)norm);
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

template <typename T>
static int log_probs_grad_frames(const ScoresView& s, const int32_t* label, const float* norm,
                                 const float* grad, const ScoresView& out, hipStream_t st) {
  const LogProbGrad<T> g{label, (const float2*)norm, grad};
  pick_frame<T, false, false>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    hipLaunchKernelGGL((log_probs_grad_frame_kernel<F>), dim3((unsigned)blocks), dim3(threads), 0,
                       st, s, g, out);
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

template <typename T, bool REF>
static int policy_frames(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,
                         const ScoresView& out, bool accumulate, hipStream_t st) {
  pick_frame<T, REF, true>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    hipLaunchKernelGGL((policy_frame_kernel<F, REF>), dim3((unsigned)blocks), dim3(threads), 0, st,
                       s, ref, g, out, accumulate);
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
