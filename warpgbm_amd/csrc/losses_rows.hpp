// Log-probabilities and the policy loss of rows held in registers: one launch
// that reads the scores once and writes the gradient (losses_rows_*.hip).
#pragma once
#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

// a row's statistics from its registers (the label's score sa apart); buf:
// five reductions' words
template <typename F, bool REF>
__device__ __forceinline__ RowStats frame_stats(const F& f, typename F::Regs& s,
                                                typename F::Regs& r, int32_t label, float sa,
                                                float (*buf)[F::kBuf]) {
  RowStats a = empty_stats();
#pragma unroll
  for (int j = 0; j < F::N; ++j) a.m = fmaxf(a.m, F::value(s, j));
  a.m = f.reduce(a.m, MaxF(), buf[0]);
  const Base b = base_of(safe_max(a.m));
  Base br = b;
  if (REF) {
#pragma unroll
    for (int j = 0; j < F::N; ++j) a.mr = fmaxf(a.mr, F::value(r, j));
    a.mr = f.reduce(a.mr, MaxF(), buf[1]);
    br = base_of(safe_max(a.mr));
  }
  if (F::kHide) f.hide(s);
  if (REF && F::kHide) f.hide(r);
  // four sums a thread: shorter chains of additions, and fewer roundings
  float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < F::N; ++j) {
    const float h = power_of(F::value(s, j), b), e = exp2_f32(h);
    z[j % 4] += f.cls(j) == label ? 0.0f : e;
    if (REF) {
      const float hr = power_of(F::value(r, j), br);
      a.zr += exp2_f32(hr);
      a.u += e == 0.0f ? 0.0f : e * (h - hr);
    }
  }
  if (F::kHide) f.hide(s);
  if (REF && F::kHide) f.hide(r);
  a.z = f.reduce((z[0] + z[1]) + (z[2] + z[3]), AddF(), buf[2]);
  if (REF) {
    a.zr = f.reduce(a.zr, AddF(), buf[3]);
    a.u = f.reduce(a.u, AddF(), buf[4]);
  }
  if (label >= 0) a.za = exp2_f32(power_of(sa, b));
  return a;
}

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
  const RowStats a = frame_stats<F, false>(f, v, v, lab, sa, buf);
  if (!in || !f.first_lane()) return;
  write_log_prob(a, sa, lab, i, log_prob, norm);
}

// (no reduction: the norm is given)
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
  const RowStats st = frame_stats<F, REF>(f, v, r, lab, sa, buf);
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
// which frame a call takes: fn(frame tag, workgroups, threads) for the smallest
// one that holds the rows (rows_fit)
// ---------------------------------------------------------------------------
template <typename T, bool REF, typename Fn>
static void pick_row_frame(const ScoresView& s, Fn fn) {
  constexpr int VE = Chunk<T>::VE;
  const int64_t chunks = (s.K + VE - 1) / VE;
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 16) return go(FrameTag<RowFrame<T, 16, 1>>());
  if (chunks <= 64) return go(FrameTag<RowFrame<T, 64, 1>>());
  if (chunks <= 256) return go(FrameTag<RowFrame<T, 64, 4>>());
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
  const int64_t blocks = (s.n + 255) / 256, tiles = (s.n + 63) / 64;
  if (!s.class_major()) {  // rows shorter than a chunk
    if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, false>>(), blocks, 256);
    return fn(FrameTag<ClassFrame<T, 8, false, false>>(), blocks, 256);
  }
  if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, true>>(), blocks, 256);
  if (s.K <= 8) return fn(FrameTag<ClassFrame<T, 8, false, true>>(), blocks, 256);
  if (s.K <= 12) return fn(FrameTag<ClassFrame<T, 12, false, true>>(), blocks, 256);
  if (s.K <= 16) return fn(FrameTag<ClassFrame<T, 16, false, true>>(), blocks, 256);
  if (s.K <= 256)
    return fn(FrameTag<ClassFrame<T, 16, true, true>>(), tiles, 64 * (int)((s.K + 15) / 16));
  fn(FrameTag<ClassFrame<T, 32, true, true>>(), tiles, 64 * (int)((s.K + 31) / 32));
}

template <typename T, bool REF, typename Fn>
static void pick_frame(const ScoresView& s, Fn fn) {
  if (s.class_major() || s.K < Chunk<T>::VE)
    pick_class_frame<T>(s, fn);
  else
    pick_row_frame<T, REF>(s, fn);
}

template <typename T>
static int log_probs_frames(const ScoresView& s, const int32_t* label, float* log_prob,
                            float* norm, hipStream_t st) {
  pick_frame<T, false>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
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
  pick_frame<T, false>(s, [&](auto tag, int64_t blocks, int threads) {
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
  pick_frame<T, REF>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    hipLaunchKernelGGL((policy_frame_kernel<F, REF>), dim3((unsigned)blocks), dim3(threads), 0, st,
                       s, ref, g, out, accumulate);
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
