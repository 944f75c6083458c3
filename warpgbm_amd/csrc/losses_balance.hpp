// The balance loss: how evenly rows fall on classes.
//   c_k = rows with class k among their top_k, f_k = c_k / (n' top_k),
//   P_k = mean of p_ik over the n' rows that count,
//   L = coef K sum_k f_k P_k,   dL/ds_ik = coef K / n' p_ik (f_k - sum_j f_j p_ij)
// (the counts are held constant).  The gradient needs every row's counts
// first, so the scores are read twice: rows in registers (losses_frames.hpp)
// give the counts, the sums of p and each row's norm; a finishing launch the
// shares; rows in registers again the gradient.  Workgroups take rows in turn
// and leave one partial sum a class, which the finishing launch joins in
// float64 in workgroup order: results do not depend on the order of execution.
// Rows that would take a workgroup more than kChain turns are further launches of
// the first pass, so that float32 sums stay short however many rows there are.
//
// 1M x 100 float32 class-major: the first pass 131 us (3.1 TB/s; the eight waves
// that share 64 rows wait for one another at three reductions), the finish 7, the
// gradient 182 (4.4 TB/s).
// 65536 x 64 bfloat16, two choices: 10, 5 and 5.
#pragma once
#include <algorithm>

#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

struct MinF {
  __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
};

// whether a thread's registers also hold the next rows: two sets of scores, the
// exponentials and the sums within what 16 waves of a workgroup can have
template <typename F>
constexpr bool kAhead = 2 * F::kWords + 2 * F::N <= 104;

// most rows that a thread adds up in float32: their roundings come to 256 * 2^-24 of
// the sum at worst (float64 sums would take the registers of two, and a loop around
// the rows' loop, in one launch, costs 500000 x 64 class-major 113 us instead of 105)
constexpr int32_t kChain = 256;

// The blocks of rows first .. end, to part [K][slots] and count [K + 1][slots] (the
// last: rows that count), a slot a workgroup from slot0 on; norm: a row's maximum
// and 1 / sum of e^(s - m) (0: left out)
template <typename F>
__global__ __launch_bounds__(F::kMax) void balance_stats_kernel(
    ScoresView s, const uint8_t* __restrict__ mask, int32_t top_k, int64_t first, int64_t end,
    int32_t slot0, int32_t slots, float* __restrict__ part, int32_t* __restrict__ count,
    float2* __restrict__ norm, uint32_t* __restrict__ ticket) {
  extern __shared__ int32_t s_count[];  // [K + 1], then [K] floats
  __shared__ float buf[4][F::kBuf];
  const int32_t K = s.K;
  float* s_part = (float*)(s_count + K + 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  for (int32_t k = threadIdx.x; k <= K; k += blockDim.x) s_count[k] = 0;
  __syncthreads();
  const F f(s);
  float acc[F::N];
#pragma unroll
  for (int j = 0; j < F::N; ++j) acc[j] = 0.0f;
  // the next rows' loads are in flight while these rows are summed
  typename F::Regs next;
  uint8_t next_want = 1;
  const auto fetch = [&](int64_t b) {
    const int64_t row = F::row(b);
    if (mask) next_want = mask[row < s.n ? row : s.n - 1];
    f.load(next, s, b);
  };
  if (kAhead<F>) fetch(first + blockIdx.x);
  for (int64_t b = first + blockIdx.x; b < end; b += gridDim.x) {
    const int64_t row = F::row(b);
    const bool in = row < s.n;
    const int64_t i = in ? row : s.n - 1;
    if (!kAhead<F>) fetch(b);
    typename F::Regs v = next;
    const bool want = in && next_want;
    if (kAhead<F> && b + gridDim.x < end) fetch(b + gridDim.x);
    f.trim(v);
    if (!want) f.drop(v);
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      m = fmaxf(m, F::value(v, j));
    }
    m = f.reduce(m, MaxF(), buf[0]);
    const float ms = safe_max(m);
    // the exponentials of up to 16 classes stay in registers; more are worked
    // out again for the sums
    constexpr bool kKeep = F::N <= 16;
    float e[kKeep ? F::N : 1], z[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      const float x = exp_diff(F::value(v, j) - ms);
      z[j % 2] += x;
      if constexpr (kKeep) e[j] = x;
    }
    z[0] = f.reduce(z[0] + z[1], AddF(), buf[1]);
    const bool live = !(z[0] == 0.0f);  // (NaN is live)
    const float iz = live ? 1.0f / z[0] : 0.0f;
    // (slices of 32 classes have 128 registers: unknown to be ms, so that the compiler
    // works the exponentials out again.  200000 x 400 class-major 440 us, 523 without.)
    float m2 = ms;
    if constexpr (!kKeep && F::kSlices) asm volatile("" : "+v"(m2));
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      float x;
      if constexpr (kKeep)
        x = e[j];
      else
        x = exp_diff(F::value(v, j) - m2);
      acc[j] = fmaf(x, iz, acc[j]);
    }
    if (in && f.first_lane()) norm[i] = make_float2(ms, iz);
    // the best classes one after the other: the largest score after the last
    // one taken, then the lowest class that has it.  A thread's classes ascend
    // with its slots, so it looks for its lowest slot (slot numbers are
    // constants of the instructions, class numbers would each take a register).
    // Class numbers are exact in float32; a NaN is not after anything.
    constexpr float kNone = 1e9f;
    float v0 = __builtin_inff();
    int32_t c0 = -1;
    for (int32_t t = 0; t < top_k; ++t) {
      float best = m;
      int slot = F::N;
      if (t == 0) {
#pragma unroll
        for (int j = F::N - 1; j >= 0; --j) slot = F::value(v, j) == best ? j : slot;
      } else {
        const int taken = f.last_slot(c0);  // of the scores equal to v0
        best = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < F::N; ++j) {
          const float x = F::value(v, j);
          if (x < v0 || (x == v0 && j > taken)) best = fmaxf(best, x);
        }
        best = f.reduce(best, MaxF(), buf[2]);
        const int from = best < v0 ? -1 : taken;
#pragma unroll
        for (int j = F::N - 1; j >= 0; --j)
          slot = F::value(v, j) == best && j > from ? j : slot;
      }
      const float c = f.reduce(slot < F::N ? (float)f.cls(slot) : kNone, MinF(), buf[3]);
      if (best > -__builtin_inff() && c < kNone && f.first_lane())
        atomicAdd(&s_count[(int32_t)c], 1);
      v0 = best;
      c0 = (int32_t)c;
    }
    if (live && f.first_lane()) atomicAdd(&s_count[K], 1);
  }
  f.sum_rows(acc, s_part);
  __syncthreads();
  for (int32_t k = threadIdx.x; k <= K; k += blockDim.x) {
    const int64_t at = (int64_t)k * slots + slot0 + blockIdx.x;
    if (k < K) part[at] = s_part[k];
    count[at] = s_count[k];
  }
}

template <typename F>
__global__ __launch_bounds__(F::kMax) void balance_grad_kernel(
    ScoresView s, const float2* __restrict__ norm, const float* __restrict__ share,
    const float* __restrict__ scale, int64_t blocks, bool accumulate, ScoresView out) {
  __shared__ float buf[2][F::kBuf];
  const F f(s);
  float fk[F::N];
#pragma unroll
  for (int j = 0; j < F::N; ++j) fk[j] = share[f.cls(j) < s.K ? f.cls(j) : s.K - 1];
  const float c = *scale;
  int turn = 0;
  typename F::Regs next;
  float2 next_norm;
  const auto fetch = [&](int64_t b) {
    const int64_t row = F::row(b);
    next_norm = norm[row < s.n ? row : s.n - 1];
    f.load(next, s, b);
  };
  if (kAhead<F>) fetch(blockIdx.x);
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x, turn ^= 1) {
    const int64_t row = F::row(b);
    const bool in = row < s.n;
    const int64_t i = in ? row : s.n - 1;
    if (!kAhead<F>) fetch(b);
    typename F::Regs v = next;
    const float2 nm = next_norm;
    if (kAhead<F> && b + gridDim.x < blocks) fetch(b + gridDim.x);
    f.trim(v);
    const bool live = in && nm.y != 0.0f;  // (NaN is live)
    float e[F::N], q = 0.0f;
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      e[j] = exp_diff(F::value(v, j) - nm.x);
      q = fmaf(fk[j], e[j], q);
    }
    // (two turns' words: a wave may be one reduction ahead of the others)
    q = f.reduce(q, AddF(), buf[turn]) * nm.y;
    if (!in) continue;
    if (!live) {
      if (!accumulate) f.store_zero(out, b);
      continue;
    }
    const float cz = c * nm.y;
    f.store(out, b, accumulate, [&](int j) { return cz * e[j] * (fk[j] - q); });
  }
}

// the frames of up to 4096 classes: f(frame tag, blocks of rows, threads).  Two
// and eight chunks a thread where there are rows enough: 200000 x 100 float32 54
// us, 61 with one, 30000 x 3000 bfloat16 254, 293 with a workgroup a row; but 8192
// x 256 bfloat16 27 with one, 30 with two.
template <typename T, typename Fn>
static void balance_frame(const ScoresView& s, Fn fn) {
  const int64_t rows = (s.n + 255) / 256;
  if (!s.class_major() && s.K < Chunk<T>::VE) {
    if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, false>>(), rows, 256);
    return fn(FrameTag<ClassFrame<T, 8, false, false>>(), rows, 256);
  }
  if (s.class_major()) {
    if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, true>>(), rows, 256);
    if (s.K <= 8) return fn(FrameTag<ClassFrame<T, 8, false, true>>(), rows, 256);
    if (s.K <= 12) return fn(FrameTag<ClassFrame<T, 12, false, true>>(), rows, 256);
    if (s.K <= 16) return fn(FrameTag<ClassFrame<T, 16, false, true>>(), rows, 256);
    return pick_slices<T>(s, fn);
  }
  const int64_t chunks = (s.K + Chunk<T>::VE - 1) / Chunk<T>::VE;
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 8) return go(FrameTag<RowFrame<T, 8, 1>>());
  if (s.n * chunks < kLossWaves * 128) {  // (two chunks a thread would not fill the GPU)
    if (chunks <= 16) return go(FrameTag<RowFrame<T, 16, 1>>());
    if (chunks <= 32) return go(FrameTag<RowFrame<T, 32, 1>>());
    if (chunks <= 64) return go(FrameTag<RowFrame<T, 64, 1>>());
  }
  if (chunks <= 16) return go(FrameTag<RowFrame<T, 8, 2>>());
  if (chunks <= 32) return go(FrameTag<RowFrame<T, 16, 2>>());
  if (chunks <= 64) return go(FrameTag<RowFrame<T, 32, 2>>());
  if (chunks <= 128) return go(FrameTag<RowFrame<T, 64, 2>>());
  if (chunks <= 256) return go(FrameTag<RowFrame<T, 64, 4>>());
  if (chunks <= 512) return go(FrameTag<RowFrame<T, 64, 8>>());
  return go(FrameTag<RowFrame<T, 256, 4>>());
}

// workgroups of the two passes: 16 waves a CU (with 64, the class-major 1M x 10
// takes 45 us instead of 37 and a gate's 65536 x 64 32 instead of 26: more
// partial sums), but 64 where the waves of a workgroup wait for one another
// (200000 x 400 class-major, 13 waves each, 505 us with 16, 421 with 64; 1M x 100,
// eight waves, 288 and 318: one rule for both is a compromise); and
// fewer partial sums where there are many classes
template <typename F>
static int64_t balance_fill(int threads) {
  return (F::kSlices ? 4 : 1) * kLossWaves * 64 / threads;
}
static inline int64_t balance_few(int32_t K) {
  return std::max<int64_t>(512, (int64_t(1) << 20) / K);
}

template <typename T>
int balance_stats(const ScoresView& s, const uint8_t* mask, int32_t top_k, const BalanceWs& w,
                  int32_t* slots, hipStream_t st) {
  balance_frame<T>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    const int64_t groups = std::min(blocks, std::min(balance_fill<F>(threads), balance_few(s.K)));
    const int64_t each = groups * kChain, last = (blocks - 1) / each;
    *slots = (int32_t)(last * groups + std::min(groups, blocks - last * each));
    for (int64_t p = 0; p <= last; ++p) {
      const int64_t first = p * each, end = std::min(blocks, first + each);
      hipLaunchKernelGGL((balance_stats_kernel<F>), dim3((unsigned)std::min(groups, end - first)),
                         dim3(threads), (2 * (size_t)s.K + 1) * 4, st, s, mask, top_k, first, end,
                         (int32_t)(p * groups), *slots, w.part, w.count, w.norm, w.ticket);
    }
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int balance_grad(const ScoresView& s, const BalanceWs& w, const ScoresView& out, bool accumulate,
                 hipStream_t st) {
  balance_frame<T>(s, [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    const int64_t groups = std::min(blocks, balance_fill<F>(threads));
    hipLaunchKernelGGL((balance_grad_kernel<F>), dim3((unsigned)groups), dim3(threads), 0, st, s,
                       w.norm, w.share, w.scale, blocks, accumulate, out);
  });
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
