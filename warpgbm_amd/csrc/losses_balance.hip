// The balance loss: its finishing launch and the host side (the passes over rows:
// losses_balance.hpp).
#include "losses_balance.hpp"

namespace wgbm {

// classes of a workgroup of the finishing launch: a wave each, its lanes along
// the workgroups' partial sums
constexpr int kFinClasses = 4;

// shares f_k, means P_k, counts, the loss and the gradient's scale (some 1000
// partial sums a class: 7 us for 100 classes, a launch's latency for few).  The
// workgroups' shares of the loss are joined by the last one to arrive, in
// workgroup order.
__global__ __launch_bounds__(256) void balance_finish_kernel(BalanceWs w, int32_t slots,
                                                             int32_t K, int32_t top_k, float coef,
                                                             BalanceOut o) {
  __shared__ double s_loss[kFinClasses];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 63, c = threadIdx.x >> 6;
  const int32_t k = blockIdx.x * kFinClasses + c;
  const bool in = k < K;
  const float* part = w.part + (int64_t)(in ? k : 0) * slots;
  const int32_t* count = w.count + (int64_t)(in ? k : 0) * slots;
  const int32_t* rows = w.count + (int64_t)K * slots;
  double a = 0.0;
  int64_t n = 0, live = 0;
#pragma unroll 4
  for (int32_t g = lane; g < slots; g += 64) {
    a += (double)part[g];
    n += count[g];
    live += rows[g];
  }
  for (int d = 32; d; d >>= 1) {
    a += __shfl_xor(a, d);
    n += __shfl_xor(n, d);
    live += __shfl_xor(live, d);
  }
  const double inv = live > 0 ? 1.0 / (double)live : 0.0;
  const double f = (double)n * inv / top_k, p = a * inv;
  if (lane == 0) {
    if (in) {
      w.share[k] = (float)f;
      o.prob[k] = (float)p;
      o.counts[k] = n;
    }
    s_loss[c] = in ? f * p : 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) *w.scale = (float)((double)coef * K * inv);
    const double l = (s_loss[0] + s_loss[1]) + (s_loss[2] + s_loss[3]);
    __hip_atomic_store(&w.loss_part[blockIdx.x], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = __hip_atomic_fetch_add(w.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last || c > 0) return;
  double t = 0.0;
  for (unsigned g = lane; g < gridDim.x; g += 64)
    t += __hip_atomic_load(&w.loss_part[g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
  if (lane == 0) *o.loss = (float)((double)coef * K * t);
}

// no rows: everything is 0
__global__ void balance_empty_kernel(int32_t K, BalanceOut o) {
  const int32_t k = blockIdx.x * 256 + threadIdx.x;
  if (k == 0) *o.loss = 0.0f;
  if (k < K) {
    o.prob[k] = 0.0f;
    o.counts[k] = 0;
  }
}

// class-major scores of more classes than a workgroup's slices hold go through
// a row-major copy: of their type, or of float32 where the gradient is added to
// another (so that it is rounded once)
constexpr int32_t kClassFrameMax = 512;
static bool through_rows(int32_t K, bool cm) { return cm && K > kClassFrameMax; }

static BalanceWs balance_ws(int64_t n, int32_t K, bool cm, void* base) {
  BalanceWs w{};
  size_t at = 0;
  const auto take = [&](size_t b) {
    const size_t o = at;
    at = (at + b + 255) & ~(size_t)255;
    return (void*)((unsigned char*)base + o);
  };
  // (at least the workgroups of the first pass: of 64 threads or more, a row each; of
  // further launches, which follow 512 workgroups or more, one for kChain rows)
  const size_t g = (size_t)std::min(n, std::min(4 * kLossWaves, balance_few(K))) +
                   (n > 512 * (int64_t)kChain ? (size_t)n / kChain : 0);
  w.ticket = (uint32_t*)take(4);
  w.scale = (float*)take(4);
  w.share = (float*)take(4 * (size_t)K);
  w.loss_part = (double*)take(8 * ((size_t)K / kFinClasses + 1));
  w.norm = (float2*)take(8 * (size_t)n);
  w.part = (float*)take(4 * g * K);
  w.count = (int32_t*)take(4 * g * (K + 1));
  if (through_rows(K, cm)) w.rows = take(4 * (size_t)n * K);
  w.bytes = at;
  return w;
}
size_t balance_workspace(const ScoresView& s) {
  return balance_ws(s.n, s.K, s.class_major(), nullptr).bytes;
}

int balance_loss(const ScoresView& s, const uint8_t* mask, int32_t top_k, float coef,
                 const BalanceOut& o, const ScoresView& out, bool accumulate, void* base,
                 hipStream_t st) {
  if (s.n == 0) {
    hipLaunchKernelGGL(balance_empty_kernel, dim3((unsigned)(s.K + 255) / 256), dim3(256), 0, st,
                       s.K, o);
    WGBM_LAUNCH_CHECK();
    return 0;
  }
  const bool cm = s.class_major(), turn = through_rows(s.K, cm);
  const BalanceWs w = balance_ws(s.n, s.K, cm, base);
  ScoresView v = s;
  if (turn) {
    v.data = w.rows;
    if (accumulate) v.dtype = kF32;
    v.rs = s.K;
    v.ks = 1;
    const int r = scores_to_rows(s, v, st);
    if (r) return r;
  }
  int32_t slots = 0;
  const auto stats = v.dtype == kF32    ? balance_stats_f32
                     : v.dtype == kBF16 ? balance_stats_bf16
                                        : balance_stats_f16;
  int r = stats(v, mask, top_k, w, &slots, st);
  if (r) return r;
  hipLaunchKernelGGL(balance_finish_kernel,
                     dim3((unsigned)((s.K + kFinClasses - 1) / kFinClasses)), dim3(256), 0, st, w,
                     slots, s.K, top_k, coef, o);
  WGBM_LAUNCH_CHECK();
  if (!out.data) return 0;
  const auto grad = v.dtype == kF32    ? balance_grad_f32
                    : v.dtype == kBF16 ? balance_grad_bf16
                                       : balance_grad_f16;
  // (in place in the row-major copy: a thread writes what it alone has read)
  r = grad(v, w, turn ? v : out, turn ? false : accumulate, st);
  if (r || !turn) return r;
  return rows_to_scores(v, out, accumulate, st);
}

}  // namespace wgbm
