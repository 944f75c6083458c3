// The balance loss: how evenly rows fall on classes.
//   c_k = rows with class k among their top_k, f_k = c_k / (n' top_k),
//   P_k = mean of p_ik over the n' rows that count,
//   L = coef K sum_k f_k P_k,   dL/ds_ik = coef K / n' p_ik (f_k - sum_j f_j p_ij)
// (the counts are held constant).  Counts are integers and the mean's partial
// sums are joined in a fixed order in float64, so results do not depend on the
// order of execution.
#include <algorithm>

#include "losses.hpp"
#include "losses_host.hpp"

namespace wgbm {

// (score, class) order of a top-k: larger scores first, lower classes first
// among equals.  A NaN is never taken.
__device__ __forceinline__ bool comes_before(float a, int32_t ka, float b, int32_t kb) {
  return a > b || (a == b && ka < kb);
}

// the best (score, class) that comes after (v0, k0) among the classes k of one
// thread; class -1 when there is none (-inf is not taken)
template <typename T>
__device__ __forceinline__ void next_best(const T* p, int64_t ks, int32_t K, int32_t first,
                                          int32_t step, float v0, int32_t k0, float& v,
                                          int32_t& kb) {
  v = -__builtin_inff();
  kb = -1;
  for (int32_t k = first; k < K; k += step) {
    const float x = to_f32(p[(int64_t)k * ks]);
    if (x > -__builtin_inff() && (k0 < 0 || comes_before(v0, k0, x, k)) &&
        (kb < 0 || comes_before(x, k, v, kb))) {
      v = x;
      kb = k;
    }
  }
}

// counts[k] and the number of rows that count (counts[K])
template <typename T, bool CM>
__global__ __launch_bounds__(256) void topk_count_kernel(ScoresView s,
                                                         const uint8_t* __restrict__ mask,
                                                         int32_t top_k,
                                                         unsigned long long* counts) {
  const int64_t i = CM ? (int64_t)blockIdx.x * 256 + threadIdx.x
                       : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= s.n || (mask && !mask[i])) return;
  const T* p = (const T*)s.data + i * s.rs;
  const int lane = threadIdx.x & 63;
  float v0 = 0.0f;
  int32_t k0 = -1;
  for (int32_t t = 0; t < top_k; ++t) {
    float v;
    int32_t k;
    next_best<T>(p, s.ks, s.K, CM ? 0 : lane, CM ? 1 : 64, v0, k0, v, k);
    if (!CM) {
      for (int o = 32; o; o >>= 1) {
        const float v2 = __shfl_xor(v, o);
        const int32_t k2 = __shfl_xor(k, o);
        if (k2 >= 0 && (k < 0 || comes_before(v2, k2, v, k))) {
          v = v2;
          k = k2;
        }
      }
    }
    if (k < 0) break;
    if (CM || lane == 0) atomicAdd(&counts[k], 1ull);
    v0 = v;
    k0 = k;
  }
}

// rows with a class that count: sum over the norms (maximum above -inf)
__global__ __launch_bounds__(256) void live_rows_kernel(const float2* __restrict__ norm, int64_t n,
                                                        unsigned long long* live) {
  int64_t c = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    c += norm[i].x == -__builtin_inff() ? 0 : 1;
  __shared__ unsigned long long s_c[4];
  unsigned long long x = (unsigned long long)c;
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) s_c[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0) atomicAdd(live, s_c[0] + s_c[1] + s_c[2] + s_c[3]);
}

// part[chunk][k] = sum of p_ik over a chunk of rows
template <typename T, bool CM>
__global__ __launch_bounds__(256) void class_sums_kernel(ScoresView s,
                                                         const float2* __restrict__ norm,
                                                         int64_t rows, float* __restrict__ part) {
  const int64_t i0 = (int64_t)blockIdx.y * rows, i1 = s.n - i0 > rows ? i0 + rows : s.n;
  const T* p = (const T*)s.data;
  float a = 0.0f;
  if (CM) {
    const int32_t k = blockIdx.x;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
      const float2 v = norm[i];
      if (v.x != -__builtin_inff()) a += loss_expf((to_f32(p[i + k * s.ks]) - v.x) - v.y);
    }
    __shared__ float s_a[4];
    for (int o = 32; o; o >>= 1) a += __shfl_xor(a, o);
    if ((threadIdx.x & 63) == 0) s_a[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0)
      part[(int64_t)blockIdx.y * s.K + k] = (s_a[0] + s_a[1]) + (s_a[2] + s_a[3]);
  } else {
    const int32_t k = blockIdx.x * 256 + threadIdx.x;
    if (k >= s.K) return;
    for (int64_t i = i0; i < i1; ++i) {
      const float2 v = norm[i];
      if (v.x != -__builtin_inff()) a += loss_expf((to_f32(p[i * s.rs + k]) - v.x) - v.y);
    }
    part[(int64_t)blockIdx.y * s.K + k] = a;
  }
}

// one workgroup: shares f_k, means P_k, the loss and the gradient's scale
__global__ __launch_bounds__(1024) void balance_finish_kernel(
    const float* __restrict__ part, int32_t chunks, const unsigned long long* __restrict__ counts,
    int32_t K, int32_t top_k, float coef, BalanceOut o, float* __restrict__ share,
    float* __restrict__ scale) {
  const double live = (double)counts[K];
  const double inv = live > 0.0 ? 1.0 / live : 0.0;
  double l = 0.0;
  for (int32_t k = threadIdx.x; k < K; k += 1024) {
    double a = 0.0;
    for (int32_t c = 0; c < chunks; ++c) a += (double)part[(int64_t)c * K + k];
    const double f = (double)counts[k] * inv / top_k;
    a *= inv;
    l += f * a;
    share[k] = (float)f;
    o.prob[k] = (float)a;
    o.counts[k] = (int64_t)counts[k];
  }
  __shared__ double s_l[16];
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
  if ((threadIdx.x & 63) == 0) s_l[threadIdx.x >> 6] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 16; ++w) t += s_l[w];
    *o.loss = (float)((double)coef * K * t);
    *scale = (float)((double)coef * K * inv);
  }
}

// rows' mean share q_i = sum_k f_k p_ik, and the gradient's coefficients
template <typename T, bool CM>
__global__ __launch_bounds__(256) void row_share_kernel(ScoresView s,
                                                        const float2* __restrict__ norm,
                                                        const float* __restrict__ share,
                                                        float* __restrict__ q) {
  const int64_t i = CM ? (int64_t)blockIdx.x * 256 + threadIdx.x
                       : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= s.n) return;
  const float2 v = norm[i];
  const T* p = (const T*)s.data + i * s.rs;
  const int lane = threadIdx.x & 63;
  float a = 0.0f;
  if (v.x != -__builtin_inff())
    for (int32_t k = CM ? 0 : lane; k < s.K; k += CM ? 1 : 64)
      a = fmaf(share[k], loss_expf((to_f32(p[(int64_t)k * s.ks]) - v.x) - v.y), a);
  if (!CM)
    for (int o = 32; o; o >>= 1) a += __shfl_xor(a, o);
  if (CM || lane == 0) q[i] = a;
}

template <typename T, bool CM>
__global__ __launch_bounds__(256) void balance_grad_kernel(ScoresView s,
                                                           const float2* __restrict__ norm,
                                                           const float* __restrict__ share,
                                                           const float* __restrict__ q,
                                                           const float* __restrict__ scale,
                                                           bool accumulate, ScoresView out) {
  const int64_t total = s.n * s.K;
  const float c = *scale;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (int64_t)gridDim.x * 256) {
    const int64_t i = CM ? t % s.n : t / s.K;
    const int32_t k = (int32_t)(CM ? t / s.n : t % s.K);
    const float2 v = norm[i];
    float x = 0.0f;
    if (v.x != -__builtin_inff()) {
      const float p = loss_expf((to_f32(((const T*)s.data)[i * s.rs + k * s.ks]) - v.x) - v.y);
      x = c * p * (share[k] - q[i]);
    }
    T* o = (T*)out.data + i * out.rs + k * out.ks;
    if (accumulate) x += to_f32(*o);
    *o = from_f32<T>(x);
  }
}

__global__ void zero_u64_kernel(unsigned long long* p, int32_t n) {
  const int32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

// row chunks of the mean's partial sums: enough workgroups, few partials
static int32_t sum_chunks(int64_t n, int32_t K, bool cm) {
  const int64_t wide = cm ? K : (K + 255) / 256;
  const int64_t want = (2048 + wide - 1) / wide;
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>(want, (n + 255) / 256));
}

// workspace: counts [K + 1], norms [n], statistics or (later) the partial sums,
// shares [K], row shares [n], scale
struct BalanceWs {
  unsigned long long* counts;
  float2* norm;
  float* q;
  float* share;
  float* scale;
  float* part;
  void* stats;
  size_t bytes;
};
static BalanceWs balance_ws(int64_t n, int32_t K, bool cm, void* base) {
  BalanceWs w{};
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t o = at;
    at = (at + b + 255) & ~(size_t)255;
    return (void*)((unsigned char*)base + o);
  };
  w.counts = (unsigned long long*)take(8 * ((size_t)K + 1));
  w.norm = (float2*)take(8 * (size_t)n);
  w.q = (float*)take(4 * (size_t)n);
  w.share = (float*)take(4 * (size_t)K);
  w.scale = (float*)take(4);
  w.part = (float*)take(4 * (size_t)K * sum_chunks(n, K, cm));
  w.stats = take(log_probs_workspace(n, K, cm));
  w.bytes = at;
  return w;
}
size_t balance_workspace(int64_t n, int32_t K, bool cm) {
  return balance_ws(n, K, cm, nullptr).bytes;
}

template <typename T, bool CM>
static int balance_t(const ScoresView& s, const uint8_t* mask, int32_t top_k, float coef,
                     const BalanceOut& o, const ScoresView& out, bool accumulate, void* base,
                     hipStream_t st) {
  const BalanceWs w = balance_ws(s.n, s.K, CM, base);
  const unsigned rows = (unsigned)(CM ? (s.n + 255) / 256 : (s.n + 3) / 4);
  hipLaunchKernelGGL(zero_u64_kernel, dim3((unsigned)(s.K + 256) / 256), dim3(256), 0, st,
                     w.counts, s.K + 1);
  WGBM_LAUNCH_CHECK();
  const int32_t chunks = s.n ? sum_chunks(s.n, s.K, CM) : 0;
  if (s.n) {
    int r = class_log_probs(s, nullptr, mask, nullptr, (float*)w.norm, w.stats, st);
    if (r) return r;
    hipLaunchKernelGGL((topk_count_kernel<T, CM>), dim3(rows), dim3(256), 0, st, s, mask, top_k,
                       w.counts);
    WGBM_LAUNCH_CHECK();
    hipLaunchKernelGGL(live_rows_kernel, dim3((unsigned)std::min<int64_t>((s.n + 255) / 256, 512)),
                       dim3(256), 0, st, w.norm, s.n, w.counts + s.K);
    WGBM_LAUNCH_CHECK();
    const int64_t span = (s.n + chunks - 1) / chunks;
    hipLaunchKernelGGL((class_sums_kernel<T, CM>),
                       dim3((unsigned)(CM ? s.K : (s.K + 255) / 256), (unsigned)chunks), dim3(256),
                       0, st, s, w.norm, span, w.part);
    WGBM_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, st, w.part, chunks, w.counts,
                     s.K, top_k, coef, o, w.share, w.scale);
  WGBM_LAUNCH_CHECK();
  if (!out.data || !s.n) return 0;
  hipLaunchKernelGGL((row_share_kernel<T, CM>), dim3(rows), dim3(256), 0, st, s, w.norm, w.share,
                     w.q);
  WGBM_LAUNCH_CHECK();
  const int64_t total = s.n * s.K;
  hipLaunchKernelGGL((balance_grad_kernel<T, CM>),
                     dim3((unsigned)std::min<int64_t>((total + 255) / 256, 8192)), dim3(256), 0, st,
                     s, w.norm, w.share, w.q, w.scale, accumulate, out);
  WGBM_LAUNCH_CHECK();
  return 0;
}

int balance_loss(const ScoresView& s, const uint8_t* mask, int32_t top_k, float coef,
                 const BalanceOut& o, const ScoresView& out, bool accumulate, void* ws,
                 hipStream_t st) {
  if (s.class_major())
    LOSS_TYPES(s.dtype, return (balance_t<T, true>(s, mask, top_k, coef, o, out, accumulate, ws,
                                                   st)));
  LOSS_TYPES(s.dtype, return (balance_t<T, false>(s, mask, top_k, coef, o, out, accumulate, ws,
                                                  st)));
}

}  // namespace wgbm
