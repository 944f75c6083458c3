// The preference loss: paired log ratios of sequences of rows.
//   u_i = logp_i - ref_i,  U_s = sum of u_i over the rows of sequence s,
//   m_p = U_preferred - U_other,  z = beta m,
//   L_p = w_p ((1 - e) softplus(-z) + e softplus(z)),
//   dL_p/dm = w_p beta (e sigmoid(z) - (1 - e) sigmoid(-z)),
//   dL/dlogp_i = sum over the pairs of i's sequence, + preferred, - other
// Sums over rows and over pairs are float64 in a fixed order (a long
// sequence's sum loses its margin's digits in float32).
#include <algorithm>

#include "losses_host.hpp"

namespace wgbm {

__global__ __launch_bounds__(256) void seq_sums_kernel(PreferenceArgs a, double* __restrict__ U) {
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= a.n_seg) return;
  const int lane = threadIdx.x & 63;
  const int64_t i1 = a.seg_start[s + 1];
  double x = 0.0;
  for (int64_t i = a.seg_start[s] + lane; i < i1; i += 64)
    x += (double)a.log_prob[i] - (a.ref ? (double)a.ref[i] : 0.0);
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if (lane == 0) U[s] = x;
}

__device__ __forceinline__ double seq_value(const PreferenceArgs& a, const double* U, int32_t s) {
  if (U) return U[s];
  return (double)a.log_prob[s] - (a.ref ? (double)a.ref[s] : 0.0);
}

__global__ __launch_bounds__(256) void pair_loss_kernel(PreferenceArgs a,
                                                        const double* __restrict__ U,
                                                        float* __restrict__ slope) {
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= a.n_pairs) return;
  const float w = a.weight ? a.weight[p] : 1.0f;
  float loss = 0.0f, margin = 0.0f, d = 0.0f;
  if (w != 0.0f) {
    const int2 q = ((const int2*)a.pairs)[p];
    const double m = seq_value(a, U, q.x) - seq_value(a, U, q.y);
    margin = (float)m;
    const float z = (float)((double)a.beta * m);
    // e^-|z|, and from it both sigmoids and both softplus without overflow
    // or a difference of nearly equal numbers
    const float e = expf(-fabsf(z)), l = log1pf(e), inv = 1.0f / (1.0f + e);
    const float big = inv, small = e * inv;  // sigmoid(|z|), sigmoid(-|z|)
    const float up = z >= 0.0f ? big : small, down = z >= 0.0f ? small : big;
    loss = w * ((1.0f - a.smooth) * (l + fmaxf(-z, 0.0f)) + a.smooth * (l + fmaxf(z, 0.0f)));
    d = w * a.beta * (a.smooth * up - (1.0f - a.smooth) * down);
  }
  a.loss[p] = loss;
  a.margin[p] = margin;
  slope[p] = d;
}

// a wave per sequence: its pairs' slopes summed, the sum written to its rows
__global__ __launch_bounds__(256) void seq_grad_kernel(PreferenceArgs a,
                                                       const float* __restrict__ slope) {
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= a.n_seg) return;
  const int lane = threadIdx.x & 63;
  const int64_t j1 = a.inc_start[s + 1];
  double x = 0.0;
  for (int64_t j = a.inc_start[s] + lane; j < j1; j += 64) {
    const int32_t q = a.inc[j];
    const double d = (double)slope[q >> 1];
    x += q & 1 ? -d : d;
  }
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  const float g = (float)x;
  if (!a.seg_start) {
    if (lane == 0) a.grad[s] = g;
    return;
  }
  const int64_t i1 = a.seg_start[s + 1];
  for (int64_t i = a.seg_start[s] + lane; i < i1; i += 64) a.grad[i] = g;
}

// rows behind the last sequence have no gradient
__global__ __launch_bounds__(256) void tail_zero_kernel(PreferenceArgs a) {
  const int64_t i = a.seg_start[a.n_seg] + (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t j = i; j < a.n_rows; j += (int64_t)gridDim.x * 256) a.grad[j] = 0.0f;
}

size_t preference_workspace(int64_t n_seg, int64_t n_pairs, bool segments) {
  return (segments ? sizeof(double) * (size_t)n_seg : 0) + sizeof(float) * (size_t)n_pairs;
}

int preference_loss(const PreferenceArgs& a, void* ws, hipStream_t st) {
  double* U = a.seg_start ? (double*)ws : nullptr;
  float* slope = (float*)((double*)ws + (U ? a.n_seg : 0));
  const unsigned seq_blocks = (unsigned)((a.n_seg + 3) / 4);
  if (U) {
    if (a.n_seg) {
      hipLaunchKernelGGL(seq_sums_kernel, dim3(seq_blocks), dim3(256), 0, st, a, U);
      WGBM_LAUNCH_CHECK();
    }
  }
  if (a.n_pairs) {
    hipLaunchKernelGGL(pair_loss_kernel, dim3((unsigned)((a.n_pairs + 255) / 256)), dim3(256), 0,
                       st, a, U, slope);
    WGBM_LAUNCH_CHECK();
  }
  if (!a.grad) return 0;
  if (a.n_seg) {
    hipLaunchKernelGGL(seq_grad_kernel, dim3(seq_blocks), dim3(256), 0, st, a, slope);
    WGBM_LAUNCH_CHECK();
  }
  if (U && a.n_rows) {
    hipLaunchKernelGGL(tail_zero_kernel, dim3(64), dim3(256), 0, st, a);
    WGBM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace wgbm
