// The preference loss: paired log ratios of sequences of rows.
//   u_i = logp_i - ref_i,  U_s = sum of u_i over the rows of sequence s,
//   m_p = U_preferred - U_other,  z = beta m,
//   L_p = w_p ((1 - e) softplus(-z) + e softplus(z)),
//   dL_p/dm = w_p beta (e sigmoid(z) - (1 - e) sigmoid(-z)),
//   dL/dlogp_i = sum over the pairs of i's sequence, + preferred, - other
// Sums over rows and over pairs are float64 in an order that the plan fixes (a
// long sequence's sum loses its margin's digits in float32; atomics would add
// in the order of execution).
//
// Bound by memory: every row is read and written once.  The plan cuts sequences
// into tasks of at most 4096 rows, a wave each.  Where every
// sequence is one task and in at most one pair, one launch does everything: a
// wave sums a pair's two sequences, and writes their gradients.  Otherwise:
// tasks' sums, (tasks joined,) pairs, sequences' slopes, rows.
#include <algorithm>

#include "losses_host.hpp"

namespace wgbm {

// sum of u over the rows [b, e), by a wave (every lane gets it)
__device__ __forceinline__ double wave_rows_sum(const PreferenceArgs& a, int64_t b, int64_t e) {
  const int lane = threadIdx.x & 63;
  double x[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t i = b + lane;
  // four rows a lane in flight
  for (; i + 192 < e; i += 256) {
    float l[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      l[j] = a.log_prob[i + 64 * j];
      r[j] = a.ref ? a.ref[i + 64 * j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += (double)l[j] - (double)r[j];
  }
  float l[3], r[3];
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    const bool in = i + 64 * j < e;
    l[j] = in ? a.log_prob[i + 64 * j] : 0.0f;
    r[j] = in && a.ref ? a.ref[i + 64 * j] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) x[j] += (double)l[j] - (double)r[j];
  double s = (x[0] + x[1]) + (x[2] + x[3]);
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  return s;
}

// sum of u over the rows [b0, b0 + n0) less that over [b1, b1 + n1), by a wave:
// one list of rows, eight a lane in flight
__device__ __forceinline__ double wave_difference(const PreferenceArgs& a, int64_t b0, int n0,
                                                  int64_t b1, int n1) {
  constexpr int U = 8;
  double x[2] = {0.0, 0.0};
  for (int i = threadIdx.x & 63; i < n0 + n1; i += 64 * U) {
    float l[U], r[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = i + 64 * j;
      const int64_t at = k < n0 ? b0 + k : b1 + (k - n0);
      l[j] = k < n0 + n1 ? a.log_prob[at] : 0.0f;
      r[j] = a.ref && k < n0 + n1 ? a.ref[at] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const double u = (double)l[j] - (double)r[j];
      x[j % 2] += i + 64 * j < n0 ? u : -u;
    }
  }
  double s = x[0] + x[1];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  return s;
}

// grad = g for the rows [b, e), by a wave
__device__ __forceinline__ void wave_rows_fill(float* grad, int64_t b, int64_t e, float g) {
  for (int64_t i = b + (threadIdx.x & 63); i < e; i += 64) grad[i] = g;
}

struct PairLoss {
  float loss, margin, slope;
};
__device__ __forceinline__ PairLoss pair_loss(const PreferenceArgs& a, double m, float w) {
  PairLoss o;
  o.margin = (float)m;
  const float z = (float)((double)a.beta * m);
  // e^-|z|, and from it both sigmoids and both softplus without overflow or a
  // difference of nearly equal numbers
  const float e = expf(-fabsf(z)), l = log1pf(e), inv = 1.0f / (1.0f + e);
  const float up = z >= 0.0f ? inv : e * inv, down = z >= 0.0f ? e * inv : inv;
  o.loss = w * ((1.0f - a.smooth) * (l + fmaxf(-z, 0.0f)) + a.smooth * (l + fmaxf(z, 0.0f)));
  o.slope = w * a.beta * (a.smooth * up - (1.0f - a.smooth) * down);
  return o;
}

// ---------------------------------------------------------------------------
// everything in one launch: a wave per pair, then a wave per idle task (rows
// of sequences without a pair, and rows behind the last sequence)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void preference_fused_kernel(PreferenceArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= a.n_pairs) {
    const int64_t k = t - a.n_pairs;
    if (a.grad && k < a.n_idle) {
      const int64_t b = a.idle[2 * k], e = a.idle[2 * k + 1];
      wave_rows_fill(a.grad, b, e, 0.0f);
    }
    return;
  }
  const int32_t s0 = a.pairs[2 * t], s1 = a.pairs[2 * t + 1];
  const int64_t b0 = a.seg_start[s0], e0 = a.seg_start[s0 + 1];
  const int64_t b1 = a.seg_start[s1], e1 = a.seg_start[s1 + 1];
  const float w = a.weight ? a.weight[t] : 1.0f;
  PairLoss o{0.0f, 0.0f, 0.0f};
  if (w != 0.0f)
    o = pair_loss(a, wave_difference(a, b0, (int)(e0 - b0), b1, (int)(e1 - b1)), w);
  if (lane == 0) {
    a.loss[t] = o.loss;
    a.margin[t] = o.margin;
  }
  if (!a.grad) return;
  wave_rows_fill(a.grad, b0, e0, o.slope);
  wave_rows_fill(a.grad, b1, e1, -o.slope);
}

// ---------------------------------------------------------------------------
// the steps apart
// ---------------------------------------------------------------------------
// part[t]: a task's sum (tasks of rows behind the last sequence: none)
__global__ __launch_bounds__(256) void task_sums_kernel(PreferenceArgs a, double* __restrict__ part) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.n_tasks || a.task[3 * t] < 0) return;
  const double x = wave_rows_sum(a, a.task[3 * t + 1], a.task[3 * t + 2]);
  if ((threadIdx.x & 63) == 0) part[t] = x;
}

// U[s]: a sequence's tasks joined, a wave each
__global__ __launch_bounds__(256) void join_tasks_kernel(PreferenceArgs a,
                                                         const double* __restrict__ part,
                                                         double* __restrict__ U) {
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= a.n_seg) return;
  double x = 0.0;
  const int64_t t1 = a.task_start[s + 1];
  for (int64_t t = a.task_start[s] + (threadIdx.x & 63); t < t1; t += 64) x += part[t];
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) U[s] = x;
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
  const int2 q = ((const int2*)a.pairs)[p];
  const float w = a.weight ? a.weight[p] : 1.0f;
  PairLoss o{0.0f, 0.0f, 0.0f};
  if (w != 0.0f) o = pair_loss(a, seq_value(a, U, q.x) - seq_value(a, U, q.y), w);
  a.loss[p] = o.loss;
  a.margin[p] = o.margin;
  slope[p] = o.slope;
}

__device__ __forceinline__ float signed_slope(const PreferenceArgs& a, const float* slope,
                                              int64_t j) {
  const int32_t q = a.inc[j];
  const float d = slope[q >> 1];
  return q & 1 ? -d : d;
}

// out[s] = sum of the slopes of sequence s's pairs.  The first workgroups take
// the pieces of the sequences in very many pairs (a sequence of one piece is
// done then), the others a share of the rest each: the plan's shares have the
// same number of sequences and incidences together, so that the incidences of
// one are consecutive, fit LDS, and are gathered with all lanes busy, however
// few or many a sequence has.
constexpr int kIncTile = 1536;  // 1024 + the pairs of one sequence (256)
__global__ __launch_bounds__(256) void seq_slopes_kernel(PreferenceArgs a,
                                                         const float* __restrict__ slope,
                                                         double* __restrict__ piece_sum,
                                                         float* __restrict__ out) {
  if ((int64_t)blockIdx.x < a.n_pieces) {
    const int64_t q = blockIdx.x, e = a.piece[3 * q + 2];
    double x[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t j = a.piece[3 * q + 1] + threadIdx.x; j < e; j += 1024) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j + 256 * k < e) x[k] += (double)signed_slope(a, slope, j + 256 * k);
    }
    double s = (x[0] + x[1]) + (x[2] + x[3]);
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    __shared__ double w[4];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    s = (w[0] + w[1]) + (w[2] + w[3]);
    if (a.piece[3 * q] >= 0)
      out[a.piece[3 * q]] = (float)s;
    else
      piece_sum[q] = s;
    return;
  }
  __shared__ float tile[kIncTile];
  const int64_t c = blockIdx.x - a.n_pieces;
  const int64_t s0 = a.share[c], s1 = a.share[c + 1];
  const int64_t r0 = a.inc_start[s0];
  const int m = (int)(a.inc_start[s1] - r0);
  float d[kIncTile / 256];
#pragma unroll
  for (int k = 0; k < kIncTile / 256; ++k) {
    const int j = threadIdx.x + 256 * k;
    d[k] = j < m ? signed_slope(a, slope, r0 + j) : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kIncTile / 256; ++k) tile[threadIdx.x + 256 * k] = d[k];
  __syncthreads();
  for (int64_t s = s0 + threadIdx.x; s < s1; s += 256) {
    if (a.is_long && a.is_long[s]) continue;
    const int lo = (int)(a.inc_start[s] - r0), hi = (int)(a.inc_start[s + 1] - r0);
    double x = 0.0;
    for (int j = lo; j < hi; ++j) x += (double)tile[j];
    out[s] = (float)x;
  }
}

// the sequences of several pieces, a wave each
__global__ __launch_bounds__(64) void seq_pieces_kernel(PreferenceArgs a,
                                                        const double* __restrict__ piece_sum,
                                                        float* __restrict__ out) {
  const int64_t k = blockIdx.x;
  double x = 0.0;
  for (int64_t q = a.multi[3 * k + 1] + threadIdx.x; q < a.multi[3 * k + 2]; q += 64)
    x += piece_sum[q];
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if (threadIdx.x == 0) out[a.multi[3 * k]] = (float)x;
}

// rows take their sequence's slope, a wave a task
__global__ __launch_bounds__(256) void task_rows_kernel(PreferenceArgs a,
                                                        const float* __restrict__ seq) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.n_tasks) return;
  const int64_t s = a.task[3 * t];
  wave_rows_fill(a.grad, a.task[3 * t + 1], a.task[3 * t + 2], s >= 0 ? seq[s] : 0.0f);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct PrefWs {
  float* slope;      // [n_pairs]
  double* part;      // [n_tasks]
  double* U;         // [n_seg]
  float* seq;        // [n_seg]
  double* piece_sum; // [n_pieces]
  size_t bytes;
};
static PrefWs pref_ws(const PreferenceArgs& a, void* base) {
  PrefWs w{};
  if (a.disjoint) return w;
  size_t at = 0;
  const auto take = [&](size_t b) {
    const size_t o = at;
    at = (at + b + 255) & ~(size_t)255;
    return (void*)((unsigned char*)base + o);
  };
  w.slope = (float*)take(4 * (size_t)a.n_pairs);
  if (a.n_pieces) w.piece_sum = (double*)take(8 * (size_t)a.n_pieces);
  if (a.seg_start) {
    w.part = (double*)take(8 * (size_t)a.n_tasks);
    w.U = a.task_start ? (double*)take(8 * (size_t)a.n_seg) : w.part;
    w.seq = (float*)take(4 * (size_t)a.n_seg);
  }
  w.bytes = at;
  return w;
}
size_t preference_workspace(const PreferenceArgs& a) { return pref_ws(a, nullptr).bytes; }

static dim3 wave_blocks(int64_t waves) { return dim3((unsigned)((waves + 3) / 4)); }

int preference_loss(const PreferenceArgs& a, void* base, hipStream_t st) {
  const dim3 wg(256);
  if (a.disjoint) {
    const int64_t waves = a.n_pairs + (a.grad ? a.n_idle : 0);
    if (!waves) return 0;
    hipLaunchKernelGGL(preference_fused_kernel, wave_blocks(waves), wg, 0, st, a);
    WGBM_LAUNCH_CHECK();
    return 0;
  }
  const PrefWs w = pref_ws(a, base);
  if (a.seg_start && a.n_pairs) {
    hipLaunchKernelGGL(task_sums_kernel, wave_blocks(a.n_tasks), wg, 0, st, a, w.part);
    WGBM_LAUNCH_CHECK();
    if (a.task_start) {
      hipLaunchKernelGGL(join_tasks_kernel, wave_blocks(a.n_seg), wg, 0, st, a, w.part, w.U);
      WGBM_LAUNCH_CHECK();
    }
  }
  if (a.n_pairs) {
    hipLaunchKernelGGL(pair_loss_kernel, dim3((unsigned)((a.n_pairs + 255) / 256)), wg, 0, st, a,
                       w.U, w.slope);
    WGBM_LAUNCH_CHECK();
  }
  if (!a.grad) return 0;
  float* seq = a.seg_start ? w.seq : a.grad;
  if (a.n_seg) {
    hipLaunchKernelGGL(seq_slopes_kernel, dim3((unsigned)(a.n_pieces + a.n_shares)), wg, 0, st, a,
                       w.slope, w.piece_sum, seq);
    WGBM_LAUNCH_CHECK();
  }
  if (a.n_multi) {
    hipLaunchKernelGGL(seq_pieces_kernel, dim3((unsigned)a.n_multi), dim3(64), 0, st, a,
                       w.piece_sum, seq);
    WGBM_LAUNCH_CHECK();
  }
  if (a.seg_start && a.n_tasks) {
    hipLaunchKernelGGL(task_rows_kernel, wave_blocks(a.n_tasks), wg, 0, st, a, seq);
    WGBM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace wgbm
