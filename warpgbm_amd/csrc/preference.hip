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
// into tasks of at most 4096 rows, 4 to 64 lanes each (the plan's choice).  Where
// every sequence is one task and in at most one pair, one launch does everything:
// the lanes of a pair sum its two sequences, and write their gradients.
// Otherwise: tasks' sums, (tasks joined,) pairs, sequences' slopes, rows.
#include <algorithm>

#include "losses_host.hpp"

namespace wgbm {

// Rows are read and written four to a lane, 16 bytes wherever they begin (this
// GPU takes such addresses): a wave has 256 rows a load.  A lane whose four would
// pass the end reads the last four instead (no branch: all loads are in flight
// together) and leaves out those that are another lane's.
struct Rows4 {
  float v[4];
};
__device__ __forceinline__ Rows4 load_rows(const float* p) {
  Rows4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}

// sum of u over the rows [b, b + n), by L lanes (each its own part)
template <int U, int L>
__device__ __forceinline__ double lane_rows_sum(const PreferenceArgs& a, int64_t b, int n) {
  const int lane = threadIdx.x & (L - 1);
  const float* lp = a.log_prob + b;
  const float* ref = a.ref ? a.ref + b : nullptr;
  if (n < 4) {
    if (lane >= n) return 0.0;
    return (double)lp[lane] - (ref ? (double)ref[lane] : 0.0);
  }
  double x[U];
#pragma unroll
  for (int j = 0; j < U; ++j) x[j] = 0.0;
  for (int k0 = 4 * lane; k0 < n; k0 += 4 * L * U) {
    Rows4 l[U], r[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = k0 + 4 * L * j, at = k < n - 4 ? k : n - 4;
      l[j] = load_rows(lp + at);
      if (ref) r[j] = load_rows(ref + at);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = k0 + 4 * L * j, skip = k < n - 4 ? 0 : k - (n - 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double u = (double)l[j].v[e] - (ref ? (double)r[j].v[e] : 0.0);
        if (e >= skip) x[j] += u;
      }
    }
  }
  double s = x[0];
#pragma unroll
  for (int j = 1; j < U; ++j) s += x[j];
  return s;
}
// the number of a group of L lanes in a grid of 256-thread workgroups (a grid's
// threads are counted in 32 bits along x: group_blocks folds longer ones)
template <int L>
__device__ __forceinline__ int64_t group_number() {
  return ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / L) + threadIdx.x / L;
}
template <int L>
__device__ __forceinline__ double lanes_sum(double s) {
  for (int o = L / 2; o; o >>= 1) s += __shfl_xor(s, o);
  return s;
}

// grad = g for the rows [b, b + n), by L lanes
template <int L>
__device__ __forceinline__ void rows_fill(float* grad, int64_t b, int n, float g) {
  float* p = grad + b;
  const Rows4 v = {{g, g, g, g}};
  for (int k = 4 * (threadIdx.x & (L - 1)); k < n; k += 4 * L) {
    if (n - k >= 4) {
      __builtin_memcpy(p + k, &v, 16);
    } else {
      for (int j = k; j < n; ++j) p[j] = g;
    }
  }
}

struct PairLoss {
  float loss, margin, slope;
};
__device__ __forceinline__ PairLoss pair_loss(const PreferenceArgs& a, double m, float w) {
  PairLoss o;
  o.margin = (float)m;
  // From here in float32, to which the loss and the slope are rounded anyway: z's
  // rounding costs 2^-24 of a loss of |z|, and 2^-24 |z| of e^-|z|, at most 2^-25 of 1.
  const float z = (float)((double)a.beta * m);
  // e^-|z|, and from it both sigmoids and both softplus without overflow or a
  // difference of nearly equal numbers
  const float e = expf(-fabsf(z)), l = log1pf(e), inv = 1.0f / (1.0f + e);
  const float up = z >= 0.0f ? inv : e * inv, down = z >= 0.0f ? e * inv : inv;
  o.loss = (1.0f - a.smooth) * (l + fmaxf(-z, 0.0f));
  // (no 0 * inf where the preferred sequence alone is possible)
  if (a.smooth != 0.0f) o.loss += a.smooth * (l + fmaxf(z, 0.0f));
  o.loss *= w;
  o.slope = w * a.beta * (a.smooth * up - (1.0f - a.smooth) * down);
  return o;
}

// ---------------------------------------------------------------------------
// everything in one launch: L lanes a pair, then as many an idle task (rows of
// sequences without a pair, and rows behind the last sequence).  50000 pairs
// of sequences of 200 rows on average, all with reference: 53 us, 4.5 TB/s (a
// copy of as many bytes 47); with a row a lane and load instead of four 63.
// ---------------------------------------------------------------------------
template <int L>
__global__ __launch_bounds__(256) void preference_fused_kernel(PreferenceArgs a) {
  const int64_t t = group_number<L>();
  if (t >= a.n_pairs) {
    const int64_t k = t - a.n_pairs;
    if (a.grad && k < a.n_idle) {
      const int64_t b = a.idle[2 * k], e = a.idle[2 * k + 1];
      rows_fill<L>(a.grad, b, (int)(e - b), 0.0f);
    }
    return;
  }
  const int32_t s0 = a.pairs[2 * t], s1 = a.pairs[2 * t + 1];
  const int64_t b0 = a.seg_start[s0], b1 = a.seg_start[s1];
  const int n0 = (int)(a.seg_start[s0 + 1] - b0), n1 = (int)(a.seg_start[s1 + 1] - b1);
  const float w = a.weight ? a.weight[t] : 1.0f;
  PairLoss o{0.0f, 0.0f, 0.0f};
  if (w != 0.0f) {
    const double x = lane_rows_sum<2, L>(a, b0, n0), y = lane_rows_sum<2, L>(a, b1, n1);
    o = pair_loss(a, lanes_sum<L>(x - y), w);
  }
  if ((threadIdx.x & (L - 1)) == 0) {
    a.loss[t] = o.loss;
    a.margin[t] = o.margin;
  }
  if (!a.grad) return;
  rows_fill<L>(a.grad, b0, n0, o.slope);
  rows_fill<L>(a.grad, b1, n1, -o.slope);
}

// ---------------------------------------------------------------------------
// the steps apart
// ---------------------------------------------------------------------------
// part[t]: a task's sum (tasks of rows behind the last sequence: none).  20001
// sequences of 25 rows 5 us (12 with a wave each): short ones are bound by the
// latency of their table, then their rows; 100 sequences of 200000 rows with
// reference 4 TB/s.
template <int L>
__global__ __launch_bounds__(256) void task_sums_kernel(PreferenceArgs a, double* __restrict__ part) {
  const int64_t t = group_number<L>();
  if (t >= a.n_tasks) return;
  const int64_t s = a.task[3 * t], b = a.task[3 * t + 1], e = a.task[3 * t + 2];
  if (s < 0) return;
  const double x = lanes_sum<L>(lane_rows_sum<L < 64 ? 2 : 4, L>(a, b, (int)(e - b)));
  if ((threadIdx.x & (L - 1)) == 0) part[t] = x;
}

// U[s]: a sequence's tasks joined, a wave each
__global__ __launch_bounds__(256) void join_tasks_kernel(PreferenceArgs a,
                                                         const double* __restrict__ part,
                                                         double* __restrict__ U) {
  const int64_t s = group_number<64>();
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

// a thread a pair: two gathered values (1M rows, 2M pairs 27 us, which is the
// gathers' line traffic: 8 bytes used of every two lines fetched)
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
// few or many a sequence has.  1M sequences, 2M pairs: 45 us, 4M gathers of a
// slope from another line each.
constexpr int kIncTile = 512;  // 256 + the pairs of one sequence (256)
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
  const int64_t s = s0 + threadIdx.x;
  if (s >= s1 || (a.is_long && a.is_long[s])) return;
  const int lo = (int)(a.inc_start[s] - r0), hi = (int)(a.inc_start[s + 1] - r0);
  double x = 0.0;
  for (int j = lo; j < hi; ++j) x += (double)tile[j];
  out[s] = (float)x;
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

// rows take their sequence's slope, L lanes a task
template <int L>
__global__ __launch_bounds__(256) void task_rows_kernel(PreferenceArgs a,
                                                        const float* __restrict__ seq) {
  const int64_t t = group_number<L>();
  if (t >= a.n_tasks) return;
  const int64_t s = a.task[3 * t], b = a.task[3 * t + 1], e = a.task[3 * t + 2];
  rows_fill<L>(a.grad, b, (int)(e - b), s >= 0 ? seq[s] : 0.0f);
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

// workgroups of n groups of L lanes
template <int L>
static dim3 group_blocks(int64_t n) {
  const int64_t b = (n + 256 / L - 1) / (256 / L), x = std::min(b, int64_t(1) << 23);
  return dim3((unsigned)x, (unsigned)((b + x - 1) / x));
}

// L: lanes of a task or pair
template <int L>
static int preference_lanes(const PreferenceArgs& a, void* base, hipStream_t st) {
  const dim3 wg(256);
  if (a.disjoint) {
    const int64_t n = a.n_pairs + (a.grad ? a.n_idle : 0);
    if (!n) return 0;
    hipLaunchKernelGGL(preference_fused_kernel<L>, group_blocks<L>(n), wg, 0, st, a);
    WGBM_LAUNCH_CHECK();
    return 0;
  }
  const PrefWs w = pref_ws(a, base);
  if (a.seg_start && a.n_pairs) {
    hipLaunchKernelGGL(task_sums_kernel<L>, group_blocks<L>(a.n_tasks), wg, 0, st, a, w.part);
    WGBM_LAUNCH_CHECK();
    if (a.task_start) {
      hipLaunchKernelGGL(join_tasks_kernel, group_blocks<64>(a.n_seg), wg, 0, st, a, w.part, w.U);
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
    hipLaunchKernelGGL(task_rows_kernel<L>, group_blocks<L>(a.n_tasks), wg, 0, st, a, seq);
    WGBM_LAUNCH_CHECK();
  }
  return 0;
}

int preference_loss(const PreferenceArgs& a, void* base, hipStream_t st) {
  switch (a.lanes) {
    case 4: return preference_lanes<4>(a, base, st);
    case 8: return preference_lanes<8>(a, base, st);
    case 16: return preference_lanes<16>(a, base, st);
    case 32: return preference_lanes<32>(a, base, st);
    default: return preference_lanes<64>(a, base, st);
  }
}

}  // namespace wgbm
