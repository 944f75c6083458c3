// Losses of class scores: log-probabilities, the clipped policy loss and the
// balance loss, each with its gradient with respect to the scores.
//
// Rows that fit the registers of the threads that share them take one launch
// (losses_rows.hpp).  Here: longer rows, both layouts.  A row's classes are cut
// into `splits` ranges whose statistics (running maximum and sums) are kept in
// the workspace, joined per row, and the gradient is written by an elementwise
// pass that reads the scores again.  The policy loss of 30000 x 3300 bfloat16
// class-major takes 392 us (a lane reads two bytes: 128 a wave and load), of 20000
// x 2000 float32 class-major against a reference 276 (2.9 TB/s of two reads of
// both and the gradient), of 2000 x 50000 bfloat16 row-major against one 422.
#include <algorithm>

#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

// statistics of the classes [k0, k1), k0 + step * j, of one row by one thread
template <typename T, bool REF>
__device__ __forceinline__ RowStats scan_classes(const T* s, const T* r, int64_t ks, int64_t rks,
                                                 int32_t k0, int32_t k1, int32_t step,
                                                 int32_t label) {
  RowStats a = empty_stats();
  constexpr int U = 8;
  for (int32_t k = k0; k < k1; k += U * step) {
    float v[U], w[U];
    float m = a.m, mr = a.mr;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const bool in = k1 - k > j * step;
      v[j] = in ? to_f32(s[(int64_t)(k + j * step) * ks]) : -__builtin_inff();
      w[j] = REF && in ? to_f32(r[(int64_t)(k + j * step) * rks]) : -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      m = fmaxf(m, v[j]);
      mr = fmaxf(mr, w[j]);
    }
    rebase_stats<REF>(a, m, mr);
    const float ms = safe_max(m), mrs = safe_max(mr);
    // (the eight's sums first: a shorter chain of additions, fewer roundings)
    RowStats e = empty_stats();
#pragma unroll
    for (int j = 0; j < U; ++j)
      add_class<REF>(e, v[j] - ms, w[j] - mrs, k + j * step == label);
    a.z += e.z;
    a.za += e.za;
    if (REF) {
      a.zr += e.zr;
      a.u += e.u;
    }
  }
  return a;
}

__device__ __forceinline__ RowStats shfl_xor_stats(const RowStats& a, int o) {
  RowStats b;
  b.m = __shfl_xor(a.m, o);
  b.z = __shfl_xor(a.z, o);
  b.za = __shfl_xor(a.za, o);
  b.mr = __shfl_xor(a.mr, o);
  b.zr = __shfl_xor(a.zr, o);
  b.u = __shfl_xor(a.u, o);
  return b;
}

// part[split][row]: the statistics of one range of a row's classes.  Rows next
// to each other: a thread per (row, range); classes next to each other: a wave.
template <typename T, bool CM, bool REF>
__global__ __launch_bounds__(256) void row_stats_kernel(ScoresView s, ScoresView ref,
                                                        const int32_t* __restrict__ label,
                                                        int32_t span, RowStats* __restrict__ part) {
  const int64_t i = CM ? (int64_t)blockIdx.x * 256 + threadIdx.x
                       : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= s.n) return;
  const int32_t k0 = blockIdx.y * span, k1 = s.K - k0 > span ? k0 + span : s.K;
  const T* p = (const T*)s.data + i * s.rs;
  const T* q = REF ? (const T*)ref.data + i * ref.rs : nullptr;
  const int32_t lab = row_label(label, i, s.K);
  RowStats a;
  if (CM) {
    a = scan_classes<T, REF>(p, q, s.ks, ref.ks, k0, k1, 1, lab);
  } else {
    a = scan_classes<T, REF>(p, q, s.ks, ref.ks, k0 + (int)(threadIdx.x & 63), k1, 64, lab);
    for (int o = 32; o; o >>= 1) a = join_stats<REF>(a, shfl_xor_stats(a, o));
  }
  if (CM || (threadIdx.x & 63) == 0) part[(int64_t)blockIdx.y * s.n + i] = a;
}

// ---------------------------------------------------------------------------
// rows: the ranges of a row joined (by a thread, or a wave's lanes over the
// ranges), then what follows from the whole row
// ---------------------------------------------------------------------------
template <bool REF>
__device__ __forceinline__ RowStats join_ranges(const RowStats* part, int64_t n, int64_t i,
                                                int32_t splits, bool wave) {
  RowStats a = empty_stats();
  const int lane = threadIdx.x & 63;
  for (int32_t j = wave ? lane : 0; j < splits; j += wave ? 64 : 1)
    a = join_stats<REF>(a, part[(int64_t)j * n + i]);
  if (wave)
    for (int o = 32; o; o >>= 1) a = join_stats<REF>(a, shfl_xor_stats(a, o));
  return a;
}

template <typename T>
__global__ __launch_bounds__(256) void log_prob_rows_kernel(ScoresView s,
                                                            const int32_t* __restrict__ label,
                                                            const RowStats* __restrict__ part,
                                                            int32_t splits, float* log_prob,
                                                            float2* norm) {
  const bool wave = splits > 1;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t i = wave ? t >> 6 : t;
  if (i >= s.n) return;
  const RowStats a = join_ranges<false>(part, s.n, i, splits, wave);
  if (wave && (threadIdx.x & 63)) return;
  const int32_t lab = row_label(label, i, s.K);
  const float sa = lab >= 0 ? to_f32(((const T*)s.data)[i * s.rs + lab * s.ks]) : 0.0f;
  write_log_prob(a, sa, lab, i, log_prob, norm);
}

template <typename T, bool REF>
__global__ __launch_bounds__(256) void policy_rows_kernel(ScoresView s, ScoresView ref,
                                                          PolicyRows g,
                                                          const RowStats* __restrict__ part,
                                                          int32_t splits,
                                                          RowCoef* __restrict__ coef) {
  const bool wave = splits > 1;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t i = wave ? t >> 6 : t;
  const bool in = i < s.n;
  const float w = !in ? 0.0f : g.weight ? g.weight[i] : 1.0f;
  const int32_t lab = in ? row_label(g.action, i, s.K) : -1;
  const bool live = w != 0.0f && lab >= 0;
  PolicyRow o{};
  RowStats a = empty_stats();
  float sa = 0.0f, ra = 0.0f, A = 0.0f, old = 0.0f;
  if (live) {
    a = join_ranges<REF>(part, s.n, i, splits, wave);
    sa = to_f32(((const T*)s.data)[i * s.rs + lab * s.ks]);
    if (REF) ra = to_f32(((const T*)ref.data)[i * ref.rs + lab * ref.ks]);
    A = g.advantage[i];
    old = g.old_log_prob[i];
    o = policy_row<REF>(a, sa, ra, A, old, w, g, i, lab, nullptr);
  }
  // rows next to a border, one after the other, each by the whole wave
  unsigned long long todo = __ballot(o.near && (!wave || (threadIdx.x & 63) == 0));
  while (todo) {
    const int src = __ffsll((unsigned long long)todo) - 1;
    todo &= todo - 1;
    const int64_t row = wave ? i : (t & ~63ll) + src;
    const double e = wave_exact_logp((const T*)s.data + row * s.rs, s.ks, s.K,
                                     __shfl(lab, src), __shfl(a.m, src));
    if ((threadIdx.x & 63) == src || wave)
      o = policy_row<REF>(a, sa, ra, A, old, w, g, i, lab, &e);
  }
  if (!in || (wave && (threadIdx.x & 63))) return;
  g.loss[i] = o.loss;
  g.log_prob[i] = o.logp;
  if (g.kl) g.kl[i] = o.kl;
  if (coef) {
    o.c.live = live && o.c.live;
    o.c.label = lab;
    coef[i] = o.c;
  }
}

// ---------------------------------------------------------------------------
// gradients, elementwise
// ---------------------------------------------------------------------------
template <bool REF>
struct PolicyGrad {
  const RowCoef* coef;
  static constexpr bool kRef = REF;
  __device__ __forceinline__ RowCoef row(const ScoresView&, int64_t i) const { return coef[i]; }
  __device__ __forceinline__ float at(const RowCoef& c, float s, float r) const {
    return coef_grad<REF>(c, s, r);
  }
};

template <typename T, bool CM, typename G>
__global__ __launch_bounds__(256) void score_grad_kernel(ScoresView s, ScoresView ref, G g,
                                                         bool accumulate, int32_t span,
                                                         ScoresView out) {
  constexpr int VE = CM ? 1 : Chunk<T>::VE;
  if (CM) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= s.n) return;
    const RowCoef c = g.row(s, i);
    const int32_t k0 = blockIdx.y * span, k1 = s.K - k0 > span ? k0 + span : s.K;
    const T* p = (const T*)s.data + i;
    const T* q = G::kRef ? (const T*)ref.data + i : nullptr;
    T* o = (T*)out.data + i;
    if (!c.live) {
      if (!accumulate)
        for (int32_t k = k0; k < k1; ++k) o[k * out.ks] = from_f32<T>(0.0f);
      return;
    }
    // eight classes' loads in flight (the stores might be to the same memory as
    // far as the compiler knows)
    constexpr int U = 8;
    for (int32_t k = k0; k < k1; k += U) {
      float v[U], r[U], x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t at = k + j < k1 ? k + j : k1 - 1;
        v[j] = to_f32(p[at * s.ks]);
        r[j] = G::kRef ? to_f32(q[at * ref.ks]) : 0.0f;
        x[j] = accumulate ? to_f32(o[at * out.ks]) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        x[j] += k + j == c.label ? c.gl : g.at(c, v[j], r[j]);
        if (k + j < k1) o[(int64_t)(k + j) * out.ks] = from_f32<T>(x[j]);
      }
    }
    return;
  }
  // 64 lanes along a row, 4 rows a workgroup
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= s.n) return;
  const RowCoef c = g.row(s, i);
  const int32_t k0 = blockIdx.y * span, k1 = s.K - k0 > span ? k0 + span : s.K;
  const T* p = (const T*)s.data + i * s.rs;
  const T* q = G::kRef ? (const T*)ref.data + i * ref.rs : nullptr;
  T* o = (T*)out.data + i * out.rs;
  for (int32_t k = k0 + (int)(threadIdx.x & 63) * VE; k < k1; k += 64 * VE) {
    const int m = k1 - k < VE ? k1 - k : VE;
    if (m < VE || !c.live) {
      for (int j = 0; j < m; ++j) {
        float x = 0.0f;
        if (c.live) {
          const float sv = to_f32(p[k + j]), rv = G::kRef ? to_f32(q[k + j]) : 0.0f;
          x = k + j == c.label ? c.gl : g.at(c, sv, rv);
        } else if (accumulate) {
          break;
        }
        if (accumulate) x += to_f32(o[k + j]);
        o[k + j] = from_f32<T>(x);
      }
      continue;
    }
    Chunk<T> v = load_chunk<T>(p + k), r, old;
    if (G::kRef) r = load_chunk<T>(q + k);
    if (accumulate) old = load_chunk<T>(o + k);
    float x[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      x[j] = k + j == c.label ? c.gl : g.at(c, v.get(j), G::kRef ? r.get(j) : 0.0f);
      if (accumulate) x[j] += old.get(j);
    }
    v.set(x);
    store_chunk<T>(o + k, v);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// a row's classes in ranges: one range where the rows alone fill the GPU, else
// ranges of at least 32 classes (row-major: 1024, a wave's 16 loads each); at
// most 2048 classes a thread, which bounds the sums' rounding
static int32_t loss_splits(int64_t n, int32_t K, bool cm) {
  const int64_t waves = std::max<int64_t>(1, cm ? (n + 63) / 64 : n);
  const int64_t want = (kLossWaves + waves - 1) / waves;
  const int64_t most = (K + (cm ? 31 : 1023)) / (cm ? 32 : 1024);
  const int64_t least = cm ? (K + 2047) / 2048 : (K + 131071) / 131072;
  return (int32_t)std::max<int64_t>(least, std::min(want, most));
}

static dim3 rows_grid(const ScoresView& s, int32_t splits) {
  return dim3((unsigned)(s.class_major() ? (s.n + 255) / 256 : (s.n + 3) / 4), (unsigned)splits);
}

template <typename T, bool REF>
static int stats_of(const ScoresView& s, const ScoresView& ref, const int32_t* label,
                    RowStats* part, hipStream_t st) {
  const int32_t splits = loss_splits(s.n, s.K, s.class_major());
  const int32_t span = (s.K + splits - 1) / splits;
  const dim3 grid = rows_grid(s, splits);
  if (s.class_major())
    hipLaunchKernelGGL((row_stats_kernel<T, true, REF>), grid, dim3(256), 0, st, s, ref, label,
                       span, part);
  else
    hipLaunchKernelGGL((row_stats_kernel<T, false, REF>), grid, dim3(256), 0, st, s, ref, label,
                       span, part);
  WGBM_LAUNCH_CHECK();
  return 0;
}

template <typename T, typename G>
static int grad_of(const ScoresView& s, const ScoresView& ref, const G& g, bool accumulate,
                   const ScoresView& out, hipStream_t st) {
  const int32_t splits = loss_splits(s.n, s.K, s.class_major());
  int32_t span = (s.K + splits - 1) / splits;
  span = (span + 7) / 8 * 8;  // whole chunks
  const dim3 grid = rows_grid(s, (s.K + span - 1) / span);
  if (s.class_major())
    hipLaunchKernelGGL((score_grad_kernel<T, true, G>), grid, dim3(256), 0, st, s, ref, g,
                       accumulate, span, out);
  else
    hipLaunchKernelGGL((score_grad_kernel<T, false, G>), grid, dim3(256), 0, st, s, ref, g,
                       accumulate, span, out);
  WGBM_LAUNCH_CHECK();
  return 0;
}

static unsigned row_blocks(int64_t n, int32_t splits) {
  return (unsigned)(((splits > 1 ? n * 64 : n) + 255) / 256);
}

template <typename T>
static int log_probs_t(const ScoresView& s, const int32_t* label, float* log_prob, float* norm,
                       void* ws, hipStream_t st) {
  RowStats* part = (RowStats*)ws;
  const int32_t splits = loss_splits(s.n, s.K, s.class_major());
  const int r = stats_of<T, false>(s, ScoresView{}, label, part, st);
  if (r) return r;
  hipLaunchKernelGGL((log_prob_rows_kernel<T>), dim3(row_blocks(s.n, splits)), dim3(256), 0, st, s,
                     label, part, splits, log_prob, (float2*)norm);
  WGBM_LAUNCH_CHECK();
  return 0;
}

// A grid's threads are counted in 32 bits: rows in registers are launched in
// parts of fewer (no frame gives a row more than 1024 threads, nor more than its
// classes and 3).  fn(first row, rows) for each part.
template <typename Fn>
static int row_parts(const ScoresView& s, Fn fn) {
  const int64_t threads = std::min<int64_t>(1024, (int64_t)s.K + 3);
  const int64_t most = ((int64_t(1) << 32) - 1) / threads / 1024 * 1024;
  for (int64_t i = 0; i < s.n; i += most) {
    const int r = fn(i, std::min(most, s.n - i));
    if (r) return r;
  }
  return 0;
}
static ScoresView rows_of(const ScoresView& s, int64_t i, int64_t n) {
  ScoresView v = s;
  if (!s.data) return v;
  v.data = (unsigned char*)s.data + i * s.rs * (s.dtype == kF32 ? 4 : 2);
  v.n = n;
  return v;
}

int class_log_probs(const ScoresView& s, const int32_t* label, float* log_prob, float* norm,
                    void* ws, hipStream_t st) {
  if (rows_fit(s, false)) {
    const auto rows = s.dtype == kF32    ? log_probs_rows_f32
                      : s.dtype == kBF16 ? log_probs_rows_bf16
                                         : log_probs_rows_f16;
    return row_parts(s, [&](int64_t i, int64_t n) {
      return rows(rows_of(s, i, n), label + i, log_prob + i, norm + 2 * i, st);
    });
  }
  LOSS_TYPES(s.dtype, return log_probs_t<T>(s, label, log_prob, norm, ws, st));
}

int class_log_probs_grad(const ScoresView& s, const int32_t* label, const float* norm,
                         const float* grad, const ScoresView& out, hipStream_t st) {
  if (rows_fit(s, false)) {
    const auto rows = s.dtype == kF32    ? log_probs_grad_rows_f32
                      : s.dtype == kBF16 ? log_probs_grad_rows_bf16
                                         : log_probs_grad_rows_f16;
    return row_parts(s, [&](int64_t i, int64_t n) {
      return rows(rows_of(s, i, n), label + i, norm + 2 * i, grad + i, rows_of(out, i, n), st);
    });
  }
  LOSS_TYPES(s.dtype, {
    const LogProbGrad<T> g{label, (const float2*)norm, grad};
    return grad_of<T>(s, ScoresView{}, g, false, out, st);
  });
}

template <typename T, bool REF>
static int policy_t(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,
                    const ScoresView& out, bool accumulate, void* ws, hipStream_t st) {
  const int32_t splits = loss_splits(s.n, s.K, s.class_major());
  RowCoef* coef = (RowCoef*)ws;
  RowStats* part = (RowStats*)(coef + s.n);
  int r = stats_of<T, REF>(s, ref, g.action, part, st);
  if (r) return r;
  hipLaunchKernelGGL((policy_rows_kernel<T, REF>), dim3(row_blocks(s.n, splits)), dim3(256), 0, st,
                     s, ref, g, part, splits, out.data ? coef : nullptr);
  WGBM_LAUNCH_CHECK();
  if (!out.data) return 0;
  return grad_of<T>(s, ref, PolicyGrad<REF>{coef}, accumulate, out, st);
}

int policy_loss(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,
                const ScoresView& out, bool accumulate, void* ws, hipStream_t st) {
  if (rows_fit(s, ref.data != nullptr)) {
    const auto rows = s.dtype == kF32    ? policy_rows_f32
                      : s.dtype == kBF16 ? policy_rows_bf16
                                         : policy_rows_f16;
    return row_parts(s, [&](int64_t i, int64_t n) {
      PolicyRows p = g;
      p.action += i;
      p.old_log_prob += i;
      p.advantage += i;
      if (p.weight) p.weight += i;
      if (p.ref_log_prob) p.ref_log_prob += i;
      p.loss += i;
      p.log_prob += i;
      if (p.kl) p.kl += i;
      return rows(rows_of(s, i, n), rows_of(ref, i, n), p, rows_of(out, i, n), accumulate, st);
    });
  }
  if (ref.data) LOSS_TYPES(s.dtype, return (policy_t<T, true>(s, ref, g, out, accumulate, ws, st)));
  LOSS_TYPES(s.dtype, return (policy_t<T, false>(s, ref, g, out, accumulate, ws, st)));
}

static size_t ranges_bytes(const ScoresView& s) {
  return sizeof(RowStats) * (size_t)s.n * loss_splits(s.n, s.K, s.class_major());
}
size_t log_probs_workspace(const ScoresView& s) {
  return rows_fit(s, false) ? 0 : ranges_bytes(s);
}
size_t policy_workspace(const ScoresView& s, bool ref) {
  return rows_fit(s, ref) ? 0 : sizeof(RowCoef) * (size_t)s.n + ranges_bytes(s);
}

}  // namespace wgbm
