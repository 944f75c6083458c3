// Gradient of what a training step makes of a row's label, alternatives and
// entropy: with upstream gradients g_j of the log-probabilities of the classes c_j
// (the label's among them), g_H of the entropy and G = sum g_j,
//   ds_k = (1 / tau) (sum of g_j with c_j = k  -  p_k (G + g_H (x_k + down)))
// x, down and p = e^(x - lse) from the row's norm (alternatives.hpp).  No sums over
// classes: rows are read once and the gradient written once.  At a class with a
// g of its own: g (1 - p) - p ((G - g) + g_H (x + down)), 1 - p from log p, so that
// a row sure of that class keeps its digits.
//
// 4099 x 32000 bfloat16 with 20 classes, the label and the entropy: 115 us (525 MB, 4.6
// TB/s: memory).  1M x 100 float32 class-major with 16 classes: 196 us (4.9 TB/s).  65536
// x 64 bfloat16, label and entropy: 5.7 us (18 MB in some 4000 waves).
#pragma once
#include "losses_lists.hpp"

namespace wgbm {

// e^x (c0 + c1 h), h = x log2(e): a class without a g of its own
struct AltGradRow {
  float m, c0, c1;
  float lse, down, g_all, g_entropy;
  bool live;
};
__device__ __forceinline__ AltGradRow alt_grad_row(const AltGradRows& g, int64_t i, float g_all,
                                                   bool any) {
  AltGradRow o;
  o.m = g.norm[3 * i];
  o.lse = g.norm[3 * i + 1];
  o.down = g.norm[3 * i + 2];
  o.g_entropy = g.grad_entropy ? g.grad_entropy[i] : 0.0f;
  o.g_all = g_all;
  o.live = o.m != -__builtin_inff() && (any || o.g_entropy != 0.0f);
  const float f = -exp_of(-o.lse) * (float)g.inv_tau;
  o.c0 = f * fmaf(o.g_entropy, o.down, g_all);
  o.c1 = f * o.g_entropy * (float)kLn2;
  return o;
}
__device__ __forceinline__ float alt_grad_at(const AltGradRow& r, const AltGradRows& g, float v) {
  const float h = (v - r.m) * g.scale;
  return exp2_f32(h) * fmaf(r.c1, fmaxf(h, kLowPower), r.c0);
}
__device__ __forceinline__ float alt_grad_listed(const AltGradRow& r, const AltGradRows& g, float v,
                                                 float own) {
  const float x = (v - r.m) * (float)g.inv_tau, lp = x - r.lse;
  const float rest = fmaf(r.g_entropy, fmaxf(x, kLowPower) + r.down, r.g_all - own);
  return (float)g.inv_tau * fmaf(own, one_less_exp(lp), -exp_of(lp) * rest);
}

// no list: only the label has a g of its own.  tile: of a long row (span 0: the rows
// are whole)
template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_grad_plain_kernel(ScoresView whole,
                                                                          AltGradRows g,
                                                                          ScoresView out_whole,
                                                                          bool accumulate,
                                                                          int32_t span) {
  const ScoresView s = span ? tile_of(whole, span, blockIdx.y) : whole;
  const ScoresView out = span ? tile_of(out_whole, span, blockIdx.y) : out_whole;
  const F f(s);
  const int64_t i = F::row(blockIdx.x);
  if (i >= s.n) return;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  int32_t lab = row_label(g.label, i, whole.K);
  const float own = lab >= 0 ? g.grad_label[i] : 0.0f;
  const float sa = lab >= 0 ? score_at<typename F::T>(whole, i, lab) : 0.0f;
  const AltGradRow r = alt_grad_row(g, i, own, own != 0.0f);
  if (!r.live && accumulate) return;
  lab -= blockIdx.y * span;
  // (one store for rows that count and rows left out: lanes of a wave may hold both)
  f.store_row(out, blockIdx.x, accumulate, lab >= 0 && lab < s.K ? lab : -1,
              r.live ? alt_grad_listed(r, g, sa, own) : 0.0f, [&](int j) {
                const float x = alt_grad_at(r, g, F::value(v, j));
                return r.live ? x : 0.0f;
              });
}

// a thread a row: the list's g are added up in registers
template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_grad_lane_kernel(ScoresView s,
                                                                         AltGradRows g,
                                                                         ScoresView out,
                                                                         bool accumulate) {
  const F f(s);
  const int64_t i = F::row(blockIdx.x);
  if (i >= s.n) return;
  const int32_t* const classes = g.classes + i * g.class_stride;
  const float* const grads = g.grad_list + i * g.grad_stride;
  using Batch = EntryBatch<float>;
  Batch b;
  b.load(classes, g.class_step, grads, g.grad_step, 0, 1, g.k);
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  float own[F::N], all = 0.0f;
  bool any = false;
#pragma unroll
  for (int j = 0; j < F::N; ++j) own[j] = 0.0f;
  const auto add = [&](int32_t c, float x) {
    if (c < 0 || c >= s.K) return;
    all += x;
    any |= x != 0.0f;
#pragma unroll
    for (int j = 0; j < F::N; ++j) own[j] += f.cls(j) == c ? x : 0.0f;
  };
  if (g.label) add(g.label[i], g.grad_label[i]);
  for (int first = 0; first < g.k; first += Batch::kSize) {
    if (first) b.load(classes, g.class_step, grads, g.grad_step, first, 1, g.k);
#pragma unroll
    for (int q = 0; q < Batch::kSize; ++q) add(first + q < g.k ? b.cls[q] : -1, b.value[q]);
  }
  const AltGradRow r = alt_grad_row(g, i, all, any);
  if (!r.live && accumulate) return;
  f.store(out, blockIdx.x, accumulate, [&](int j) {
    const float x = F::value(v, j);
    const float y = own[j] != 0.0f ? alt_grad_listed(r, g, x, own[j]) : alt_grad_at(r, g, x);
    return r.live ? y : 0.0f;
  });
}

// class-major rows in slices: the list's gradients are worked out by the threads that
// have the entries, and written by those that have the classes (SliceMap).  A label
// beside the list is entry k.
template <typename F>
static size_t grad_slices_lds(int32_t k, int threads) {
  return ((size_t)SliceMap<F>::kWords * threads + 2 * 64 * (size_t)(k + 1) + 2 * (size_t)threads) *
         4;
}

template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_grad_slices_kernel(ScoresView s,
                                                                           AltGradRows g,
                                                                           ScoresView out,
                                                                           bool accumulate) {
  using Map = SliceMap<F>;
  extern __shared__ uint32_t lds[];
  const int k = g.k, all = k + 1, lane = threadIdx.x & 63;
  const Map map{lds};
  // the entries' gradients, and their scores, later the classes' gradients
  float* const own = (float*)(lds + Map::kWords * blockDim.x) + lane;
  float* const score = own + 64 * all;
  float* const buf = (float*)(lds + Map::kWords * blockDim.x) + 128 * all;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  const int64_t i = in ? row : s.n - 1;
  const int32_t* const classes = g.classes + i * g.class_stride;
  const float* const grads = g.grad_list + i * g.grad_stride;
  using Batch = EntryBatch<float>;
  Batch b;
  b.load(classes, g.class_step, grads, g.grad_step, f.w, f.S, k);
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  map.clear();
  __syncthreads();
  float sum[2] = {0.0f, 0.0f};  // of the g, and how many are not 0
  bool twice = false;
  for (int first = f.w; first < k; first += Batch::kSize * f.S) {
    if (first != f.w) b.load(classes, g.class_step, grads, g.grad_step, first, f.S, k);
#pragma unroll
    for (int q = 0; q < Batch::kSize; ++q) {
      const int j = first + q * f.S;
      if (j >= k) break;
      float x = 0.0f;
      if ((uint32_t)b.cls[q] < (uint32_t)s.K) {
        x = b.value[q];
        sum[0] += x;
        sum[1] += x != 0.0f ? 1.0f : 0.0f;
        twice |= map.put(f, b.cls[q], j);
      }
      own[64 * j] = x;
      score[64 * j] = 0.0f;
    }
  }
  if (__syncthreads_or(twice)) {
    // the first of the entries that name a class takes its place, and all their g
    for (int j = f.w; j < k; j += f.S) {
      const int32_t c = classes[j * g.class_step];
      bool first = (uint32_t)c < (uint32_t)s.K;
      for (int o = 0; o < j; ++o) first &= classes[o * g.class_step] != c;
      if (!first) continue;
      map.set(f, c, j);
      // (later entries' own numbers: only first entries' are changed)
      float more = 0.0f;
      for (int o = j + 1; o < k; ++o)
        if (classes[o * g.class_step] == c) more += own[64 * o];
      own[64 * j] += more;
    }
    __syncthreads();
  }
  if (f.w == 0) {
    // the label, an entry of its own unless the list has it
    const int32_t c = row_label(g.label, i, s.K);
    const float x = c >= 0 ? g.grad_label[i] : 0.0f;
    sum[0] += x;
    sum[1] += x != 0.0f ? 1.0f : 0.0f;
    own[64 * k] = x;
    score[64 * k] = 0.0f;
    if (c >= 0) {
      const int e = map.get(f, c);
      if (e)
        own[64 * (e - 1)] += x;
      else
        map.set(f, c, k);
    }
  }
  __syncthreads();
  uint32_t mine[Map::kWords];
  map.mine(mine);
#pragma unroll
  for (int j = 0; j < F::N; ++j) {
    const int e = Map::entry(mine, j);
    if (e) score[64 * (e - 1)] = F::value(v, j);
  }
  f.reduce_all(sum, AddF(), buf);
  const AltGradRow r = alt_grad_row(g, i, sum[0], sum[1] != 0.0f);
  for (int j = f.w; j <= k; j += f.S)
    score[64 * j] = alt_grad_listed(r, g, score[64 * j], own[64 * j]);
  __syncthreads();
  // (one store for rows that count and rows left out: lanes of a wave may hold both)
  if (!in || (!r.live && accumulate)) return;
  f.store(out, blockIdx.x, accumulate, [&](int j) {
    const int e = Map::entry(mine, j);
    float y = alt_grad_at(r, g, F::value(v, j));
    if (e) y = score[64 * (e - 1)];
    return r.live ? y : 0.0f;
  });
}

// Rows that threads share.  The listed classes are taken out of the rows (a bit a
// slot, set through LDS, found again by the thread that has the class), which
// leaves their places 0 or as they were, and their gradients are written to
// memory after the others': each is rounded once.
template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_grad_list_kernel(ScoresView whole,
                                                                         AltGradRows g,
                                                                         ScoresView out_whole,
                                                                         bool accumulate,
                                                                         int32_t span) {
  using T = typename F::T;
  extern __shared__ uint32_t lds[];  // classes, gradients, scores of the lists; bits of the slots
  __shared__ float buf[2 * F::kBuf];
  const int k = g.k;
  int32_t* const l_cls = (int32_t*)lds;
  float* const l_own = (float*)(l_cls + F::kListRows * k);
  float* const l_score = l_own + F::kListRows * k;
  uint32_t* const bits = (uint32_t*)(l_score + F::kListRows * k);
  const int32_t k0 = span ? (int32_t)blockIdx.y * span : 0;
  const ScoresView s = span ? tile_of(whole, span, blockIdx.y) : whole;
  const ScoresView out = span ? tile_of(out_whole, span, blockIdx.y) : out_whole;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  const int64_t i = in ? row : s.n - 1;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
#pragma unroll
  for (int b = 0; b < F::kMaskWords; ++b) bits[b * blockDim.x + threadIdx.x] = 0;
  const int32_t lab = row_label(g.label, i, whole.K);
  const float g_label = lab >= 0 ? g.grad_label[i] : 0.0f;
  const float sa = lab >= 0 ? score_at<T>(whole, i, lab) : 0.0f;
  __syncthreads();
  float sum[2] = {0.0f, 0.0f};  // of the g, and how many are not 0
  bool twice = false;
  int word;
  uint32_t bit;
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    int32_t c = g.classes[i * g.class_stride + j * g.class_step];
    float own = 0.0f, sc = 0.0f;
    if (c < 0 || c >= whole.K) c = -1;
    if (c >= 0) {
      own = g.grad_list[i * g.grad_stride + j * g.grad_step];
      sum[0] += own;
      sum[1] += own != 0.0f ? 1.0f : 0.0f;
      if (c >= k0 && c - k0 < s.K) {
        f.locate(c - k0, word, bit);
        twice |= (atomicOr(&bits[word], bit) & bit) != 0;
        sc = score_at<T>(whole, i, c);
      } else {
        c = -1;  // another tile's
      }
    }
    l_cls[f.entry_at(j, k)] = c;
    l_own[f.entry_at(j, k)] = own;
    l_score[f.entry_at(j, k)] = sc;
  }
  if (__syncthreads_or(twice)) {
    // a class that is listed again: the first entry takes all its g
    uint32_t again = 0;
    int n = 0;
    for (int j = f.entry(); j < k; j += f.entry_step(), ++n) {
      const int32_t c = l_cls[f.entry_at(j, k)];
      if (c >= 0 && listed_before(f, l_cls, j, k, c)) again |= 1u << n;
    }
    __syncthreads();
    n = 0;
    for (int j = f.entry(); j < k; j += f.entry_step(), ++n) {
      const int32_t c = l_cls[f.entry_at(j, k)];
      if (c < 0 || again >> n & 1) continue;
      // (later entries' own numbers: only first entries' are changed)
      float more = 0.0f;
      for (int o = j + 1; o < k; ++o)
        if (l_cls[f.entry_at(o, k)] == c) more += l_own[f.entry_at(o, k)];
      l_own[f.entry_at(j, k)] += more;
    }
    __syncthreads();
    n = 0;
    for (int j = f.entry(); j < k; j += f.entry_step(), ++n)
      if (again >> n & 1) l_cls[f.entry_at(j, k)] = -1;
  }
  // the label: an entry of its own unless the list has it
  bool mine = false;
  const bool label_here = lab >= k0 && lab - k0 < s.K && lab >= 0;
  if (f.entry() == 0 && label_here) {
    f.locate(lab - k0, word, bit);
    mine = (bits[word] & bit) == 0;
    if (mine) atomicOr(&bits[word], bit);
  }
  f.reduce_all(sum, AddF(), buf);
  __syncthreads();
  uint32_t out_bits[F::kMaskWords];
#pragma unroll
  for (int b = 0; b < F::kMaskWords; ++b) out_bits[b] = bits[b * blockDim.x + threadIdx.x];
  const AltGradRow r = alt_grad_row(g, i, sum[0] + g_label, sum[1] != 0.0f || g_label != 0.0f);
  f.take_out(v, out_bits);
  // (one store for rows that count and rows left out: lanes of a wave may hold both)
  if (in && (r.live || !accumulate))
    f.store(out, blockIdx.x, accumulate, [&](int j) {
      return r.live ? alt_grad_at(r, g, F::value(v, j)) : 0.0f;
    });
  __syncthreads();
  if (!in || !r.live) return;
  // (the scores were read before: the gradient may be written over them)
  const auto write = [&](int32_t c, float sc, float own) {
    float x = alt_grad_listed(r, g, sc, own);
    T* q = (T*)out.data + i * out.rs + (c - k0) * out.ks;
    if (accumulate) x += to_f32(*q);
    *q = from_f32<T>(x);
  };
  for (int j = f.entry(); j < k; j += f.entry_step()) {
    const int at = f.entry_at(j, k);
    const int32_t c = l_cls[at];
    if (c >= 0) write(c, l_score[at], l_own[at] + (c == lab ? g_label : 0.0f));
  }
  if (mine) write(lab, sa, g_label);
}

// frames of class-major rows and of row-major ones up to 1024 chunks.  Nothing is summed
// over a row, so waves wait for one another at the lists only: few threads with two chunks
// each, up to 32 with eight, then workgroups.  Gradient with eight
// listed classes, us, with the threads and chunks taken, half the threads and twice the
// chunks, twice the threads and half the chunks (-: the same, or no such frame):
//   float32                           bfloat16
//   1M x 27        103    -  108      1M x 55        119    -  123
//   1M x 59        154  187  194      1M x 119       186  212  228
//   504201 x 119   132  141  192      502092 x 239   159  164  219
//   251046 x 239   122  119  191      250520 x 479   143  134  216
//   125260 x 479   103  116  117      125130 x 959   112  132  138
//   60060 x 999    108    -  101      60030 x 1999   121    -  105
//   30015 x 1999   102  105    -      30006 x 3999   130  117    -   (half: a wave a row)
//   15003 x 3999    95  106  158      15000 x 7999   120  123  196   (half: a wave a row)
// Without a list the order is the same, but for 16-bit rows of 257 to 1024 chunks: a wave a
// row takes 90 and 93 us there, workgroups 104 and 107.
template <typename T, typename Fn>
static void pick_short_frame(const ScoresView& s, Fn fn) {
  constexpr int VE = Chunk<T>::VE;
  if (thread_rows(s)) return pick_thread_rows<T>(s, fn);
  if (s.class_major()) return pick_list_slices<T>(s, fn);
  const int64_t chunks = (s.K + VE - 1) / VE;
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 8) return go(FrameTag<RowFrame<T, 4, 2>>());
  if (chunks <= 16) return go(FrameTag<RowFrame<T, 8, 2>>());
  if (chunks <= 32) return go(FrameTag<RowFrame<T, 16, 2>>());
  if (chunks <= 64) return go(FrameTag<RowFrame<T, 32, 2>>());
  if (chunks <= 128) return go(FrameTag<RowFrame<T, 32, 4>>());
  if (chunks <= 256) return go(FrameTag<RowFrame<T, 32, 8>>());
  if (chunks <= 512) return go(FrameTag<RowFrame<T, 256, 2>>());
  go(FrameTag<RowFrame<T, 256, 4>>());
}

template <typename T>
static int alternatives_grad_frames(const ScoresView& s, const AltGradRows& g,
                                    const ScoresView& out, bool accumulate, hipStream_t st) {
  const auto launch = [&](auto tag, int64_t blocks, int threads, int32_t span, int32_t tiles) {
    using F = typename decltype(tag)::type;
    const dim3 grid((unsigned)blocks, (unsigned)tiles);
    if (g.k == 0) {
      hipLaunchKernelGGL((alternatives_grad_plain_kernel<F>), grid, dim3(threads), 0, st, s, g, out,
                         accumulate, span);
    } else if constexpr (F::kLaneRows && !F::kSlices) {
      hipLaunchKernelGGL((alternatives_grad_lane_kernel<F>), grid, dim3(threads), 0, st, s, g, out,
                         accumulate);
    } else if constexpr (F::kSlices) {
      hipLaunchKernelGGL((alternatives_grad_slices_kernel<F>), grid, dim3(threads),
                         grad_slices_lds<F>(g.k, threads), st, s, g, out, accumulate);
    } else {
      const size_t lds = (size_t)F::kListRows * g.k * 12 + (size_t)F::kMaskWords * threads * 4;
      hipLaunchKernelGGL((alternatives_grad_list_kernel<F>), grid, dim3(threads), lds, st, s, g,
                         out, accumulate, span);
    }
  };
  // (nothing is summed over a row: long rows go in parts)
  using Tile = RowFrame<T, 256, 4>;
  static_assert(Tile::N * 256 == kGradTileChunks * Chunk<T>::VE, "a tile");
  int32_t span;
  const int32_t tiles = row_tiles(s, true, &span);
  if (tiles == 1) {
    pick_short_frame<T>(s, [&](auto tag, int64_t blocks, int threads) {
      launch(tag, blocks, threads, 0, 1);
    });
  } else {
    launch(FrameTag<Tile>(), s.n, 256, span, tiles);
  }
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
