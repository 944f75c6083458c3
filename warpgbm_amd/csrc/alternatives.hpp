// Alternatives of a row's scores: with x = (s - m) / tau, m = max s,
//   lse = log sum e^x,  down = sum p (-x),  p = e^(x - lse)
//   entropy = lse + down, log-probability of class c = x_c - lse
// for the row's label and its k best classes (the lower class first among equal
// scores).  Both terms of the entropy are sums of numbers >= 0, and lse is
// log1p of the sum without the largest term, 1: nothing cancels, for a row sure
// of its class as for an even one.  Rows are read once into registers
// (losses_frames.hpp).
//
// 1M x 10 float32 class-major, three alternatives: 19 us (88 MB, 4.5 TB/s: memory).  8191
// x 16001 bfloat16, 64 alternatives: 73 us (267 MB, 3.6 TB/s): vector instructions are
// issued in four fifths of the cycles.  1 x 50001 float32: 9.3 us, one workgroup's
// latency.  A turn a class is what long lists of class-major rows cost: 1M x 100 float32
// 90 us without alternatives, 116 with three, 295 with 16.
#pragma once
#include "losses_lists.hpp"

namespace wgbm {

// a row's sums: of e^x over the scores below the maximum; of e^x h, h = x log2(e);
// and how many scores equal the maximum
struct AltSums {
  float z, u, ties;
};
__device__ __forceinline__ void add_score(AltSums& a, float v, float m, float ms, float c) {
  const float h = (v - ms) * c, e = exp2_f32(h);
  a.z += v == m ? 0.0f : e;
  a.ties += v == m ? 1.0f : 0.0f;
  a.u = fmaf(e, fmaxf(h, kLowPower), a.u);
}

struct AltRow {
  float m;      // the maximum, 0 for a row without a class
  double lse;
  float down;
  bool live;    // (a row of NaN is live: it shows in the results)
};
__device__ __forceinline__ AltRow alt_row(const AltSums& a, float m) {
  AltRow o;
  o.live = m > -__builtin_inff() || a.z != a.z;
  o.m = safe_max(m);
  const float rest = a.z + (a.ties - 1.0f);
  o.lse = log_1p(rest);
  o.down = -a.u * (float)kLn2 / (1.0f + rest);
  return o;
}
__device__ __forceinline__ float alt_log_prob(const AltRow& r, const AltRows& g, float v) {
  return (float)(((double)v - (double)r.m) * g.inv_tau - r.lse);
}
// the row's results but for its alternatives, by one thread
__device__ __forceinline__ void write_alt_row(const AltRow& r, const AltRows& g, int64_t i,
                                              int32_t label, float sa) {
  g.entropy[i] = r.live ? (float)(r.lse + (double)r.down) : 0.0f;
  g.norm[3 * i] = r.live ? r.m : -__builtin_inff();
  g.norm[3 * i + 1] = r.live ? (float)r.lse : 0.0f;
  g.norm[3 * i + 2] = r.live ? r.down : 0.0f;
  if (g.label) g.label_log_prob[i] = r.live && label >= 0 ? alt_log_prob(r, g, sa) : 0.0f;
}
__device__ __forceinline__ void write_alternative(const AltRow& r, const AltRows& g, int64_t i,
                                                  int t, int32_t cls, float v) {
  const int64_t at = i * g.k + t;
  g.classes[at] = cls;
  g.log_prob[at] = cls >= 0 ? alt_log_prob(r, g, v) : -__builtin_inff();
}

// ---------------------------------------------------------------------------
// Few classes a row, or few alternatives: the best classes one after the other.
// Each thread knows the best of its classes that are not taken; the best of those is
// the row's, and the thread that had it looks through its classes again (five
// instructions a slot).  Classes ascend with slots, so the first of equal scores is
// the lowest class.
// ---------------------------------------------------------------------------
template <typename F>
struct Turns {
  static constexpr int kWords = (F::N + 31) / 32;
  uint32_t taken[kWords];  // a bit a slot
  float best;
  int slot;  // -1: none is left
  __device__ __forceinline__ void look(const typename F::Regs& v) {
    best = -__builtin_inff();
    slot = -1;
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      // (a taken class's score reads as NaN, which is larger than nothing)
      const int32_t gone = __builtin_amdgcn_sbfe((int32_t)taken[j / 32], j % 32, 1);
      const float x = __builtin_bit_cast(
          float, __builtin_bit_cast(int32_t, F::value(v, j)) | gone);
      const bool more = x > best;
      best = more ? x : best;
      slot = more ? j : slot;
    }
  }
  __device__ __forceinline__ void take(const typename F::Regs& v) {
#pragma unroll
    for (int q = 0; q < kWords; ++q) taken[q] |= slot / 32 == q ? 1u << (slot % 32) : 0u;
    look(v);
  }
};

// words of LDS: two turns' best scores and classes, three sums, of slices
template <typename F>
static size_t turns_lds(int threads) {
  return F::kSlices ? 7 * 4 * (size_t)threads : 0;
}

template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_turns_kernel(ScoresView s, AltRows g) {
  extern __shared__ uint32_t lds[];
  float* const words = (float*)lds;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  const bool in = row < s.n;
  if (!F::kBarrier && !in) return;
  const int64_t i = in ? row : s.n - 1;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  const int32_t lab = row_label(g.label, i, s.K);
  const float sa = lab >= 0 ? score_at<typename F::T>(s, i, lab) : 0.0f;
  f.trim(v);
  Turns<F> turn{};
  turn.look(v);
  float* const sums = words + 4 * blockDim.x;
  const float m = f.reduce(turn.best, MaxF(), words), ms = safe_max(m);
  AltSums a{0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < F::N; ++j) add_score(a, F::value(v, j), m, ms, g.scale);
  float sum[3] = {a.z, a.u, a.ties};
  f.template reduce_all<3>(sum, AddF(), sums);
  const AltRow r = alt_row(AltSums{sum[0], sum[1], sum[2]}, m);
  const bool write = in && f.first_lane();
  if (write) write_alt_row(r, g, i, lab, sa);
  constexpr int32_t kNone = 0x7fffffff;
  for (int32_t t = 0; t < g.k; ++t) {
    // the row's best, and the lowest class that has it
    float best = turn.best;
    const int32_t mine = turn.slot >= 0 ? f.cls(turn.slot) : kNone;
    int32_t c = mine;
    if constexpr (F::kSlices) {
      // (two turns' words: a wave may be one turn ahead of the others)
      float* const bv = words + t % 2 * 2 * blockDim.x;
      int32_t* const bc = (int32_t*)(bv + blockDim.x);
      const int lane = threadIdx.x & 63;
      bv[threadIdx.x] = best;
      bc[threadIdx.x] = c;
      __syncthreads();
      for (int u = 0; u < f.S; ++u) {
        const float x = bv[u * 64 + lane];
        const int32_t k = bc[u * 64 + lane];
        const bool more = x > best || (x == best && k < c);
        best = more ? x : best;
        c = more ? k : c;
      }
    } else if constexpr (!F::kLaneRows) {
      best = lanes_reduce<F::G>(best, MaxF());
      // (class numbers are exact in float32)
      c = (int32_t)lanes_reduce<F::G>(turn.slot >= 0 && turn.best == best ? (float)mine : 1e9f,
                                      [](float x, float y) { return fminf(x, y); });
      if (c >= s.K) c = kNone;
    }
    if (write) write_alternative(r, g, i, t, c != kNone ? c : -1, best);
    if (c == mine && c != kNone) turn.take(v);
  }
}

// ---------------------------------------------------------------------------
// Longer rows: candidates.  The k-th largest of the maxima of 128 or more parts of
// the row is no larger than the k-th largest score, so the classes from there on
// (some more than k in rows without an order) are copied to LDS, and a
// candidate's place is the number of candidates with a larger key.  Rows with
// more candidates than the copy holds take their best classes in turns from memory.
//
// A part is what a thread has (or four neighbouring ones): 4 to 32 classes in a row at a
// time.  Where class numbers carry no order of scores, k parts hold little more than k
// candidates; where the best classes lie next to each other they share parts, and the
// candidates grow to the square.  64 best of bfloat16 rows, us, classes in any order, with
// scores that fall as the logarithm of the class's number beside noise of a unit,
// without noise, and all equal: 30000 x 3001 87, 133, 4270, 4340; 8191 x 16001 63, 72, 179,
// 5940; 4099 x 32000 80, 127, 5710, 5740 (the last two of each, but for 179: turns).
// ---------------------------------------------------------------------------
// a number no larger than the k-th largest of the wave's M keys a lane (its upper
// 16 bits: 2^-7 of the value), as a score
template <int M>
__device__ __forceinline__ float kth_at_least(const uint32_t (&key)[M], int32_t k) {
  uint32_t t = 0;
  for (int b = 31; b >= 16; --b) {
    const uint32_t next = t | 1u << b;
    int n = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) n += __popcll(__ballot(key[j] >= next));
    if (n >= k) t = next;
  }
  // (fewer than k parts with a class: every class is a candidate)
  return t <= kOrderNegInf ? -__FLT_MAX__ : score_of(t);
}

__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t other = (uint64_t)__shfl_xor((unsigned long long)key, o);
    key = other > key ? other : key;
  }
  return key;
}

// the places of n candidates, by the thread group's threads t, t + step, ...
__device__ __forceinline__ void rank_candidates(const uint64_t* cand, int n, int t, int step,
                                                const AltRow& r, const AltRows& g, int64_t i) {
  for (int q = t; q < n || q < g.k; q += step) {
    if (q >= n) {  // (the row has fewer classes)
      write_alternative(r, g, i, q, -1, 0.0f);
      continue;
    }
    const uint64_t mine = cand[q];
    int place = 0;
    for (int o = 0; o < n; ++o) place += cand[o] > mine;
    if (place < g.k)
      write_alternative(r, g, i, place, class_of(mine), score_of((uint32_t)(mine >> 32)));
  }
}

// workgroup's or wave's largest key below `below` (0: none), best(below) being a
// thread's
template <int NW, typename Fn>
__device__ __forceinline__ uint64_t next_key(uint64_t below, uint64_t* buf, Fn best) {
  uint64_t key = wave_max_key(best(below));
  if (NW == 1) return key;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = key;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) key = buf[w] > key ? buf[w] : key;
  return key;
}

// the row's best classes in turns, read from memory again
template <typename T, int NW>
__device__ __forceinline__ void take_turns(const ScoresView& s, const AltRow& r, const AltRows& g,
                                           int64_t i, int t, uint64_t* buf) {
  uint64_t below = ~0ull;
  for (int32_t e = 0; e < g.k; ++e) {
    below = next_key<NW>(below, buf, [&](uint64_t under) {
      uint64_t best = 0;
      for (int32_t k = t; k < s.K; k += 64 * NW) {
        const float x = score_at<T>(s, i, k);
        const uint64_t key = key_of(x, k);
        if (x > -__builtin_inff() && key < under && key > best) best = key;
      }
      return best;
    });
    if (t == 0)
      write_alternative(r, g, i, e, below ? class_of(below) : -1,
                        score_of((uint32_t)(below >> 32)));
  }
}

template <typename F>
__global__ __launch_bounds__(F::kMax) void alternatives_candidates_kernel(ScoresView s,
                                                                          AltRows g) {
  using T = typename F::T;
  constexpr int NW = F::G / 64, R = F::kRows, VE = F::VE, kHold = NW == 1 ? 256 : 512;
  static_assert(F::G >= 64, "a row is a wave's or a workgroup's");
  __shared__ uint64_t cand[R][kHold];
  __shared__ uint32_t part[NW == 1 ? 1 : 256];
  __shared__ uint64_t key_buf[NW];
  __shared__ float buf[2][2 * F::kBuf], most[F::kBuf];
  __shared__ int counts[R];
  __shared__ float from_share;
  const F f(s);
  const int64_t row = F::row(blockIdx.x);
  if (row >= s.n) return;  // (a whole wave or workgroup)
  const int64_t i = row;
  typename F::Regs v;
  f.load(v, s, blockIdx.x);
  const int32_t lab = row_label(g.label, i, s.K);
  const float sa = lab >= 0 ? score_at<T>(s, i, lab) : 0.0f;
  int* const count = &counts[threadIdx.x / F::G];
  if (f.first_lane()) *count = 0;
  f.trim(v);
  // the chunks' maxima: a candidate is looked for in a chunk that has one
  float top[F::NC];
  float m = -__builtin_inff();
#pragma unroll
  for (int c = 0; c < F::NC; ++c) {
    top[c] = F::value(v, c * VE);
#pragma unroll
    for (int e = 1; e < VE; ++e) top[c] = fmaxf(top[c], F::value(v, c * VE + e));
    m = fmaxf(m, top[c]);
  }
  const float own = m;
  float from = 0.0f;
  if constexpr (NW == 1) {
    if (g.k > 0) {
      // two parts a lane, the halves of its classes; eight (four in float32 rows of a chunk
      // a lane) for lists of more than half of the lanes that have classes, or nearly all
      // parts would be in the list and most classes candidates.  64 alternatives of 20047
      // x 257 float16 30 us, 67 with two parts; of 30000 x 3001 bfloat16 79 and 90; but of
      // 30000 x 1000 55 and 52, and 20 of 20047 x 257 19 and 18.
      constexpr int P = F::N < 8 ? F::N : 8;
      uint32_t key[P];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float x = F::value(v, p * F::N / P);
#pragma unroll
        for (int j = p * F::N / P + 1; j < (p + 1) * F::N / P; ++j) x = fmaxf(x, F::value(v, j));
        // (a part of NaN alone has no class)
        key[p] = order_of(fmaxf(x, -__builtin_inff()));
      }
      const int32_t lanes = (s.K + VE - 1) / VE;
      if (2 * g.k > (lanes < 64 ? lanes : 64)) {
        from = kth_at_least<P>(key, g.k);
      } else {
        uint32_t two[2] = {key[0], key[P / 2]};
#pragma unroll
        for (int p = 1; p < P / 2; ++p) {
          two[0] = key[p] > two[0] ? key[p] : two[0];
          two[1] = key[P / 2 + p] > two[1] ? key[P / 2 + p] : two[1];
        }
        from = kth_at_least<2>(two, g.k);
      }
    }
  } else {
    // 256 parts: a thread's classes, or those of four threads
    const float four = NW > 4 ? lanes_reduce<4>(m, MaxF()) : m;
    if (NW <= 4 || (threadIdx.x & 3) == 0)
      part[NW > 4 ? threadIdx.x >> 2 : threadIdx.x] = order_of(four);
  }
  m = f.reduce(m, MaxF(), most);
  const float ms = safe_max(m);
  if (NW > 1 && threadIdx.x < 64 && g.k > 0) {
    const uint32_t key[4] = {part[threadIdx.x], part[threadIdx.x + 64], part[threadIdx.x + 128],
                             part[threadIdx.x + 192]};
    const float t = kth_at_least<4>(key, g.k);
    if (threadIdx.x == 0) from_share = t;
  }
  if (F::N >= 32) f.hide(v);
  float z[2] = {0.0f, 0.0f}, u[2] = {0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < F::N; ++j) {
    const float h = (F::value(v, j) - ms) * g.scale, e = exp2_f32(h);
    z[j % 2] += e;
    u[j % 2] = fmaf(e, fmaxf(h, kLowPower), u[j % 2]);
  }
  float sum[2] = {z[0] + z[1], u[0] + u[1]};
  f.template reduce_all<2>(sum, AddF(), buf[0]);
  // the sum without its largest term: where it is small next to that, once more
  // from the scores below the maximum (a row without a class: 0 or NaN)
  AltSums a{sum[0] - 1.0f, sum[1], 1.0f};
  if (!(a.z >= 0.125f)) {
    f.hide(v);  // (or the compiler would keep the first pass's numbers for this one)
    float again[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < F::N; ++j) {
      const float x = F::value(v, j);
      again[0] += x == m ? 0.0f : exp2_f32((x - ms) * g.scale);
      again[1] += x == m ? 1.0f : 0.0f;
    }
    f.template reduce_all<2>(again, AddF(), buf[1]);
    a.z = again[0];
    a.ties = again[1];
  }
  const AltRow r = alt_row(a, m);
  if (f.first_lane()) write_alt_row(r, g, i, lab, sa);
  if (g.k == 0) return;
  if (NW > 1) from = from_share;
  uint64_t* const list = cand[threadIdx.x / F::G];
  if (own >= from) {
    uint32_t has = 0;
#pragma unroll
    for (int c = 0; c < F::NC; ++c) has |= top[c] >= from ? 1u << c : 0u;
    const T* p = (const T*)s.data + i * s.rs;
    for (; has; has &= has - 1) {
      const int c = __ffs(has) - 1;
      const int32_t k = f.first(c), skip = f.skip(c);
      const Chunk<T> x = load_chunk<T>(p + (uint32_t)k);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float y = x.get(e);
        if (y >= from && e >= skip) {
          const int at = atomicAdd(count, 1);
          if (at < kHold) list[at] = key_of(y, k + e);
        }
      }
    }
  }
  if (NW > 1)
    __syncthreads();
  else
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // (a wave's own list)
  const int n = *(volatile int*)count;
  if (n <= kHold)
    rank_candidates(list, n, threadIdx.x % F::G, F::G, r, g, i);
  else
    take_turns<T, NW>(s, r, g, i, threadIdx.x % F::G, key_buf);
}

// ---------------------------------------------------------------------------
// Rows longer than a workgroup's registers: a workgroup a row, tile after tile,
// twice (the maximum and where candidates begin; then sums and candidates)
// ---------------------------------------------------------------------------
template <typename T>
using AltTile = RowFrame<T, 1024, 4>;

template <typename T>
__global__ __launch_bounds__(1024) void alternatives_long_kernel(ScoresView s, AltRows g,
                                                                 int32_t span, int32_t tiles) {
  using F = AltTile<T>;
  constexpr int NW = 16, kHold = 1024;
  __shared__ uint64_t list[kHold];
  __shared__ uint32_t part[256];
  __shared__ uint64_t key_buf[NW];
  __shared__ float buf[3 * F::kBuf], most[F::kBuf];
  __shared__ int count;
  __shared__ float from_share;
  const int64_t i = blockIdx.x;
  const int32_t lab = row_label(g.label, i, s.K);
  const float sa = lab >= 0 ? score_at<T>(s, i, lab) : 0.0f;
  if (threadIdx.x == 0) count = 0;
  float m = -__builtin_inff();
  for (int32_t t = 0; t < tiles; ++t) {
    const ScoresView p = tile_of(s, span, t);
    const F f(p);
    typename F::Regs v;
    f.load(v, p, i);
    f.trim(v);  // (a class counts in one part only)
#pragma unroll
    for (int j = 0; j < F::N; ++j) m = fmaxf(m, F::value(v, j));
  }
  const float own = m;
  const float four = lanes_reduce<4>(m, MaxF());
  if ((threadIdx.x & 3) == 0) part[threadIdx.x >> 2] = order_of(four);
  const F whole(s);
  m = whole.reduce(m, MaxF(), most);
  const float ms = safe_max(m);
  if (threadIdx.x < 64 && g.k > 0) {
    const uint32_t key[4] = {part[threadIdx.x], part[threadIdx.x + 64], part[threadIdx.x + 128],
                             part[threadIdx.x + 192]};
    const float t = kth_at_least<4>(key, g.k);
    if (threadIdx.x == 0) from_share = t;
  }
  __syncthreads();
  const float from = g.k > 0 ? from_share : __builtin_inff();
  const bool some = g.k > 0 && own >= from;
  // (the tiles' sums are joined in float64: a row may have 2^24 classes)
  double z = 0.0, u = 0.0;
  float ties = 0.0f;
  for (int32_t t = 0; t < tiles; ++t) {
    const ScoresView p = tile_of(s, span, t);
    const F f(p);
    typename F::Regs v;
    f.load(v, p, i);
    f.trim(v);
    AltSums a[2] = {};
#pragma unroll
    for (int j = 0; j < F::N; ++j) add_score(a[j % 2], F::value(v, j), m, ms, g.scale);
    z += (double)(a[0].z + a[1].z);
    u += (double)(a[0].u + a[1].u);
    ties += a[0].ties + a[1].ties;
    if (some) {
#pragma unroll
      for (int j = 0; j < F::N; ++j) {
        const float x = F::value(v, j);
        if (x >= from) {
          const int at = atomicAdd(&count, 1);
          if (at < kHold) list[at] = key_of(x, t * span + f.cls(j));
        }
      }
    }
  }
  float sum[3] = {(float)z, (float)u, ties};
  whole.template reduce_all<3>(sum, AddF(), buf);
  const AltRow r = alt_row(AltSums{sum[0], sum[1], sum[2]}, m);
  if (threadIdx.x == 0) write_alt_row(r, g, i, lab, sa);
  if (g.k == 0) return;
  const int n = count;
  if (n <= kHold) {
    rank_candidates(list, n, threadIdx.x, 1024, r, g, i);
    return;
  }
  take_turns<T, NW>(s, r, g, i, threadIdx.x, key_buf);
}

// ---------------------------------------------------------------------------
// which kernel a call takes.  From 64 chunks on: as few threads as hold a row's chunks in 8
// each, 16 where no workgroup has more.  20 best of 60M float32 (120M bfloat16) scores,
// us, so, with a quarter of the threads and four times the chunks, and the other way round:
//   of 1000 (2000) classes   59 (74), -, 117 (135)
//   of 2000 (4000)           50 (57), -, 70 (86)
//   of 4000 (8000)           47 (61), 48 (65), 126 (149)
//   of 8000 (16000)          43 (50), -, 73 (92)
//   of 16000 (32000)         50 (64), 43 (53), -
// (256 threads of sixteen chunks would be faster for the last ones, 3750 rows each)
// ---------------------------------------------------------------------------
template <typename T>
static int alternatives_frames(const ScoresView& s, const AltRows& g, hipStream_t st) {
  constexpr int VE = Chunk<T>::VE;
  const auto turns = [&](auto tag, int64_t blocks, int threads) {
    using F = typename decltype(tag)::type;
    hipLaunchKernelGGL((alternatives_turns_kernel<F>), dim3((unsigned)blocks), dim3(threads),
                       turns_lds<F>(threads), st, s, g);
  };
  const auto candidates = [&](auto tag) {
    using F = typename decltype(tag)::type;
    hipLaunchKernelGGL((alternatives_candidates_kernel<F>),
                       dim3((unsigned)((s.n + F::kRows - 1) / F::kRows)), dim3(F::kThreads), 0, st,
                       s, g);
  };
  const int64_t chunks = (s.K + VE - 1) / VE;
  if (thread_rows(s)) {
    pick_thread_rows<T>(s, turns);
  } else if (s.class_major()) {
    pick_list_slices<T>(s, turns);
  } else if (chunks <= 32) {
    pick_few_threads<T>(s, chunks, turns);
  } else if (chunks <= 64) {
    candidates(FrameTag<RowFrame<T, 64, 1>>());
  } else if (chunks <= 128) {
    candidates(FrameTag<RowFrame<T, 64, 2>>());
  } else if (chunks <= 256) {
    candidates(FrameTag<RowFrame<T, 64, 4>>());
  } else if (chunks <= 512) {
    candidates(FrameTag<RowFrame<T, 64, 8>>());
  } else if (chunks <= 1024) {
    candidates(FrameTag<RowFrame<T, 256, 4>>());
  } else if (chunks <= 2048) {
    candidates(FrameTag<RowFrame<T, 256, 8>>());
  } else if (chunks <= 4096) {
    candidates(FrameTag<RowFrame<T, 1024, 4>>());
  } else if (chunks <= 8192) {
    candidates(FrameTag<RowFrame<T, 1024, 8>>());
  } else if (chunks <= 16384) {
    candidates(FrameTag<RowFrame<T, 1024, 16>>());
  } else {
    static_assert(AltTile<T>::N * 1024 == kTileChunks * VE, "a tile");
    int32_t span;
    const int32_t tiles = row_tiles(s, false, &span);
    hipLaunchKernelGGL((alternatives_long_kernel<T>), dim3((unsigned)s.n), dim3(1024), 0, st, s, g,
                       span, tiles);
  }
  WGBM_LAUNCH_CHECK();
  return 0;
}

}  // namespace wgbm
