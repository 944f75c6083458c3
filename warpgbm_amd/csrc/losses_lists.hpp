// Lists of a row's classes: its best alternatives, and a teacher's.  Arguments
// and arithmetic shared by alternatives*.hpp and distill.hpp.
//
// Scores are divided by a temperature: with m = max s, x = (s - m) / tau and
// e^x = 2^h, h = (s - m) c, c = log2(e) / tau (the difference first, as
// in exp_diff).
#pragma once
#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

// below this power an exponential is 0 in float32; products with it take the
// power no lower (0 * infinity would be NaN)
constexpr float kLowPower = -1000.0f;

// log(1 + z) of a float32 sum z >= 0 with all its digits, large or small: the
// logarithm of the rounded sum (its exponent apart) and what the rounding left out
__device__ __forceinline__ double log_1p(float z) {
  const float w = 1.0f + z;
  return log_of(w) + (double)((z - (w - 1.0f)) * __builtin_amdgcn_rcpf(w));
}

// phi(x) = e^x - 1 - x for |x| <= 1
__device__ __forceinline__ float phi_small(float x) {
  float p = 1.0f / 39916800.0f;
  p = fmaf(p, x, 1.0f / 3628800.0f);
  p = fmaf(p, x, 1.0f / 362880.0f);
  p = fmaf(p, x, 1.0f / 40320.0f);
  p = fmaf(p, x, 1.0f / 5040.0f);
  p = fmaf(p, x, 1.0f / 720.0f);
  p = fmaf(p, x, 1.0f / 120.0f);
  p = fmaf(p, x, 1.0f / 24.0f);
  p = fmaf(p, x, 1.0f / 6.0f);
  p = fmaf(p, x, 0.5f);
  return p * x * x;
}
// 1 - e^x
__device__ __forceinline__ float one_less_exp(float x) {
  return fabsf(x) <= 1.0f ? -(x + phi_small(x)) : 1.0f - exp_of(x);
}

// ---------------------------------------------------------------------------
// ordered keys: a larger score has a larger one, and among equal scores the
// lower class; -0 and 0 are equal
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
constexpr uint32_t kOrderNegInf = 0x007fffffu;  // of -infinity; what lies below are NaNs'
__device__ __forceinline__ uint64_t key_of(float v, int32_t k) {
  return (uint64_t)order_of(v) << 32 | (0xffffffffu - (uint32_t)k);
}
__device__ __forceinline__ int32_t class_of(uint64_t key) {
  return (int32_t)(0xffffffffu - (uint32_t)key);
}

// classes that a row lists twice: whether entry j's class c is that of an
// earlier one
template <typename F>
__device__ __forceinline__ bool listed_before(const F& f, const int32_t* cls, int j, int k,
                                              int32_t c) {
  for (int o = 0; o < j; ++o)
    if (cls[f.entry_at(o, k)] == c) return true;
  return false;
}

// Entries first, first + step, ... of a row's list (k of them), four at a time: a batch's
// loads are in flight together, the first batch's before the row's scores are waited for.
template <typename V>
struct EntryBatch {
  static constexpr int kSize = 4;
  int32_t cls[kSize];
  V value[kSize];
  __device__ __forceinline__ void load(const int32_t* classes, int64_t class_step, const V* values,
                                       int64_t value_step, int first, int step, int k) {
#pragma unroll
    for (int q = 0; q < kSize; ++q) {
      const int j = first + q * step < k ? first + q * step : k - 1;
      cls[q] = classes[j * class_step];
      value[q] = values[j * value_step];
    }
  }
};

// ---------------------------------------------------------------------------
// Lists of class-major rows in slices: the thread that has a listed class knows its
// score, another one its entry.  They meet in LDS: a byte for each slot of each
// thread holds the number of the entry that names it (0: none), and a table of k x 64
// numbers takes scores to the entries and gradients back, so that every class is
// read and written once, by its own thread in whole lines.  (Reading and writing
// listed classes by their addresses, 64 lines an instruction: 1M x 100 float32 with 16
// listed took 302 us instead of 267.)
// ---------------------------------------------------------------------------
template <typename F>
struct SliceMap {
  static constexpr int kWords = (F::N + 3) / 4;  // of a thread's bytes
  uint32_t* words;                               // kWords x blockDim.x
  __device__ __forceinline__ void clear() const {
#pragma unroll
    for (int q = 0; q < kWords; ++q) words[q * blockDim.x + threadIdx.x] = 0;
  }
  __device__ __forceinline__ int at(const F& f, int32_t c, int& shift) const {
    int wave, slot;
    f.locate(c, wave, slot);
    shift = slot % 4 * 8;
    return slot / 4 * blockDim.x + wave * 64 + (threadIdx.x & 63);
  }
  // entry j of this lane's row names class c; whether another one did before
  __device__ __forceinline__ bool put(const F& f, int32_t c, int j) const {
    int shift;
    const int word = at(f, c, shift);
    return atomicOr(&words[word], (uint32_t)(j + 1) << shift) >> shift & 255;
  }
  // the same for the only entry that may (after a barrier)
  __device__ __forceinline__ void set(const F& f, int32_t c, int j) const {
    int shift;
    const int word = at(f, c, shift);
    ((uint8_t*)&words[word])[shift / 8] = (uint8_t)(j + 1);
  }
  __device__ __forceinline__ int get(const F& f, int32_t c) const {
    int shift;
    const int word = at(f, c, shift);
    return words[word] >> shift & 255;
  }
  __device__ __forceinline__ void mine(uint32_t (&m)[kWords]) const {
#pragma unroll
    for (int q = 0; q < kWords; ++q) m[q] = words[q * blockDim.x + threadIdx.x];
  }
  static __device__ __forceinline__ int entry(const uint32_t (&m)[kWords], int slot) {
    return m[slot / 4] >> (slot % 4 * 8) & 255;
  }
};

// Which slices rows with lists take: fn(frame tag, workgroups, threads).  What a row's
// list costs is shared by its waves, but each wave joins what all have, so fewer waves
// with more classes each than pick_slices takes: 4, 8, 12 or 16, which fill the SIMDs
// evenly.  Distillation, us: 1M x 100 float32, 16 listed, 4 waves of 26 242, 8 of 13 280,
// 2 of 50 310, 5 of 20 297; 300000 x 200 8 waves of 26 134, 16 of 13 214; 150000 x 400
// 12 of 36 141, 13 of 32 197; 500000 x 64 4 of 16 78, 8 of 8 103.
template <typename T, typename Fn>
static void pick_list_slices(const ScoresView& s, Fn fn) {
  const auto go = [&](auto tag, int S) { fn(tag, (s.n + 63) / 64, 64 * S); };
  const int S = s.K <= 128 ? 4 : s.K <= 256 ? 8 : s.K <= 432 ? 12 : 16;
  const int N = (s.K + S - 1) / S;
  if (N <= 8) return go(FrameTag<ClassFrame<T, 8, true, true>>(), S);
  if (N <= 10) return go(FrameTag<ClassFrame<T, 10, true, true>>(), S);
  if (N <= 13) return go(FrameTag<ClassFrame<T, 13, true, true>>(), S);
  if (N <= 16) return go(FrameTag<ClassFrame<T, 16, true, true>>(), S);
  if (N <= 20) return go(FrameTag<ClassFrame<T, 20, true, true>>(), S);
  if (N <= 26) return go(FrameTag<ClassFrame<T, 26, true, true>>(), S);
  if (N <= 32) return go(FrameTag<ClassFrame<T, 32, true, true>>(), S);
  go(FrameTag<ClassFrame<T, 36, true, true>>(), S);
}

// Whether a thread takes a whole row: class-major up to 16 classes, and row-major ones
// up to 12 (a lane's loads are 48 bytes apart at most), which share what a row costs as
// a whole with nobody.  1M x 10 row-major, a thread a row and four: best three classes
// float32 20 and 35 us, bfloat16 20 and 47; distillation 48 and 66, 33 and 71; gradient 40
// and 43, 25 and 46; but of 1M x 16 float32 38 and 36, 113 and 60, 97 and 42.
static inline bool thread_rows(const ScoresView& s) {
  return s.K <= (s.class_major() ? 16 : 12);
}
template <typename T, typename Fn>
static void pick_thread_rows(const ScoresView& s, Fn fn) {
  if (s.class_major()) return pick_class_frame<T>(s, fn);
  const int64_t blocks = (s.n + 255) / 256;
  if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, false>>(), blocks, 256);
  if (s.K <= 8) return fn(FrameTag<ClassFrame<T, 8, false, false>>(), blocks, 256);
  fn(FrameTag<ClassFrame<T, 12, false, false>>(), blocks, 256);
}

// Row-major rows of up to 32 chunks with work for each row as a whole: few threads a
// row, so that a wave spends it on more rows, where there are rows enough.  300000 x 30
// float32, 4 threads of two chunks and 8 of one: best four classes 20 and 27 us,
// distillation 27 and 38; 200000 x 60, 4 of four and 8 of two: 25 and 30, 30 and 32;
// 300000 x 100, 8 of four and 16 of two: 55 and 74, 56 and 80.
template <typename T, typename Fn>
static void pick_few_threads(const ScoresView& s, int64_t chunks, Fn fn) {
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  const bool many = s.n * chunks >= kLossWaves * 128;
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 8)
    return many ? go(FrameTag<RowFrame<T, 4, 2>>()) : go(FrameTag<RowFrame<T, 8, 1>>());
  if (chunks <= 16)
    return many ? go(FrameTag<RowFrame<T, 4, 4>>()) : go(FrameTag<RowFrame<T, 8, 2>>());
  many ? go(FrameTag<RowFrame<T, 8, 4>>()) : go(FrameTag<RowFrame<T, 16, 2>>());
}

// a part of a row's classes as a matrix of its own: tile t of tiles, at least 8
// classes each
__device__ __forceinline__ ScoresView tile_of(const ScoresView& s, int32_t span, int32_t t) {
  ScoresView v = s;
  const int32_t k0 = t * span;
  v.data = (unsigned char*)s.data + (int64_t)k0 * (s.dtype == kF32 ? 4 : 2);
  v.K = s.K - k0 < span ? s.K - k0 : span;
  return v;
}

}  // namespace wgbm
