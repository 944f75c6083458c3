// Frames: how a row's scores sit in the registers of the threads that share
// it.  A frame loads a row's classes once; the losses make their passes
// (maximum, sums, gradient) over the registers.
#pragma once
#include "losses.hpp"

namespace wgbm {

// 16 bytes of a row: VE classes next to each other.  Rows of an odd length
// start at any multiple of the element size; global loads and stores of this
// GPU take such addresses.
template <typename T>
struct Chunk {
  static constexpr int VE = 16 / (int)sizeof(T);
  // (kept as words: an array of 16-bit elements would take a register each)
  uint32_t w[4];
  __device__ __forceinline__ float get(int e) const;  // element e as float32
  __device__ __forceinline__ T element(int e) const {
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(T, w[e]);
    else
      return __builtin_bit_cast(T, (uint16_t)(w[e / 2] >> (16 * (e % 2))));
  }
  __device__ __forceinline__ void set(const float* x);  // all elements, each rounded once
};
template <>
__device__ __forceinline__ float Chunk<float>::get(int e) const {
  return __builtin_bit_cast(float, w[e]);
}
template <>
__device__ __forceinline__ float Chunk<__bf16>::get(int e) const {
  return __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}
template <>
__device__ __forceinline__ float Chunk<_Float16>::get(int e) const {
  return (float)element(e);
}
template <>
__device__ __forceinline__ void Chunk<float>::set(const float* x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, x[e]);
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <>
__device__ __forceinline__ void Chunk<__bf16>::set(const float* x) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = __builtin_bit_cast(
        uint32_t, __builtin_convertvector((f32x2){x[2 * e], x[2 * e + 1]}, bf16x2));
}
template <>
__device__ __forceinline__ void Chunk<_Float16>::set(const float* x) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = __builtin_bit_cast(
        uint32_t, __builtin_convertvector((f32x2){x[2 * e], x[2 * e + 1]}, f16x2));
}
template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p) {
  Chunk<T> c;
  __builtin_memcpy(c.w, p, 16);
  return c;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c) {
  __builtin_memcpy(p, c.w, 16);
}
// The compiler keeps what one pass over the registers worked out (converted
// scores, exponentials) for the next one, in registers of their own; after
// hidden() the next pass starts from the scores again.
template <typename T>
__device__ __forceinline__ void hidden(Chunk<T>& c) {
  asm volatile("" : "+v"(c.w[0]), "+v"(c.w[1]), "+v"(c.w[2]), "+v"(c.w[3]));
}

// label of row i, -1 where it has none
__device__ __forceinline__ int32_t row_label(const int32_t* label, int64_t i, int32_t K) {
  if (!label) return -1;
  const int32_t a = label[i];
  return a >= 0 && a < K ? a : -1;
}

template <typename T>
__device__ __forceinline__ float score_at(const ScoresView& s, int64_t i, int32_t k) {
  return to_f32(((const T*)s.data)[i * s.rs + k * s.ks]);
}

// results of class_log_probs for one row
__device__ __forceinline__ void write_log_prob(const RowStats& a, float sa, int32_t label,
                                               int64_t i, float* log_prob, float2* norm) {
  const bool live = row_live(a);
  const float m = safe_max(a.m);
  log_prob[i] = live && label >= 0 ? (float)row_log_prob(a, sa) : 0.0f;
  norm[i] = live ? make_float2(m, (float)log_of(a.z + a.za))
                 : make_float2(-__builtin_inff(), 0.0f);
}

// g (1[k = a] - softmax), the log-probability's gradient, from the row's norm
template <typename T>
struct LogProbGrad {
  const int32_t* label;
  const float2* norm;
  const float* grad;
  static constexpr bool kRef = false;
  __device__ __forceinline__ RowCoef row(const ScoresView& s, int64_t i) const {
    RowCoef c{};
    const int32_t a = row_label(label, i, s.K);
    const float g = grad[i];
    const float2 v = norm[i];
    if (a < 0 || g == 0.0f || v.x == -__builtin_inff()) return c;
    c.m = v.x;
    c.c0 = -g * expf(-v.y);
    // the label's from its own logarithm: 1 - p without a difference
    c.gl = -g * expm1f((score_at<T>(s, i, a) - v.x) - v.y);
    c.label = a;
    c.live = 1;
    return c;
  }
  __device__ __forceinline__ float at(const RowCoef& c, float s, float) const {
    return coef_grad<false>(c, s, 0.0f);
  }
};

// log p of the label in float64, by the 64 lanes of a wave
template <typename T>
__device__ __forceinline__ double wave_exact_logp(const T* p, int64_t ks, int32_t K,
                                                            int32_t label, float m) {
  double z = 0.0;
  for (int32_t k = threadIdx.x & 63; k < K; k += 64)
    z += exp((double)to_f32(p[(int64_t)k * ks]) - (double)m);
  for (int o = 32; o; o >>= 1) z += __shfl_xor(z, o);
  return (double)to_f32(p[(int64_t)label * ks]) - (double)m - log(z);
}

// ---------------------------------------------------------------------------
// reductions over a group of G lanes (a power of two up to 64, aligned); every
// lane gets the same bits (each step combines two values that commute)
// ---------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
struct AddF {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct MaxF {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
template <int G, typename Op>
__device__ __forceinline__ float lanes_reduce(float x, Op op) {
  if (G >= 2) x = op(x, dpp_f32<0xB1>(x));   // lanes 1 0 3 2
  if (G >= 4) x = op(x, dpp_f32<0x4E>(x));   // lanes 2 3 0 1
  if (G >= 8) x = op(x, dpp_f32<0x141>(x));  // the other quad of eight
  if (G >= 16) x = op(x, dpp_f32<0x140>(x));  // the other half of sixteen
  if (G >= 32) x = op(x, __shfl_xor(x, 16));
  if (G >= 64) x = op(x, __shfl_xor(x, 32));
  return x;
}

// over a whole workgroup of NW waves: each wave's value through LDS (buf: NW
// words that no other reduction of this row uses), joined in wave order
template <int NW, typename Op>
__device__ __forceinline__ float waves_reduce(float x, Op op, float* buf) {
  x = lanes_reduce<64>(x, op);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  x = buf[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) x = op(x, buf[w]);
  return x;
}

// a frame as a value, for the functions that pick one
template <typename F>
struct FrameTag {
  using type = F;
};

// ---------------------------------------------------------------------------
// RowFrame: classes next to each other.  G threads share a row; thread t holds
// the chunks t, t + G, ... (NC of them): classes (c * G + t) * VE .. + VE.
//
// Every load is whole and unconditional, so that all of a thread's are in
// flight together: a chunk that would pass the row's end is read VE classes
// before it (K >= VE), and its classes that belong to other threads (or to
// none) are then set to -inf.  Class of (chunk c, element e) = first(c) + e;
// elements below skip(c) are not this thread's.
// ---------------------------------------------------------------------------
template <typename T_, int G_, int NC_>
struct RowFrame {
  using T = T_;
  static constexpr int G = G_, NC = NC_, VE = Chunk<T>::VE, N = NC * VE;
  static constexpr int kWords = 4 * NC;  // registers of a thread's scores
  static constexpr int kThreads = G <= 256 ? 256 : G, kMax = kThreads;
  static constexpr bool kBarrier = G > 64, kSlices = false, kLaneRows = false;
  static constexpr int kShared = 1;  // rows that the waves of a workgroup share
  static constexpr int kRows = kThreads / G;  // rows of a workgroup
  static constexpr int kBuf = G > 64 ? G / 64 : 1;
  int32_t t, K;  // this thread's place in its group

  __device__ __forceinline__ RowFrame(const ScoresView& s) : t(threadIdx.x % G), K(s.K) {}
  static __device__ __forceinline__ int64_t row(int64_t block) {
    return block * kRows + threadIdx.x / G;
  }
  __device__ __forceinline__ bool first_lane() const { return t == 0; }
  __device__ __forceinline__ int32_t want(int c) const { return (c * G + t) * VE; }
  __device__ __forceinline__ int32_t first(int c) const {
    const int32_t k = want(c);
    return k < K - VE ? k : K - VE;
  }
  __device__ __forceinline__ int32_t skip(int c) const { return want(c) - first(c); }

  struct Regs {
    Chunk<T> c[NC];
  };
  // the row's first element (rows of a whole wave: an address in scalar
  // registers, the classes a 32-bit offset)
  __device__ __forceinline__ T* at(const ScoresView& s, int64_t b) const {
    int64_t i;
    if (G >= 64)
      i = b * kRows + (kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / G) : 0);
    else
      i = row(b);
    return (T*)s.data + (i < s.n ? i : s.n - 1) * s.rs;
  }
  __device__ __forceinline__ void load(Regs& r, const ScoresView& s, int64_t b) const {
    const T* p = at(s, b);
#pragma unroll
    for (int c = 0; c < NC; ++c) r.c[c] = load_chunk<T>(p + (uint32_t)first(c));
  }
  __device__ __forceinline__ void trim(Regs& r) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int32_t sk = skip(c);
      if (__any(sk > 0)) {
        uint32_t(&w)[4] = r.c[c].w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (VE == 4) {
            w[e] = e < sk ? kNegInf : w[e];
          } else {
            const uint32_t one = (w[e] & 0xffff0000u) | (kNegInf & 0xffffu);
            w[e] = sk >= 2 * e + 2 ? kNegInf : sk == 2 * e + 1 ? one : w[e];
          }
        }
      }
    }
  }
  // -inf, or two of them
  static constexpr uint32_t kNegInf = sizeof(T) == 4                  ? 0xff800000u
                                      : __is_same(T, _Float16) ? 0xfc00fc00u
                                                               : 0xff80ff80u;
  // whether each pass starts from the scores again (8191 x 16001 bfloat16, 64
  // classes a thread: 121 us without, 115 with, five waves instead of three)
  static constexpr bool kHide = N >= 64;
  __device__ __forceinline__ void hide(Regs& r) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) hidden(r.c[c]);
  }
  // whether class k (-1: none) is one of this thread's
  __device__ __forceinline__ bool has(int32_t k) const { return k >= 0 && (k / VE) % G == t; }
  // a row that is left out has no class
  __device__ __forceinline__ void drop(Regs& r) const {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) r.c[c].w[e] = kNegInf;
  }
  static __device__ __forceinline__ float value(const Regs& r, int j) {
    return r.c[j / VE].get(j % VE);
  }
  __device__ __forceinline__ int32_t cls(int j) const { return first(j / VE) + j % VE; }
  // this thread's last slot with a class up to k (-1: none)
  __device__ __forceinline__ int last_slot(int32_t k) const {
    const int32_t q = k / VE;
    if (q < t) return -1;
    const int c = (q - t) / G;
    return c * VE + (c * G + t == q ? k - first(c) : VE - 1);
  }

  // reductions over the row; buf as for waves_reduce (kBuf words each)
  template <typename Op>
  __device__ __forceinline__ float reduce(float x, Op op, float* buf) const {
    // (buf is null where rows are one wave's)
    if (G <= 64) return lanes_reduce<(G < 64 ? G : 64)>(x, op);
    return waves_reduce<(G > 64 ? G / 64 : 1)>(x, op, buf);
  }
  // NV of them at once, in two steps with a barrier between where kBarrier; buf: kBuf
  // words a value (a workgroup's threads for slices), free again after one more barrier
  template <int NV, typename Op>
  __device__ __forceinline__ void put_all(float (&x)[NV], Op op, float* buf) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = lanes_reduce<(G < 64 ? G : 64)>(x[v], op);
    if (G > 64 && (threadIdx.x & 63) == 0)
#pragma unroll
      for (int v = 0; v < NV; ++v) buf[v * kBuf + (threadIdx.x >> 6)] = x[v];
  }
  template <int NV, typename Op>
  __device__ __forceinline__ void join_all(float (&x)[NV], Op op, const float* buf) const {
    if (G <= 64) return;
    // (a wave's value a lane: 16 waves' values in registers would cost the rows' room)
#pragma unroll
    for (int v = 0; v < NV; ++v)
      x[v] = lanes_reduce<kBuf>(buf[v * kBuf + (threadIdx.x & (kBuf - 1))], op);
  }
  template <int NV, typename Op>
  __device__ __forceinline__ void reduce_all(float (&x)[NV], Op op, float* buf) const {
    put_all(x, op, buf);
    if (G > 64) __syncthreads();
    join_all(x, op, buf);
  }

  // Lists of a row's classes (losses_lists.hpp): its entries j = t, t + G, ... are
  // this thread's.
  static constexpr int kListRows = kRows, kListLanes = G < 64 ? G : 64;
  __device__ __forceinline__ int entry() const { return t; }
  __device__ __forceinline__ int entry_step() const { return G; }
  // place of entry j in a table of the workgroup's lists of k
  __device__ __forceinline__ int entry_at(int j, int k) const { return threadIdx.x / G * k + j; }
  // a bit for each of a thread's slots; class k's is bit `bit` of word `word` among the
  // workgroup's (kMaskWords a thread, those of a number next to each other)
  static constexpr int kMaskWords = (N + 31) / 32;
  __device__ __forceinline__ void locate(int32_t k, int& word, uint32_t& bit) const {
    const int32_t q = k / VE, w = q * VE, from = w < K - VE ? w : K - VE;
    const int slot = q / G * VE + (k - from);
    word = (slot >> 5) * kThreads + threadIdx.x / G * G + q % G;
    bit = 1u << (slot & 31);
  }
  // classes whose bits are set are no longer this row's
  __device__ __forceinline__ void take_out(Regs& r, const uint32_t (&m)[kMaskWords]) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t b = (m[c * VE / 32] >> (c * VE % 32)) & ((1u << VE) - 1);
      if (__any(b != 0)) {
        uint32_t(&w)[4] = r.c[c].w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (VE == 4) {
            w[e] = b >> e & 1 ? kNegInf : w[e];
          } else {
            const uint32_t keep = (b >> (2 * e) & 1 ? 0u : 0xffffu) |
                                  (b >> (2 * e + 1) & 1 ? 0u : 0xffff0000u);
            w[e] = (w[e] & keep) | (kNegInf & ~keep);
          }
        }
      }
    }
  }

  // sum[k] = the workgroup's sum of acc over its rows, for every class.  Lanes
  // at the same place in their groups first, then the waves one after the
  // other: the same order every time.
  __device__ __forceinline__ void sum_rows(float (&acc)[N], float* sum) const {
    if (G < 64) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        for (int o = G; o < 64; o <<= 1) acc[j] += __shfl_xor(acc[j], o);
    }
    constexpr int kTurns = G <= 64 ? kThreads / 64 : 1;  // waves that hold the same classes
    for (int w = 0; w < kTurns; ++w) {
      if (G > 64 || ((int)(threadIdx.x >> 6) == w && (threadIdx.x & 63) < (G < 64 ? G : 64))) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j % VE >= skip(j / VE)) sum[cls(j)] = w ? sum[cls(j)] + acc[j] : acc[j];
      }
      __syncthreads();
    }
  }
  // sum of e^(s - m) over the row in float64, from memory; buf: kBuf words
  __device__ __forceinline__ double wide_sum(const ScoresView& s, int64_t i, float m,
                                             double* buf) const {
    const T* p = (const T*)s.data + i * s.rs;
    double z = 0.0;
    for (int32_t k = t; k < K; k += G) z += exp((double)to_f32(p[k]) - (double)m);
    for (int o = (G < 64 ? G : 64) / 2; o; o >>= 1) z += __shfl_xor(z, o);
    if (G <= 64) return z;
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = z;
    __syncthreads();
    z = 0.0;
    for (int w = 0; w < kBuf; ++w) z += buf[w];
    return z;
  }

  // out[cls(j)] (+)= f(j) for this thread's classes
  template <typename F>
  __device__ __forceinline__ void store(const ScoresView& o, int64_t b, bool accumulate, F f) const {
    T* p = at(o, b);
    const auto values = [&](int c, T* q) {
      float x[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = f(c * VE + e);
      if (accumulate) {
        const Chunk<T> old = load_chunk<T>(q);
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] += old.get(e);
      }
      Chunk<T> v;
      v.set(x);
      return v;
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      T* q = p + (uint32_t)first(c);
      if (skip(c) == 0) store_chunk<T>(q, values(c, q));
    }
    // a part of a chunk at the row's end, one thread's
    const int32_t part = K % VE;
    if (part && __any((K / VE) % G == t)) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c * G + t != K / VE) continue;
        T* q = p + (uint32_t)first(c);
        const Chunk<T> v = values(c, q);
#pragma unroll
        for (int e = 1; e < VE; ++e)
          if (e >= VE - part) q[e] = v.element(e);
      }
    }
  }
  // the same, and gl for class `label`: its thread writes it after its chunk
  template <typename F>
  __device__ __forceinline__ void store_row(const ScoresView& o, int64_t b, bool accumulate,
                                            int32_t label, float gl, F f) const {
    const bool mine = has(label);
    T* q = at(o, b) + (mine ? label : 0);
    if (mine && accumulate) gl += to_f32(*q);
    store(o, b, accumulate, f);
    if (mine) *q = from_f32<T>(gl);
  }
  __device__ __forceinline__ void store_zero(const ScoresView& o, int64_t b) const {
    store(o, b, false, [](int) { return 0.0f; });
  }
};

// ---------------------------------------------------------------------------
// ClassFrame: a thread per row and slice of its classes, the rows of a class
// next to each other (one load instruction reads 64 rows of a class).  The
// slices w = 0 .. S-1 are the waves of a workgroup; slice w holds the classes
// w, w + S, ... (N of them).  With S = 1 a workgroup's waves hold rows of
// their own; short rows may then also have their classes next to each other
// (ADJ false: any strides).  Classes past the last are read as the last one and
// set to -inf.
// ---------------------------------------------------------------------------
template <typename T_, int N_, bool SLICES, bool ADJ>
struct ClassFrame {
  using T = T_;
  static constexpr int N = N_, kWords = N_;
  static constexpr int kMax = SLICES ? 1024 : 256;
  static constexpr bool kBarrier = SLICES, kSlices = SLICES, kLaneRows = true;
  static constexpr int kShared = SLICES ? 64 : 1;
  static constexpr int kBuf = SLICES ? 16 * 64 : 1;
  int32_t w, S, K;

  __device__ __forceinline__ ClassFrame(const ScoresView& s)
      : w(SLICES ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0),
        S(SLICES ? blockDim.x >> 6 : 1),
        K(s.K) {}
  static __device__ __forceinline__ int64_t row(int64_t block) {
    return SLICES ? block * 64 + (threadIdx.x & 63) : block * 256 + threadIdx.x;
  }
  __device__ __forceinline__ bool first_lane() const { return w == 0; }
  __device__ __forceinline__ int32_t cls(int j) const { return w + j * S; }
  // this thread's last slot with a class up to k (-1: none)
  __device__ __forceinline__ int last_slot(int32_t k) const { return k < w ? -1 : (k - w) / S; }

  struct Regs {
    T c[N];
  };
  // the first row of this wave's 64, and this lane's offset from it (the last
  // row for lanes past the end): class addresses stay in scalar registers
  __device__ __forceinline__ T* at(const ScoresView& s, int64_t b) const {
    return (T*)s.data + first_row(s, b) * s.rs;
  }
  // (a wave wholly past the end: the last row of the matrix)
  static __device__ __forceinline__ int64_t first_row(const ScoresView& s, int64_t b) {
    if (SLICES) return b * 64;
    const int64_t i = b * 256 + 64 * __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    return i < s.n ? i : s.n - 1;
  }
  static __device__ __forceinline__ auto offset(const ScoresView& s, int64_t b) {
    const int64_t left = s.n - 1 - first_row(s, b);
    const uint32_t lane = threadIdx.x & 63, l = lane < left ? lane : (uint32_t)left;
    if constexpr (ADJ)
      return l;
    else
      return (int64_t)l * s.rs;
  }
  __device__ __forceinline__ void load(Regs& r, const ScoresView& s, int64_t b) const {
    const T* p = at(s, b);
    const auto o = offset(s, b);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int32_t k = cls(j) < K ? cls(j) : K - 1;
      r.c[j] = (p + k * s.ks)[o];
    }
  }
  __device__ __forceinline__ void trim(Regs& r) const {
#pragma unroll
    for (int j = 0; j < N; ++j) r.c[j] = cls(j) < K ? r.c[j] : (T)(-__builtin_inff());
  }
  static constexpr bool kHide = false;
  __device__ __forceinline__ void hide(Regs&) const {}
  __device__ __forceinline__ void drop(Regs& r) const {
#pragma unroll
    for (int j = 0; j < N; ++j) r.c[j] = (T)(-__builtin_inff());
  }
  static __device__ __forceinline__ float value(const Regs& r, int j) { return to_f32(r.c[j]); }

  template <typename Op>
  __device__ __forceinline__ float reduce(float x, Op op, float* buf) const {
    if (!SLICES) return x;
    const int lane = threadIdx.x & 63;
    buf[w * 64 + lane] = x;
    __syncthreads();
    x = buf[lane];
    for (int v = 1; v < S; ++v) x = op(x, buf[v * 64 + lane]);
    return x;
  }
  template <int NV, typename Op>
  __device__ __forceinline__ void put_all(float (&x)[NV], Op, float* buf) const {
    if (!SLICES) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) buf[v * blockDim.x + threadIdx.x] = x[v];
  }
  template <int NV, typename Op>
  __device__ __forceinline__ void join_all(float (&x)[NV], Op op, const float* buf) const {
    if (!SLICES) return;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = buf[v * blockDim.x + lane];
    for (int u = 1; u < S; ++u) {
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v] = op(x[v], buf[v * blockDim.x + u * 64 + lane]);
    }
  }
  template <int NV, typename Op>
  __device__ __forceinline__ void reduce_all(float (&x)[NV], Op op, float* buf) const {
    put_all(x, op, buf);
    if (SLICES) __syncthreads();
    join_all(x, op, buf);
  }
  // lists (losses_lists.hpp): the wave and slot of class k (k / S of k < 512 by a
  // multiplication)
  __device__ __forceinline__ void locate(int32_t k, int& wave, int& slot) const {
    slot = (k * ((65535 + S) / S)) >> 16;
    wave = k - slot * S;
  }
  // slot j is no longer one of this row's classes
  __device__ __forceinline__ void take_out(Regs& r, int j, bool out) const {
    r.c[j] = out ? (T)(-__builtin_inff()) : r.c[j];
  }
  // sum[k] = the workgroup's sum of acc over its rows, for every class
  __device__ __forceinline__ void sum_rows(float (&acc)[N], float* sum) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      acc[j] = lanes_reduce<64>(acc[j], AddF());
      __builtin_amdgcn_sched_barrier(0);  // (N at once would take the registers of two waves)
    }
    const int kTurns = SLICES ? 1 : 4;
    for (int u = 0; u < kTurns; ++u) {
      if ((SLICES || (int)(threadIdx.x >> 6) == u) && (threadIdx.x & 63) == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (cls(j) < K) sum[cls(j)] = u ? sum[cls(j)] + acc[j] : acc[j];
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ double wide_sum(const ScoresView& s, int64_t i, float m,
                                             double* buf) const {
    const T* p = (const T*)s.data + i * s.rs;
    double z = 0.0;
    for (int32_t k = w; k < K; k += S) z += exp((double)to_f32(p[k * s.ks]) - (double)m);
    if (!SLICES) return z;
    const int lane = threadIdx.x & 63;
    buf[w * 64 + lane] = z;
    __syncthreads();
    z = 0.0;
    for (int v = 0; v < S; ++v) z += buf[v * 64 + lane];
    return z;
  }
  template <typename F>
  __device__ __forceinline__ void store(const ScoresView& o, int64_t b, bool accumulate, F f) const {
    store_row(o, b, accumulate, -1, 0.0f, f);
  }
  template <typename F>
  __device__ __forceinline__ void store_row(const ScoresView& o, int64_t b, bool accumulate,
                                            int32_t label, float gl, F f) const {
    T* p = at(o, b);
    const auto l = offset(o, b);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (cls(j) < K) {
        T* q = p + cls(j) * o.ks + l;
        const float y = f(j), x = cls(j) == label ? gl : y;
        *q = from_f32<T>(accumulate ? x + to_f32(*q) : x);
      }
    }
  }
  __device__ __forceinline__ void store_zero(const ScoresView& o, int64_t b) const {
    store(o, b, false, [](int) { return 0.0f; });
  }
};

// which slices class-major rows of 17 to 512 classes take: fn(frame tag,
// workgroups, threads).  4, 8, 12 or 16 waves, which fill the SIMDs evenly, of as
// few classes each as hold the row.  1M x 100 float32, 8 waves of 13 classes, 10 of 10,
// 7 of 16, 13 of 8: balance loss 319, 325, 330, 349 us; policy loss of 500000 x 100
// 94, 125, 108, 158; of 1M x 30, 4 waves of 8, 3 of 10, 3 of 13, 2 of 16: 65, 66,
// 70, 75; of 160000 x 150, 12 of 13, 16 of 10, 10 of 16: 58, 68, 61.
template <typename T, typename Fn>
static void pick_slices(const ScoresView& s, Fn fn) {
  const int64_t tiles = (s.n + 63) / 64;
  if (s.K > 256)
    return fn(FrameTag<ClassFrame<T, 32, true, true>>(), tiles, 64 * (int)((s.K + 31) / 32));
  const int S = s.K <= 64 ? 4 : s.K <= 128 ? 8 : s.K <= 192 ? 12 : 16;
  if (s.K <= 8 * S) return fn(FrameTag<ClassFrame<T, 8, true, true>>(), tiles, 64 * S);
  if (s.K <= 10 * S) return fn(FrameTag<ClassFrame<T, 10, true, true>>(), tiles, 64 * S);
  if (s.K <= 13 * S) return fn(FrameTag<ClassFrame<T, 13, true, true>>(), tiles, 64 * S);
  fn(FrameTag<ClassFrame<T, 16, true, true>>(), tiles, 64 * S);
}

// ---------------------------------------------------------------------------
// which frame a call takes: fn(frame tag, workgroups, threads) for the smallest
// one that holds the rows (rows_fit).  Row-major rows take two to eight chunks a
// thread rather than one, so that a wave has more loads in flight and spends
// what a row costs as a whole on more rows: with one chunk a thread the policy
// loss of 300000 x 100 float32 takes 57 us instead of 43, of 100000 x 500
// bfloat16 57 and 40, the log-probabilities' gradient 59 and 44, 47 and 38; 30000 x
// 3000 bfloat16, eight chunks of a wave's threads instead of two of a
// workgroup's, whose waves wait for one another: 95 and 65 (not the gradient
// without sums: 66 and 68).  Up to eight chunks a thread each: log-probabilities'
// gradient of 300000 x 30 float32 19 us, 20 with two.
// ---------------------------------------------------------------------------
template <typename T, bool REF, bool SUMS, typename Fn>
static void pick_row_frame(const ScoresView& s, Fn fn) {
  constexpr int VE = Chunk<T>::VE;
  const int64_t chunks = (s.K + VE - 1) / VE;
  const auto go = [&](auto tag) {
    using F = typename decltype(tag)::type;
    fn(tag, (s.n + F::kRows - 1) / F::kRows, F::kThreads);
  };
  if (chunks <= 4) return go(FrameTag<RowFrame<T, 4, 1>>());
  if (chunks <= 8) return go(FrameTag<RowFrame<T, 8, 1>>());
  if (chunks <= 16) return go(FrameTag<RowFrame<T, 8, 2>>());
  if (chunks <= 32) return go(FrameTag<RowFrame<T, 16, 2>>());
  if (chunks <= 64) return go(FrameTag<RowFrame<T, 32, 2>>());
  if (chunks <= 128) return go(FrameTag<RowFrame<T, 32, 4>>());
  if (chunks <= 256) return go(FrameTag<RowFrame<T, 32, 8>>());
  if constexpr (!SUMS) {
    if (chunks <= 512) return go(FrameTag<RowFrame<T, 256, 2>>());
  }
  if (chunks <= 512) return go(FrameTag<RowFrame<T, 64, 8>>());
  if (chunks <= 1024) return go(FrameTag<RowFrame<T, 256, 4>>());
  if (chunks <= 2048) return go(FrameTag<RowFrame<T, 256, 8>>());
  if (REF || chunks <= 4096) return go(FrameTag<RowFrame<T, 1024, 4>>());
  if constexpr (!REF) {
    if (chunks <= 8192) return go(FrameTag<RowFrame<T, 1024, 8>>());
    go(FrameTag<RowFrame<T, 1024, 16>>());
  }
}

template <typename T, typename Fn>
static void pick_class_frame(const ScoresView& s, Fn fn) {
  const int64_t blocks = (s.n + 255) / 256;
  if (!s.class_major()) {  // rows shorter than a chunk
    if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, false>>(), blocks, 256);
    return fn(FrameTag<ClassFrame<T, 8, false, false>>(), blocks, 256);
  }
  if (s.K <= 4) return fn(FrameTag<ClassFrame<T, 4, false, true>>(), blocks, 256);
  if (s.K <= 8) return fn(FrameTag<ClassFrame<T, 8, false, true>>(), blocks, 256);
  if (s.K <= 12) return fn(FrameTag<ClassFrame<T, 12, false, true>>(), blocks, 256);
  if (s.K <= 16) return fn(FrameTag<ClassFrame<T, 16, false, true>>(), blocks, 256);
  pick_slices<T>(s, fn);
}

template <typename T, bool REF, bool SUMS, typename Fn>
static void pick_frame(const ScoresView& s, Fn fn) {
  if (s.class_major() || s.K < Chunk<T>::VE)
    pick_class_frame<T>(s, fn);
  else
    pick_row_frame<T, REF, SUMS>(s, fn);
}

}  // namespace wgbm
