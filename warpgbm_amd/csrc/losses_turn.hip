// Transposes of class-major scores of more classes than a workgroup's slices
// hold: the losses work on a row-major copy of them.
#include <type_traits>

#include "losses_frames.hpp"
#include "losses_host.hpp"

namespace wgbm {

// b(i, k) (+)= a(i, k) between class-major scores (or gradient) and a row-major
// copy, by tiles of 64 x 64 through LDS; tile `first` + block, the rows' tiles next to
// each other (60000 x 2000 bfloat16: the balance loss takes 598 us with its two
// transposes, 204 of row-major scores)
template <typename A, typename B, bool TO_ROWS>
__global__ __launch_bounds__(256) void transpose_kernel(ScoresView a, ScoresView b,
                                                        bool accumulate, int32_t row_tiles,
                                                        int32_t first) {
  __shared__ float tile[64][65];
  const int64_t i0 = (int64_t)(blockIdx.x % (uint32_t)row_tiles) * 64;
  const int32_t k0 = (first + (int32_t)(blockIdx.x / (uint32_t)row_tiles)) * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const A* p = (const A*)a.data;
  B* q = (B*)b.data;
#pragma unroll 4
  for (int r = y; r < 64; r += 4) {
    // x along the dimension that is contiguous in a
    const int64_t i = i0 + (TO_ROWS ? x : r);
    const int32_t k = k0 + (TO_ROWS ? r : x);
    if (i < a.n && k < a.K) tile[r][x] = to_f32(p[i * a.rs + k * a.ks]);
  }
  __syncthreads();
#pragma unroll 4
  for (int r = y; r < 64; r += 4) {
    const int64_t i = i0 + (TO_ROWS ? r : x);
    const int32_t k = k0 + (TO_ROWS ? x : r);
    if (i < a.n && k < a.K) {
      B* o = q + i * b.rs + k * b.ks;
      const float v = tile[x][r];
      *o = from_f32<B>(accumulate ? v + to_f32(*o) : v);
    }
  }
}

// T: the class-major side's type; the row-major side has it too, or float32.
// Launches of at most 2^23 workgroups of 256 threads: a grid's threads are counted in
// 32 bits.
template <typename T, bool TO_ROWS>
static int transpose(const ScoresView& a, const ScoresView& b, bool accumulate, hipStream_t st) {
  const int64_t row_tiles = (a.n + 63) / 64, class_tiles = ((int64_t)a.K + 63) / 64;
  const auto go = [&](auto rows, int64_t part_rows, int64_t from) {
    using R = decltype(rows);
    using A = std::conditional_t<TO_ROWS, T, R>;
    using B = std::conditional_t<TO_ROWS, R, T>;
    const int64_t most = std::max<int64_t>(1, (int64_t(1) << 23) / part_rows);
    ScoresView p = rows_of(a, from * 64, std::min(a.n - from * 64, part_rows * 64));
    ScoresView q = rows_of(b, from * 64, p.n);
    for (int64_t k = 0; k < class_tiles; k += most)
      hipLaunchKernelGGL((transpose_kernel<A, B, TO_ROWS>),
                         dim3((unsigned)(part_rows * std::min(most, class_tiles - k))), dim3(256),
                         0, st, p, q, accumulate, (int32_t)part_rows, (int32_t)k);
  };
  for (int64_t from = 0; from < row_tiles; from += int64_t(1) << 23) {
    const int64_t part = std::min(int64_t(1) << 23, row_tiles - from);
    if ((TO_ROWS ? b : a).dtype == kF32)
      go(float(), part, from);
    else
      go(T(), part, from);
  }
  WGBM_LAUNCH_CHECK();
  return 0;
}

int scores_to_rows(const ScoresView& a, const ScoresView& b, hipStream_t st) {
  LOSS_TYPES(a.dtype, return (transpose<T, true>(a, b, false, st)));
}
int rows_to_scores(const ScoresView& a, const ScoresView& b, bool accumulate, hipStream_t st) {
  LOSS_TYPES(b.dtype, return (transpose<T, false>(a, b, accumulate, st)));
}

}  // namespace wgbm
