// Host declarations of the losses (losses.hip, losses_balance.hip, losses_lists.hip,
// losses_turn.hip, preference.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "losses.hpp"

namespace wgbm {

// waves that fill the GPU (256 CUs, 16 waves each)
constexpr int64_t kLossWaves = 4096;

// runs a statement with T the element type of a dtype code
#define LOSS_TYPES(dtype, ...)        \
  do {                                \
    if ((dtype) == kF32) {            \
      using T = float;                \
      __VA_ARGS__;                    \
    } else if ((dtype) == kBF16) {    \
      using T = __bf16;               \
      __VA_ARGS__;                    \
    } else {                          \
      using T = _Float16;             \
      __VA_ARGS__;                    \
    }                                 \
  } while (0)

size_t log_probs_workspace(const ScoresView& s);
int class_log_probs(const ScoresView& s, const int32_t* label, float* log_prob, float* norm,
                    void* ws, hipStream_t st);
int class_log_probs_grad(const ScoresView& s, const int32_t* label, const float* norm,
                         const float* grad, const ScoresView& out, hipStream_t st);

// Whether rows fit the registers of the threads that share them (one launch,
// losses_rows.hpp).  Class-major: 16 waves' slices of 32 classes.  Row-major:
// 1024 threads of 16 chunks of 16 bytes (64 of the 128 registers that a thread
// has), of 4 with a second matrix.  (8 with a second matrix would fit now that the
// sums against a reference are pinned: 2000 x 50000 bfloat16 220 us, the ranged path,
// which takes them, 422.)
// Shorter rows than a chunk: a thread each.
inline bool rows_fit(const ScoresView& s, bool ref) {
  const int32_t VE = s.dtype == kF32 ? 4 : 8;
  if (s.class_major()) return s.K <= 512;
  return s.K < VE || (s.K + VE - 1) / VE <= (ref ? 4096 : 16384);
}
#define LOSS_ROWS(t)                                                                             \
  int log_probs_grad_rows_##t(const ScoresView& s, const int32_t* label, const float* norm,      \
                              const float* grad, const ScoresView& out, hipStream_t st);         \
  int log_probs_rows_##t(const ScoresView& s, const int32_t* label, float* log_prob, float* norm, \
                         hipStream_t st);                                                        \
  int policy_rows_##t(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,           \
                      const ScoresView& out, bool accumulate, hipStream_t st)
LOSS_ROWS(f32);
LOSS_ROWS(bf16);
LOSS_ROWS(f16);

// Lists of a row's classes: at most kMaxList entries.  scale = log2(e) / tau.
constexpr int32_t kMaxList = 64;
struct AltRows {
  const int32_t* label;  // null: none
  int32_t k;
  float scale;
  double inv_tau;
  int32_t* classes;  // [n][k]
  float* log_prob;   // [n][k]
  float* entropy;
  float* label_log_prob;
  float* norm;  // [n][3]
};
struct AltGradRows {
  const float* norm;
  const int32_t* label;  // null: none
  const float* grad_label;
  const int32_t* classes;  // row i's entry j at classes + i * class_stride + j * class_step
  int64_t class_stride, class_step;
  const float* grad_list;
  int64_t grad_stride, grad_step;
  int32_t k;
  const float* grad_entropy;  // null: 0
  float scale;
  double inv_tau;
};
struct DistillRows {
  const int32_t* classes;
  int64_t class_stride, class_step;
  const float* logits;
  int64_t logit_stride, logit_step;
  int32_t k;
  bool rest;              // the classes that are not listed count
  const float* log_norm;  // null: log_norm_all for every row
  double log_norm_all;
  const float* weight;  // null: 1
  float scale;
  double inv_tau;
  float tau;
  float* loss;
};
#define LOSS_LISTS(t)                                                                          \
  int alternatives_##t(const ScoresView& s, const AltRows& g, hipStream_t st);                 \
  int alternatives_grad_##t(const ScoresView& s, const AltGradRows& g, const ScoresView& out,  \
                            bool accumulate, hipStream_t st);                                  \
  int distill_##t(const ScoresView& s, const DistillRows& g, const ScoresView& out,            \
                  bool accumulate, hipStream_t st)
LOSS_LISTS(f32);
LOSS_LISTS(bf16);
LOSS_LISTS(f16);
// (class-major rows of more classes than slices hold go through a row-major copy)
size_t lists_workspace(const ScoresView& s, bool grad);
int class_alternatives(const ScoresView& s, const AltRows& g, void* ws, hipStream_t st);
int class_alternatives_grad(const ScoresView& s, const AltGradRows& g, const ScoresView& out,
                            bool accumulate, void* ws, hipStream_t st);
int distill_loss(const ScoresView& s, const DistillRows& g, const ScoresView& out, bool accumulate,
                 void* ws, hipStream_t st);
// Rows of more 16-byte chunks than this are cut in tiles of chunks: of the gradient of
// alternatives, which sums nothing over a row, and of the other two.
constexpr int32_t kGradTileChunks = 1024, kWholeChunks = 16384, kTileChunks = 4096;
// Tiles of a row of K classes, of `span` classes each but the last, at most `most`: as
// even as whole chunks allow.  The last one holds 8 classes at least (a frame reads a
// row's end by a whole chunk): where fewer would be left over, shorter tiles leave more
// to it.
inline int32_t cut_tiles(int32_t K, int32_t most, int32_t* span) {
  const int32_t n = (K + most - 1) / most;
  *span = ((K + n - 1) / n + 7) / 8 * 8;
  while (K % *span != 0 && K % *span < 8) *span -= 8;
  return (K + *span - 1) / *span;
}
// the same for scores (1 tile: whole rows)
inline int32_t row_tiles(const ScoresView& s, bool grad, int32_t* span) {
  const int32_t VE = s.dtype == kF32 ? 4 : 8;
  *span = s.K;
  if (s.class_major() || (s.K + VE - 1) / VE <= (grad ? kGradTileChunks : kWholeChunks)) return 1;
  return cut_tiles(s.K, (grad ? kGradTileChunks : kTileChunks) * VE, span);
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
inline ScoresView rows_of(const ScoresView& s, int64_t i, int64_t n) {
  ScoresView v = s;
  if (!s.data) return v;
  v.data = (unsigned char*)s.data + i * s.rs * (s.dtype == kF32 ? 4 : 2);
  v.n = n;
  return v;
}

// class-major scores to a row-major copy of their type or of float32, and a
// row-major gradient back (added to b where accumulate)
int scores_to_rows(const ScoresView& a, const ScoresView& b, hipStream_t st);
int rows_to_scores(const ScoresView& a, const ScoresView& b, bool accumulate, hipStream_t st);

size_t policy_workspace(const ScoresView& s, bool ref);
int policy_loss(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,
                const ScoresView& out, bool accumulate, void* ws, hipStream_t st);

struct BalanceOut {
  float* loss;
  int64_t* counts;
  float* prob;
};
// working memory of a balance loss
struct BalanceWs {
  uint32_t* ticket;
  float* scale;
  float* share;       // [K]
  double* loss_part;  // [K / 4 + 1]
  float2* norm;       // [n]
  float* part;        // [K][slots]
  int32_t* count;     // [K + 1][slots]
  void* rows;         // a row-major copy of the scores, where one is needed
  size_t bytes;
};
#define LOSS_BALANCE(t)                                                                          \
  int balance_stats_##t(const ScoresView& s, const uint8_t* mask, int32_t top_k,                 \
                        const BalanceWs& w, int32_t* slots, hipStream_t st);                     \
  int balance_grad_##t(const ScoresView& s, const BalanceWs& w, const ScoresView& out,           \
                       bool accumulate, hipStream_t st)
LOSS_BALANCE(f32);
LOSS_BALANCE(bf16);
LOSS_BALANCE(f16);
size_t balance_workspace(const ScoresView& s);
int balance_loss(const ScoresView& s, const uint8_t* mask, int32_t top_k, float coef,
                 const BalanceOut& o, const ScoresView& out, bool accumulate, void* ws,
                 hipStream_t st);

// (the tables as in wgbm_preference_args)
struct PreferenceArgs {
  const float* log_prob;
  const float* ref;
  int64_t n_rows;
  const int64_t* seg_start;  // null: every row is a sequence of its own
  int64_t n_seg;
  const int32_t* pairs;
  int64_t n_pairs;
  const int32_t* inc;
  const int64_t* inc_start;
  const int64_t* share;
  int64_t n_shares;
  const uint8_t* is_long;
  const int64_t* task;
  int64_t n_tasks;
  const int64_t* task_start;  // null: task t < n_seg is sequence t
  const int64_t* piece;
  int64_t n_pieces;
  const int64_t* multi;
  int64_t n_multi;
  const int64_t* idle;
  int64_t n_idle;
  bool disjoint;
  const float* weight;
  float beta, smooth;
  int32_t lanes;  // 4 .. 64
  float* loss;
  float* margin;
  float* grad;
};
size_t preference_workspace(const PreferenceArgs& a);
int preference_loss(const PreferenceArgs& a, void* ws, hipStream_t st);

}  // namespace wgbm
