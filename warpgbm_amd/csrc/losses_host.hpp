// Host declarations of the losses (losses.hip, losses_balance.hip,
// preference.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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
