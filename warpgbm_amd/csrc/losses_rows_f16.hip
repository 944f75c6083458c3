// Log-probabilities and the policy loss of rows in registers, _Float16 scores.
#include "losses_rows.hpp"

namespace wgbm {

int log_probs_rows_f16(const ScoresView& s, const int32_t* label, float* log_prob, float* norm,
                      hipStream_t st) {
  return log_probs_frames<_Float16>(s, label, log_prob, norm, st);
}

int log_probs_grad_rows_f16(const ScoresView& s, const int32_t* label, const float* norm,
                           const float* grad, const ScoresView& out, hipStream_t st) {
  return log_probs_grad_frames<_Float16>(s, label, norm, grad, out, st);
}

int policy_rows_f16(const ScoresView& s, const ScoresView& ref, const PolicyRows& g,
                   const ScoresView& out, bool accumulate, hipStream_t st) {
  return ref.data ? policy_frames<_Float16, true>(s, ref, g, out, accumulate, st)
                  : policy_frames<_Float16, false>(s, ref, g, out, accumulate, st);
}

}  // namespace wgbm
