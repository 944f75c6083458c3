// Alternatives of class scores and their gradient, float scores.
#include "alternatives.hpp"
#include "alternatives_grad.hpp"

namespace wgbm {

int alternatives_f32(const ScoresView& s, const AltRows& g, hipStream_t st) {
  return alternatives_frames<float>(s, g, st);
}

int alternatives_grad_f32(const ScoresView& s, const AltGradRows& g, const ScoresView& out,
                      bool accumulate, hipStream_t st) {
  return alternatives_grad_frames<float>(s, g, out, accumulate, st);
}

}  // namespace wgbm
