// Alternatives of class scores and their gradient, _Float16 scores.
#include "alternatives.hpp"
#include "alternatives_grad.hpp"

namespace wgbm {

int alternatives_f16(const ScoresView& s, const AltRows& g, hipStream_t st) {
  return alternatives_frames<_Float16>(s, g, st);
}

int alternatives_grad_f16(const ScoresView& s, const AltGradRows& g, const ScoresView& out,
                      bool accumulate, hipStream_t st) {
  return alternatives_grad_frames<_Float16>(s, g, out, accumulate, st);
}

}  // namespace wgbm
