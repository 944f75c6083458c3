// Alternatives of class scores and their gradient, __bf16 scores.
#include "alternatives.hpp"
#include "alternatives_grad.hpp"

namespace wgbm {

int alternatives_bf16(const ScoresView& s, const AltRows& g, hipStream_t st) {
  return alternatives_frames<__bf16>(s, g, st);
}

int alternatives_grad_bf16(const ScoresView& s, const AltGradRows& g, const ScoresView& out,
                      bool accumulate, hipStream_t st) {
  return alternatives_grad_frames<__bf16>(s, g, out, accumulate, st);
}

}  // namespace wgbm
