// Distillation from listed classes, __bf16 scores.
#include "distill.hpp"

namespace wgbm {

int distill_bf16(const ScoresView& s, const DistillRows& g, const ScoresView& out, bool accumulate,
            hipStream_t st) {
  return distill_frames<__bf16>(s, g, out, accumulate, st);
}

}  // namespace wgbm
