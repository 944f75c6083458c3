// Distillation from listed classes, float scores.
#include "distill.hpp"

namespace wgbm {

int distill_f32(const ScoresView& s, const DistillRows& g, const ScoresView& out, bool accumulate,
            hipStream_t st) {
  return distill_frames<float>(s, g, out, accumulate, st);
}

}  // namespace wgbm
