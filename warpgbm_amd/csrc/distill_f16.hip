// Distillation from listed classes, _Float16 scores.
#include "distill.hpp"

namespace wgbm {

int distill_f16(const ScoresView& s, const DistillRows& g, const ScoresView& out, bool accumulate,
            hipStream_t st) {
  return distill_frames<_Float16>(s, g, out, accumulate, st);
}

}  // namespace wgbm
