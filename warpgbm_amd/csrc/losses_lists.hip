// Host side of the losses with lists of a row's classes (alternatives.hpp,
// alternatives_grad.hpp, distill.hpp): launches in parts, and class-major rows of
// more classes than a workgroup's slices hold, which go through a row-major copy
// (of their type, or of float32 where the gradient is added to another, so that it is
// rounded once).
#include "losses_host.hpp"

namespace wgbm {

static bool through_rows(const ScoresView& s) { return s.class_major() && s.K > 512; }

size_t lists_workspace(const ScoresView& s, bool grad) {
  if (!through_rows(s)) return 0;
  return (size_t)s.n * s.K * (grad || s.dtype == kF32 ? 4 : 2);
}

static ScoresView row_copy(const ScoresView& s, bool wide, void* ws) {
  ScoresView v = s;
  v.data = ws;
  if (wide) v.dtype = kF32;
  v.rs = s.K;
  v.ks = 1;
  return v;
}

int class_alternatives(const ScoresView& s, const AltRows& g, void* ws, hipStream_t st) {
  ScoresView v = s;
  if (through_rows(s)) {
    v = row_copy(s, false, ws);
    const int r = scores_to_rows(s, v, st);
    if (r) return r;
  }
  const auto rows = v.dtype == kF32    ? alternatives_f32
                    : v.dtype == kBF16 ? alternatives_bf16
                                       : alternatives_f16;
  return row_parts(v, [&](int64_t i, int64_t n) {
    AltRows p = g;
    if (p.label) {
      p.label += i;
      p.label_log_prob += i;
    }
    p.classes += i * g.k;
    p.log_prob += i * g.k;
    p.entropy += i;
    p.norm += 3 * i;
    return rows(rows_of(v, i, n), p, st);
  });
}

// a gradient of rows: fn(scores, gradient, whether it is added), in place in the
// copy where there is one (a thread writes what it alone has read)
template <typename Fn>
static int with_rows(const ScoresView& s, const ScoresView& out, bool accumulate, void* ws,
                     hipStream_t st, Fn fn) {
  if (!through_rows(s)) return fn(s, out, accumulate);
  const ScoresView v = row_copy(s, accumulate, ws);
  int r = scores_to_rows(s, v, st);
  if (r) return r;
  r = fn(v, out.data ? v : out, false);
  if (r || !out.data) return r;
  return rows_to_scores(v, out, accumulate, st);
}

int class_alternatives_grad(const ScoresView& s, const AltGradRows& g, const ScoresView& out,
                            bool accumulate, void* ws, hipStream_t st) {
  return with_rows(s, out, accumulate, ws, st, [&](const ScoresView& v, const ScoresView& o,
                                                   bool add) {
    const auto rows = v.dtype == kF32    ? alternatives_grad_f32
                      : v.dtype == kBF16 ? alternatives_grad_bf16
                                         : alternatives_grad_f16;
    return row_parts(v, [&](int64_t i, int64_t n) {
      AltGradRows p = g;
      p.norm += 3 * i;
      if (p.label) {
        p.label += i;
        p.grad_label += i;
      }
      if (p.k) {
        p.classes += i * g.class_stride;
        p.grad_list += i * g.grad_stride;
      }
      if (p.grad_entropy) p.grad_entropy += i;
      return rows(rows_of(v, i, n), p, rows_of(o, i, n), add, st);
    });
  });
}

int distill_loss(const ScoresView& s, const DistillRows& g, const ScoresView& out, bool accumulate,
                 void* ws, hipStream_t st) {
  return with_rows(s, out, accumulate, ws, st, [&](const ScoresView& v, const ScoresView& o,
                                                   bool add) {
    const auto rows = v.dtype == kF32    ? distill_f32
                      : v.dtype == kBF16 ? distill_bf16
                                         : distill_f16;
    return row_parts(v, [&](int64_t i, int64_t n) {
      DistillRows p = g;
      p.classes += i * g.class_stride;
      p.logits += i * g.logit_stride;
      if (p.log_norm) p.log_norm += i;
      if (p.weight) p.weight += i;
      p.loss += i;
      return rows(rows_of(v, i, n), p, rows_of(o, i, n), add, st);
    });
  });
}

}  // namespace wgbm
