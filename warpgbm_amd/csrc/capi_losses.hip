// extern "C" entry points of the losses (declared in include/warpgbm_amd.h).
#include "../../include/warpgbm_amd.h"
#include <cmath>

#include "losses_host.hpp"

using namespace wgbm;

static_assert(WGBM_MAX_LIST == kMaxList, "list length");
static_assert(WGBM_F32 == kF32 && WGBM_BF16 == kBF16 && WGBM_F16 == kF16, "type codes");

// most classes of a row, and of the balance loss
constexpr int32_t kMaxClasses = 1 << 24;
constexpr int32_t kMaxBalanceClasses = 4096;
constexpr int32_t kMaxTopK = 8;

static inline hipStream_t S(void* s) { return (hipStream_t)s; }

// a scores argument as the kernels take it; what is checked here is all that
// keeps their accesses inside [data, data + extent)
static int view_of(const wgbm_scores* s, const char* what, ScoresView* v) {
  WGBM_REQUIRE(s, "%s: null pointer", what);
  WGBM_REQUIRE(s->dtype == WGBM_F32 || s->dtype == WGBM_BF16 || s->dtype == WGBM_F16,
               "%s: type code %d is none of WGBM_F32, WGBM_BF16, WGBM_F16", what, s->dtype);
  WGBM_REQUIRE(s->n_rows >= 0 && s->n_rows < (int64_t(1) << 31), "%s: n_rows out of range", what);
  WGBM_REQUIRE(s->n_classes >= 1 && s->n_classes <= kMaxClasses,
               "%s: n_classes must be in [1, %d]", what, kMaxClasses);
  const bool row = s->class_stride == 1 && s->row_stride >= s->n_classes;
  const bool cls = s->row_stride == 1 && s->class_stride >= (s->n_rows > 0 ? s->n_rows : 1);
  WGBM_REQUIRE(row || cls,
               "%s: strides (%lld, %lld) are neither those of rows (n, 1) nor of classes (1, k) "
               "next to each other without overlap",
               what, (long long)s->row_stride, (long long)s->class_stride);
  WGBM_REQUIRE(s->row_stride < (int64_t(1) << 40) && s->class_stride < (int64_t(1) << 40),
               "%s: stride out of range", what);
  WGBM_REQUIRE(s->data || s->n_rows == 0, "%s: null data", what);
  const int es = s->dtype == WGBM_F32 ? 4 : 2;
  WGBM_REQUIRE(((uintptr_t)s->data % es) == 0, "%s: data is not aligned to its type", what);
  *v = ScoresView{s->data, s->dtype, s->n_rows, s->n_classes, s->row_stride, s->class_stride};
  return 0;
}

// a second matrix of the same shape, type and order
static int same_kind(const ScoresView& a, const ScoresView& b, const char* what) {
  WGBM_REQUIRE(a.dtype == b.dtype && a.n == b.n && a.K == b.K,
               "%s must have the shape and type of the scores", what);
  WGBM_REQUIRE(a.class_major() == b.class_major(),
               "%s must have the order (rows or classes next to each other) of the scores", what);
  return 0;
}

static int balance_classes(const ScoresView& s) {
  WGBM_REQUIRE(s.K <= kMaxBalanceClasses, "balance_loss: at most %d classes, got %d",
               kMaxBalanceClasses, s.K);
  return 0;
}

#define TRY(expr)         \
  do {                    \
    const int _r = (expr); \
    if (_r) return _r;    \
  } while (0)

extern "C" {

int64_t wgbm_class_log_probs_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s)) return -1;
  return (int64_t)log_probs_workspace(s);
}

int wgbm_class_log_probs(const wgbm_scores* scores, const int32_t* labels, float* log_prob,
                         float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  ScoresView s;
  TRY(view_of(scores, "scores", &s));
  if (s.n == 0) return 0;
  WGBM_REQUIRE(labels && log_prob && norm, "class_log_probs: null pointer");
  const int64_t need = (int64_t)log_probs_workspace(s);
  WGBM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "class_log_probs: workspace too small");
  return class_log_probs(s, labels, log_prob, norm, workspace, S(stream));
}

int wgbm_class_log_probs_grad(const wgbm_scores* scores, const int32_t* labels, const float* norm,
                              const float* grad_log_prob, const wgbm_scores* grad, void* stream) {
  ScoresView s, g;
  TRY(view_of(scores, "scores", &s));
  TRY(view_of(grad, "grad", &g));
  TRY(same_kind(s, g, "grad"));
  if (s.n == 0) return 0;
  WGBM_REQUIRE(labels && norm && grad_log_prob, "class_log_probs_grad: null pointer");
  return class_log_probs_grad(s, labels, norm, grad_log_prob, g, S(stream));
}

int64_t wgbm_policy_loss_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s)) return -1;
  return (int64_t)policy_workspace(s, true);
}

int wgbm_policy_loss(const wgbm_scores* scores, const wgbm_policy_args* a, float* loss,
                     float* log_prob, float* kl, const wgbm_scores* grad, int32_t accumulate,
                     void* workspace, int64_t workspace_bytes, void* stream) {
  ScoresView s, r{}, g{};
  TRY(view_of(scores, "scores", &s));
  WGBM_REQUIRE(a, "policy_loss: null arguments");
  if (a->ref_scores) {
    TRY(view_of(a->ref_scores, "ref_scores", &r));
    TRY(same_kind(s, r, "ref_scores"));
    WGBM_REQUIRE(!a->ref_log_prob, "policy_loss: ref_scores and ref_log_prob exclude each other");
  }
  if (grad) {
    TRY(view_of(grad, "grad", &g));
    TRY(same_kind(s, g, "grad"));
  }
  WGBM_REQUIRE(a->clip_low >= 0.0 && a->clip_low <= 1.0,
               "policy_loss: clip_low must be in [0, 1]");
  WGBM_REQUIRE(a->clip_high >= 0.0 && std::isfinite(a->clip_high),
               "policy_loss: clip_high must be non-negative and finite");
  WGBM_REQUIRE(std::isfinite(a->kl_coef) && a->kl_coef >= 0.0f,
               "policy_loss: kl_coef must be non-negative and finite");
  if (s.n == 0) return 0;
  WGBM_REQUIRE(a->actions && a->old_log_prob && a->advantage && loss && log_prob,
               "policy_loss: null pointer");
  const int64_t need = (int64_t)policy_workspace(s, a->ref_scores != nullptr);
  WGBM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "policy_loss: workspace too small");
  PolicyRows p{};
  p.action = a->actions;
  p.old_log_prob = a->old_log_prob;
  p.advantage = a->advantage;
  p.weight = a->weight;
  p.ref_log_prob = a->ref_log_prob;
  p.clip_lo = 1.0 - a->clip_low;
  p.clip_hi = 1.0 + a->clip_high;
  p.log_lo = (float)std::log(p.clip_lo);
  p.log_hi = (float)std::log(p.clip_hi);
  p.kl_coef = a->kl_coef;
  p.loss = loss;
  p.log_prob = log_prob;
  p.kl = kl;
  return policy_loss(s, r, p, g, accumulate != 0, workspace, S(stream));
}

int64_t wgbm_balance_loss_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s) || balance_classes(s)) return -1;
  return (int64_t)balance_workspace(s);
}

int wgbm_balance_loss(const wgbm_scores* scores, const uint8_t* mask, int32_t top_k, float coef,
                      float* loss, int64_t* counts, float* prob, const wgbm_scores* grad,
                      int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
  ScoresView s, g{};
  TRY(view_of(scores, "scores", &s));
  if (grad) {
    TRY(view_of(grad, "grad", &g));
    TRY(same_kind(s, g, "grad"));
  }
  TRY(balance_classes(s));
  WGBM_REQUIRE(top_k >= 1 && top_k <= kMaxTopK && top_k <= s.K,
               "balance_loss: top_k must be in [1, min(%d, n_classes)], got %d", kMaxTopK, top_k);
  WGBM_REQUIRE(std::isfinite(coef), "balance_loss: coef must be finite");
  WGBM_REQUIRE(loss && counts && prob && workspace, "balance_loss: null pointer");
  WGBM_REQUIRE(workspace_bytes >= (int64_t)balance_workspace(s),
               "balance_loss: workspace too small");
  return balance_loss(s, mask, top_k, coef, BalanceOut{loss, counts, prob}, g, accumulate != 0,
                      workspace, S(stream));
}

// log2(e) / tau and 1 / tau of a temperature
static int tempered(double temperature, const char* what, float* scale, double* inv) {
  WGBM_REQUIRE(temperature >= 1e-6 && temperature <= 1e6,
               "%s: temperature must be in [1e-6, 1e6]", what);
  *inv = 1.0 / temperature;
  *scale = (float)(1.44269504088896340736 / temperature);
  return 0;
}
static int list_length(int32_t k, int32_t least, const char* what) {
  WGBM_REQUIRE(k >= least && k <= kMaxList, "%s: the lists' length must be in [%d, %d], got %d",
               what, least, kMaxList, k);
  return 0;
}
static int list_strides(int64_t stride, int64_t step, int64_t n, int32_t k, const char* what) {
  WGBM_REQUIRE((step == 1 && stride >= k) || (stride == 1 && step >= n),
               "%s: a list's strides (%lld, %lld) are neither those of rows nor of entries next to "
               "each other without overlap",
               what, (long long)stride, (long long)step);
  WGBM_REQUIRE(stride < (int64_t(1) << 40) && step < (int64_t(1) << 40),
               "%s: a list's stride is out of range", what);
  return 0;
}

int32_t wgbm_lists_tiles(const wgbm_scores* scores, int32_t grad, int32_t* span) {
  ScoresView s;
  int32_t most;
  if (view_of(scores, "scores", &s)) return -1;
  return row_tiles(s, grad != 0, span ? span : &most);
}

int64_t wgbm_class_alternatives_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s)) return -1;
  return (int64_t)lists_workspace(s, false);
}

int wgbm_class_alternatives(const wgbm_scores* scores, const int32_t* labels, int32_t top_k,
                            double temperature, int32_t* classes, float* log_prob, float* entropy,
                            float* label_log_prob, float* norm, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  ScoresView s;
  TRY(view_of(scores, "scores", &s));
  TRY(list_length(top_k, 0, "class_alternatives"));
  WGBM_REQUIRE(top_k <= s.K, "class_alternatives: top_k must be at most n_classes (%d), got %d", s.K,
               top_k);
  AltRows g{};
  TRY(tempered(temperature, "class_alternatives", &g.scale, &g.inv_tau));
  if (s.n == 0) return 0;
  WGBM_REQUIRE(entropy && norm && (top_k == 0 || (classes && log_prob)) &&
                   (!labels || label_log_prob),
               "class_alternatives: null pointer");
  const int64_t need = (int64_t)lists_workspace(s, false);
  WGBM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "class_alternatives: workspace too small");
  g.label = labels;
  g.k = top_k;
  g.classes = classes;
  g.log_prob = log_prob;
  g.entropy = entropy;
  g.label_log_prob = label_log_prob;
  g.norm = norm;
  return class_alternatives(s, g, workspace, S(stream));
}

int64_t wgbm_class_alternatives_grad_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s)) return -1;
  return (int64_t)lists_workspace(s, true);
}

int wgbm_class_alternatives_grad(const wgbm_scores* scores,
                                 const wgbm_alternatives_grad_args* a, const wgbm_scores* grad,
                                 int32_t accumulate, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  ScoresView s, o;
  TRY(view_of(scores, "scores", &s));
  TRY(view_of(grad, "grad", &o));
  TRY(same_kind(s, o, "grad"));
  WGBM_REQUIRE(a, "class_alternatives_grad: null arguments");
  TRY(list_length(a->list_length, 0, "class_alternatives_grad"));
  AltGradRows g{};
  TRY(tempered(a->temperature, "class_alternatives_grad", &g.scale, &g.inv_tau));
  if (a->list_length) {
    TRY(list_strides(a->classes_stride, a->classes_step, s.n, a->list_length,
                     "class_alternatives_grad"));
    TRY(list_strides(a->grad_stride, a->grad_step, s.n, a->list_length,
                     "class_alternatives_grad"));
  }
  if (s.n == 0) return 0;
  WGBM_REQUIRE(a->norm && (!a->labels || a->grad_label_log_prob) &&
                   (a->list_length == 0 || (a->classes && a->grad_log_prob)),
               "class_alternatives_grad: null pointer");
  const int64_t need = (int64_t)lists_workspace(s, true);
  WGBM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "class_alternatives_grad: workspace too small");
  g.norm = a->norm;
  g.label = a->labels;
  g.grad_label = a->grad_label_log_prob;
  g.classes = a->classes;
  g.class_stride = a->classes_stride;
  g.class_step = a->classes_step;
  g.grad_list = a->grad_log_prob;
  g.grad_stride = a->grad_stride;
  g.grad_step = a->grad_step;
  g.k = a->list_length;
  g.grad_entropy = a->grad_entropy;
  return class_alternatives_grad(s, g, o, accumulate != 0, workspace, S(stream));
}

int64_t wgbm_distill_loss_workspace(const wgbm_scores* scores) {
  ScoresView s;
  if (view_of(scores, "scores", &s)) return -1;
  return (int64_t)lists_workspace(s, true);
}

int wgbm_distill_loss(const wgbm_scores* scores, const wgbm_distill_args* a, float* loss,
                      const wgbm_scores* grad, int32_t accumulate, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  ScoresView s, o{};
  TRY(view_of(scores, "scores", &s));
  if (grad) {
    TRY(view_of(grad, "grad", &o));
    TRY(same_kind(s, o, "grad"));
  }
  WGBM_REQUIRE(a, "distill_loss: null arguments");
  TRY(list_length(a->list_length, 1, "distill_loss"));
  TRY(list_strides(a->classes_stride, a->classes_step, s.n, a->list_length, "distill_loss"));
  TRY(list_strides(a->logits_stride, a->logits_step, s.n, a->list_length, "distill_loss"));
  DistillRows g{};
  TRY(tempered(a->temperature, "distill_loss", &g.scale, &g.inv_tau));
  WGBM_REQUIRE(a->log_norm || !a->rest || std::isfinite(a->log_norm_all),
               "distill_loss: log_norm must be finite");
  if (s.n == 0) return 0;
  WGBM_REQUIRE(a->classes && a->logits && loss, "distill_loss: null pointer");
  const int64_t need = (int64_t)lists_workspace(s, true);
  WGBM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
               "distill_loss: workspace too small");
  g.classes = a->classes;
  g.class_stride = a->classes_stride;
  g.class_step = a->classes_step;
  g.logits = a->logits;
  g.logit_stride = a->logits_stride;
  g.logit_step = a->logits_step;
  g.k = a->list_length;
  g.rest = a->rest != 0;
  g.log_norm = a->rest ? a->log_norm : nullptr;
  g.log_norm_all = a->log_norm_all;
  g.weight = a->weight;
  g.tau = (float)a->temperature;
  g.loss = loss;
  return distill_loss(s, g, o, accumulate != 0, workspace, S(stream));
}

static PreferenceArgs preference_args(const wgbm_preference_args* a) {
  PreferenceArgs p{};
  p.log_prob = a->log_prob;
  p.ref = a->ref_log_prob;
  p.n_rows = a->n_rows;
  p.seg_start = a->sequence_start;
  p.n_seg = a->n_sequences;
  p.pairs = a->pairs;
  p.n_pairs = a->n_pairs;
  p.inc = a->incidence;
  p.inc_start = a->incidence_start;
  p.share = a->share;
  p.n_shares = a->n_shares;
  p.is_long = a->is_long;
  p.task = a->task;
  p.n_tasks = a->n_tasks;
  p.task_start = a->task_start;
  p.piece = a->piece;
  p.n_pieces = a->n_pieces;
  p.multi = a->multi;
  p.n_multi = a->n_multi;
  p.idle = a->idle;
  p.n_idle = a->n_idle;
  p.disjoint = a->disjoint != 0;
  p.weight = a->weight;
  p.beta = a->beta;
  p.smooth = a->label_smoothing;
  p.lanes = a->lanes ? a->lanes : 64;
  return p;
}

static int check_preference(const wgbm_preference_args* a) {
  WGBM_REQUIRE(a, "preference_loss: null arguments");
  WGBM_REQUIRE(a->n_rows >= 0 && a->n_rows < (int64_t(1) << 40), "preference_loss: bad n_rows");
  WGBM_REQUIRE(a->n_sequences >= 0 && a->n_sequences < (int64_t(1) << 30),
               "preference_loss: bad n_sequences");
  WGBM_REQUIRE(a->n_pairs >= 0 && a->n_pairs < (int64_t(1) << 30), "preference_loss: bad n_pairs");
  for (const int64_t size : {a->n_shares, a->n_tasks, a->n_pieces, a->n_multi, a->n_idle})
    WGBM_REQUIRE(size >= 0 && size < (int64_t(1) << 31), "preference_loss: bad table sizes");
  WGBM_REQUIRE(a->sequence_start || (a->n_sequences == a->n_rows && !a->disjoint),
               "preference_loss: without sequence_start every row is a sequence");
  WGBM_REQUIRE(std::isfinite(a->beta) && a->beta > 0.0f,
               "preference_loss: beta must be positive and finite");
  WGBM_REQUIRE(a->label_smoothing >= 0.0f && a->label_smoothing <= 0.5f,
               "preference_loss: label_smoothing must be in [0, 0.5]");
  WGBM_REQUIRE(a->lanes == 0 || a->lanes == 4 || a->lanes == 8 || a->lanes == 16 ||
                   a->lanes == 32 || a->lanes == 64,
               "preference_loss: lanes must be 4, 8, 16, 32 or 64 (or 0)");
  return 0;
}

int64_t wgbm_preference_loss_workspace(const wgbm_preference_args* a) {
  if (check_preference(a)) return -1;
  return (int64_t)preference_workspace(preference_args(a));
}

int wgbm_preference_loss(const wgbm_preference_args* a, float* loss, float* margin, float* grad,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  TRY(check_preference(a));
  PreferenceArgs p = preference_args(a);
  p.loss = loss;
  p.margin = margin;
  p.grad = grad;
  WGBM_REQUIRE(a->n_rows == 0 || a->log_prob, "preference_loss: null pointer");
  WGBM_REQUIRE(a->n_pairs == 0 || (a->pairs && loss && margin), "preference_loss: null pointer");
  WGBM_REQUIRE(a->disjoint || !a->sequence_start || a->n_rows == 0 || a->task,
               "preference_loss: sequences need their tasks");
  WGBM_REQUIRE(a->disjoint || !grad || a->n_sequences == 0 ||
                   (a->incidence_start && a->share && a->n_shares > 0 &&
                    (a->n_pairs == 0 || a->incidence) && (a->n_pieces == 0 || a->is_long)),
               "preference_loss: the gradient needs the pairs of each sequence");
  WGBM_REQUIRE((a->n_pieces == 0 || a->piece) && (a->n_multi == 0 || a->multi) &&
                   (a->n_idle == 0 || a->idle) && (a->n_tasks == 0 || a->task),
               "preference_loss: null table");
  const int64_t need = (int64_t)preference_workspace(p);
  WGBM_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
               "preference_loss: workspace too small");
  return preference_loss(p, workspace, S(stream));
}

}  // extern "C"
