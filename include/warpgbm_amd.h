/*
 * warpgbm_amd -- C ABI of the MI355X (gfx950) hot path of WarpGBM.
 *
 * All pointers are device pointers (HIP global memory) unless stated
 * otherwise; `stream` is a hipStream_t passed as void* (NULL = default
 * stream).  Every call is asynchronous on `stream` and returns 0 on success,
 * a hipError_t value on a HIP failure, or WGBM_EINVAL / WGBM_ENOMEM; the
 * message is available from wgbm_last_error() (thread-local).  Calls never
 * print, and they validate shapes and ranges before launching anything.
 *
 * Arithmetic contract (see the reference semantics cited at each entry):
 *  - histogram gradient sums are exact sums of the residuals quantised to
 *    q = rint(r * 2^s) with a power-of-two scale s chosen from a maximum
 *    |r| M (at most 28 significant bits per value), rounded once to
 *    float32; counts are exact.  Results do not depend on row order or
 *    launch shape.  M is taken per output block: the whole call when it has
 *    one segment and one era, else each segment / each era separately (an
 *    era or segment of small residuals keeps its precision next to another
 *    one's outliers).  Within one such block a bin's error is at most
 *    count * M * 2^-29, so a bin that holds only residuals far below M (e.g.
 *    1e-3 values in the same era as a 1e6 one) can lose them, where the
 *    reference's float32 atomics keep ~24 bits of that bin's own scale.  A
 *    non-finite residual makes its block's sums NaN.
 *  - split gains/directions are bit-identical to a sequential float32 scan.
 *  - predictions add trees in tree order (deterministic).
 */
#ifndef WARPGBM_AMD_H
#define WARPGBM_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WGBM_EINVAL 1000
#define WGBM_ENOMEM 1001

/* Library version string. */
const char* wgbm_version(void);
/* Message of the last failed call on this thread ("" if none). */
const char* wgbm_last_error(void);

/* ------------------------------------------------------------------------
 * Reference-compatible operators.  Each replaces one function bound by the
 * reference's pybind module (warpgbm/cuda/node_kernel.cpp:41-47).
 * ------------------------------------------------------------------------ */

/* compute_histogram3 -- replaces launch_histogram_kernel_cuda_configurable
 * (warpgbm/cuda/histogram_kernel.cu:63-104, bound at node_kernel.cpp:43).
 * For each position p < n_samples, row s = sample_indices[p], era
 * e = era_indices[s] (ignored when num_eras == 1), and each output feature
 * f < n_feats with code b = bin_indices[s * n_feats_master + feature_indices[f]]:
 * if 0 <= b < num_bins:  grad_hist[e,f,b] += residual[s];  hess_hist[e,f,b] += 1.
 * grad_hist / hess_hist: float32 [num_eras, n_feats, num_bins], ACCUMULATED
 * into (the caller zeroes them, as the reference's caller does).  Rows whose
 * era is outside [0, num_eras) are skipped, and so are feature indices
 * outside [0, n_feats_master) (their outputs keep their values; the
 * reference reads such codes out of bounds).  Only the selected columns are
 * histogrammed (in any order, repeats allowed).  threads_per_block and
 * rows_per_thread are accepted for signature compatibility and ignored. */
int wgbm_compute_histogram3(const int8_t* bin_indices, int64_t n_rows, int64_t n_feats_master,
                            const float* residuals, const int32_t* sample_indices,
                            int64_t n_samples, const int32_t* feature_indices, int64_t n_feats,
                            const int32_t* era_indices, int32_t num_eras, float* grad_hist,
                            float* hess_hist, int32_t num_bins, int32_t threads_per_block,
                            int32_t rows_per_thread, void* stream);

/* compute_split -- replaces launch_directional_split_kernel
 * (warpgbm/cuda/best_split_kernel.cu:61-88, bound at node_kernel.cpp:42).
 * G, H: float32 [num_eras, n_feats, num_bins]; per_era_gain and
 * per_era_direction: float32 [num_eras, n_feats, num_bins - 1], overwritten.
 * min_split_gain is accepted and unused, as in the reference kernel. */
int wgbm_compute_split(const float* G, const float* H, int32_t num_eras, int32_t n_feats,
                       int32_t num_bins, float min_split_gain, float min_child_samples,
                       float eps, float* per_era_gain, float* per_era_direction,
                       int32_t threads, void* stream);

/* custom_cuda_binner -- replaces launch_bin_column_kernel
 * (warpgbm/cuda/binner.cu:27-52, bound at node_kernel.cpp:44).
 * bin_indices[i] = number of leading edges with X[i] >= edge (NaN -> 0). */
int wgbm_custom_cuda_binner(const float* X, int64_t n, const float* bin_edges, int32_t n_edges,
                            int8_t* bin_indices, void* stream);

/* predict_forest -- replaces predict_with_forest (warpgbm/cuda/predict.cu:48-76,
 * bound at node_kernel.cpp:45).  tree_tensor: float32 [n_trees, max_nodes, 6]
 * rows (feature, bin, left, right, is_leaf, leaf_value) as written by the
 * reference's flatten_tree; out[i] += learning_rate * leaf, trees added in
 * tree order.  A walk that leaves the table contributes NaN. */
int wgbm_predict_forest(const int8_t* bin_indices, int64_t n, int64_t n_feats,
                        const float* tree_tensor, int64_t n_trees, int64_t max_nodes,
                        float learning_rate, float* out, void* stream);

/* ------------------------------------------------------------------------
 * Batched entry points (no single reference counterpart; each batches the
 * per-node / per-feature / per-tree reference calls named in its comment).
 * ------------------------------------------------------------------------ */

/* Native code layout: codes written by wgbm_bin_matrix (num_bins = n_edges
 * + 1) or wgbm_copy_prebinned (for num_bins).  Every byte of every row is in
 * [0, num_bins + 1]: a code c in [0, num_bins) is stored as c, a negative
 * code as num_bins, a code >= num_bins and every padding byte as
 * num_bins + 1.  The column-major copy keeps the raw codes. */
#define WGBM_CODES_NATIVE 1

/* Multi-segment histogram: the positions order[seg[k] .. seg[k+1]) are the
 * rows of segment k (a node; cf. the per-node sample_indices of
 * warpgbm/core.py:551-562).  codes: int8 [n_rows, stride] row-major,
 * features 0..n_feats-1; codes outside [0, num_bins) are skipped.  flags:
 * 0 for any int8 codes, or WGBM_CODES_NATIVE when the codes are in the native
 * layout for this num_bins (a faster kernel that relies on every byte being
 * in [0, num_bins + 1]).  G, H: float32 [n_seg, n_feats, num_bins],
 * accumulated into.  seg is a device int64 array [n_seg + 1]; n_pos is
 * seg[n_seg] (known to the caller). */
int wgbm_histogram_segments(const int8_t* codes, int64_t n_rows, int64_t stride, int32_t n_feats,
                            const float* residuals, const int32_t* order, const int64_t* seg,
                            int32_t n_seg, int64_t n_pos, int32_t num_bins, int32_t flags,
                            float* G, float* H, void* stream);

/* wgbm_histogram_segments that allocates nothing.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Same arguments and results as wgbm_histogram_segments; the
 * call's working memory (tile plan, partial histograms, gathered residuals)
 * is a fixed device array of WGBM_NOALLOC_SCRATCH_BYTES that every GPU the
 * library runs on holds until the process ends.  A call needing more (about
 * 4 bytes per row of a row list plus 256 KiB per histogram tile of 1000
 * features at 32 bins; the 1M x 1000 root and 16-node calls need 32 and
 * 40 MiB)
 * returns WGBM_EINVAL with the sizes in wgbm_last_error().  Calls that
 * overlap on one GPU (other streams, other threads) share the array and
 * race: serialise them. */
#define WGBM_NOALLOC_SCRATCH_BYTES (64 * 1024 * 1024)
int wgbm_histogram_segments_noalloc(const int8_t* codes, int64_t n_rows, int64_t stride,
                                    int32_t n_feats, const float* residuals, const int32_t* order,
                                    const int64_t* seg, int32_t n_seg, int64_t n_pos,
                                    int32_t num_bins, int32_t flags, float* G, float* H,
                                    void* stream);

/* Quantile edges (the torch.quantile call of warpgbm/core.py:529-534) from
 * columns already sorted ascending (NaN last): sorted float32 [n_feats, n];
 * q float32 [nq]; edges float32 [n_feats, nq]. */
int wgbm_quantile_edges(const float* sorted, int64_t n, int32_t n_feats, const float* q,
                        int32_t nq, float* edges, void* stream);

/* Quantile edges of every column of X float32 [n, n_feats] (row stride
 * x_stride elements) without sorting: the order statistics torch.quantile
 * interpolates between are found by radix selection (4 passes over an
 * order-preserving key of each column), then interpolated as above.
 * Bit-identical to torch.quantile(X[:, f], q); n <= 2^24. */
int wgbm_quantile_edges_matrix(const float* X, int64_t n, int32_t n_feats, int64_t x_stride,
                               const float* q, int32_t nq, float* edges, void* stream);

/* wgbm_quantile_edges_matrix in two steps, for a matrix that reaches the
 * device in row blocks (the staged upload of warpgbm/core.py:527-534's input,
 * whose torch.quantile call needs the whole column): each block's values are
 * staged as soon as it lands, the edges taken once every row is staged.
 *
 * stage_rows: rows [row0, row0 + rows) of the matrix, X pointing at the first
 * of them (row stride x_stride elements), into the column-major staging array
 * cols uint32 [n_feats][cols_stride] at column offset row0, and the running
 * per-column extremes kmin / kmax uint32 [n_feats] (order-preserving keys;
 * the caller sets them to 0xffffffff / 0 before the first block).  row0 is a
 * multiple of 4; cols_stride is a multiple of 32 and at least the final row
 * count n.  Blocks may be staged in any order, on one stream.
 * edges_staged: the edges of all n staged rows, bit-identical to
 * wgbm_quantile_edges_matrix on the whole matrix.  n <= 2^24. */
int wgbm_quantile_stage_rows(const float* X, int64_t rows, int32_t n_feats, int64_t x_stride,
                             int64_t row0, uint32_t* cols, int64_t cols_stride, uint32_t* kmin,
                             uint32_t* kmax, void* stream);
int wgbm_quantile_edges_staged(const uint32_t* cols, int64_t n, int32_t n_feats,
                               int64_t cols_stride, const uint32_t* kmin, const uint32_t* kmax,
                               const float* q, int32_t nq, float* edges, void* stream);

/* Batched binner (the per-feature loop of warpgbm/core.py:527-538 and
 * 908-913 in one launch).  X float32 [n, n_feats] with row stride x_stride
 * (elements); edges float32 [n_feats, n_edges] sorted per feature.  Writes
 * codes_rm int8 [n, codes_stride] in the native layout for num_bins =
 * n_edges + 1 (codes in [0, n_edges], padding bytes n_edges + 2) and, if
 * codes_cm is not NULL, codes_cm int8 [n_feats, n] (column-major copy). */
int wgbm_bin_matrix(const float* X, int64_t n, int32_t n_feats, int64_t x_stride,
                    const float* edges, int32_t n_edges, int8_t* codes_rm, int64_t codes_stride,
                    int8_t* codes_cm, void* stream);

/* Pre-binned int8 input (warpgbm/core.py:502-505): copy [n, n_feats] with
 * row stride x_stride bytes into the native row-major layout for num_bins
 * (2..127) and the raw column-major copy, as wgbm_bin_matrix.  If over_flag
 * (one int32 on the device) is not NULL it ends as 1 when some value is
 * >= num_bins, else 0: the reference's "every column max < num_bins" test
 * (core.py:501-503) made in the same pass. */
int wgbm_copy_prebinned(const int8_t* X, int64_t n, int32_t n_feats, int64_t x_stride,
                        int8_t* codes_rm, int64_t codes_stride, int8_t* codes_cm,
                        int32_t num_bins, int32_t* over_flag, void* stream);

/* Single-launch ensemble inference over heap-ordered trees (replaces the
 * per-tree launches of warpgbm/core.py:1010-1026 and the single launch of
 * :928-930).  Tree t = round * K + k, node h has children 2h+1 / 2h+2;
 * feat[t*H + h] >= 0 splits on that feature (left if code <= bin), -1 is a
 * leaf with value leaf[t*H + h].  out float32 [n, K] row-major, pre-filled
 * with the initial scores; tree contributions added round by round.  codes:
 * native layout for num_bins (negative codes go left, codes >= num_bins go
 * right, as the raw int8 compare of the reference). */
int wgbm_predict_heap(const int8_t* codes, int64_t n, int64_t codes_stride, int32_t num_bins,
                      const int32_t* feat, const int32_t* bin, const float* leaf,
                      int32_t n_rounds, int32_t K, int32_t H, int32_t max_depth,
                      float learning_rate, float* out, void* stream);

/* The kernel a wgbm_predict_heap call of these sizes takes (codes on 16
 * bytes): 0 = a thread per (row, class) over the heap tables, 1 = row blocks,
 * trees in chunks, 2 = row blocks, all trees resident in LDS, 3 = column
 * blocks; -1 for sizes out of range.  Every kernel gives the same result.  No
 * device call is made. */
int wgbm_predict_heap_path(int64_t n, int64_t codes_stride, int32_t n_rounds, int32_t K,
                           int32_t max_depth);

/* In-place row softmax of float32 [n, K] (warpgbm/metrics.py:12-15). */
int wgbm_softmax_rows(float* x, int64_t n, int32_t K, void* stream);

/* Per-era split-gain importance (replaces the per-node .item() loop of
 * warpgbm/core.py:624-627): acc float32 [num_eras, n_feats] (device, in/out)
 * gets acc[e][f] += gain[node[i] * num_eras + e] for i in [feat_start[f],
 * feat_start[f+1]), one float32 add after the other in that order.  gain:
 * float32 rows of num_eras per node; node: int64 gain-row indices grouped by
 * feature, each group in the order the reference visits the nodes (trees in
 * order, nodes depth-first, left first); feat_start: int64 [n_feats + 1]. */
int wgbm_importance_add(float* acc, int32_t n_feats, int32_t num_eras, const float* gain,
                        const int64_t* node, const int64_t* feat_start, void* stream);

/* ------------------------------------------------------------------------
 * Losses of class scores and of paired scores, with their gradients (no
 * counterpart in the reference, whose losses are squared error and softmax
 * cross entropy): what a boosting round with the engine's objective 2 fits.
 *
 * All sums are float32 (sums over the rows of a sequence and over the pairs of a
 * sequence: float64; the balance loss's over all rows: float32 for at most 256
 * rows one after the other, float64 from there), in an order that depends on the sizes
 * only: results are the same in every run.  Gradients are rounded to the
 * scores' type once.  The calls allocate nothing and may be captured into a
 * HIP graph; `workspace` (device memory, 16-byte aligned, of the bytes that the
 * matching _workspace call returns: 0, none, for most, -1 for arguments it
 * refuses) is written before it is read and must not be shared by calls that may
 * overlap.
 * ------------------------------------------------------------------------ */
#define WGBM_F32 0
#define WGBM_BF16 1
#define WGBM_F16 2

/* Scores [n_rows, n_classes] of one of the types above, or a gradient of
 * them: element (i, k) at data[i * row_stride + k * class_stride], strides in
 * elements.  Either class_stride is 1 (row-major, row_stride >= n_classes) or
 * row_stride is 1 (class-major, class_stride >= n_rows: the engine's scores).
 * n_classes at most 2^24.  A score of -inf is a class that the row may not
 * take; a row whose scores are all -inf has no class and counts as left out
 * (results 0).  NaN shows in the results of its row. */
typedef struct wgbm_scores {
  void* data;
  int32_t dtype;
  int64_t n_rows;
  int32_t n_classes;
  int64_t row_stride;
  int64_t class_stride;
} wgbm_scores;

/* log_prob[i] = log softmax(scores[i])[labels[i]], and norm [n_rows][2]: the
 * row's maximum m and log(sum exp(s - m)).  A row whose label is outside
 * [0, n_classes) has log_prob 0; a row without a class has log_prob 0 and norm
 * (-inf, 0). */
int64_t wgbm_class_log_probs_workspace(const wgbm_scores* scores);
int wgbm_class_log_probs(const wgbm_scores* scores, const int32_t* labels, float* log_prob,
                         float* norm, void* workspace, int64_t workspace_bytes, void* stream);
/* grad[i][k] = grad_log_prob[i] * (1[k = labels[i]] - softmax(scores[i])[k]);
 * 0 for rows without a label or a class and where grad_log_prob is 0.  norm as
 * written by wgbm_class_log_probs. */
int wgbm_class_log_probs_grad(const wgbm_scores* scores, const int32_t* labels, const float* norm,
                              const float* grad_log_prob, const wgbm_scores* grad, void* stream);

/* Clipped policy loss with a KL term, per row, and its gradient:
 *   ratio = exp(logp[action] - old_log_prob),
 *   loss = weight * (-min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef * KL),
 * KL = exp(x) - x - 1 with x = ref_log_prob - logp[action] (the sampled
 * estimate), or sum_k p_k (log p_k - log q_k) for q = softmax(ref_scores), or
 * absent when neither is given.  Whether a ratio is clipped is decided as in
 * float64.  weight NULL: 1.  A row of weight 0 or whose action is outside
 * [0, n_classes) is not read: loss, log_prob, kl and gradient 0.  A class of
 * probability 0 takes no part in the exact KL; one that only the reference
 * excludes makes it infinite, as do finite scores of a reference so low that the
 * sum of e^(s_k - max s) (log p_k - log q_k) passes float32's range.  kl may be
 * NULL; grad NULL: no gradient; accumulate != 0 adds to grad instead of
 * overwriting it.  grad must not overlap an input. */
typedef struct wgbm_policy_args {
  const int32_t* actions;          /* [n_rows] */
  const float* old_log_prob;       /* [n_rows] */
  const float* advantage;          /* [n_rows] */
  const float* weight;             /* [n_rows] or NULL */
  const float* ref_log_prob;       /* [n_rows] or NULL */
  const wgbm_scores* ref_scores;   /* of the scores' shape, type and order, or NULL */
  double clip_low;                 /* [0, 1] */
  double clip_high;                /* [0, inf) */
  float kl_coef;
} wgbm_policy_args;
/* (what a call with ref_scores takes; without them a call takes none where
 * wgbm_class_log_probs_workspace returns 0) */
int64_t wgbm_policy_loss_workspace(const wgbm_scores* scores);
int wgbm_policy_loss(const wgbm_scores* scores, const wgbm_policy_args* args, float* loss,
                     float* log_prob, float* kl, const wgbm_scores* grad, int32_t accumulate,
                     void* workspace, int64_t workspace_bytes, void* stream);

/* Balance loss over the n' rows with mask != 0 (mask NULL: all) that have a
 * class: counts[k] (int64) = rows with class k among their top_k classes (the
 * lower class first among equal scores; -inf and NaN are never taken), f_k =
 * counts[k] / (n' top_k), prob[k] = mean of softmax(scores)[k],
 *   *loss = coef * n_classes * sum_k f_k prob[k],
 * grad as for the policy loss, with f held constant (0 in rows left out; with
 * accumulate those keep what they hold).  n_classes at most 4096, top_k at
 * most 8.  Without a row that counts everything is 0. */
int64_t wgbm_balance_loss_workspace(const wgbm_scores* scores);
int wgbm_balance_loss(const wgbm_scores* scores, const uint8_t* mask, int32_t top_k, float coef,
                      float* loss, int64_t* counts, float* prob, const wgbm_scores* grad,
                      int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream);

/* Lists of a row's classes: at most WGBM_MAX_LIST of them.  Entry j of row i of an
 * argument is at i * stride + j * step; either step is 1 (stride >= list_length) or
 * stride is 1 (step >= n_rows).  Temperatures are in [1e-6, 1e6] and divide the scores. */
#define WGBM_MAX_LIST 64

/* The parts that the losses with lists cut a row of row-major scores into where registers
 * do not hold it whole, wgbm_class_alternatives_grad (grad != 0) or the other two: their
 * number, and in *span (or NULL) the classes of each but the last, which has 8 at least
 * and span at most.  1 and n_classes where rows are whole, -1 for scores that the losses
 * refuse.  No device call is made. */
int32_t wgbm_lists_tiles(const wgbm_scores* scores, int32_t grad, int32_t* span);

/* With p = softmax(scores[i] / temperature): the top_k classes of largest score, in
 * descending order, the lower class first among equal scores, with log p of each
 * (classes, log_prob [n_rows][top_k]; -1 and -inf where the row has fewer classes;
 * NaN is never taken); the entropy of p; log p of the row's label (labels NULL: not
 * written; 0 for a label outside [0, n_classes)); and norm [n_rows][3]: the row's
 * largest score m, log(sum exp((s - m) / temperature)) and sum p (m - s) /
 * temperature.  top_k in [0, min(WGBM_MAX_LIST, n_classes)]; with 0 classes and
 * log_prob are not written.  A row without a class has entropy 0, label log-probability
 * 0 and norm (-inf, 0, 0). */
int64_t wgbm_class_alternatives_workspace(const wgbm_scores* scores);
int wgbm_class_alternatives(const wgbm_scores* scores, const int32_t* labels, int32_t top_k,
                            double temperature, int32_t* classes, float* log_prob, float* entropy,
                            float* label_log_prob, float* norm, void* workspace,
                            int64_t workspace_bytes, void* stream);

/* Gradient with respect to the scores of
 *   grad_label_log_prob[i] log p[label] + sum_j grad_log_prob[i][j] log p[classes[i][j]]
 *     + grad_entropy[i] entropy
 * (each term absent where its pointers are NULL or list_length is 0), from the norm
 * that wgbm_class_alternatives wrote at the same temperature.  Entries outside [0,
 * n_classes) do not count; a class that is listed twice counts twice.  Rows without a
 * class, and rows whose upstream gradients are all 0, have gradient 0 (with accumulate
 * they keep what they hold).  grad as for the policy loss. */
typedef struct wgbm_alternatives_grad_args {
  const float* norm;                  /* [n_rows][3] */
  const int32_t* labels;              /* [n_rows] or NULL */
  const float* grad_label_log_prob;   /* [n_rows], with labels */
  const int32_t* classes;             /* [n_rows][list_length] */
  int64_t classes_stride;
  int64_t classes_step;
  const float* grad_log_prob;         /* [n_rows][list_length] */
  int64_t grad_stride;
  int64_t grad_step;
  int32_t list_length;                /* [0, WGBM_MAX_LIST] */
  const float* grad_entropy;          /* [n_rows] or NULL */
  double temperature;
} wgbm_alternatives_grad_args;
int64_t wgbm_class_alternatives_grad_workspace(const wgbm_scores* scores);
int wgbm_class_alternatives_grad(const wgbm_scores* scores,
                                 const wgbm_alternatives_grad_args* args, const wgbm_scores* grad,
                                 int32_t accumulate, void* workspace, int64_t workspace_bytes,
                                 void* stream);

/* Divergence of p = softmax(scores[i] / T), T = temperature, from a teacher's listed
 * classes c_j with logits l_j, per row, and its gradient:
 *   loss = weight T^2 (sum_j q_j log(q_j / p_cj) + Q log(Q / P))
 * with q_j = exp(l_j / T - log_norm[i]), Q = 1 - sum_j q_j the teacher's share of all
 * other classes and P the scores' (rest != 0), or q = softmax(l / T) over the list and
 * Q = 0 (rest == 0).  log_norm[i] is log(sum over all the teacher's classes of
 * exp(l / T)); log_norm NULL: log_norm_all for every row (0: the logits are T times
 * log-probabilities).  A Q below 2^-20 is taken as rounding, and as 0.
 * Entries outside [0, n_classes) are unused; a class that is listed again counts the
 * first time only.  Listed classes of score -inf do not count, nor does Q where no
 * other class has a score above -inf: what is left of q and Q is scaled to sum 1.
 * A row of weight 0 (weight NULL: 1) is not read; one without a class or of whose
 * list nothing counts is left out: loss and gradient 0.  grad as for the policy loss
 * (NULL: none). */
typedef struct wgbm_distill_args {
  const int32_t* classes;  /* [n_rows][list_length] */
  int64_t classes_stride;
  int64_t classes_step;
  const float* logits;     /* [n_rows][list_length] */
  int64_t logits_stride;
  int64_t logits_step;
  int32_t list_length;     /* [1, WGBM_MAX_LIST] */
  int32_t rest;
  const float* log_norm;   /* [n_rows] or NULL */
  double log_norm_all;
  const float* weight;     /* [n_rows] or NULL */
  double temperature;
} wgbm_distill_args;
int64_t wgbm_distill_loss_workspace(const wgbm_scores* scores);
int wgbm_distill_loss(const wgbm_scores* scores, const wgbm_distill_args* args, float* loss,
                      const wgbm_scores* grad, int32_t accumulate, void* workspace,
                      int64_t workspace_bytes, void* stream);

/* Preference loss of pairs of sequences of rows (paired log ratios): with
 * u_i = log_prob[i] - ref_log_prob[i] and U_s the sum of u over the rows
 * sequence_start[s] .. sequence_start[s + 1] of sequence s (none: U_s = 0),
 *   margin[p] = U[preferred] - U[other],
 *   loss[p] = weight[p] * ((1 - e) log(1 + exp(-beta margin)) + e log(1 + exp(beta margin))),
 * e = label_smoothing, and grad[i] = sum over the pairs that hold i's sequence.
 * Rows behind the last sequence have gradient 0.  Without sequence_start every
 * row is a sequence.  A pair of weight 0 is not read.  grad NULL: no gradient.
 *
 * The tables (device memory) lay the pairs and sequences out for the kernels;
 * warpgbm_amd.losses.PreferencePlan builds them, once for all calls, and the
 * call takes them as valid:
 *  pairs [n_pairs][2]: sequence numbers 0 .. n_sequences - 1;
 *  incidence [2 n_pairs]: the numbers 2 * pair + side (0 preferred, 1 other)
 *    grouped by sequence, the sequences in very many pairs (`long`) last;
 *  incidence_start [n_sequences + 1]: each sequence's range of them, empty for
 *    the long ones;
 *  share [n_shares + 1]: sequence numbers that cut the sequences into runs with
 *    at most 256 sequences and 512 of the incidences of incidence_start;
 *  is_long [n_sequences]: 1 for the long ones (NULL: none);
 *  piece [n_pieces][3]: (sequence, or -1 where it has several pieces; first and
 *    end incidence) of the long sequences; multi [n_multi][3]: (sequence, first
 *    and end piece) of those with several;
 *  task [n_tasks][3], with sequence_start only: (sequence; first and end row),
 *    every row of every sequence in one task, in sequence order, at least one a
 *    sequence, then the rows behind the last one with sequence -1; task_start
 *    [n_sequences + 1]: each sequence's tasks, NULL where each has one;
 *  disjoint != 0: each sequence has one task and at most one pair (none of the
 *    tables above is read but pairs); idle [n_idle][2] then holds the row ranges
 *    that no pair covers. */
typedef struct wgbm_preference_args {
  const float* log_prob;            /* [n_rows] */
  const float* ref_log_prob;        /* [n_rows] or NULL (0) */
  int64_t n_rows;
  const int64_t* sequence_start;    /* [n_sequences + 1] or NULL */
  int64_t n_sequences;
  const int32_t* pairs;
  int64_t n_pairs;
  const int32_t* incidence;
  const int64_t* incidence_start;
  const int64_t* share;
  int64_t n_shares;
  const uint8_t* is_long;
  const int64_t* task;
  int64_t n_tasks;
  const int64_t* task_start;
  const int64_t* piece;
  int64_t n_pieces;
  const int64_t* multi;
  int64_t n_multi;
  const int64_t* idle;
  int64_t n_idle;
  int32_t disjoint;
  const float* weight;              /* [n_pairs] or NULL (1) */
  float beta;
  float label_smoothing;            /* [0, 0.5] */
  int32_t lanes;                    /* threads of a task, or of a pair where disjoint:
                                       4, 8, 16, 32 or 64 (0: 64); results may differ in the
                                       last bits of the float64 sums */
} wgbm_preference_args;
int64_t wgbm_preference_loss_workspace(const wgbm_preference_args* args);
int wgbm_preference_loss(const wgbm_preference_args* args, float* loss, float* margin, float* grad,
                         void* workspace, int64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Level-wise boosting engine (the caller of the four operators:
 * warpgbm/core.py grow_forest 692-744, grow_forest_multiclass 746-818,
 * grow_tree 597-658).
 * ------------------------------------------------------------------------ */
typedef struct wgbm_engine wgbm_engine;

typedef struct wgbm_engine_config {
  int64_t n_rows;
  int32_t n_feats;
  int64_t codes_stride;       /* multiple of 16, >= n_feats */
  int32_t num_bins;           /* 2..127 */
  int32_t num_eras;
  int32_t max_depth;
  int32_t n_trees;            /* 1 (regression), K (softmax), any (gradients) */
  int32_t objective;          /* 0 regression, 1 softmax, 2 gradients given */
  float min_child_weight;
  float min_split_gain;
  float l2_reg;
  float learning_rate;
  const int8_t* codes_rm;     /* [n_rows, codes_stride], native layout */
  const int8_t* codes_cm;     /* [n_feats, n_rows] */
  const int32_t* root_order;  /* [n_rows] row ids sorted by era, ascending inside */
  const int64_t* era_start;   /* [num_eras + 1] */
  /* device bytes for the per-level split buffers (level histograms, staged
   * per-era gains, era-block sums, criteria); 0 = 4 GiB.  A depth with more
   * (tree, node)s than fit is processed in chunks of nodes, each histogrammed
   * directly; the trees do not depend on it.  max_depth is limited only by
   * int32 node and segment numbering (n_trees * 2^max_depth * num_eras <
   * 2^31) and by the device memory of the per-node bookkeeping, which
   * wgbm_engine_create checks against the free memory. */
  int64_t level_bytes;
} wgbm_engine_config;

/* Heap-ordered record of the trees grown in one round; H = 2^(max_depth+1)-1.
 * feat: split feature, -1 leaf, -2 absent; count: rows in the node;
 * gain: per-era gains of the chosen split [n_trees, H, num_eras]. */
typedef struct wgbm_tree_record {
  int32_t* feat;   /* [n_trees, H] */
  int32_t* bin;    /* [n_trees, H] */
  float* leaf;     /* [n_trees, H] */
  int64_t* count;  /* [n_trees, H] */
  float* gain;     /* [n_trees, H, num_eras] */
  int32_t H;
} wgbm_tree_record;

int wgbm_engine_create(wgbm_engine** out, const wgbm_engine_config* cfg);
/* One boosting round.  target: float32 y [n_rows] (regression) or int32
 * labels [n_rows] (softmax) or float32 gradients [n_trees, n_rows] of a loss,
 * to whose negative the trees are fitted (objective 2); pred: float32 [n_rows]
 * (regression) or class-major [n_trees, n_rows] (softmax, gradients: the
 * scores of class k are row k, so each class tree's leaf updates stay inside
 * one row), updated in place; feat_sel: int32 [n_sel] features of this round's trees (colsample_bytree
 * subset, local order). */
int wgbm_engine_round(wgbm_engine* eng, const void* target, float* pred, const int32_t* feat_sel,
                      int32_t n_sel, const wgbm_tree_record* rec, void* stream);
/* Tuning knobs: key 1 = histogram tile rows (0 = automatic); key 2 = codes
 * read by the era path when num_bins <= 7 (0 = the int8 codes, 1 = a
 * pair-code copy, one byte per feature pair; default 1); key 3 = the
 * per-level node scan of one-era fits (1 = a thread per node, default; 0 = a
 * wave per node); key 4 = one-era split search and leaf / record step (1 =
 * one fused launch, default; 0 = two launches); key 5 = the one-era root
 * (1 = its positions and totals in one launch and the root level's
 * histogram tiles planned once per engine, default; 0 = a root partition
 * pass, block scan and totals launch, and a plan per round); key 6 = the
 * one-era split levels' partition (1 = one pass that routes and places every
 * row, each node's children filled from its two ends, on levels of at most
 * 1024 (tree, node)s, default; 0 = route, block prefix and a stable
 * scatter); key 7 = the era levels' partition (1 = the route reserves each
 * (node, era) segment's child ranges and leaves its sums for the node scan,
 * no block prefix, default; 0 = route, block prefix, node scan, scatter);
 * key 8 = one-era rounds of at most 20480 rows and 512 (feature, tree)s (1 =
 * one launch per level where that is the faster, default; 0 = the level chain;
 * setting any of keys 1 to 7 takes the level chain too, whose parts they choose).
 * Keys 1 and 2 size the era path's tile buffers again (a synchronisation and an
 * allocation; without room the levels go without tiles).
 * Set before the first round; every setting grows the same trees. */
int wgbm_engine_set_tuning(wgbm_engine* eng, int32_t key, int64_t value);
void wgbm_engine_destroy(wgbm_engine* eng);

/* ------------------------------------------------------------------------
 * Instrumentation: HIP-event timing of selected kernels (tags
 * "hist_tiles", "engine_hist_tiles"; in mode 1 also the engine's era path
 * per depth d: "des_rows_L<d>", the per-era gain kernel, and "des_sums_L<d>",
 * the era sums, pick and finish).  mode 0 off; 1: events recorded on the
 * kernel's stream right before and after its launch; 2: events attached to
 * the kernel's dispatch (hipExtLaunchKernel).  Reading synchronises the
 * events.
 * ------------------------------------------------------------------------ */
void wgbm_timer_enable(int32_t mode);
int wgbm_timer_read(const char* tag, double* total_ms, int64_t* count);
void wgbm_timer_reset(void);
/* Rate of 64-bit LDS atomic adds (per second, whole GPU) in the tile
 * histogram's LDS layout with synthetic bins and no global traffic: the
 * ceiling of the histogram kernel's LDS stage.  Synchronises `stream`. */
int wgbm_probe_lds_atomics(int32_t blocks, int32_t iters, double* ops_per_s, void* stream);
/* Achievable HBM read rate (bytes per second, whole GPU): `iters` launches
 * that each stream the device buffer `buf` (16-byte aligned, `bytes` long;
 * the last bytes % 16 are not read) once with 16-byte loads and no other
 * memory traffic: the practical ceiling of a read-bound kernel.  No
 * counterpart in the reference.  Synchronises `stream`. */
int wgbm_probe_hbm_read(const void* buf, int64_t bytes, int32_t iters, double* bytes_per_s,
                        void* stream);
/* Free the library's scratch buffers (all devices / streams). */
void wgbm_release_scratch(void);

#ifdef __cplusplus
}
#endif

#endif /* WARPGBM_AMD_H */
