"""Losses of class scores and of paired scores, with their gradients.

What a boosting round of the objectives "policy", "preference" and
"policy_preference" fits its trees to, as operators on GPU tensors: each call
returns the per-row (per-pair) losses and the gradient with respect to the
scores, computed by the HIP library through the C ABI of
``include/warpgbm_amd.h``.  The reference has no counterpart (its losses are
squared error and softmax cross entropy, warpgbm/core.py:186-214, 719).

Scores are [n rows, K classes] in float32, bfloat16 or float16, with either the
classes of a row next to each other (``scores`` contiguous, or rows with a
stride) or the rows of a class (``scores_cm.t()`` of the engine's class-major
[K, n]).  Per-row inputs are contiguous.  A score of -inf is a class that the
row may not take; a row whose scores are all -inf counts as left out.  Rows
left out (weight 0, mask false, label outside [0, K)) are not read: their
results and gradients are 0, whatever their scores hold.

Launches go on torch's current stream of the scores' device; nothing
synchronises except the construction of a :class:`PreferencePlan`.  Outputs and
working memory come from torch's allocator, so calls may be captured into a
HIP graph.  Nothing is recorded for autograd.  A gradient that is given to be
added to must not share memory with an input.  Shared memory, wrong types,
shapes, devices or layouts raise ``RuntimeError``.
"""
from __future__ import annotations

import ctypes as C
import functools
from collections import namedtuple

import numpy as np
import torch

from . import _lib

ClassLogProbs = namedtuple("ClassLogProbs", ["log_prob", "norm"])
PolicyLoss = namedtuple("PolicyLoss", ["loss", "log_prob", "kl", "grad"])
BalanceLoss = namedtuple("BalanceLoss", ["loss", "counts", "prob", "grad"])
PreferenceLoss = namedtuple("PreferenceLoss", ["loss", "margin", "grad"])

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _vector(t, name, dtype, n, device):
    """A contiguous [n] tensor of dtype on device; its address."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    if t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError(f"{name} must have shape ({n},), got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def _strides(n, K, rs, ks, name):
    """The strides of [n, K] scores as the library takes them: that of a
    dimension of one element says nothing and is replaced."""
    given = (rs, ks)
    if n == 0:
        return K, 1
    if K == 1:
        ks = 1
        if n == 1:
            rs = 1
    elif n == 1:
        rs = K if ks == 1 else 1
    if not ((ks == 1 and rs >= K) or (rs == 1 and ks >= n)):
        raise RuntimeError(f"{name} must have the classes of a row or the rows of a class next to "
                           f"each other (no overlap), got strides {given}")
    return rs, ks


def _matrix(t, name):
    """The C view of a [n, K] tensor of scores."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a torch.Tensor")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor, got device {t.device}")
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    n, K = t.shape
    if K < 1:
        raise RuntimeError(f"{name} must have at least one class")
    rs, ks = _strides(n, K, *t.stride(), name)
    return _lib.Scores(t.data_ptr(), code, n, K, rs, ks)


def _like(v, scores):
    """A new matrix of the scores' shape, type and order, and its view."""
    n, K = scores.shape
    if v.row_stride == 1 and v.class_stride != 1:
        t = torch.empty_strided((n, K), (1, max(n, 2)), dtype=scores.dtype, device=scores.device)
        return t, _lib.Scores(t.data_ptr(), v.dtype, n, K, 1, max(n, 2))
    t = torch.empty((n, K), dtype=scores.dtype, device=scores.device)
    return t, _lib.Scores(t.data_ptr(), v.dtype, n, K, K, 1)


def _lines(t):
    """A tensor's memory as (address, bytes of a line, lines, bytes from line to
    line): its rows, or the columns where those are contiguous; one line where
    it is contiguous as a whole."""
    es = t.element_size()
    if t.dim() != 2 or t.is_contiguous():
        return t.data_ptr(), t.numel() * es, 1, t.numel() * es
    (n, K), (rs, ks) = t.shape, t.stride()
    if K > 1 and ks != 1:
        n, K, rs = K, n, ks
    return t.data_ptr(), K * es, n, rs * es


def _meet(a, b):
    """Whether two tensors share memory (rows of one between rows of another do
    not)."""
    p, w, m, s = _lines(a)
    q, x, k, t = _lines(b)
    if not (w and m and x and k) or p + (m - 1) * s + w <= q or q + (k - 1) * t + x <= p:
        return False
    if m == 1 or k == 1 or s == t:
        # r: the last line of b, counted from a's i-th, that begins before that one ends
        step = t if m == 1 else s
        r = min(max((w - 1 - (q - p)) // step, 1 - m), k - 1)
        return q - p + r * step < w and q - p + r * step + x > 0
    at = p + np.arange(m) * s
    j = np.clip((at + w - 1 - q) // t, 0, k - 1) * t + q
    return bool(np.any((j < at + w) & (j + x > at)))


def _grad(grad, v, scores, with_grad, *inputs):
    """The gradient's matrix: a given one (added to), a new one, or none.  inputs:
    what else the call reads."""
    if grad is None:
        return _like(v, scores) if with_grad else (None, None)
    if not with_grad:
        raise RuntimeError("grad given, but with_grad is False")
    g = _matrix(grad, "grad")
    if grad.device != scores.device or grad.dtype != scores.dtype or grad.shape != scores.shape:
        raise RuntimeError("grad must have the shape, dtype and device of scores")
    if (g.row_stride == 1 and g.class_stride != 1) != (v.row_stride == 1 and v.class_stride != 1):
        raise RuntimeError("grad must have its rows or classes next to each other as scores has")
    # (tensors of other allocations, which most are, cost a tenth of _meet)
    whole = grad.untyped_storage()
    lo = whole.data_ptr()
    hi = lo + whole.nbytes()
    for t in (scores, *inputs):
        if t is None:
            continue
        at = t.data_ptr()
        if at >= hi or (at < lo and at + t.untyped_storage().nbytes() <= lo):
            continue
        if _meet(grad, t):
            raise RuntimeError("grad must not share the scores' memory" if t is scores
                               else "grad must not share memory with an input")
    return grad, g


class _on:
    """The scores' device as the current one (HIP launches go to the device
    that is current), at no cost where it already is."""

    def __init__(self, device):
        self.index = device.index
        self.back = None

    def __enter__(self):
        now = torch.cuda.current_device()
        if self.index is not None and now != self.index:
            torch.cuda.set_device(self.index)
            self.back = now

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)


@functools.lru_cache(maxsize=4096)
def _bytes_of(entry, dtype, n, K, class_major):
    """What a _workspace entry returns for scores of a shape and order (a call
    into the library costs more than the small losses' launches).  A refusal is
    raised, and so not kept: its message is the library's last one now."""
    v = _lib.Scores(16, dtype, n, K, 1 if class_major else K, max(n, 2) if class_major else 1)
    nbytes = getattr(_lib.load(), entry)(C.byref(v))
    if nbytes < 0:
        _lib.check(1000, entry)
    return nbytes


def _bytes(entry, v):
    return _bytes_of(entry, v.dtype, v.n_rows, v.n_classes,
                     v.row_stride == 1 and v.class_stride != 1)


def _workspace(entry, v, device):
    """Working memory of a call: (tensor or None, address, bytes)."""
    nbytes = _bytes(entry, v)
    if nbytes == 0:
        return None, None, 0
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), nbytes


def class_log_probs(scores, labels) -> ClassLogProbs:
    """Log-probability of each row's label under softmax(scores), and the norm
    [n, 2] of every row (its maximum m and log(sum exp(s - m))), which
    :func:`class_log_probs_grad` takes.  labels: int32 [n]; a row whose label is
    outside [0, K) has none and log-probability 0."""
    v = _matrix(scores, "scores")
    n, dev = scores.shape[0], scores.device
    lab = _vector(labels, "labels", torch.int32, n, dev)
    lib = _lib.load()
    with _on(dev):
        log_prob = torch.empty(n, dtype=torch.float32, device=dev)
        norm = torch.empty((n, 2), dtype=torch.float32, device=dev)
        ws, at, size = _workspace("wgbm_class_log_probs_workspace", v, dev)
        rc = lib.wgbm_class_log_probs(C.byref(v), lab, log_prob.data_ptr(), norm.data_ptr(), at,
                                      size, _lib.current_stream_ptr(dev))
    _lib.check(rc, "class_log_probs")
    return ClassLogProbs(log_prob, norm)


def class_log_probs_grad(scores, labels, norm, grad_log_prob) -> torch.Tensor:
    """Gradient with respect to the scores of sum_i grad_log_prob[i] *
    log_prob[i], in the scores' type and order."""
    v = _matrix(scores, "scores")
    n, dev = scores.shape[0], scores.device
    lab = _vector(labels, "labels", torch.int32, n, dev)
    g = _vector(grad_log_prob, "grad_log_prob", torch.float32, n, dev)
    if not isinstance(norm, torch.Tensor) or tuple(norm.shape) != (n, 2):
        raise RuntimeError(f"norm must be a ({n}, 2) tensor")
    nrm = _vector(norm.view(-1) if norm.is_contiguous() else norm, "norm", torch.float32, 2 * n,
                  dev)
    lib = _lib.load()
    with _on(dev):
        out, ov = _like(v, scores)
        rc = lib.wgbm_class_log_probs_grad(C.byref(v), lab, nrm, g, C.byref(ov),
                                           _lib.current_stream_ptr(dev))
    _lib.check(rc, "class_log_probs_grad")
    return out


def policy_loss(scores, actions, old_log_prob, advantage, *, weight=None, ref_log_prob=None,
                ref_scores=None, clip=(0.2, 0.2), kl_coef=0.0, grad=None,
                with_grad=True) -> PolicyLoss:
    """Clipped policy loss with a KL term, per row, and its gradient.

    ratio = exp(logp[action] - old_log_prob) and
    ``loss = weight * (-min(ratio * advantage, clip(ratio, 1 - clip[0], 1 +
    clip[1]) * advantage) + kl_coef * KL)``; KL is the sampled estimate
    exp(x) - x - 1 with x = ref_log_prob - logp[action], or the divergence of
    softmax(scores) from softmax(ref_scores) over all classes (ref_scores: the
    scores' shape, type and order), or absent when neither is given.  Whether a
    ratio is clipped is decided as in float64.

    actions int32 [n]; old_log_prob, advantage, weight, ref_log_prob float32
    [n].  Rows of weight 0 are left out.  ``loss``, ``log_prob`` and ``kl`` (None
    without a reference; not weighted) are float32 [n]; ``grad`` is the gradient
    of the losses' sum, added to a given ``grad``, None with
    ``with_grad=False``."""
    v = _matrix(scores, "scores")
    n, dev = scores.shape[0], scores.device
    if ref_scores is not None and ref_log_prob is not None:
        raise RuntimeError("ref_scores and ref_log_prob exclude each other")
    try:
        low, high = (float(c) for c in clip)
    except (TypeError, ValueError):
        raise RuntimeError(f"clip must be a pair of numbers, got {clip!r}") from None
    f32 = torch.float32
    rv = None
    if ref_scores is not None:
        rv = _matrix(ref_scores, "ref_scores")
        if ref_scores.device != dev:
            raise RuntimeError(f"ref_scores must be on {dev}, got {ref_scores.device}")
    args = _lib.PolicyArgs(
        _vector(actions, "actions", torch.int32, n, dev),
        _vector(old_log_prob, "old_log_prob", f32, n, dev),
        _vector(advantage, "advantage", f32, n, dev),
        _vector(weight, "weight", f32, n, dev) if weight is not None else None,
        _vector(ref_log_prob, "ref_log_prob", f32, n, dev) if ref_log_prob is not None else None,
        C.pointer(rv) if rv is not None else None, low, high, float(kl_coef))
    lib = _lib.load()
    with _on(dev):
        out, gv = _grad(grad, v, scores, with_grad, actions, old_log_prob, advantage, weight,
                        ref_log_prob, ref_scores)
        loss = torch.empty(n, dtype=f32, device=dev)
        log_prob = torch.empty(n, dtype=f32, device=dev)
        kl = None
        if ref_scores is not None or ref_log_prob is not None:
            kl = torch.empty(n, dtype=f32, device=dev)
        # (rows whose log-probabilities need none take none without reference scores)
        ws, at, size = None, None, 0
        if ref_scores is not None or _bytes("wgbm_class_log_probs_workspace", v):
            ws, at, size = _workspace("wgbm_policy_loss_workspace", v, dev)
        rc = lib.wgbm_policy_loss(
            C.byref(v), C.byref(args), loss.data_ptr(), log_prob.data_ptr(),
            kl.data_ptr() if kl is not None else None,
            C.byref(gv) if gv is not None else None, int(grad is not None), at, size,
            _lib.current_stream_ptr(dev))
    _lib.check(rc, "policy_loss")
    return PolicyLoss(loss, log_prob, kl, out)


def balance_loss(scores, *, top_k=1, mask=None, coef=1.0, grad=None,
                 with_grad=True) -> BalanceLoss:
    """How evenly rows fall on classes: ``loss = coef * K * sum_k f_k * prob_k``
    with f_k the share of class k among the top_k choices of the rows that count
    (``counts``, int64 [K]; the lower class first among equal scores) and prob_k
    the mean of softmax(scores) (float32 [K]).  The least value, coef, is that
    of even classes.

    mask: bool [n], the rows that count (None: all).  The gradient (of prob, the
    counts held constant) is added to a given ``grad``.  At most 4096 classes,
    top_k at most 8 and K."""
    v = _matrix(scores, "scores")
    n, dev = scores.shape[0], scores.device
    K = scores.shape[1]
    if not 1 <= top_k <= min(8, K):
        raise RuntimeError(f"top_k must be in [1, min(8, n_classes)], got {top_k}")
    at_mask = _vector(mask, "mask", torch.bool, n, dev) if mask is not None else None
    lib = _lib.load()
    with _on(dev):
        out, gv = _grad(grad, v, scores, with_grad, mask)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty(K, dtype=torch.int64, device=dev)
        prob = torch.empty(K, dtype=torch.float32, device=dev)
        ws, at, size = _workspace("wgbm_balance_loss_workspace", v, dev)
        rc = lib.wgbm_balance_loss(
            C.byref(v), at_mask, int(top_k), float(coef), loss.data_ptr(), counts.data_ptr(),
            prob.data_ptr(), C.byref(gv) if gv is not None else None, int(grad is not None),
            at, size, _lib.current_stream_ptr(dev))
    _lib.check(rc, "balance_loss")
    return BalanceLoss(loss, counts, prob, out)


class PreferencePlan:
    """Pairs of sequences laid out for :func:`preference_loss`, once for all
    rounds of a fit.

    pairs: integers [P, 2], (preferred, other) sequence numbers; n_rows: rows of
    the log-probabilities; segments: offsets [S + 1] of the sequences' rows
    (from 0, not descending, at most n_rows; an empty sequence has a log ratio
    of 0, rows behind the last one belong to none), or None when every row is a
    sequence of its own.  Arrays or tensors; ``device`` where they are not
    already on a GPU.  The construction checks them (it waits for the GPU), sorts
    the pairs' sides by sequence and keeps copies: 1.6 ms for 2M pairs of 1M rows on
    the GPU (2.9 from host arrays), 0.8 for 100000 sequences of 20M rows in 50000 pairs,
    where the loss takes 0.07 and 0.06.  Pairs that change in every step pay that
    each time."""

    def __init__(self, pairs, n_rows, segments=None, device=None):
        pairs = self._whole_numbers(pairs, "pairs")
        if pairs.dim() != 2 or pairs.shape[1] != 2:
            raise RuntimeError(f"pairs must have shape (P, 2), got {tuple(pairs.shape)}")
        if device is None:
            device = pairs.device if pairs.is_cuda else torch.device("cuda")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.n_rows = int(n_rows)
        if self.n_rows < 0:
            raise RuntimeError("n_rows must not be negative")
        P = pairs.shape[0]
        if P >= 1 << 30:
            raise RuntimeError("at most 2^30 - 1 pairs")
        self.n_pairs = P
        seg = None
        S = self.n_rows
        if segments is not None:
            seg = self._whole_numbers(segments, "segments").to(device=device, dtype=torch.int64)
            if seg.dim() != 1 or seg.shape[0] < 1:
                raise RuntimeError("segments must be the offsets [S + 1] of S sequences")
            S = seg.shape[0] - 1
            seg = seg.clone()
        if S >= 1 << 30:
            raise RuntimeError("at most 2^30 - 1 sequences")
        self.n_sequences = S
        self.sequence_start = seg
        pairs = pairs.to(device=device, dtype=torch.int64)
        # (each .tolist() waits for the GPU)
        if seg is not None:
            length = seg.diff()
            first, last, least, longest = torch.stack(
                [seg[0], seg[-1], length.min() if S else seg[0], length.max() if S else seg[0]]
            ).tolist()
            if first != 0 or last > self.n_rows or (S and least < 0):
                raise RuntimeError(f"segments must ascend from 0 to at most n_rows={self.n_rows}")
        if P:
            least, most = torch.stack(list(pairs.aminmax())).tolist()
            if least < 0 or most >= S:
                raise RuntimeError(f"pairs must hold sequence numbers in [0, {S})")
        self.pairs = pairs.to(torch.int32).contiguous().clone()
        self.task = self.task_start = self.piece = self.multi = self.idle = None
        self.disjoint = False
        self.workspace_bytes = None
        self.lanes = 0
        degree = self._incidences(device)
        if seg is not None:
            self._tasks(seg, length, last, longest, degree, device)
        if device.type == "cuda":  # the tables are whole for every stream that reads them
            torch.cuda.current_stream(device).synchronize()

    # most rows of a task; pairs of a sequence from which on it is summed by
    # workgroups of its own, and the pairs of one of these
    _TASK, _LONG, _PIECE = 4096, 256, 8192
    # sequences and pairs' sides, together, of a workgroup that sums the others
    _SHARE = 256

    @staticmethod
    def _cut(first, end, size):
        """The ranges [first, end) cut into pieces of size (at least one each):
        (number of the range, first, end) of every piece, and the ranges' offsets
        in that list."""
        n = ((end - first + size - 1) // size).clamp(min=1)
        start = torch.zeros(n.shape[0] + 1, dtype=torch.int64, device=n.device)
        torch.cumsum(n, 0, out=start[1:])
        of = torch.repeat_interleave(torch.arange(n.shape[0], device=n.device), n)
        at = first[of] + (torch.arange(of.shape[0], device=n.device) - start[of]) * size
        return torch.stack([of, at, torch.minimum(at + size, end[of])], 1), start

    def _incidences(self, device):
        """The numbers 2 * pair + side grouped by sequence, in pair order (a
        stable sort), the sequences in very many pairs last.  Returns the largest
        number of pairs of a sequence."""
        S = self.n_sequences
        ends = self.pairs.reshape(-1)
        degree = torch.bincount(ends, minlength=S) if S else ends.long()
        most = int(degree.max()) if S else 0
        key = ends
        if most > self._LONG:
            long = degree > self._LONG
            key = torch.where(long[ends.long()], ends.long() + S, ends.long())
        self.incidence = torch.sort(key, stable=True).indices.to(torch.int32)
        short = degree if most <= self._LONG else degree.masked_fill(long, 0)
        self.incidence_start = torch.zeros(S + 1, dtype=torch.int64, device=device)
        torch.cumsum(short, 0, out=self.incidence_start[1:])
        # a run's first sequence: the first whose number and incidences before it
        # reach the run's start
        before = self.incidence_start + torch.arange(S + 1, device=device)
        runs = (S + (2 * self.n_pairs if most <= self._LONG else int(before[-1]) - S)
                + self._SHARE - 1) // self._SHARE
        cuts = torch.arange(runs + 1, device=device) * self._SHARE
        self.share = torch.searchsorted(before, cuts).clamp(max=S)
        self.is_long = None
        if most > self._LONG:
            self.is_long = long.to(torch.uint8)
            who = long.nonzero()[:, 0]
            end = self.incidence_start[-1] + degree[who].cumsum(0)
            self.piece, start = self._cut(end - degree[who], end, self._PIECE)
            several = start.diff() > 1
            of = self.piece[:, 0]
            self.piece[:, 0] = torch.where(several[of], torch.full_like(of, -1), who[of])
            self.multi = torch.stack([who, start[:-1], start[1:]], 1)[several].contiguous()
        return most

    def _tasks(self, seg, length, last, longest, most, device):
        """The rows of every sequence, and those behind the last one, in tasks
        of :meth:`_lanes` threads."""
        S, n = self.n_sequences, self.n_rows
        self.lanes = self._lanes(last / max(S, 1), min(longest, self._TASK))
        tail = None
        if last < n:
            # (no longer than the sequences' tasks: they have as many threads)
            size = min(self._TASK, max(longest, 64))
            tail = self._cut(seg[-1:], torch.full_like(seg[-1:], n), size)[0]
            tail[:, 0] = -1
        if longest > self._TASK:
            task, self.task_start = self._cut(seg[:-1], seg[1:], self._TASK)
        else:
            task = torch.stack([torch.arange(S, device=device), seg[:-1], seg[1:]], 1)
        if most <= 1 and self.task_start is None:
            self.disjoint = True
            free = torch.diff(self.incidence_start) == 0
            free &= length > 0
            task = task[free]
        self.task = (task if tail is None else torch.cat([task, tail])).contiguous()
        if self.disjoint:
            self.idle, self.task = self.task[:, 1:].contiguous(), None

    @staticmethod
    def _lanes(mean, longest):
        """Threads of a task or pair: a row is read by four to a thread, and a wave
        of 64 for sequences of 20 rows leaves most of it idle.  Measured, us, with
        64, 32, 16, 8 and 4 threads: 50000 pairs of 200 rows 55, 54, 63, 80; of 100
        rows 44, 34, 36, 46; of 50 rows, 100000 pairs, 74, 47, 39, 44; of 20 rows,
        250000 pairs, 159, 96, 63, 59, 65; 1M sequences of 5 rows in 1M pairs 503, 278,
        174, 115, 86.
        A sequence much longer than the mean must not keep its threads busy alone
        for more than some 16 turns."""
        lanes = 4 if mean <= 10 else 8 if mean <= 32 else 16 if mean <= 64 else \
            32 if mean <= 128 else 64
        while lanes < 64 and longest > 128 * lanes:
            lanes *= 2
        return lanes

    @staticmethod
    def _whole_numbers(a, name):
        t = a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))
        if t.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"{name} must be int32 or int64, got {t.dtype}")
        return t


def _table(t):
    return (None, 0) if t is None else (t.data_ptr(), t.shape[0])


def preference_loss(log_prob, plan, *, ref_log_prob=None, weight=None, beta=1.0,
                    label_smoothing=0.0, with_grad=True) -> PreferenceLoss:
    """Loss of the plan's pairs, and its gradient with respect to log_prob.

    With U_s the sum over sequence s of log_prob - ref_log_prob, ``margin =
    U[preferred] - U[other]`` and ``loss = weight * ((1 - e) * softplus(-beta *
    margin) + e * softplus(beta * margin))``, e = label_smoothing, one per pair;
    ``grad`` is the gradient of the losses' sum (None with
    ``with_grad=False``).  log_prob, ref_log_prob: float32 [n_rows], any scores
    of rows (a scorer's without a reference give the pairwise logistic loss);
    weight: float32 [P], pairs of weight 0 are left out (margin 0)."""
    if not isinstance(plan, PreferencePlan):
        raise RuntimeError("plan must be a PreferencePlan")
    if plan.device.type != "cuda":
        raise RuntimeError(f"the plan must be on a GPU, got device {plan.device}")
    n, dev = plan.n_rows, plan.device
    f32 = torch.float32
    lp = _vector(log_prob, "log_prob", f32, n, dev)
    rp = _vector(ref_log_prob, "ref_log_prob", f32, n, dev) if ref_log_prob is not None else None
    P = plan.n_pairs
    w = _vector(weight, "weight", f32, P, dev) if weight is not None else None
    seg = plan.sequence_start
    args = _lib.PreferenceArgs(
        lp, rp, n, seg.data_ptr() if seg is not None else None, plan.n_sequences,
        plan.pairs.data_ptr(), P, plan.incidence.data_ptr(), plan.incidence_start.data_ptr(),
        plan.share.data_ptr(), plan.share.shape[0] - 1,
        plan.is_long.data_ptr() if plan.is_long is not None else None,
        *_table(plan.task), plan.task_start.data_ptr() if plan.task_start is not None else None,
        *_table(plan.piece), *_table(plan.multi), *_table(plan.idle), int(plan.disjoint), w,
        float(beta), float(label_smoothing), plan.lanes)
    lib = _lib.load()
    with _on(dev):
        loss = torch.empty(P, dtype=f32, device=dev)
        margin = torch.empty(P, dtype=f32, device=dev)
        grad = torch.empty(n, dtype=f32, device=dev) if with_grad else None
        size = plan.workspace_bytes  # (of the plan alone)
        if size is None:
            size = lib.wgbm_preference_loss_workspace(C.byref(args))
            if size < 0:
                _lib.check(1000, "preference_loss")
            plan.workspace_bytes = size
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        rc = lib.wgbm_preference_loss(C.byref(args), loss.data_ptr(), margin.data_ptr(),
                                      grad.data_ptr() if grad is not None else None,
                                      ws.data_ptr() if ws is not None else None, size,
                                      _lib.current_stream_ptr(dev))
    _lib.check(rc, "preference_loss")
    return PreferenceLoss(loss, margin, grad)
