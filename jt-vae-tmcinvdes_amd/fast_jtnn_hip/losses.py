"""Log-probabilities of chosen labels under rows of logits, and the fine-tuning losses built on them.

The training losses of the model are teacher-forced cross entropies (``jtnn_dec.py``, ``segment_cross_entropy``).  What
comes after them - scoring molecules (or any token sequences) under a model, learning from pairs of which one is
preferred, learning from rewards of sampled ones - needs the log-probability of every chosen label:

* ``token_log_probs(logits, labels)``: one value per row.
* ``sequence_log_probs(logits, labels, plan)``: their sums per sequence.
* ``preference_loss(...)``: paired log ratios against a reference model.
* ``policy_loss(...)``: clipped probability ratios with a KL term.

Logits are [N, V] in fp32, fp16 or bf16, rows at any stride; labels are [N] int32 or int64, a negative label leaves its
row out (log-probability 0, gradient 0, its logits are never read).  A label >= V gives NaN.  Gradients come back in the
logits' type and layout.  Statistics are fp32, sums over a sequence fp64; no atomics, so results repeat bit for bit.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _capi as K


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor  # 0-d, differentiable
    log_probs: torch.Tensor  # [n_seq] log-probability of every sequence, ``other_log_probs`` included (detached)
    margins: torch.Tensor  # [n_pairs] beta times the difference of the two log ratios (detached)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor  # 0-d, differentiable
    log_probs: torch.Tensor  # [N] (detached)
    kl: torch.Tensor  # 0-d: weighted sum of the KL estimates (detached)
    clipped: torch.Tensor  # 0-d: summed weight of the rows whose ratio was clipped (detached)


class SequencePlan:
    """Which sequence every row of a batch belongs to, checked on the host and uploaded once.

    ``row_seq``: host integers [N], sequence of every row, -1 for rows that belong to none; rows of a sequence need not
    be consecutive (the tree decoder orders its rows by decoding step).  ``pairs``: host integers [P, 2], (preferred,
    other) sequence of every pair; a sequence may appear in several pairs."""

    def __init__(self, row_seq, n_seq, device, pairs=None):
        row_seq = np.ascontiguousarray(_host(row_seq))
        if row_seq.ndim != 1 or row_seq.dtype.kind not in "iu":
            raise ValueError("row_seq: a list of integers is expected, got %s %s" % (row_seq.dtype, row_seq.shape))
        n_seq = int(n_seq)
        if n_seq < 0:
            raise ValueError("n_seq is %d" % n_seq)
        if row_seq.size and (int(row_seq.min()) < -1 or int(row_seq.max()) >= n_seq):
            raise IndexError("row_seq outside [-1, %d)" % n_seq)
        self.n_rows, self.n_seq = int(row_seq.size), n_seq
        row_seq = row_seq.astype(np.int32)
        # rows without a sequence get the extra key n_seq, whose group is left out
        keyptr, order = K.prep_group_by_key(np.where(row_seq < 0, n_seq, row_seq), n_seq + 1)
        self.n_pairs = None
        if pairs is not None:
            pairs = np.ascontiguousarray(_host(pairs))
            if pairs.size == 0:
                pairs = np.zeros((0, 2), dtype=np.int32)
            if pairs.ndim != 2 or pairs.shape[1] != 2 or pairs.dtype.kind not in "iu":
                raise ValueError("pairs: integers [P, 2] are expected, got %s %s" % (pairs.dtype, pairs.shape))
            if pairs.size and (int(pairs.min()) < 0 or int(pairs.max()) >= n_seq):
                raise IndexError("pairs name sequences outside [0, %d)" % n_seq)
            self.n_pairs = int(pairs.shape[0])
            pairs = pairs.astype(np.int32).reshape(-1)
            seq_ptr, seq_pairs = K.prep_group_by_key(pairs, max(n_seq, 1))  # entry 2 p + side
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("SequencePlan lives on an MI355X only (got %s); there is no CPU path" % device)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
        device = self.device
        parts = [row_seq, keyptr[:n_seq + 1], order]
        if self.n_pairs is not None:
            parts += [pairs, seq_ptr, seq_pairs]
        ends = np.cumsum([0] + [-(-max(a.size, 1) // 4) * 4 for a in parts])  # tables start at 16-byte boundaries
        host = np.zeros(int(ends[-1]), dtype=np.int32)
        for a, at in zip(parts, ends):
            host[at:at + a.size] = a
        with torch.cuda.device(device):
            # one copy that is over when the constructor returns: the plan may be used on any stream
            self._store = torch.from_numpy(host).to(device)
            self._stream = K.stream_ptr()
        views = [self._store[at:at + max(a.size, 1)] for a, at in zip(parts, ends)]
        self.row_seq, self.seq_ptr, self.seq_rows = views[:3]
        self.pairs, self.pair_ptr, self.pair_list = views[3:] if self.n_pairs is not None else (None,) * 3

    def on_current_stream(self):
        """Tells the allocator when the tables are read on another stream than the one they were made on."""
        if K.stream_ptr() != self._stream:
            self._store.record_stream(torch.cuda.current_stream(self.device))


def _host(a):
    return a.detach().cpu().numpy() if isinstance(a, torch.Tensor) else np.asarray(a)


def _check(what, logits, labels):
    """Refuses what the kernels cannot take."""
    if not isinstance(logits, torch.Tensor) or not isinstance(labels, torch.Tensor):
        raise TypeError("%s: tensors are expected" % what)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("%s: logits [N, V] with V > 0 are expected, got %s" % (what, tuple(logits.shape)))
    if logits.dtype not in K.DTYPE_CODE:
        raise TypeError("%s: logits in float32, float16 or bfloat16 are expected, got %s" % (what, logits.dtype))
    if labels.dim() != 1 or labels.shape[0] != logits.shape[0]:
        raise ValueError("%s: %s labels for %d rows" % (what, tuple(labels.shape), logits.shape[0]))
    if labels.dtype not in (torch.int32, torch.int64):
        raise TypeError("%s: int32 or int64 labels are expected, got %s" % (what, labels.dtype))
    if logits.shape[0] >= 2 ** 31 or logits.shape[1] >= 2 ** 31:
        raise ValueError("%s: logits %s exceed 32-bit row or column numbers" % (what, tuple(logits.shape)))


def _on_device(what, logits, **others):
    """The last check of every entry point: all inputs on the logits' GPU."""
    if logits.device.type != "cuda":
        raise RuntimeError("fast_jtnn_hip.%s runs on an MI355X only (logits are on %s); there is no CPU path"
                           % (what, logits.device))
    for name, t in others.items():
        if t is not None and t.device != logits.device:
            raise RuntimeError("%s: logits are on %s, %s on %s" % (what, logits.device, name, t.device))


def _check_plan(what, plan, logits, pairs=False):
    if not isinstance(plan, SequencePlan):
        raise TypeError("%s: a SequencePlan is expected, got %s" % (what, type(plan).__name__))
    if plan.n_rows != logits.shape[0]:
        raise ValueError("%s: the plan describes %d rows, the logits have %d" % (what, plan.n_rows, logits.shape[0]))
    if pairs and plan.n_pairs is None:
        raise ValueError("%s: the plan was built without pairs" % what)


def _check_vector(what, name, t, n):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s: %s [%d] is expected, got %s" % (what, name, n, getattr(t, "shape", type(t).__name__)))
    if not t.is_floating_point():
        raise TypeError("%s: %s must be floating point, got %s" % (what, name, t.dtype))


def _fp32(t):
    """A per-row or per-sequence input as the kernels read it (None stays None)."""
    return None if t is None else t.detach().float().contiguous()


def _number(what, name, v, lo, hi=float("inf")):
    v = float(v)
    if not (lo <= v <= hi) or v in (float("inf"), float("-inf")):
        raise ValueError("%s: %s = %r is outside [%g, %g]" % (what, name, v, lo, hi))
    return v


def _rows(logits):
    """The logits as rows of unit column stride (a copy only where columns are strided or rows overlap)."""
    x = logits.detach()
    n, v = x.shape
    if (v > 1 and x.stride(1) != 1) or (n > 1 and x.stride(0) < v):
        x = x.contiguous()
    return x


def _arg(x, labels):
    """(jtvae_logits_t, tensors to keep alive until the launch is enqueued)."""
    labels = labels.detach().contiguous()
    n, v = x.shape
    ld = max(x.stride(0), v) if n > 1 else v
    return K.logits_arg(x.data_ptr(), ld, n, v, K.DTYPE_CODE[x.dtype], labels.data_ptr(),
                        64 if labels.dtype == torch.int64 else 32), labels


def _like_rows(x):
    """(uninitialised gradient in the layout of ``x``, its leading dimension): the few padding columns of the package's
    row buffers are kept - the kernel writes them as zero - so that the products that follow take it without a copy."""
    ld = _like_ld(x)
    return torch.empty((x.shape[0], ld), dtype=x.dtype, device=x.device)[:, :x.shape[1]], ld


def _like_ld(x):
    n, v = x.shape
    ld = x.stride(0) if n > 1 else v
    return ld if v <= ld < v + 64 else v


def _logits_grad(x, labels, owner, stats, coef, upstream):
    d, ld = _like_rows(x)
    if coef.numel() == 0:  # no sequences, so no row counts: an address that is never read
        coef = coef.new_zeros(1)
    g, keep = _arg(x, labels)
    K.label_log_probs_bwd(g, K.ptr(owner), stats.data_ptr(), coef.data_ptr(), K.ptr(upstream), d.data_ptr(), ld, ld)
    return d


def _stats(x, labels, owner, want32, want64):
    n, dev = x.shape[0], x.device
    stats = torch.empty((n, 2), dtype=torch.float32, device=dev)
    lp32 = torch.empty((n,), dtype=torch.float32, device=dev) if want32 else None
    lp64 = torch.empty((max(n, 1),), dtype=torch.float64, device=dev) if want64 else None
    g, keep = _arg(x, labels)
    K.label_log_probs(g, K.ptr(owner), stats.data_ptr(), K.ptr(lp32), K.ptr(lp64))
    return stats, lp32, lp64


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        x = _rows(logits)
        with torch.cuda.device(x.device):
            stats, lp, _ = _stats(x, labels, None, True, False)
        ctx.save_for_backward(x if x.data_ptr() != logits.data_ptr() else logits, labels, stats)
        return lp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp):
        logits, labels, stats = ctx.saved_tensors
        with torch.cuda.device(logits.device):
            coef = dlp.detach().float().contiguous()
            return _logits_grad(logits.detach(), labels, None, stats, coef, None), None


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """[N] fp32: log softmax(logits[i])[labels[i]], 0 where the label is negative.  Differentiable in ``logits``."""
    _check("token_log_probs", logits, labels)
    _on_device("token_log_probs", logits, labels=labels)
    return _TokenLogProbs.apply(logits, labels)


class _SequenceLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, plan):
        x = _rows(logits)
        with torch.cuda.device(x.device):
            plan.on_current_stream()
            stats, _, lp64 = _stats(x, labels, plan.row_seq, False, True)
            sums = torch.empty((plan.n_seq,), dtype=torch.float32, device=x.device)
            K.sequence_sums(lp64.data_ptr(), plan.seq_ptr.data_ptr(), plan.seq_rows.data_ptr(), plan.n_seq, None, None,
                            sums.data_ptr(), n_rows=x.shape[0])
        ctx.save_for_backward(x if x.data_ptr() != logits.data_ptr() else logits, labels, stats)
        ctx.plan = plan
        return sums

    @staticmethod
    @once_differentiable
    def backward(ctx, dsums):
        logits, labels, stats = ctx.saved_tensors
        with torch.cuda.device(logits.device):
            coef = dsums.detach().float().contiguous()
            return _logits_grad(logits.detach(), labels, ctx.plan.row_seq, stats, coef, None), None, None


def sequence_log_probs(logits: torch.Tensor, labels: torch.Tensor, plan: SequencePlan) -> torch.Tensor:
    """[plan.n_seq] fp32: sum of the rows' label log-probabilities per sequence (0 for a sequence without rows).
    Differentiable in ``logits``."""
    _check("sequence_log_probs", logits, labels)
    _check_plan("sequence_log_probs", plan, logits)
    _on_device("sequence_log_probs", logits, labels=labels, plan=plan)
    return _SequenceLogProbs.apply(logits, labels, plan)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, other, labels, plan, ref, beta, smoothing, scale):
        x, dev, S, P = _rows(logits), logits.device, plan.n_seq, plan.n_pairs
        with torch.cuda.device(dev):
            plan.on_current_stream()
            oth, ref = _fp32(other), _fp32(ref)
            stats, _, lp64 = _stats(x, labels, plan.row_seq, False, True)
            sums64 = torch.empty((S,), dtype=torch.float64, device=dev)
            dmargin = torch.empty((P,), dtype=torch.float64, device=dev)
            sums, coef = (torch.empty((S,), dtype=torch.float32, device=dev) for _ in range(2))
            margins = torch.empty((P,), dtype=torch.float32, device=dev)
            loss = torch.empty((), dtype=torch.float32, device=dev)
            K.sequence_sums(lp64.data_ptr(), plan.seq_ptr.data_ptr(), plan.seq_rows.data_ptr(), S, K.ptr(oth),
                            sums64.data_ptr(), sums.data_ptr(), n_rows=x.shape[0])
            K.preference_pairs(sums64.data_ptr(), ref.data_ptr(), plan.pairs.data_ptr(), P, plan.pair_ptr.data_ptr(),
                               plan.pair_list.data_ptr(), S, beta, smoothing, scale, loss.data_ptr(),
                               margins.data_ptr(), dmargin.data_ptr(), coef.data_ptr())
        ctx.save_for_backward(x if x.data_ptr() != logits.data_ptr() else logits, labels, stats, coef)
        ctx.plan, ctx.other_dtype = plan, None if other is None else other.dtype
        ctx.mark_non_differentiable(sums, margins)
        ctx.set_materialize_grads(False)
        return loss, sums, margins

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 8
        logits, labels, stats, coef = ctx.saved_tensors
        d = dother = None
        with torch.cuda.device(logits.device):
            up = dloss.detach().float().contiguous()
            if ctx.needs_input_grad[0]:
                d = _logits_grad(logits.detach(), labels, ctx.plan.row_seq, stats, coef, up)
            if ctx.needs_input_grad[1]:
                dother = (coef * up).to(ctx.other_dtype)
        return d, dother, None, None, None, None, None, None


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, plan: SequencePlan, ref_log_probs: torch.Tensor,
                    beta: float = 0.1, label_smoothing: float = 0.0, other_log_probs: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> PreferenceLoss:
    """Paired log ratios: with S_q the log-probability of sequence q (plus ``other_log_probs[q]``, what the sequence's
    probability owes to decisions outside these logits, e.g. the stop predictions of the tree decoder) and

        D_p = beta ((S - ref_log_probs)[preferred] - (S - ref_log_probs)[other]),

    the loss is ``scale * sum_p -(1 - label_smoothing) log sigmoid(D_p) - label_smoothing log sigmoid(-D_p)``; ``scale``
    defaults to one over the number of pairs.  Differentiable in ``logits`` and ``other_log_probs``."""
    what = "preference_loss"
    _check(what, logits, labels)
    _check_plan(what, plan, logits, pairs=True)
    _check_vector(what, "ref_log_probs", ref_log_probs, plan.n_seq)
    if other_log_probs is not None:
        _check_vector(what, "other_log_probs", other_log_probs, plan.n_seq)
    beta = _number(what, "beta", beta, 0.0)
    smoothing = _number(what, "label_smoothing", label_smoothing, 0.0, 1.0)
    scale = 1.0 / max(plan.n_pairs, 1) if scale is None else _number(what, "scale", scale, -float("inf"))
    _on_device(what, logits, labels=labels, plan=plan, ref_log_probs=ref_log_probs, other_log_probs=other_log_probs)
    return PreferenceLoss(*_PreferenceLoss.apply(logits, other_log_probs, labels, plan, ref_log_probs, beta, smoothing,
                                                 scale))


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, old, adv, ref, weights, lo, hi, kl_coef, scale):
        x, dev, n = _rows(logits), logits.device, logits.shape[0]
        with torch.cuda.device(dev):
            old, adv, ref, weights = (_fp32(t) for t in (old, adv, ref, weights))
            stats = torch.empty((n, 2), dtype=torch.float32, device=dev)
            lp, coef = (torch.empty((n,), dtype=torch.float32, device=dev) for _ in range(2))
            loss, kl, clipped = (torch.empty((), dtype=torch.float32, device=dev) for _ in range(3))
            nbytes = K.policy_loss_workspace_bytes(n)
            ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
            g, keep = _arg(x, labels)
            policy = K.Policy(old.data_ptr(), adv.data_ptr(), K.ptr(ref), K.ptr(weights), lo, hi, kl_coef, scale)
            # a row's coefficient depends on that row alone: its gradient is made while the row is in registers
            d, ld = _like_rows(x) if ctx.needs_input_grad[0] else (None, 0)
            K.policy_loss(g, policy, stats.data_ptr(), lp.data_ptr(), coef.data_ptr(), loss.data_ptr(), kl.data_ptr(),
                          clipped.data_ptr(), K.ptr(d), ld, ld, ws.data_ptr(), nbytes)
        ctx.save_for_backward(x if x.data_ptr() != logits.data_ptr() else logits, labels, stats, coef)
        ctx.gradient = d
        ctx.mark_non_differentiable(lp, kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, lp, kl, clipped

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 10
        logits, labels, stats, coef = ctx.saved_tensors
        d, ctx.gradient = ctx.gradient, None
        with torch.cuda.device(logits.device):
            up = dloss.detach().float().contiguous()
            x = logits.detach()
            if d is None:  # a second pass through the graph: the first one's gradient has been given away
                d = _logits_grad(x, labels, None, stats, coef, up)
            else:  # stands as it is where the upstream factor is 1, which only the device knows
                g, keep = _arg(x, labels)
                ld = _like_ld(x)
                K.label_log_probs_bwd(g, None, stats.data_ptr(), coef.data_ptr(), up.data_ptr(), d.data_ptr(), ld, ld,
                                      unless_one=True)
        return (d,) + (None,) * 9


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor,
                ref_log_probs: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None, clip=0.2,
                kl_coef: float = 0.0, scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss of sampled labels: with r = exp(lp - old_log_probs), A the advantages and
    k = exp(ref - lp) - (ref - lp) - 1 (a never negative estimate of the KL divergence from the reference model),

        loss = scale * sum over rows of weights (kl_coef k - min(r A, min(max(r, 1 - clip), 1 + clip) A)).

    ``clip`` is one number or (low, high); without ``ref_log_probs`` there is no KL term (``kl_coef`` must be 0).  Rows
    with a negative label do not count; ``weights`` (default 1) carry masks and means.  Differentiable in ``logits``."""
    what = "policy_loss"
    _check(what, logits, labels)
    given = dict(old_log_probs=old_log_probs, advantages=advantages, ref_log_probs=ref_log_probs, weights=weights)
    for name, t in given.items():
        if t is not None or name in ("old_log_probs", "advantages"):
            _check_vector(what, name, t, logits.shape[0])
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    lo, hi = _number(what, "clip", lo, 0.0, 1.0), _number(what, "clip", hi, 0.0)
    kl_coef = _number(what, "kl_coef", kl_coef, 0.0)
    scale = _number(what, "scale", scale, -float("inf"))
    if kl_coef and ref_log_probs is None:
        raise ValueError("%s: kl_coef needs ref_log_probs" % what)
    _on_device(what, logits, labels=labels, **given)
    return PolicyLoss(*_PolicyLoss.apply(logits, labels, old_log_probs, advantages, ref_log_probs, weights, lo, hi,
                                         kl_coef, scale))
