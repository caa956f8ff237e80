"""Log-probabilities of chosen labels under rows of logits, and the fine-tuning losses built on them.

The training losses of the model are teacher-forced cross entropies (``jtnn_dec.py``, ``segment_cross_entropy``).  What
comes after them - scoring molecules (or any token sequences) under a model, learning from pairs of which one is
preferred, learning from rewards of sampled ones - needs the log-probability of every chosen label:

* ``token_log_probs(logits, labels)``: one value per row.
* ``sequence_log_probs(logits, labels, plan)``: their sums per sequence.
* ``preference_loss(...)``: paired log ratios against a reference model.
* ``policy_loss(...)``: clipped probability ratios with a KL term.

Logits are [N, V] in fp32, fp16 or bf16, rows at any stride; labels are [N] int32 or int64, a negative label leaves its
row out (log-probability 0, gradient 0, its logits are never read).  A label >= V gives NaN.  Where the upstream gradient
or a weight is zero the gradient is zero, whatever the row holds.  Gradients come back in the logits' type and layout, and
are differentiable once, in reverse mode only.  Statistics are fp32, sums over a sequence fp64; no atomics, so
results repeat bit for bit.  Every call only enqueues work on the current stream and may be captured; a captured plan
lives as long as the graph.  Making a ``SequencePlan`` is not such a call: its tables are grouped on the host and copied
with a wait.
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi as K


def _differentiable_once(backward):
    """torch's ``once_differentiable``, entered only where a graph of the backward pass is being built: the backward
    runs on autograd's own thread, where every Python call counts."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def call(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return call


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
        row_seq, n_seq = _numbers("rows", _host(row_seq), 1), int(n_seq)
        if n_seq >= 2 ** 31 - 1:
            raise ValueError("%d sequences exceed 32-bit numbers" % n_seq)
        if row_seq.shape == (0,):  # an empty list has no type of its own
            row_seq = row_seq.astype(np.int32)
        if row_seq.ndim != 1 or row_seq.dtype.kind not in "iu":
            raise ValueError("row_seq: a list of integers is expected, got %s %s" % (row_seq.dtype, row_seq.shape))
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
            pairs = _numbers("pairs", _host(pairs), 2)  # every pair has two entries in the tables
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
        self.arg = K.Sequences(self.row_seq.data_ptr(), self.seq_ptr.data_ptr(), self.seq_rows.data_ptr(), n_seq,
                               K.ptr(self.pairs), self.n_pairs or 0, K.ptr(self.pair_ptr), K.ptr(self.pair_list))

    def on_current_stream(self):
        """Tells the allocator when the tables are read on another stream than the one they were made on."""
        if K.stream_ptr() != self._stream:
            self._store.record_stream(torch.cuda.current_stream(self.device))


def _host(a):
    return a.detach().cpu().numpy() if isinstance(a, torch.Tensor) else np.asarray(a)


def _numbers(what, a, per):
    """A host array whose entries, ``per`` of a kind, have 32-bit numbers."""
    if a.ndim and a.shape[0] * per >= 2 ** 31:
        raise ValueError("%d %s exceed 32-bit numbers" % (a.shape[0], what))
    return np.ascontiguousarray(a)


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
    # scoring enters no autograd function, which would refuse it; asking without a level costs 0.6 us
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("%s: there is no forward-mode derivative" % what)
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
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().float().contiguous()


def _number(what, name, v, lo, hi=float("inf")):
    v = float(v)
    if not (lo <= v <= hi) or v in (float("inf"), float("-inf")):
        raise ValueError("%s: %s = %r is outside [%g, %g]" % (what, name, v, lo, hi))
    return v


_NOTHING = contextlib.nullcontext()


def guard(device):
    """The device as the current one; nothing is switched where it is already."""
    return _NOTHING if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _wants_grad(t):
    return t.requires_grad and torch.is_grad_enabled()


def _rows(logits):
    """The logits themselves, or a copy where columns are strided or rows overlap."""
    (n, v), (s0, s1) = logits.shape, logits.stride()
    if (s1 != 1 and v > 1) or (s0 < v and n > 1):
        return logits.detach().contiguous()
    return logits


def _arg(x, labels):
    """(jtvae_logits_t, the labels as it names them: kept alive until the last launch that reads them)."""
    labels = labels.contiguous()
    n, v = x.shape
    return K.Logits(x.data_ptr(), K.DTYPE_CODE[x.dtype], x.stride(0) if n > 1 else v, n, v, labels.data_ptr(),
                    64 if labels.dtype is torch.int64 else 32), labels


def _grad_rows(x):
    """(uninitialised gradient in the layout of ``x``, its leading dimension): the few padding columns of the package's
    row buffers are kept - the kernel writes them as zero - so that the products that follow take it without a copy."""
    n, v = x.shape
    ld = x.stride(0) if n > 1 else v
    if not v < ld < v + 64:
        return torch.empty((n, v), dtype=x.dtype, device=x.device), v
    return torch.empty((n, ld), dtype=x.dtype, device=x.device)[:, :v], ld


def _scratch(device, *counts):
    """One buffer of 64-bit words for the pieces of the given lengths; (buffer, address of every piece)."""
    buf = torch.empty((sum(counts) + 1,), dtype=torch.float64, device=device)
    at, out = buf.data_ptr(), []
    for c in counts:
        out.append(at)
        at += 8 * c
    return buf, out


class _Gradient:
    """The gradient of a call's logits.  What can be made ready is made with the forward pass: autograd runs the backward
    pass on a thread of its own, which has just been woken and takes two to three times as long over the same Python.
    Buffers of up to ``EARLY_BYTES`` are among it (both passes of ``token_log_probs`` 24 x 385: 103 -> 100 us, of
    ``preference_loss`` 320 x 385: 141 -> 135, an empty autograd function on the same machine: 50); larger ones
    are not held between the passes.  Nothing made early serves where one of the passes is captured into a graph and the other
    is not, or into another one: a replay would write a buffer that is no memory of the graph's, or find one that has been
    changed."""

    EARLY_BYTES = 4 << 20

    __slots__ = ("g", "keep", "place", "buffer", "ld", "made", "capture")

    def __init__(self, x, labels, g, keep, want, made=False):
        """``made``: the buffer will hold the gradient for an upstream factor of one when the forward pass ends."""
        self.g, self.keep, self.place = g, keep, self._place(x, labels)
        self.buffer, self.made, self.capture = None, made, K.capture_id()
        if want and (made or g.n_rows * g.n_cols * x.element_size() <= self.EARLY_BYTES):
            self.buffer, self.ld = _grad_rows(x)

    @staticmethod
    def _place(x, labels):
        """What ``g`` says of the saved tensors.  The strides belong to it: a copy may take the freed logits' address and
        lie there without their padding."""
        return x.data_ptr(), x.stride(), labels.data_ptr()

    def _moved(self, x, labels):
        """(logits as rows, jtvae_logits_t, labels it names) of saved tensors that come back elsewhere; hooks may return
        them in any layout, but not as anything else."""
        what = "backward pass"
        _check(what, x, labels)
        _on_device(what, x, labels=labels)
        if x.shape != (self.g.n_rows, self.g.n_cols) or K.DTYPE_CODE[x.dtype] != self.g.dtype:
            raise RuntimeError("%s: the saved logits came back as %s %s" % (what, x.dtype, tuple(x.shape)))
        x = _rows(x)
        return (x, *_arg(x, labels))

    def early(self, buffer):
        """A buffer made with the forward pass, if the backward pass that now runs may use it."""
        return buffer if buffer is not None and self.capture == K.capture_id() else None

    def __call__(self, x, labels, owner, stats, coef, up, scaled=None, n_scaled=0):
        """The gradient from saved statistics and coefficients (addresses), on the device and stream of the forward pass,
        which autograd has made the current ones."""
        d, self.buffer = self.early(self.buffer), None
        unless_one = self.made and d is not None
        if d is None:  # not held or not fit, or given away by an earlier pass through the same graph
            d, self.ld = _grad_rows(x)
        g = self.g
        if self._place(x, labels) != self.place:
            x, g, labels = self._moved(x, labels)
        K.label_log_probs_bwd(g, owner, stats, coef, up, d.data_ptr(), self.ld, self.ld, int(unless_one), scaled,
                              n_scaled)
        return d


def _tokens(x, labels):
    """(log-probabilities, buffer of the statistics, jtvae_logits_t, labels it names)."""
    dev, n = x.device, x.shape[0]
    lp = torch.empty((n,), dtype=torch.float32, device=dev)
    buf, (stats,) = _scratch(dev, n)
    g, keep = _arg(x, labels)
    K.label_log_probs(g, None, stats, lp.data_ptr(), None)
    return lp, buf, g, keep


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        x = _rows(logits)
        with guard(x.device):
            lp, ctx.ws, g, keep = _tokens(x, labels)
            ctx.gradient = _Gradient(x, labels, g, keep, True)
        ctx.save_for_backward(x, labels)
        return lp

    @staticmethod
    @_differentiable_once
    def backward(ctx, dlp):
        x, labels = ctx.saved_tensors
        coef = dlp.contiguous()
        return ctx.gradient(x, labels, None, ctx.ws.data_ptr(), coef.data_ptr(), None), None


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """[N] fp32: log softmax(logits[i])[labels[i]], 0 where the label is negative.  Differentiable in ``logits``."""
    _check("token_log_probs", logits, labels)
    _on_device("token_log_probs", logits, labels=labels)
    if _wants_grad(logits):
        return _TokenLogProbs.apply(logits, labels)
    with guard(logits.device):  # scoring: nothing to record
        return _tokens(_rows(logits), labels)[0]


def _sequences(x, labels, plan):
    """(sums, buffer that begins with the statistics, jtvae_logits_t, labels it names)."""
    dev, n = x.device, x.shape[0]
    plan.on_current_stream()
    sums = torch.empty((plan.n_seq,), dtype=torch.float32, device=dev)
    buf, (stats, ws) = _scratch(dev, n, n)
    g, keep = _arg(x, labels)
    K.sequence_log_probs(g, plan.arg, stats, sums.data_ptr(), ws, 8 * n)
    return sums, buf, g, keep


class _SequenceLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, plan):
        x = _rows(logits)
        with guard(x.device):
            sums, ctx.ws, g, keep = _sequences(x, labels, plan)
            ctx.gradient = _Gradient(x, labels, g, keep, True)
        ctx.save_for_backward(x, labels)
        ctx.plan = plan
        return sums

    @staticmethod
    @_differentiable_once
    def backward(ctx, dsums):
        x, labels = ctx.saved_tensors
        stats, coef = ctx.ws.data_ptr(), dsums.contiguous()
        # without sequences no row counts and the coefficients are never read: any address will do
        return ctx.gradient(x, labels, ctx.plan.arg.row_seq, stats, coef.data_ptr() or stats, None), None, None


def sequence_log_probs(logits: torch.Tensor, labels: torch.Tensor, plan: SequencePlan) -> torch.Tensor:
    """[plan.n_seq] fp32: sum of the rows' label log-probabilities per sequence (0 for a sequence without rows).
    Differentiable in ``logits``."""
    _check("sequence_log_probs", logits, labels)
    _check_plan("sequence_log_probs", plan, logits)
    _on_device("sequence_log_probs", logits, labels=labels, plan=plan)
    if _wants_grad(logits):
        return _SequenceLogProbs.apply(logits, labels, plan)
    with guard(logits.device):  # scoring: nothing to record
        return _sequences(_rows(logits), labels, plan)[0]


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, other, labels, plan, ref, beta, smoothing, scale, want, want_other):
        x, dev, n, S, P = _rows(logits), logits.device, logits.shape[0], plan.n_seq, plan.n_pairs
        with guard(dev):
            plan.on_current_stream()
            oth, ref = _fp32(other), _fp32(ref)
            sums = torch.empty((S,), dtype=torch.float32, device=dev)
            margins = torch.empty((P,), dtype=torch.float32, device=dev)
            loss = torch.empty((), dtype=torch.float32, device=dev)
            ctx.ws, (stats, coef, ws) = _scratch(dev, n, (S + 1) // 2, n + S + P)
            g, keep = _arg(x, labels)
            K.preference_loss(g, plan.arg, K.Preference(ref.data_ptr(), K.ptr(oth), beta, smoothing, scale), stats,
                              sums.data_ptr(), margins.data_ptr(), coef, loss.data_ptr(), ws, 8 * (n + S + P))
            ctx.gradient = _Gradient(x, labels, g, keep, want)
            ctx.dother = torch.empty((S,), dtype=torch.float32, device=dev) if want_other else None
        ctx.save_for_backward(x, labels)
        ctx.plan, ctx.at, ctx.other_dtype = plan, (stats, coef), None if other is None else other.dtype
        ctx.mark_non_differentiable(sums, margins)
        ctx.set_materialize_grads(False)
        return loss, sums, margins

    @staticmethod
    @_differentiable_once
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 10
        x, labels = ctx.saved_tensors
        plan, d, (stats, coef) = ctx.plan, None, ctx.at
        want, want_other = ctx.needs_input_grad[:2]
        dother, ctx.dother = ctx.gradient.early(ctx.dother), None
        if want_other and dother is None:  # a second pass through the graph
            dother = torch.empty((plan.n_seq,), dtype=torch.float32, device=x.device)
        if want:
            d = ctx.gradient(x, labels, plan.arg.row_seq, stats, coef, dloss.data_ptr(), K.ptr(dother),
                             plan.n_seq if want_other else 0)
        elif want_other:
            none = K.Logits(None, K.F32, 1, 0, 1, None, 32)  # no rows: the sequences' coefficients alone
            K.label_log_probs_bwd(none, None, None, coef, dloss.data_ptr(), None, 1, 1, 0, K.ptr(dother), plan.n_seq)
        if want_other and ctx.other_dtype is not torch.float32:
            dother = dother.to(ctx.other_dtype)
        return d, dother, None, None, None, None, None, None, None, None


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, plan: SequencePlan, ref_log_probs: torch.Tensor,
                    beta: float = 0.1, label_smoothing: float = 0.0, other_log_probs: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> PreferenceLoss:
    """Paired log ratios: with S_q the log-probability of sequence q (plus ``other_log_probs[q]``, what the sequence's
    probability owes to decisions outside these logits, e.g. the stop predictions of the tree decoder) and

        D_p = beta ((S - ref_log_probs)[preferred] - (S - ref_log_probs)[other]),

    the loss is ``scale * sum_p -(1 - label_smoothing) log sigmoid(D_p) - label_smoothing log sigmoid(-D_p)``; ``scale``
    defaults to one over the number of pairs.  Differentiable in ``logits`` and ``other_log_probs``; ``ref_log_probs``
    [plan.n_seq] are constants, read in fp32."""
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
    return PreferenceLoss(*_PreferenceLoss.apply(
        logits, other_log_probs, labels, plan, ref_log_probs, beta, smoothing, scale, _wants_grad(logits),
        other_log_probs is not None and _wants_grad(other_log_probs)))


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, old, adv, ref, weights, lo, hi, kl_coef, scale, want):
        x, dev, n = _rows(logits), logits.device, logits.shape[0]
        with guard(dev):
            old, adv, ref, weights = (_fp32(t) for t in (old, adv, ref, weights))
            lp = torch.empty((n,), dtype=torch.float32, device=dev)
            loss, kl, clipped = (torch.empty((), dtype=torch.float32, device=dev) for _ in range(3))
            nbytes = K.policy_loss_workspace_bytes(n)
            ctx.ws, (stats, coef, ws) = _scratch(dev, n, (n + 1) // 2, nbytes // 8)
            g, keep = _arg(x, labels)
            # a row's coefficient depends on that row alone: its gradient is made while the row is in registers
            ctx.gradient = made = _Gradient(x, labels, g, keep, want, made=True)
            ld = made.ld if want else 0
            policy = K.Policy(old.data_ptr(), adv.data_ptr(), K.ptr(ref), K.ptr(weights), lo, hi, kl_coef, scale)
            K.policy_loss(g, policy, stats, lp.data_ptr(), coef, loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(),
                          K.ptr(made.buffer), ld, ld, ws, nbytes)
        ctx.save_for_backward(x, labels)
        ctx.at = stats, coef
        ctx.mark_non_differentiable(lp, kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, lp, kl, clipped

    @staticmethod
    @_differentiable_once
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 11
        x, labels = ctx.saved_tensors
        # a fresh gradient stands as it is where the upstream factor is 1, which only the device knows
        return (ctx.gradient(x, labels, None, *ctx.at, dloss.data_ptr()),) + (None,) * 10


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor,
                ref_log_probs: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None, clip=0.2,
                kl_coef: float = 0.0, scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss of sampled labels: with r = exp(lp - old_log_probs), A the advantages and
    k = exp(ref - lp) - (ref - lp) - 1 (a never negative estimate of the KL divergence from the reference model),

        loss = scale * sum over rows of weights (kl_coef k - min(r A, min(max(r, 1 - clip), 1 + clip) A)).

    ``clip`` is one number or (low, high); without ``ref_log_probs`` there is no KL term (``kl_coef`` must be 0).  Rows
    with a negative label or a weight of zero do not count, whatever their other inputs hold; ``weights`` (default 1) carry
    masks and means.  Differentiable in ``logits``; the
    other inputs are constants.  The gradient is made along with the loss, for a factor of one on it: a factor is best
    given as ``scale`` (another one in the backward pass is right too, and makes the gradient a second time).  Until the
    backward pass the graph holds that gradient, which is as large as the logits and no saved tensor: hooks that offload
    those, and checkpointing, do not see it."""
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
                                         kl_coef, scale, _wants_grad(logits)))
