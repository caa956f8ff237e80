"""CPU: what the fine-tuning losses and the AdamW step refuse, before any launch - the Python entry points on host
tensors (the device check comes last, so every other refusal shows here) and the C ABI with addresses it must not use."""
import ctypes

import numpy as np
import pytest
import torch

from fast_jtnn_hip import AdamW, SequencePlan, losses
from fast_jtnn_hip import _capi as K

X, Y = torch.zeros(4, 7), torch.zeros(4, dtype=torch.int64)
F = torch.zeros(4)


def _plan(n_rows=4, n_seq=2, pairs=True):
    """A plan as the constructor leaves it, without its device tables."""
    p = SequencePlan.__new__(SequencePlan)
    p.n_rows, p.n_seq, p.n_pairs, p.device = n_rows, n_seq, 1 if pairs else None, torch.device("cpu")
    return p


@pytest.mark.parametrize("logits,labels,error", [
    (torch.zeros(4), Y, ValueError), (torch.zeros(4, 0), Y, ValueError), (torch.zeros(2, 2, 2), Y, ValueError),
    (X.double(), Y, TypeError), (X.int(), Y, TypeError), (X, Y[:3], ValueError), (X, Y[:, None], ValueError),
    (X, Y.float(), TypeError), (X, Y.to(torch.int16), TypeError), (X.numpy(), Y, TypeError), (X, Y.numpy(), TypeError),
])
def test_logits_and_labels_refused(logits, labels, error):
    calls = [lambda: losses.token_log_probs(logits, labels),
             lambda: losses.sequence_log_probs(logits, labels, _plan()),
             lambda: losses.preference_loss(logits, labels, _plan(), torch.zeros(2)),
             lambda: losses.policy_loss(logits, labels, F, F)]
    for call in calls:
        with pytest.raises(error):
            call()


def test_no_cpu_path():
    for call in (lambda: losses.token_log_probs(X, Y), lambda: losses.sequence_log_probs(X, Y, _plan()),
                 lambda: losses.preference_loss(X, Y, _plan(), torch.zeros(2)),
                 lambda: losses.policy_loss(X, Y, F, F), lambda: SequencePlan([0, 1], 2, "cpu"),
                 lambda: AdamW([torch.nn.Parameter(torch.zeros(3))])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_plans_refused():
    for row_seq, n_seq, pairs, error in (([0, 2], 2, None, IndexError), ([-2, 0], 2, None, IndexError),
                                         ([0.5], 1, None, ValueError), ([[0]], 1, None, ValueError),
                                         ([0], -1, None, ValueError), ([0], 2, [[0, 2]], IndexError),
                                         ([0], 2, [[-1, 0]], IndexError), ([0], 2, [[0, 1, 1]], ValueError),
                                         ([0], 2, [[0.0, 1.0]], ValueError), ([0], 2, [0, 1], ValueError)):
        with pytest.raises(error):
            SequencePlan(np.asarray(row_seq), n_seq, "cpu", pairs=pairs)
    with pytest.raises(ValueError, match="plan describes"):
        losses.sequence_log_probs(X, Y, _plan(n_rows=3))
    with pytest.raises(TypeError, match="SequencePlan"):
        losses.sequence_log_probs(X, Y, [0, 0, 1, 1])
    with pytest.raises(ValueError, match="without pairs"):
        losses.preference_loss(X, Y, _plan(pairs=False), torch.zeros(2))


def test_loss_arguments_refused():
    two = torch.zeros(2)
    for kw in (dict(beta=-1.0), dict(beta=float("nan")), dict(label_smoothing=1.5), dict(label_smoothing=-0.1),
               dict(scale=float("inf")), dict(ref_log_probs=torch.zeros(3)), dict(other_log_probs=torch.zeros(3)),
               dict(other_log_probs=[0.0, 0.0])):
        args = dict(ref_log_probs=two)
        args.update(kw)
        with pytest.raises(ValueError):
            losses.preference_loss(X, Y, _plan(), **args)
    with pytest.raises(TypeError):
        losses.preference_loss(X, Y, _plan(), two.long())
    for kw in (dict(clip=1.5), dict(clip=-0.1), dict(clip=(0.2, -1.0)), dict(kl_coef=-1.0), dict(kl_coef=0.1),
               dict(weights=torch.zeros(5)), dict(advantages=torch.zeros(4, 1)), dict(old_log_probs=None),
               dict(scale=float("nan"))):
        args = dict(old_log_probs=F, advantages=F)
        args.update(kw)
        with pytest.raises(ValueError):
            losses.policy_loss(X, Y, **args)
    with pytest.raises(TypeError):
        losses.policy_loss(X, Y, F, F.long())


def test_adamw_arguments_refused():
    p = lambda *a, **k: torch.nn.Parameter(torch.zeros(*a, **k))  # noqa: E731
    for params, kw, error in (([p(2)], dict(lr=-1.0), ValueError), ([p(2)], dict(betas=(1.0, 0.9)), ValueError),
                              ([p(2)], dict(betas=(0.9, -0.1)), ValueError), ([p(2)], dict(eps=-1e-8), ValueError),
                              ([p(2)], dict(weight_decay=-1), ValueError), ([p(2)], dict(state_bits=16), ValueError),
                              ([p(2)], dict(rounding="up"), ValueError),
                              ([p(2)], dict(max_norm=0.0), ValueError), ([p(2)], dict(max_norm=float("nan")), ValueError),
                              ([p(2, dtype=torch.float64)], {}, TypeError),
                              ([p(2), p(2, dtype=torch.bfloat16)], {}, TypeError),
                              ([torch.nn.Parameter(torch.zeros(3, 4).t())], {}, ValueError)):
        with pytest.raises(error):
            AdamW(params, **kw)


@pytest.mark.filterwarnings("ignore:optimizer contains")
def test_adamw_refuses_a_parameter_given_twice():
    """Two blocks would work on its elements at once."""
    p = torch.nn.Parameter(torch.zeros(2))
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, torch.nn.Parameter(torch.zeros(2)), p])


def test_c_entry_points_refuse_before_launch():
    lib = K.lib
    ok = K.Logits(256, K.F32, 8, 4, 7, 256, 64)

    def lp(g, stats=256):
        return lib.jtvae_label_log_probs(ctypes.byref(g), None, stats, 256, None, None)

    assert lib.jtvae_label_log_probs(None, None, 256, 256, None, None) == K.E_NULL
    assert lp(ok, None) == K.E_NULL
    assert lp(K.Logits(256, K.F32, 6, 4, 7, 256, 64)) == K.E_SHAPE  # ld < n_cols
    assert lp(K.Logits(256, K.F32, 8, -1, 7, 256, 64)) == K.E_SHAPE
    assert lp(K.Logits(256, K.F32, 8, 4, 0, 256, 64)) == K.E_SHAPE
    assert lp(K.Logits(256, 3, 8, 4, 7, 256, 64)) == K.E_RANGE
    assert lp(K.Logits(256, K.F32, 8, 4, 7, 256, 16)) == K.E_RANGE
    assert lp(K.Logits(None, K.F32, 8, 4, 7, 256, 64)) == K.E_NULL
    assert lp(K.Logits(258, K.F32, 8, 4, 7, 256, 64)) == K.E_ALIGN
    assert lp(K.Logits(258, K.BF16, 8, 4, 7, 260, 64)) == K.E_ALIGN
    assert lp(K.Logits(None, K.F32, 8, 0, 7, None, 64)) == 0  # no rows: nothing to do
    bwd = lib.jtvae_label_log_probs_bwd
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 0, 256, 7, 8, None, 0, None) == K.E_SHAPE  # width > ld_dx
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 0, 256, 8, 6, None, 0, None) == K.E_SHAPE  # width < n_cols
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 0, 257, 8, 8, None, 0, None) == K.E_ALIGN
    assert bwd(ctypes.byref(ok), None, None, 256, None, 0, 256, 8, 8, None, 0, None) == K.E_NULL
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 1, 256, 8, 8, None, 0, None) == K.E_NULL  # unless_one without upstream
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 0, 256, 8, 8, 256, -1, None) == K.E_SHAPE
    assert bwd(ctypes.byref(ok), None, 256, 256, None, 0, 256, 8, 8, None, 2, None) == K.E_NULL
    seqs = K.Sequences(256, 256, 256, 2, 256, 1, 256, 256)
    pref = K.Preference(256, None, 0.1, 0.0, 1.0)
    none = K.Logits(None, K.F32, 8, 0, 7, None, 64)

    def sums(q=seqs, ws=32, sums=256, stats=256):
        return lib.jtvae_sequence_log_probs(ctypes.byref(ok), ctypes.byref(q), stats, sums, 256, ws, None)

    assert K.lib.jtvae_sequence_log_probs_workspace_bytes(4) == 32
    assert sums(ws=31) == K.E_WORKSPACE and sums(sums=None) == K.E_NULL and sums(stats=None) == K.E_NULL
    assert sums(q=K.Sequences(None, 256, 256, 2, None, 0, None, None)) == K.E_NULL
    assert sums(q=K.Sequences(256, 256, 256, -1, None, 0, None, None)) == K.E_SHAPE
    assert lib.jtvae_sequence_log_probs(ctypes.byref(none), ctypes.byref(K.Sequences()), None, None, None, 0, None) == 0

    def pairs(q=seqs, p=pref, ws=56, loss=256, coef=256):
        return lib.jtvae_preference_loss(ctypes.byref(ok), ctypes.byref(q), ctypes.byref(p), 256, 256, 256, coef, loss, 256,
                                         ws, None)

    assert K.lib.jtvae_preference_loss_workspace_bytes(4, 2, 1) == 56
    assert pairs(ws=55) == K.E_WORKSPACE and pairs(loss=None) == K.E_NULL and pairs(coef=None) == K.E_NULL
    assert pairs(p=K.Preference(None, None, 0.1, 0.0, 1.0)) == K.E_NULL
    assert pairs(p=K.Preference(256, None, 0.1, 1.5, 1.0)) == K.E_RANGE
    assert pairs(q=K.Sequences(256, 256, 256, 2, None, 1, 256, 256)) == K.E_NULL
    assert pairs(q=K.Sequences(256, 256, 256, 2, 256, -1, 256, 256)) == K.E_SHAPE
    pol = K.Policy(256, 256, None, None, 0.2, 0.2, 0.0, 1.0)
    need = K.policy_loss_workspace_bytes(4)
    assert need > 0 and K.policy_loss_workspace_bytes(0) == 0

    def policy(p=pol, g=ok, ws=need, stats=256, loss=256):
        return lib.jtvae_policy_loss(ctypes.byref(g), ctypes.byref(p), stats, 256, 256, loss, 256, 256, None, 0, 0, 256, ws, None)

    assert policy(ws=need - 1) == K.E_WORKSPACE and policy(stats=None) == K.E_NULL and policy(loss=None) == K.E_NULL
    assert policy(p=K.Policy(None, 256, None, None, 0.2, 0.2, 0.0, 1.0)) == K.E_NULL
    assert policy(p=K.Policy(256, 256, None, None, 1.2, 0.2, 0.0, 1.0)) == K.E_RANGE
    ptr = (ctypes.c_int64 * 2)(0, 1)
    grads = (ctypes.c_void_p * 1)(None)

    def group(**kw):
        a = dict(tensors=256, chunks=256, chunk_ptr=ctypes.addressof(ptr), grads=ctypes.addressof(grads), steps=256,
                 bias=256, n_tensors=1, n_chunks=1, dtype=K.F32, state_bits=32, use_master=0, stochastic=0, lr_device=None, lr=1e-3,
                 beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0)
        a.update(kw)
        return K.AdamwGroup(*[a[n] for n, _ in K.AdamwGroup._fields_])

    for kw, code in ((dict(tensors=None), K.E_NULL), (dict(chunks=None), K.E_NULL), (dict(grads=None), K.E_NULL),
                     (dict(dtype=7), K.E_RANGE), (dict(state_bits=16), K.E_RANGE), (dict(n_tensors=-1), K.E_SHAPE),
                     (dict(n_chunks=2), K.E_SHAPE), (dict(beta1=1.0), K.E_RANGE), (dict(eps=-1.0), K.E_RANGE),
                     (dict(steps=None), K.E_NULL)):
        assert lib.jtvae_adamw_step(ctypes.byref(group(**kw)), 1, 0.0, None, None, None) == code, kw
    step = lambda n, norm, partials=256, out=256: lib.jtvae_adamw_step(  # noqa: E731
        ctypes.byref(group()), n, norm, partials, out, None)
    assert lib.jtvae_adamw_step(None, 1, 0.0, None, None, None) == K.E_NULL
    assert lib.jtvae_adamw_step(None, 0, 0.0, None, None, None) == 0
    assert step(-1, 0.0) == K.E_SHAPE and step(1, -1.0) == K.E_RANGE and step(1, float("nan")) == K.E_RANGE
    assert step(1, 1.0, partials=None) == K.E_NULL and step(1, 1.0, out=None) == K.E_NULL


def test_trainer_optimizers_refused():
    from fast_jtnn_hip import trainer

    m = torch.nn.Linear(3, 2)
    with pytest.raises(ValueError, match="is none of"):
        trainer.Trainer(m, optimizer="sgd")
    with pytest.raises(ValueError, match="weight_decay"):
        trainer.Trainer(m, weight_decay=0.1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        trainer.Trainer(m, optimizer="adamw")
    assert isinstance(trainer.Trainer(m).optimizer, torch.optim.Adam)


def test_decoder_entry_points_refuse_cpu():
    from fast_jtnn_hip import JTNNDecoder, synthetic

    d = JTNNDecoder(synthetic.FakeVocab(5), 16, 4, torch.nn.Embedding(5, 16))
    for call in (lambda: d.log_likelihood([], torch.zeros(0, 4)), lambda: d.trace_scores([], torch.zeros(0, 4)),
                 lambda: d.preference_loss([], torch.zeros(0, 4), [[0, 1]], torch.zeros(2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
