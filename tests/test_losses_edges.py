"""CPU: calls of the losses at the edges of what they take (the device check comes last)."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from fast_jtnn_hip import SequencePlan, losses


def _plan(n_rows, n_seq):
    """A plan as the constructor leaves it, without its device tables."""
    p = SequencePlan.__new__(SequencePlan)
    p.n_rows, p.n_seq, p.n_pairs, p.device = n_rows, n_seq, 1, torch.device("cpu")
    return p


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """With and without reverse mode recording: no call returns a value that has lost its tangent."""
    x, labels, f = torch.zeros(4, 7), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    calls = [lambda t: losses.token_log_probs(t, labels), lambda t: losses.sequence_log_probs(t, labels, _plan(4, 2)),
             lambda t: losses.preference_loss(t, labels, _plan(4, 2), f[:2]), lambda t: losses.policy_loss(t, labels, f, f)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            for call in calls:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(forward_ad.make_dual(leaf, torch.ones_like(x)))
                with pytest.raises(RuntimeError, match="no CPU path"):
                    call(leaf)  # no tangent of its own


def test_a_plan_of_an_empty_list():
    """Nothing to refuse but the device: a batch may have no rows."""
    for rows, pairs in (([], None), ([], []), ((), [[0, 1]])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            SequencePlan(rows, 2, "cpu", pairs=pairs)
    for rows in ([[]], [["a"]]):
        with pytest.raises(ValueError, match="row_seq"):
            SequencePlan(rows, 2, "cpu")


def test_plans_beyond_32_bit_numbers_refused():
    """Before anything of that size is made (the arrays here are one number, repeated)."""
    zero = np.zeros((), np.int32)
    for rows, n_seq, pairs in (([0], 2 ** 31 - 1, None), ([0], 2 ** 32 + 1, None), (np.broadcast_to(zero, (2 ** 31,)), 1, None),
                               ([0], 1, np.broadcast_to(zero, (2 ** 30, 2)))):
        with pytest.raises(ValueError, match="32-bit"):
            SequencePlan(rows, n_seq, "cpu", pairs=pairs)
    with pytest.raises(ValueError, match="n_seq is"):
        SequencePlan([0], -2 ** 33, "cpu")
