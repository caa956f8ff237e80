"""GPU: calls of the label log-probabilities and the losses at the edges of what they take."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_saved_logits_without_their_padding():
    """Hooks that move only the floating tensors to the host: rows of 385 columns, 388 apart, come back side by side,
    perhaps where the freed ones lay, while the labels never move."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, sequence_log_probs, token_log_probs

    x = torch.randn(24, 388, device="cuda")
    labels = torch.randint(0, 385, (24,), device="cuda")
    plan = SequencePlan(np.arange(24) % 2, 2, "cuda", pairs=[[0, 1]])
    two, f = torch.zeros(2, device="cuda"), torch.full((24,), -6.0, device="cuda")

    def pack(t):
        return t.cpu() if t.is_floating_point() else t

    for call in (lambda y: token_log_probs(y, labels).sum(), lambda y: sequence_log_probs(y, labels, plan).sum(),
                 lambda y: preference_loss(y, labels, plan, two).loss, lambda y: policy_loss(y, labels, f, f, clip=(1.0, 50.0)).loss * 2):
        got = []
        for moved in (False, True):
            leaf = x.clone().requires_grad_()
            y = (leaf * 1.0)[:, :385]
            if moved:
                with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
                    loss = call(y)
            else:
                loss = call(y)
            del y
            loss.backward()
            got.append(leaf.grad)
        assert torch.equal(*got) and bool((got[0][:, :385] != 0).all())


def test_as_many_columns_as_a_row_may_have():
    """2^31 - 1 equal logits: their sum and every result but the log-probability's last place are exact; what lies
    2^31 elements in front of the gradient, where column numbers that wrap around would point, stays as it was."""
    from fast_jtnn_hip import _capi as K
    from fast_jtnn_hip import token_log_probs

    v = (1 << 31) - 1
    x = torch.zeros(1, v, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    labels = torch.tensor([v - 1], device="cuda")
    lp = token_log_probs(x, labels)
    assert abs(float(lp) + 31 * np.log(2.0)) <= 2.0 ** -20
    (d,) = torch.autograd.grad(lp.sum(), x)
    assert float(d[0, v - 1]) == 1 and int((d[0, :v - 1] != -2.0 ** -31).sum()) == 0
    del d
    buf = torch.ones(2 << 31, dtype=torch.bfloat16, device="cuda")
    out = buf[1 << 31:]
    stats, coef = torch.tensor([0.0, 2.0 ** 31], device="cuda"), torch.ones(1, device="cuda")
    g = K.Logits(x.data_ptr(), K.BF16, v, 1, v, labels.data_ptr(), 64)
    K.label_log_probs_bwd(g, None, stats.data_ptr(), coef.data_ptr(), None, out.data_ptr(), v, v)
    assert int((buf[:1 << 31] != 1).sum()) == 0 and float(out[v]) == 1
    assert float(out[v - 1]) == 1 and int((out[:v - 1] != -2.0 ** -31).sum()) == 0
