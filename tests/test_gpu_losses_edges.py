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
