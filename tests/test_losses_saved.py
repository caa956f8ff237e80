"""CPU: where the backward pass of the losses takes the saved logits from, the launch itself replaced."""
import pytest
import torch

from fast_jtnn_hip import _capi as K
from fast_jtnn_hip import losses


@pytest.fixture
def launches(monkeypatch):
    """Arguments of the launches that would be made, on host tensors."""
    seen = []
    monkeypatch.setattr(K, "label_log_probs_bwd", lambda g, *a, **k: seen.append((g.x, g.ld, g.labels, g.label_bits)))
    monkeypatch.setattr(losses, "_on_device", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return seen


def _gradient(x, labels):
    return losses._Gradient(x, labels, *losses._arg(x, labels), False)


def test_the_same_place_with_another_distance_between_rows(launches):
    """Padded rows (388 for 385 columns) are freed and their copy, which a hook brings back, lies at the same address
    without the padding."""
    buf, labels = torch.zeros(24 * 388), torch.zeros(24, dtype=torch.int64)
    x, back = buf.view(24, 388)[:, :385], buf[:24 * 385].view(24, 385)
    grad = _gradient(x, labels)
    for t, ld in ((x, 388), (back, 385), (x, 388)):
        grad(t, labels, None, 1, 1, None)
        assert launches.pop() == (buf.data_ptr(), ld, labels.data_ptr(), 64)


def test_strided_columns_and_labels(launches):
    """Copies whose columns are strided, labels that were copied once: what is launched are rows and plain labels."""
    x, labels = torch.zeros(6, 8), torch.arange(12, dtype=torch.int32)[::2]
    grad = _gradient(x, labels)
    grad(x, labels, None, 1, 1, None)
    assert launches.pop() == (x.data_ptr(), 8, grad.keep.data_ptr(), 32) and grad.keep.is_contiguous()
    turned = torch.zeros(8, 6).t()
    grad(turned, labels, None, 1, 1, None)
    at, ld, y, _ = launches.pop()
    assert at != turned.data_ptr() and ld == 8 and y != labels.data_ptr()


def test_saved_tensors_that_come_back_as_something_else(launches):
    x, labels = torch.zeros(6, 8), torch.zeros(6, dtype=torch.int64)
    grad = _gradient(x, labels)
    for t, y, error in ((torch.zeros(6, 9), labels, RuntimeError), (torch.zeros(5, 8), labels[:5], RuntimeError),
                        (torch.zeros(6, 8, dtype=torch.bfloat16), labels, RuntimeError), (x.double(), labels, TypeError),
                        (x, labels.float(), TypeError), (x, torch.zeros(5, dtype=torch.int64), ValueError)):
        with pytest.raises(error):
            grad(t, y, None, 1, 1, None)
    assert not launches


def test_saved_tensors_left_on_the_host(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    x, labels = torch.zeros(6, 8), torch.zeros(6, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        _gradient(x, labels)(x.clone(), labels, None, 1, 1, None)


def test_buffers_made_early_serve_the_same_capture_alone(launches, monkeypatch):
    """Both passes eager or in one capture: the buffer of the forward pass.  Else one of the backward pass's own, made as
    a whole (the launch is not told that it stands already)."""
    x, labels = torch.zeros(6, 8), torch.zeros(6, dtype=torch.int64)
    for made in (False, True):
        for there, here, same in ((None, None, True), (3, 3, True), (None, 3, False), (3, None, False), (3, 4, False)):
            monkeypatch.setattr(K, "capture_id", lambda: there)
            grad = losses._Gradient(x, labels, *losses._arg(x, labels), True, made=made)
            early, flags = grad.buffer, []
            monkeypatch.setattr(K, "label_log_probs_bwd", lambda *a: flags.append(a[8]))
            monkeypatch.setattr(K, "capture_id", lambda: here)
            d = grad(x, labels, None, 1, 1, None)
            assert (d is early) == same and flags == [int(made and same)]
            assert grad(x, labels, None, 1, 1, None) is not d  # given away once


def test_capture_id_refused():
    assert K.lib.jtvae_stream_capture_id(None, None) == K.E_NULL
