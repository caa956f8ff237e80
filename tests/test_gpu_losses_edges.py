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


def test_an_upstream_factor_of_zero_over_rows_that_count():
    """The usual guard of a loss that is not finite: nothing of a NaN, an infinity or a label outside the vocabulary comes
    through a factor of zero - neither into the logits' gradient nor into the other terms'."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss

    x = torch.randn(6, 385, device="cuda")
    x[2] = float("nan")
    x[3, 5] = float("inf")
    labels = torch.arange(6, device="cuda")
    labels[4] = 1000
    old = torch.full((6,), -2.0, device="cuda")
    old[5] = -2000.0  # the ratio overflows
    zero, ref = torch.zeros((), device="cuda"), torch.zeros(2, device="cuda")
    x.requires_grad_()
    loss = policy_loss(x, labels, old, old, ref_log_probs=old, kl_coef=0.1).loss
    assert not bool(torch.isfinite(loss))
    guarded = torch.where(torch.isfinite(loss), loss, zero)
    assert bool((torch.autograd.grad(loss, x, zero, retain_graph=True)[0] == 0).all())
    assert bool((torch.autograd.grad(guarded, x)[0] == 0).all())
    plan = SequencePlan([0, 0, 0, 1, 1, 1], 2, "cuda", pairs=[[0, 1]])
    for dtype in (torch.float32, torch.float64):
        other = torch.zeros(2, dtype=dtype, device="cuda", requires_grad=True)
        for logits, leaves in ((x, (x, other)), (x, (x,)), (x.detach(), (other,))):
            loss = preference_loss(logits, labels, plan, ref, other_log_probs=other).loss
            assert not bool(torch.isfinite(loss))
            for d in torch.autograd.grad(loss, leaves, zero):
                assert bool((d == 0).all())


def test_only_the_other_terms_scaled():
    """Their gradient alone, with a factor: the coefficients times it, as beside the logits' gradient; without sequences."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    x = torch.randn(40, 385, device="cuda")
    labels = torch.randint(0, 385, (40,), device="cuda")
    plan = SequencePlan(np.arange(40) % 8, 8, "cuda", pairs=np.arange(8).reshape(4, 2))
    other, ref, three = torch.randn(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda"), torch.tensor(-3.0, device="cuda")
    alone = torch.autograd.grad(preference_loss(x, labels, plan, ref, other_log_probs=other).loss, other, three)[0]
    x.requires_grad_()
    both = torch.autograd.grad(preference_loss(x, labels, plan, ref, other_log_probs=other).loss, (x, other), three)[1]
    assert torch.equal(alone, both) and bool((alone != 0).all())
    none = SequencePlan(np.full(40, -1), 0, "cuda", pairs=np.zeros((0, 2), np.int32))
    other = torch.zeros(0, device="cuda", requires_grad=True)
    loss = preference_loss(x.detach(), labels, none, other.detach(), other_log_probs=other).loss
    assert torch.autograd.grad(loss, other)[0].shape == (0,)


@pytest.mark.parametrize("n", [4096, 4097, 70000])
def test_no_sequences_over_many_rows(n):
    """Rows of which none belongs to a sequence, on both sides of the rule that gives the sums a launch of their own."""
    from fast_jtnn_hip import SequencePlan, preference_loss, sequence_log_probs

    x = torch.randn(n, 7, device="cuda", requires_grad=True)
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    plan = SequencePlan(np.full(n, -1), 0, "cuda", pairs=np.zeros((0, 2), np.int32))
    r = preference_loss(x, labels, plan, torch.zeros(0, device="cuda"))
    assert float(r.loss) == 0 and r.log_probs.shape == (0,) and r.margins.shape == (0,)
    assert bool((torch.autograd.grad(r.loss, x)[0] == 0).all())
    sums = sequence_log_probs(x, labels, plan)
    assert sums.shape == (0,) and bool((torch.autograd.grad(sums.sum(), x)[0] == 0).all())


def test_capture_ids():
    """One number per capture, on every stream that takes part; none outside, and none on a stream that does not."""
    from fast_jtnn_hip import _capi as K

    x = torch.zeros(5, device="cuda")
    a, b, apart = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    seen = []
    assert K.capture_id() is None
    for _ in range(3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=a):
            x.add_(1)
            seen.append(K.capture_id())
            b.wait_stream(a)
            with torch.cuda.stream(b):
                assert K.capture_id() == seen[-1]
                x.add_(1)
            with torch.cuda.stream(apart):
                assert K.capture_id() is None
            a.wait_stream(b)
            assert K.capture_id() == seen[-1]
    assert len(set(seen)) == 3 and None not in seen and K.capture_id() is None


def test_passes_captured_into_two_graphs():
    """The forward pass in one graph, the backward pass in another: every replay of the second writes the whole gradient,
    whatever became of the last replay's; a replay of both follows the logits."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, sequence_log_probs, token_log_probs

    n, v = 24, 385
    x = torch.randn(n, v, device="cuda", requires_grad=True)
    labels = torch.randint(0, v, (n,), device="cuda")
    plan = SequencePlan(np.arange(n) % 4, 4, "cuda", pairs=[[0, 1], [2, 3]])
    ref, old = torch.zeros(4, device="cuda"), torch.full((n,), -6.0, device="cuda")
    other = torch.zeros(4, device="cuda", requires_grad=True)
    calls = [(lambda: token_log_probs(x, labels).sum(), [x]),
             (lambda: sequence_log_probs(x, labels, plan).sum(), [x]),
             (lambda: preference_loss(x, labels, plan, ref, other_log_probs=other).loss, [x, other]),
             (lambda: policy_loss(x, labels, old, old).loss, [x]),
             (lambda: policy_loss(x, labels, old, old).loss * 3, [x])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        [torch.autograd.grad(f(), leaves) for f, leaves in calls]
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=side):
        losses = [f() for f, _ in calls]
    with torch.cuda.graph(second, stream=side):
        got = [torch.autograd.grad(loss, leaves, retain_graph=True) for loss, (_, leaves) in zip(losses, calls)]
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(n, v, device="cuda"))
        want = [torch.autograd.grad(f(), leaves) for f, leaves in calls]
        first.replay()
        for again in range(2):
            second.replay()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(got, want)):
                for p, q in zip(a, b):
                    assert torch.equal(p, q), (k, again, i)
                    p.fill_(float("nan"))


def test_forward_mode_is_refused_with_a_plan_too():
    """Scoring without reverse mode, plan and logits on the GPU; a level alone changes nothing."""
    from torch.autograd import forward_ad

    from fast_jtnn_hip import SequencePlan, sequence_log_probs, token_log_probs

    x, labels = torch.randn(4, 7, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    plan = SequencePlan([0, 0, 1, 1], 2, "cuda")
    calls = [lambda t: token_log_probs(t, labels), lambda t: sequence_log_probs(t, labels, plan)]
    want = [f(x) for f in calls]
    with forward_ad.dual_level():
        for f, w in zip(calls, want):
            assert torch.equal(f(x), w)
            with pytest.raises(NotImplementedError):
                f(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("v", [9, 4099, 70001])
def test_the_estimate_of_an_impossible_label(v):
    """A label whose logit is -inf (log-probability -inf) that the reference model gives a chance: an infinite estimate and
    an infinite loss with a penalty, the loss of its ratio (zero) without one; the other rows' estimates stay."""
    from fast_jtnn_hip import policy_loss

    inf = float("inf")
    x = torch.randn(4, v, device="cuda")
    x[1, 2] = -inf
    labels, f = torch.full((4,), 2, device="cuda"), torch.full((4,), -8.0, device="cuda")
    a = torch.tensor([-1.0, 1.0, 1.0, -2.0], device="cuda")
    out, rest = (policy_loss(t, y, q, b, ref_log_probs=q, clip=(1.0, 1e9)) for t, y, q, b in (
        (x, labels, f, a), (x[[0, 2, 3]], labels[:3], f[:3], a[[0, 2, 3]])))
    assert float(out.kl) == inf and float(out.log_probs[1]) == -inf
    assert abs(float(out.loss) - float(rest.loss)) <= 2.0 ** -22 * abs(float(rest.loss))
    assert float(policy_loss(x, labels, f, a, ref_log_probs=f, kl_coef=0.1, clip=(1.0, 1e9)).loss) == inf
    keep = torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda")
    out = policy_loss(x, labels, f, a, ref_log_probs=f, weights=keep, kl_coef=0.1)
    assert bool(torch.isfinite(out.kl)) and bool(torch.isfinite(out.loss))


@pytest.mark.parametrize("smoothing", [0.0, 0.125, 1.0])
def test_coefficients_of_far_margins(smoothing):
    """Against the derivative in 64 bits, relative to itself: two logistic values, each good to a few 2^-53, and one rounding
    to 32 bits (2^-24, and 2^-149 where the result leaves the normal range)."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    margins = torch.tensor([-90.0, -60.0, -37.0, -25.0, -15.0, -1.0, 0.0, 0.5, 10.0, 20.0, 30.0, 37.0, 45.0, 90.0], device="cuda")
    p = len(margins)
    pairs = np.arange(2 * p).reshape(p, 2)
    x = torch.zeros(2 * p, 3, device="cuda")
    other = torch.zeros(2 * p, device="cuda", requires_grad=True)
    ref = torch.zeros(2 * p, device="cuda")
    ref[1::2] = margins
    r = preference_loss(x, torch.zeros(2 * p, dtype=torch.int64, device="cuda"), SequencePlan(np.arange(2 * p), 2 * p, "cuda",
                        pairs=pairs), ref, beta=1.0, label_smoothing=smoothing, other_log_probs=other, scale=1.0)
    (d,) = torch.autograd.grad(r.loss, other)
    m = margins.double()
    want = smoothing / (1 + torch.exp(-m)) - (1 - smoothing) / (1 + torch.exp(m))
    assert torch.equal(r.margins, margins)
    assert bool(((d[::2].double() - want).abs() <= want.abs() * 2.0 ** -23 + 2.0 ** -149).all()) and torch.equal(d[::2], -d[1::2])


def test_a_plan_of_an_empty_list():
    from fast_jtnn_hip import SequencePlan, sequence_log_probs

    x, labels = torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    assert torch.equal(sequence_log_probs(x, labels, SequencePlan([], 3, "cuda")), torch.zeros(3, device="cuda"))
    assert sequence_log_probs(x, labels, SequencePlan([], 0, "cuda", pairs=[])).shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_differences_of_long_sums(dtype):
    """Equal logits: a row's sum is its number of columns exactly, so its log-probability is off by the logarithm's 2^-53
    alone, and a sequence's by one more per addition.  Sums of hundreds of thousands of such rows lie beyond the last place
    of 32-bit numbers; their differences to references nearby do not: log-probabilities rounded to 32 bits (each off by
    1e-8 and more, the same way) would show as 1e-3."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    n, v = 300_000, 3
    x = torch.full((n, v), 0.5, dtype=dtype, device="cuda")
    labels = torch.arange(n, device="cuda") % v
    row_seq = np.where(np.arange(n) % 3 < 2, 0, 1)
    want = -np.log(3.0) * np.bincount(row_seq).astype(np.float64)
    ref = torch.tensor([want[0] - 0.375, want[1] + 1.25], device="cuda", dtype=torch.float32)
    near = want - ref.double().cpu().numpy()
    r = preference_loss(x, labels, SequencePlan(row_seq, 2, "cuda", pairs=[[0, 1]]), ref, beta=1.0)
    exact = near[0] - near[1]
    off = n * abs(want).max() * 2.0 ** -52  # 1.5e-5
    assert abs(float(r.margins[0]) - exact) <= abs(exact) * 2.0 ** -24 + off
    assert abs(float(r.loss) - np.log1p(np.exp(-exact))) <= 2.0 ** -22 + off
