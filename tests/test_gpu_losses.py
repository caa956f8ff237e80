"""GPU: log-probabilities of labels under rows of logits and the losses built on them, against the definitions in 64
bits.

Tolerances.  With d = max - x, an exponent's argument is off by at most 2^-23 d (one subtraction, one product), the
exponential by 2^-23, and a row's sum of V terms, none negative, by 2^-24 per addition on the longest chain, which is
below V / 64 + 64 here.  So s is off by at most S(V) = 2^-23 (ln V + 2 + V / 128 + 32) relative (sum of p d is at most
ln V + 1), a log-probability by S(V) plus its own rounding, and a probability by S(V) + 2^-23 (d + 4) relative.  A result
in type t is then rounded by at most finfo(t).eps / 2."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(1, 1), (3, 2), (1, 64), (5, 63), (24, 385), (7, 780), (130, 257), (33, 1025), (9, 4099), (2, 50021), (1, 131072),
         (300, 2049)]


def sum_error(v):
    return 2.0 ** -23 * (math.log(v) + 2 + v / 128 + 32)


def make(n, v, dtype, seed, ld=None, offset=0):
    """Logits of a trained model (labels mostly well above the noise) as rows of ``ld`` in a larger buffer."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or v
    buf = torch.randn(n * ld + offset, generator=g, device="cuda").mul_(2)
    labels = torch.randint(0, v, (n,), generator=g, device="cuda")
    x = buf[offset:].view(n, ld)[:, :v]
    if n:
        x[torch.arange(n, device="cuda"), labels] += torch.randn(n, generator=g, device="cuda") * 2 + 4
    buf = buf.to(dtype)
    return buf[offset:].view(n, ld)[:, :v], labels


def exact(x, labels):
    """(log-probabilities, softmax, distance from the maximum) in 64 bits; rows without a label: 0, 0, 0."""
    x = x.detach().double()
    n = x.shape[0]
    keep = labels >= 0
    at = labels.clamp(min=0).long()
    lp = torch.log_softmax(x, 1)[torch.arange(n, device=x.device), at]
    soft = torch.softmax(x, 1)
    return torch.where(keep, lp, 0.0), soft, x.max(1, keepdim=True).values - x


def exact_grad(soft, labels, coef):
    g = -soft.clone()
    g[torch.arange(len(labels), device=g.device), labels.clamp(min=0).long()] += 1
    return torch.where((labels >= 0)[:, None], g * coef.double()[:, None], 0.0)


def check_grad(d, soft, dist, labels, coef, dtype):
    want = exact_grad(soft, labels, coef)
    fi = torch.finfo(dtype)
    k = coef.double().abs()[:, None]
    dist = torch.where(torch.isfinite(dist), dist, 0.0)
    tol = k * soft * (sum_error(d.shape[1]) + 2.0 ** -23 * (dist + 4)) + want.abs() * (fi.eps / 2 + 2.0 ** -22)
    tol = tol + (fi.smallest_normal if dtype != torch.float16 else 2.0 ** -24) + 2.0 ** -125 * k
    # the label's own element: c - c p, whose parts are rounded to 32 bits
    tol[torch.arange(len(labels), device=d.device), labels.clamp(min=0).long()] += 2.0 ** -22 * k[:, 0]
    bad = ~((d.double() - want).abs() <= tol)
    assert not bad.any(), ((d.double() - want).abs() / tol).max()
    assert (d[labels < 0] == 0).all()


def check_lp(lp, want, v):
    assert ((lp.double() - want).abs() <= sum_error(v) + want.abs() * 2.0 ** -24).all(), (lp.double() - want).abs().max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", SIZES)
def test_token_log_probs(n, v, dtype):
    from fast_jtnn_hip import token_log_probs

    for ld, offset in ((v, 0), (v + 3, 1)):
        x, labels = make(n, v, dtype, 1000 + n + v, ld, offset)
        if n > 1:
            labels[::7] = -100
        x.requires_grad_()
        coef = torch.randn(n, device="cuda")
        lp = token_log_probs(x, labels)
        (d,) = torch.autograd.grad(lp, x, coef)
        want, soft, dist = exact(x, labels)
        assert lp.dtype == torch.float32 and d.dtype == dtype and d.shape == x.shape
        check_lp(lp, want, v)
        check_grad(d, soft, dist, labels, coef, dtype)
        lp2 = token_log_probs(x, labels.to(torch.int32))
        assert torch.equal(lp, lp2) and torch.equal(d, torch.autograd.grad(lp2, x, coef)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 385, 3001, 40000])
def test_masked_logits(v, dtype):
    """Vocabularies masked with -inf or the type's lowest value, rows with nothing left, infinities and NaN."""
    from fast_jtnn_hip import token_log_probs

    x, labels = make(12, v, dtype, 5)
    low = torch.finfo(dtype).min
    inf = float("inf")
    labels[:] = 1
    x[1, 2:] = -inf  # two words left
    x[2, 2:] = low
    x[3, :] = low  # all equal: uniform
    x[4, 0] = -inf
    x[5, 1] = -inf  # the label itself
    labels[5] = 1
    x[6, :] = -inf  # nothing left, no label: not read
    labels[6] = -1
    x[7, :] = float("nan")
    labels[7] = -100
    x[8, :] = -inf  # nothing left, but a label: no distribution
    x[9, 0] = float("nan")
    x[10, 0] = inf
    labels[11] = v + 3  # no such word
    x.requires_grad_()
    lp = token_log_probs(x, labels)
    coef = torch.full((12,), 0.5, device="cuda")
    (d,) = torch.autograd.grad(lp, x, coef)
    fine = [0, 1, 2, 3, 4, 6, 7]
    clean = x.detach().clone()
    clean[[6, 7]] = 0
    want, soft, dist = exact(clean, labels.clamp(max=v - 1))
    check_lp(lp[fine], want[fine], v)
    dist = dist.clamp(max=2000)  # farther terms are exactly zero
    check_grad(d[fine], soft[fine], dist[fine], labels[fine], coef[fine], dtype)
    assert lp[5] == -inf
    check_grad(d[5:6], soft[5:6], dist[5:6], labels[5:6], coef[5:6], dtype)
    assert torch.isnan(lp[[8, 9, 10, 11]]).all() and torch.isnan(d[[8, 9, 11]]).any(1).all()
    assert torch.isnan(d[11]).all()


def test_layouts():
    """Strided columns, rows that overlap (a broadcast row), a transposed view, no rows, one row of a wide buffer."""
    from fast_jtnn_hip import token_log_probs

    x, labels = make(6, 90, torch.float32, 3)
    coef = torch.randn(6, device="cuda")
    base = exact(x, labels)

    def run(leaf, view):
        lp = token_log_probs(view, labels)
        (d,) = torch.autograd.grad(lp, view, coef, retain_graph=True)
        lp.backward(coef)
        return lp, d

    leaf = x.t().contiguous().requires_grad_()
    lp, d = run(leaf, leaf.t())
    check_lp(lp, base[0], 90)
    check_grad(d, base[1], base[2], labels, coef, torch.float32)
    assert torch.equal(leaf.grad, d.t())
    leaf = torch.stack([x, x + 1], 2).reshape(6, 180).requires_grad_()
    lp, d = run(leaf, leaf[:, ::2])
    check_grad(d, base[1], base[2], labels, coef, torch.float32)
    assert torch.equal(leaf.grad[:, ::2], d) and (leaf.grad[:, 1::2] == 0).all()
    leaf = x[2].clone().requires_grad_()
    view = leaf.expand(6, 90)
    lp, d = run(leaf, view)
    want, soft, dist = exact(view, labels)
    check_lp(lp, want, 90)
    check_grad(d, soft, dist, labels, coef, torch.float32)
    assert ((leaf.grad.double() - exact_grad(soft, labels, coef).sum(0)).abs()
            <= 6 * 2.0 ** -20 * coef.abs().sum().item()).all()
    wide = torch.randn(3, 5000, device="cuda")
    lp = token_log_probs(wide[1:2, 7:97], labels[:1])
    check_lp(lp, exact(wide[1:2, 7:97], labels[:1])[0], 90)
    empty = torch.zeros(0, 9, device="cuda", requires_grad=True)
    lp = token_log_probs(empty, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (0,)
    lp.sum().backward()
    assert empty.grad.shape == (0, 9)


def test_padding_columns_of_row_buffers_become_zero():
    """The package's products hand over rows padded to 16 bytes: the gradient keeps that layout, padding zero."""
    from fast_jtnn_hip import token_log_probs

    x, labels = make(5, 385, torch.float32, 8, ld=388)
    x.requires_grad_()
    (d,) = torch.autograd.grad(token_log_probs(x, labels).sum(), x)
    assert d.stride() == (388, 1)
    assert (d.as_strided((5, 3), (388, 1), 385) == 0).all()


def test_offsets_beyond_32_bits():
    """Rows 2^28 elements apart: the last one starts beyond 2^31."""
    from fast_jtnn_hip import token_log_probs

    n, v, ld = 10, 1000, 1 << 28
    buf = torch.empty((n - 1) * ld + v, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((n, v), (ld, 1))
    src, labels = make(n, v, torch.bfloat16, 11)
    x.copy_(src)
    x.requires_grad_()
    lp = token_log_probs(x, labels)
    (d,) = torch.autograd.grad(lp.sum(), x)
    want, soft, dist = exact(src, labels)
    check_lp(lp, want, v)
    check_grad(d, soft, dist, labels, torch.ones(n, device="cuda"), torch.bfloat16)


def sequences(n, s, seed):
    rs = np.random.RandomState(seed)
    row_seq = rs.randint(-1, max(s - 1, 1), size=n).astype(np.int32)  # the last sequence stays empty
    if s == 1:
        row_seq = np.minimum(row_seq, 0)
    return row_seq


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,s", [(1, 3, 1), (40, 385, 6), (700, 130, 300), (20, 20011, 4), (3000, 70, 2)])
def test_sequence_log_probs(n, v, s, dtype):
    from fast_jtnn_hip import SequencePlan, sequence_log_probs

    x, labels = make(n, v, dtype, n + v)
    row_seq = sequences(n, s, n)
    labels[torch.from_numpy(row_seq).cuda() < 0] = 0  # a row outside every sequence counts nowhere, label or not
    if n > 5:
        labels[3] = -1
        x[int(np.argmax(row_seq < 0))] = float("nan")
    x.requires_grad_()
    plan = SequencePlan(row_seq, s, "cuda")
    got = sequence_log_probs(x, labels, plan)
    coef = torch.randn(s, device="cuda")
    (d,) = torch.autograd.grad(got, x, coef)
    member = torch.from_numpy(row_seq).cuda().long()
    used = torch.where(member >= 0, labels, -1)
    want, soft, dist = exact(torch.nan_to_num(x.detach()), used)
    total = torch.zeros(s + 1, dtype=torch.float64, device="cuda").index_add_(0, torch.where(member < 0, s, member), want)[:s]
    longest = np.bincount(row_seq[row_seq >= 0], minlength=1).max()
    assert ((got.double() - total).abs() <= longest * sum_error(v) + total.abs() * 2.0 ** -24).all()
    check_grad(d, soft, dist, used, torch.where(member < 0, 0.0, coef[member.clamp(min=0)]), dtype)


def preference_oracle(x, labels, row_seq, pairs, ref, beta, smooth, other, scale):
    x = x.detach().double().requires_grad_()
    member = torch.from_numpy(row_seq).cuda().long()
    keep = (member >= 0) & (labels >= 0)
    lp = torch.log_softmax(x, 1)[torch.arange(len(labels), device="cuda"), labels.clamp(min=0)]
    s = torch.zeros(len(ref), dtype=torch.float64, device="cuda").index_add(0, member[keep], lp[keep])
    o = other.detach().double().requires_grad_()
    s = s + o
    p = torch.from_numpy(pairs).cuda().long()
    margin = beta * ((s - ref.double())[p[:, 0]] - (s - ref.double())[p[:, 1]])
    ls = torch.nn.functional.logsigmoid
    loss = scale * -((1 - smooth) * ls(margin) + smooth * ls(-margin)).sum()
    grads = torch.autograd.grad(loss, (x, o, s))
    return loss.detach(), s.detach(), margin.detach(), grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,s,p", [(2, 5, 2, 1), (160, 385, 16, 8), (900, 60, 301, 1500), (64, 20011, 8, 5),
                                     (5000, 33, 4, 7)])
def test_preference_loss(n, v, s, p, dtype):
    """Sequences that stand in several pairs, on both sides, or with themselves; empty ones; rows out of order."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    rs = np.random.RandomState(n)
    x, labels = make(n, v, dtype, n * 3 + v)
    row_seq = sequences(n, s, n + 1) if n > 2 else np.array([0, 1], dtype=np.int32)
    pairs = rs.randint(0, s, size=(p, 2)).astype(np.int32)
    if p > 4:
        pairs[1] = (1, 1)
        pairs[2] = pairs[0]
        labels[4] = -1
    plan = SequencePlan(row_seq, s, "cuda", pairs=pairs)
    other = torch.randn(s, device="cuda").requires_grad_()
    member = torch.from_numpy(row_seq).cuda().long()
    lp, soft, dist = exact(x, torch.where(member >= 0, labels, -1))
    sums = torch.zeros(s + 1, dtype=torch.float64, device="cuda").index_add_(0, torch.where(member < 0, s, member), lp)[:s]
    ref = (sums + torch.randn(s, device="cuda") * 3).float()
    x.requires_grad_()
    longest = max(1, np.bincount(row_seq[row_seq >= 0], minlength=1).max())
    for beta, smooth, scale in ((0.1, 0.0, None), (0.7, 0.2, 2.5)):
        r = preference_loss(x, labels, plan, ref, beta=beta, label_smoothing=smooth, other_log_probs=other, scale=scale)
        d, do = torch.autograd.grad(r.loss * 3, (x, other))
        k = scale or 1.0 / p
        loss, want_s, margin, (_, go, gs) = preference_oracle(x, labels, row_seq, pairs, ref, beta, smooth, other, k)
        s_err = longest * sum_error(v)
        assert ((r.log_probs.double() - want_s).abs() <= s_err + want_s.abs() * 2.0 ** -24).all()
        m_err = 2 * beta * s_err
        assert ((r.margins.double() - margin).abs() <= m_err + margin.abs() * 2.0 ** -24).all()
        # |d loss / d margin| <= k per pair
        assert (r.loss.double() - loss).abs() <= p * k * m_err + loss.abs() * 2.0 ** -23
        # d^2 loss / d margin^2 <= k / 4 per pair that names the sequence, times beta, times the upstream 3
        named = torch.from_numpy(np.bincount(pairs.reshape(-1), minlength=s)).cuda().double()
        c_err = 3 * (named * k * beta * m_err / 4 + gs.abs() * 2.0 ** -22) + 1e-12
        assert ((do.double() - 3 * go).abs() <= c_err).all()
        coef = torch.where(member < 0, 0.0, 3 * gs[member.clamp(min=0)])
        used = torch.where(member >= 0, labels, -1)
        want = exact_grad(soft, used, coef)
        e = torch.where(member < 0, 0.0, c_err[member.clamp(min=0)])
        fi = torch.finfo(dtype)
        tol = (coef.abs()[:, None] * soft * (sum_error(v) + 2.0 ** -23 * (dist + 4)) + e[:, None]
               + coef.abs()[:, None] * 2.0 ** -21 + want.abs() * fi.eps / 2
               + (fi.smallest_normal if dtype != torch.float16 else 2.0 ** -24))
        assert ((d.double() - want).abs() <= tol).all()


def test_preference_far_margins_and_no_pairs():
    """A sequence that has become impossible (log-probability -inf) gives an infinite margin: no NaN in the loss, the
    full coefficient; without pairs the loss is zero and so is the gradient."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    x, labels = make(4, 9, torch.float32, 2)
    labels[:] = 1
    x[2, 1] = -float("inf")
    x.requires_grad_()
    ref = torch.zeros(2, device="cuda")
    plan = SequencePlan([0, 0, 1, 1], 2, "cuda", pairs=[[0, 1]])
    r = preference_loss(x, labels, plan, ref)
    assert r.margins[0] == float("inf") and r.loss == 0 and r.log_probs[1] == -float("inf")
    plan = SequencePlan([0, 0, 1, 1], 2, "cuda", pairs=[[1, 0]])
    r = preference_loss(x, labels, plan, ref, beta=0.25)
    assert r.margins[0] == -float("inf") and r.loss == float("inf")
    (d,) = torch.autograd.grad(r.loss, x)
    _, soft, dist = exact(x, labels)
    coef = torch.tensor([0.25, 0.25, -0.25, -0.25], device="cuda")
    check_grad(d, soft, dist.clamp(max=2000), labels, coef, torch.float32)
    plan = SequencePlan([0, 0, 1, 1], 2, "cuda", pairs=np.zeros((0, 2), np.int32))
    r = preference_loss(x, labels, plan, ref)
    (d,) = torch.autograd.grad(r.loss, x)
    assert r.loss == 0 and r.margins.shape == (0,) and (d == 0).all()


def policy_oracle(x, labels, old, adv, ref, w, lo, hi, kc, scale):
    x = x.detach().double()
    lp = torch.log_softmax(x, 1)[torch.arange(len(labels), device="cuda"), labels.clamp(min=0)]
    lp = torch.where(labels >= 0, lp, 0.0).requires_grad_()
    keep = (labels >= 0).double()
    ww = scale * keep * (1.0 if w is None else w.double())
    r, a = torch.exp(lp - old.double()), adv.double()
    cut = torch.clamp(r, 1 - lo, 1 + hi) * a
    k3 = torch.zeros_like(lp) if ref is None else torch.exp(ref.double() - lp) - (ref.double() - lp) - 1
    loss = (ww * (kc * k3 - torch.minimum(r * a, cut))).sum()
    (g,) = torch.autograd.grad(loss, lp)
    return loss.detach(), lp.detach(), (ww * k3).sum().detach(), (ww * (cut < r * a)).sum().detach(), g, ww, r.detach()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(1, 2), (64, 385), (500, 61), (40, 20011), (3, 131072), (2000, 300), (600, 4099)])
def test_policy_loss(n, v, dtype):
    from fast_jtnn_hip import policy_loss

    x, labels = make(n, v, dtype, n + 7 * v)
    if n > 3:
        labels[2] = -5
        x[2] = float("nan")
    lp = exact(torch.nan_to_num(x), labels)[0]
    g = torch.Generator(device="cuda").manual_seed(n)
    step = 0.3 * torch.randn(n, generator=g, device="cuda")
    for border in (math.log(0.8), math.log(1.2), math.log(0.9), math.log(1.4)):  # no ratio where the gradient jumps
        step = torch.where((step - border).abs() < 2e-3, step + 5e-3, step)
    old = (lp - step).float()
    ref = (lp + 0.3 * torch.randn(n, generator=g, device="cuda")).float()
    adv = torch.randn(n, generator=g, device="cuda")
    w = torch.rand(n, generator=g, device="cuda")
    x.requires_grad_()
    _, soft, dist = exact(torch.nan_to_num(x.detach()), labels)
    for clip, kc, rf, wt, scale, up in ((0.2, 0.05, ref, w, 1.0 / n, 1.0), ((0.1, 0.4), 0.0, None, None, 1.0, -2.5),
                                        (0.2, 0.0, ref, None, 0.5, 1.0)):
        out = policy_loss(x, labels, old, adv, ref_log_probs=rf, weights=wt, clip=clip, kl_coef=kc, scale=scale)
        (d,) = torch.autograd.grad(out.loss * up, x)
        lo, hi = clip if isinstance(clip, tuple) else (clip, clip)
        loss, want_lp, kl, clipped, coef, ww, r = policy_oracle(torch.nan_to_num(x.detach()), labels, old, adv, rf, wt, lo,
                                                                hi, kc, scale)
        check_lp(out.log_probs, want_lp, v)
        s = sum_error(v)
        ra = (r * adv.double()).abs()
        assert (out.loss.double() - loss).abs() <= (ww * s * 2 * (ra + kc * 3)).sum() + loss.abs() * 2.0 ** -23 + 1e-12
        assert (out.kl.double() - kl).abs() <= (ww * s * 3).sum() + kl.abs() * 2.0 ** -23 + 1e-12
        assert (out.clipped.double() - clipped).abs() <= clipped * 2.0 ** -23
        c_err = abs(up) * (ww * s * 2 * (ra + kc * 3)) + (coef * up).abs() * 2.0 ** -22
        want = exact_grad(soft, labels, coef * up)
        fi = torch.finfo(dtype)
        tol = ((coef * up).abs()[:, None] * (soft * (s + 2.0 ** -23 * (dist + 4)) + 2.0 ** -21) + c_err[:, None]
               + want.abs() * fi.eps / 2 + (fi.smallest_normal if dtype != torch.float16 else 2.0 ** -24))
        assert ((d.double() - want).abs() <= tol).all()
        assert (d[labels < 0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(1, 4096), (1, 8191), (1, 8192), (2, 8209), (4, 128000), (64, 20011), (65, 20011), (3, 600011)])
def test_sums_of_a_few_long_rows(n, v, dtype):
    """Long rows with others that do not count, -inf, NaN and a single finite logit among them; a row's value is the same
    among few and alone, and the gradient works from the statistics left behind."""
    from fast_jtnn_hip import SequencePlan, sequence_log_probs

    x, labels = make(n, v, dtype, n + v, ld=v + 1, offset=1)
    owner = np.arange(n) % 3
    x[0, v // 2:] = float("-inf")
    labels[0] = v // 3
    if n > 3:
        owner[1] = -1
        x[1] = float("nan")
        x[2] = float("-inf")
        x[2, v - 1] = 3.0
        labels[2] = v - 1
        labels[3] = -1
    x.requires_grad_()
    sums = sequence_log_probs(x, labels, SequencePlan(owner, 4, "cuda"))
    counted = torch.tensor(owner, device="cuda") >= 0
    keep = torch.where(counted, labels, -1)
    lp, soft, dist = exact(torch.nan_to_num(x.detach(), nan=0.0, posinf=None, neginf=float("-inf")), keep)
    want = torch.zeros(4, dtype=torch.float64, device="cuda").index_add_(0, torch.tensor(owner, device="cuda").clamp(min=0), lp)
    rows = -(-n // 3)
    assert ((sums.double() - want).abs() <= rows * sum_error(v) + want.abs() * 2.0 ** -23).all()
    alone = [sequence_log_probs(x[i:i + 1], labels[i:i + 1], SequencePlan([0], 1, "cuda")) for i in range(min(n, 3))]
    if n <= 3:
        assert torch.equal(torch.cat(alone), sums[:n])
    (d,) = torch.autograd.grad(sums.sum(), x)
    check_grad(d, soft, dist, keep, torch.ones(n, device="cuda"), dtype)
    bad = x.detach().clone()
    bad[0, 5] = float("nan")
    assert torch.isnan(sequence_log_probs(bad[:1], labels[:1], SequencePlan([0], 1, "cuda"))).all()


@pytest.mark.parametrize("n,v,dtype", [(40, 385, torch.float32), (9, 4099, torch.bfloat16), (6, 30011, torch.float16),
                                       (4, 70001, torch.float32)])
def test_nothing_comes_from_behind_a_mask(n, v, dtype):
    """Weights of zero, upstream gradients of zero and sequences in no pair, over infinities and NaN: the others' values are
    those of the batch without the masked rows."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, sequence_log_probs, token_log_probs

    x, labels = make(n, v, dtype, n * v)
    x = x.contiguous()
    old, adv, ref = torch.full((n,), -3.0, device="cuda"), torch.randn(n, device="cuda"), torch.full((n,), -2.5, device="cuda")
    masked = torch.arange(n, device="cuda") % 2 == 1
    w = torch.where(masked, 0.0, 0.5)
    bad = x.clone()
    bad[1::2] = float("nan")
    bad[1] = float("-inf")
    bad[3, 0] = float("inf")
    labels[3] = v + 5
    olds, advs, refs = (torch.where(masked, b, t) for t, b in ((old, -math.inf), (adv, math.nan), (ref, math.inf)))
    bad.requires_grad_()
    kept = x[::2].detach().requires_grad_()  # a view: rows at the same distance from 16-byte boundaries, so the same bits

    def same(d, want):
        assert (d[1::2] == 0).all() and torch.equal(d[::2], want)

    out = policy_loss(bad, labels, olds, advs, ref_log_probs=refs, weights=w, kl_coef=0.1)
    few = policy_loss(kept, labels[::2], old[::2], adv[::2], ref_log_probs=ref[::2], weights=w[::2], kl_coef=0.1)
    for f in ("loss", "kl", "clipped"):
        a, b = float(getattr(out, f)), float(getattr(few, f))
        assert abs(a - b) <= 2.0 ** -22 * abs(b) and math.isfinite(b)  # the same terms, perhaps in another order
    for up in (1.0, -2.0):  # made with the forward pass, and made again
        one = torch.tensor(up, device="cuda")
        same(torch.autograd.grad(out.loss, bad, one, retain_graph=True)[0],
             torch.autograd.grad(few.loss, kept, one, retain_graph=True)[0])
    lp = token_log_probs(bad, labels)
    a = torch.where(masked, 0.0, lp).sum()
    same(torch.autograd.grad(a, bad)[0], torch.autograd.grad(token_log_probs(kept, labels[::2]).sum(), kept)[0])
    a = sequence_log_probs(bad, labels, SequencePlan(np.arange(n) % 2, 2, "cuda"))[0]
    b = sequence_log_probs(kept, labels[::2], SequencePlan(np.zeros(len(kept), np.int32), 1, "cuda"))[0]
    assert torch.equal(a, b)
    same(torch.autograd.grad(a, bad)[0], torch.autograd.grad(b, kept)[0])
    # sequences 0 and 2 are a pair, 1 and 3 (the masked rows) are in none
    plan = SequencePlan(np.arange(n) % 4, 4, "cuda", pairs=[[0, 2]])
    less = SequencePlan(np.arange(n)[::2] % 4 // 2, 2, "cuda", pairs=[[0, 1]])
    r = preference_loss(bad, labels, plan, torch.tensor([0.0, math.nan, 0.0, math.inf], device="cuda"))
    q = preference_loss(kept, labels[::2], less, torch.zeros(2, device="cuda"))
    assert torch.equal(r.loss, q.loss)
    same(torch.autograd.grad(r.loss, bad)[0], torch.autograd.grad(q.loss, kept)[0])


def test_an_infinite_estimate_without_a_penalty():
    """kl_coef = 0: an infinite KL estimate is reported and does not touch the loss."""
    from fast_jtnn_hip import policy_loss

    x, labels = make(8, 385, torch.float32, 3)
    x.requires_grad_()
    old, adv = torch.full((8,), -2.0, device="cuda"), torch.ones(8, device="cuda")
    ref = torch.full((8,), -math.inf, device="cuda")
    out, want = policy_loss(x, labels, old, adv, ref_log_probs=ref), policy_loss(x, labels, old, adv)
    assert float(out.kl) == math.inf and torch.equal(out.loss, want.loss)
    assert torch.equal(torch.autograd.grad(out.loss, x)[0], torch.autograd.grad(want.loss, x)[0])


def test_no_rows():
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, sequence_log_probs

    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    f = torch.zeros(0, device="cuda")
    plan = SequencePlan(np.zeros(0, np.int32), 3, "cuda", pairs=[[0, 1], [2, 2]])
    assert torch.equal(sequence_log_probs(x, y, plan), torch.zeros(3, device="cuda"))
    r = preference_loss(x, y, plan, torch.tensor([0.0, 2.0, 0.0], device="cuda"), beta=1.0)
    want = (math.log1p(math.exp(-2.0)) + math.log(2.0)) / 2
    assert abs(float(r.loss) - want) < 1e-6
    out = policy_loss(x, y, f, f)
    assert float(out.loss) == 0 and out.log_probs.shape == (0,)
    for t in (r.loss, out.loss):
        assert torch.autograd.grad(t, x)[0].shape == (0, 5)
    none = SequencePlan(np.full(4, -1, np.int32), 0, "cuda", pairs=np.zeros((0, 2), np.int32))
    z = torch.randn(4, 5, device="cuda", requires_grad=True)
    r = preference_loss(z, torch.zeros(4, dtype=torch.int64, device="cuda"), none, torch.zeros(0, device="cuda"))
    assert float(r.loss) == 0 and (torch.autograd.grad(r.loss, z)[0] == 0).all()


def test_gradients_against_differences():
    """Central differences of the calls themselves, step h = 2^-6: the loss (about 1) is off by 2^-22, so a difference
    by 2^-22 / h = 2^-16, and the cubic term by h^2 / 6 |f'''| with |f'''| below 4 here."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss

    x, labels = make(4, 6, torch.float32, 21)
    labels[3] = -1
    plan = SequencePlan([0, 1, 0, 1], 2, "cuda", pairs=[[0, 1]])
    f = torch.tensor([-1.0, -2.0, -1.5, 0.0], device="cuda")
    adv = torch.tensor([0.5, -0.6, 0.4, 1.0], device="cuda")
    ref = torch.tensor([-3.0, -2.5], device="cuda")
    calls = [lambda t: preference_loss(t, labels, plan, ref, beta=0.5, label_smoothing=0.1).loss,
             lambda t: policy_loss(t, labels, f, adv, ref_log_probs=f - 0.2, clip=(0.95, 20.0), kl_coef=0.1, scale=0.3).loss]
    h = 2.0 ** -6
    for call in calls:
        leaf = x.clone().requires_grad_()
        (d,) = torch.autograd.grad(call(leaf), leaf)
        for i in range(4):
            for j in range(6):
                up, down = x.clone(), x.clone()
                up[i, j] += h
                down[i, j] -= h
                diff = (call(up).double() - call(down).double()) / (2 * h)
                assert abs(float(diff) - float(d[i, j])) <= 2.0 ** -16 + h * h / 6 * 4, (i, j)


def test_backward_twice_and_no_second_derivative():
    """retain_graph: the second pass with another upstream factor gives its own gradient and leaves the first alone."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, token_log_probs

    n, v = 30, 700
    x, labels = make(n, v, torch.bfloat16, 4)
    x.requires_grad_()
    old = torch.full((n,), -2.0, device="cuda")
    adv = torch.randn(n, device="cuda")
    plan = SequencePlan(np.arange(n) % 4, 4, "cuda", pairs=[[0, 1], [2, 3]])
    for call in (lambda: policy_loss(x, labels, old, adv, clip=(0.9, 50.0)).loss,
                 lambda: preference_loss(x, labels, plan, torch.zeros(4, device="cuda")).loss):
        loss = call()
        (a,) = torch.autograd.grad(loss, x, retain_graph=True)
        keep = a.clone()
        (b,) = torch.autograd.grad(loss, x, torch.tensor(4.0, device="cuda"), retain_graph=True)
        (c,) = torch.autograd.grad(loss, x)
        assert torch.equal(a, keep) and torch.equal(a, c) and torch.equal(b, 4 * a)  # a power of two: exact
        assert a.data_ptr() != b.data_ptr() and a.data_ptr() != c.data_ptr()
        again = call()
        (d,) = torch.autograd.grad(again, x)
        assert torch.equal(a, d)  # no atomics: bit for bit
    lp = token_log_probs(x.float(), labels)
    y = x.detach().float().requires_grad_()
    (g,) = torch.autograd.grad(token_log_probs(y, labels).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert lp.requires_grad


def test_changed_logits_are_noticed():
    from fast_jtnn_hip import policy_loss, token_log_probs

    x, labels = make(5, 40, torch.float32, 6)
    f = torch.zeros(5, device="cuda")
    for call in (lambda t: token_log_probs(t, labels).sum(), lambda t: policy_loss(t, labels, f, f + 1).loss * 2):
        leaf = x.clone().requires_grad_()
        y = leaf * 1.0
        loss = call(y)
        with torch.no_grad():
            y.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_only_the_other_terms_need_a_gradient():
    from fast_jtnn_hip import SequencePlan, preference_loss

    x, labels = make(6, 40, torch.float32, 6)
    plan = SequencePlan([0, 0, 0, 1, 1, 1], 2, "cuda", pairs=[[0, 1]])
    other = torch.zeros(2, dtype=torch.float64, device="cuda", requires_grad=True)
    loss = preference_loss(x, labels, plan, torch.zeros(2, device="cuda"), other_log_probs=other).loss
    loss.backward()
    assert other.grad.dtype == torch.float64 and float(other.grad.sum()) == 0 and float(other.grad.abs().sum()) > 0


def test_on_another_stream():
    """Inputs and plan made on the default stream, used on a side stream, and freed there while work is queued."""
    from fast_jtnn_hip import SequencePlan, preference_loss

    x, labels = make(400, 3001, torch.float16, 9)
    x.requires_grad_()
    ref = torch.zeros(8, device="cuda")
    pairs = [[0, 1], [2, 3], [4, 5], [6, 7]]
    row_seq = np.arange(400) % 8

    def run():
        plan = SequencePlan(row_seq, 8, "cuda", pairs=pairs)
        r = preference_loss(x, labels, plan, ref)
        return r.loss.detach(), torch.autograd.grad(r.loss, x)[0]

    loss, d = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in got:
        assert torch.equal(a, loss) and torch.equal(b, d)


@pytest.mark.parametrize("n,v,dtype", [(50, 385, torch.float32), (6, 30011, torch.bfloat16), (700, 3001, torch.float16)])
def test_captured_and_replayed(n, v, dtype):
    """Forward and backward of all three in one graph, replayed on changed inputs with eager work in between."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, token_log_probs

    x, labels = make(n, v, dtype, 14)
    x = x.contiguous().requires_grad_()
    plan = SequencePlan(np.arange(n) % 4, 4, "cuda", pairs=[[0, 1], [2, 3]])
    ref = torch.zeros(4, device="cuda")
    old, adv = torch.full((n,), -3.0, device="cuda"), torch.randn(n, device="cuda")

    def step():
        lp = token_log_probs(x, labels)
        a = torch.autograd.grad(lp, x, adv)[0]
        r = preference_loss(x, labels, plan, ref)
        b = torch.autograd.grad(r.loss, x)[0]
        p = policy_loss(x, labels, old, adv, ref_log_probs=old, kl_coef=0.1)
        c = torch.autograd.grad(p.loss, x)[0]
        q = policy_loss(x, labels, old, adv)
        e = torch.autograd.grad(q.loss * 0.5, x)[0]
        return [t.detach() for t in (lp, a, r.loss, r.margins, b, p.loss, p.kl, c, e)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(make(n, v, dtype, 100 + k)[0])
            labels.copy_(make(n, v, dtype, 100 + k)[1])
            labels[k] = -1
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), (k, i)


def test_backward_captured_alone():
    """An eager forward pass whose backward pass is captured: every replay writes the whole gradient, into memory of the
    graph's own, whatever became of the last replay's."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, sequence_log_probs, token_log_probs

    n, v = 24, 385
    x, labels = make(n, v, torch.float32, 15)
    x = x.contiguous().requires_grad_()
    plan = SequencePlan(np.arange(n) % 4, 4, "cuda", pairs=[[0, 1], [2, 3]])
    ref, adv = torch.zeros(4, device="cuda"), torch.randn(n, device="cuda")
    old = torch.full((n,), -3.0, device="cuda")
    other = torch.zeros(4, device="cuda", requires_grad=True)
    calls = [(lambda: token_log_probs(x, labels).sum(), [x]),
             (lambda: sequence_log_probs(x, labels, plan).sum(), [x]),
             (lambda: preference_loss(x, labels, plan, ref, other_log_probs=other).loss, [x, other]),
             (lambda: policy_loss(x, labels, old, adv).loss, [x])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses = [f() for f, _ in calls]
        want = [torch.autograd.grad(f(), leaves) for f, leaves in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = [torch.autograd.grad(loss, leaves, retain_graph=True) for loss, (_, leaves) in zip(losses, calls)]
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            for p, q in zip(a, b):
                assert torch.equal(p, q), (k, i)
                p.fill_(float("nan"))


def test_more_rows_than_one_launch_takes():
    """68 million rows of two columns: more work-items than a grid may have, so several launches."""
    from fast_jtnn_hip import policy_loss, token_log_probs

    n = 68_000_000
    x = torch.zeros(n, 2, dtype=torch.float16, device="cuda")
    labels = torch.zeros(n, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    spots = [slice(0, 1000), slice(n // 2 - 500, n // 2 + 500), slice((1 << 25) - 500, (1 << 25) + 500), slice(n - 1000, n)]
    for s in spots:
        x[s] = torch.randn(1000, 2, generator=g, device="cuda").half()
        labels[s] = torch.randint(0, 2, (1000,), generator=g, device="cuda").int()
    x.requires_grad_()
    coef = torch.ones(n, device="cuda")
    lp = token_log_probs(x, labels)
    (d,) = torch.autograd.grad(lp, x, coef)
    out = policy_loss(x, labels, torch.full((n,), -0.5, device="cuda"), coef, clip=(0.9, 9.0))
    (e,) = torch.autograd.grad(out.loss, x)
    for s in spots:
        want, soft, dist = exact(x[s], labels[s])
        check_lp(lp[s], want, 2)
        check_lp(out.log_probs[s], want, 2)
        check_grad(d[s], soft, dist, labels[s].long(), coef[s], torch.float16)
        check_grad(e[s], soft, dist, labels[s].long(), -torch.exp(want + 0.5).float(), torch.float16)
    assert abs(float(out.loss) + math.exp(0.5) * float(torch.exp(lp.double()).sum())) <= 1e-5 * n


def test_nothing_is_made_for_a_gradient_nobody_wants():
    from fast_jtnn_hip import policy_loss

    x, labels = make(2000, 30000, torch.bfloat16, 3)
    f = torch.full((2000,), -2.0, device="cuda")
    x.requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        a = policy_loss(x, labels, f, f)
    assert not a.loss.requires_grad and torch.cuda.max_memory_allocated() - before < 4 << 20
    b = policy_loss(x, labels, f, f)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.log_probs, b.log_probs)


def test_inputs_on_the_host_are_refused():
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, token_log_probs

    x, labels = make(4, 9, torch.float32, 2)
    plan = SequencePlan([0, 0, 1, 1], 2, "cuda", pairs=[[0, 1]])
    f, two = torch.zeros(4, device="cuda"), torch.zeros(2, device="cuda")
    for call in (lambda: token_log_probs(x, labels.cpu()), lambda: preference_loss(x, labels, plan, two.cpu()),
                 lambda: preference_loss(x, labels, plan, two, other_log_probs=two.cpu()),
                 lambda: policy_loss(x, labels, f, f.cpu()), lambda: policy_loss(x, labels, f, f, weights=f.cpu())):
        with pytest.raises(RuntimeError, match="logits are on"):
            call()


def test_calls_are_timed_like_the_others():
    from fast_jtnn_hip import AdamW, SequencePlan, preference_loss
    from fast_jtnn_hip import _capi as K

    x, labels = make(40, 500, torch.float16, 2)
    x = torch.nn.Parameter(x.clone())
    plan = SequencePlan(np.arange(40) % 2, 2, "cuda", pairs=[[0, 1]])
    opt = AdamW([x], max_norm=1.0)
    with K.KernelTimer() as t:
        preference_loss(x, labels, plan, torch.zeros(2, device="cuda")).loss.backward()
        opt.step()
    got = t.summary()
    assert set(got) == {"preference_loss", "label_log_probs_bwd", "adamw_step"}
    assert got["label_log_probs_bwd"]["bytes"] >= 2 * 40 * 500 * 2
    assert got["adamw_step"]["bytes"] >= 40 * 500 * (2 * 2 + 8 + 16)


def test_saved_tensors_that_come_back_elsewhere():
    """Hooks that move saved tensors to the host and back: the backward pass reads them where they are now."""
    from fast_jtnn_hip import SequencePlan, policy_loss, preference_loss, token_log_probs

    x, labels = make(30, 700, torch.float32, 5)
    plan = SequencePlan(np.arange(30) % 2, 2, "cuda", pairs=[[0, 1]])
    two, f = torch.zeros(2, device="cuda"), torch.full((30,), -1.0, device="cuda")
    for call in (lambda y: token_log_probs(y, labels).sum(), lambda y: preference_loss(y, labels, plan, two).loss,
                 lambda y: policy_loss(y, labels, f, f).loss * 2):
        got = []
        for moved in (False, True):
            leaf = x.clone().requires_grad_()
            if moved:
                with torch.autograd.graph.save_on_cpu():
                    loss = call(leaf * 1.0)
            else:
                loss = call(leaf * 1.0)
            junk = torch.full((40, 900), 7.0, device="cuda")  # takes the place of what was freed
            loss.backward()
            got.append(leaf.grad)
            del junk
        assert torch.equal(*got)


def test_two_threads_at_once():
    """Calls from two host threads on streams of their own."""
    import threading

    from fast_jtnn_hip import policy_loss

    x, labels = make(300, 5000, torch.bfloat16, 6)
    f = torch.full((300,), -2.0, device="cuda")
    leaf = x.clone().requires_grad_()
    want = torch.autograd.grad(policy_loss(leaf, labels, f, f).loss, leaf)[0]
    torch.cuda.synchronize()
    bad = []

    def work(seed):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            y = x.clone().requires_grad_()
            for _ in range(20):
                r = policy_loss(y, labels, f, f)
                (d,) = torch.autograd.grad(r.loss, y)
                s.synchronize()
                if not torch.equal(d, want):
                    bad.append(seed)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad
