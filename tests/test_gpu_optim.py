"""GPU: the AdamW step against its formulas in 64 bits.

Tolerances.  Every element takes a handful of 32-bit operations on 32-bit states: a moment is off by at most
4 * 2^-24 of the sum of its two terms' magnitudes (two rounded factors, two roundings), the second moment likewise with
one more product (6 * 2^-24), the update m / (sqrt(v) b + eps) by 2^-24 times 16 of what the terms of m allow, the
weight by two roundings of its own.  With the clip, the factor adds 2^-23 to the gradient and 2^-22 to its square."""
import copy
import io
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1,), (3, 5), (255,), (256,), (257,), (4096,), (4097,), (450, 385), (0,), (12289,), (1000, 33)]


def params_of(shapes, dtype, seed, flat_offset=None):
    """Parameters with gradients; ``flat_offset``: all of them views of one buffer at odd places."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    numels = [int(np.prod(s)) for s in shapes]
    if flat_offset is not None:
        wb = (torch.randn(sum(numels) + flat_offset, generator=g, device="cuda") * 0.1).to(dtype)
        gb = (torch.randn(sum(numels) + flat_offset, generator=g, device="cuda") * 0.01).to(dtype)
    out, at = [], flat_offset
    for s, n in zip(shapes, numels):
        if flat_offset is not None:
            p = torch.nn.Parameter(wb[at:at + n].view(s))
            p.grad = gb[at:at + n].view(s)
            at += n
        else:
            p = torch.nn.Parameter((torch.randn(s, generator=g, device="cuda") * 0.1).to(dtype))
            p.grad = (torch.randn(s, generator=g, device="cuda") * 0.01).to(dtype)
        out.append(p)
    return out


def deq(state, name):
    """Values an 8-bit state stands for, in 64 bits, and the scale of every element."""
    q, sc = state[name].double().reshape(-1), state[name + "_scale"].double()
    per = sc.repeat_interleave(256)[:q.numel()]
    return q * per, per


def snapshot(opt, p):
    s = opt.state[p]
    d = {k: v.clone() for k, v in s.items()}
    d["w"] = (s["master"] if "master" in s else p.detach()).double().reshape(-1).clone()
    return d


def moments(d, bits):
    if bits == 32:
        return d["exp_avg"].double().reshape(-1), d["exp_avg_sq"].double().reshape(-1)
    return deq(d, "exp_avg")[0], deq(d, "exp_rms")[0] ** 2


def half_step(q):
    """Half the distance between neighbouring e4m3 values around |q|."""
    e = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
    return torch.exp2(e - 3) / 2


def check_step(opt, params, before, grads, lr, betas, eps, wd, bits, factor=1.0, fac_err=0.0):
    b1, b2 = betas
    for p, d, g in zip(params, before, grads):
        s = opt.state[p]
        if g is None or p.numel() == 0:
            for k in d:
                if k != "w" and p.numel():
                    assert torch.equal(s[k].view(torch.uint8) if s[k].dtype == torch.float8_e4m3fn else s[k],
                                       d[k].view(torch.uint8) if d[k].dtype == torch.float8_e4m3fn else d[k])
            continue
        t = int(d["step"]) + 1
        assert int(s["step"]) == t
        g = g.double().reshape(-1) * factor
        m0, v0 = moments(d, bits)
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        m_err = (4 * U + fac_err) * (b1 * m0.abs() + (1 - b1) * g.abs()) + 2.0 ** -149
        v_err = (6 * U + 2 * fac_err) * v + 2.0 ** -149
        den = torch.sqrt(v / (1 - b2 ** t)) + eps
        upd = lr / (1 - b1 ** t) * m / den
        w = d["w"] * (1 - lr * wd) - upd
        # 1 - b of a beta near 1, rounded to 32 bits, moves nothing else: bias corrections are formed in 64 bits
        u_err = lr / (1 - b1 ** t) * (m_err + 12 * U * m.abs()) / den + upd.abs() * (v_err / v.clamp(min=1e-300)).clamp(max=1)
        w_err = u_err + 4 * U * d["w"].abs() + 2 * U * w.abs()
        now = s["master"] if "master" in s else p.detach()
        if "master" in s or p.dtype == torch.float32:
            assert ((now.double().reshape(-1) - w).abs() <= w_err).all(), (p.shape, p.dtype)
        if "master" in s:
            assert torch.equal(p.detach(), s["master"].to(p.dtype))
        elif p.dtype != torch.float32:
            fi = torch.finfo(p.dtype)
            assert ((now.double().reshape(-1) - w).abs() <= w_err + w.abs() * fi.eps / 2 * 1.001 + 2.0 ** -25).all()
        if bits == 32:
            assert ((s["exp_avg"].double().reshape(-1) - m).abs() <= m_err).all()
            assert ((s["exp_avg_sq"].double().reshape(-1) - v).abs() <= v_err).all()
            continue
        r = torch.sqrt(v)
        for name, want, err in (("exp_avg", m, m_err), ("exp_rms", r, r * (4 * U + fac_err) + 1e-22)):
            got, per = deq(s, name)
            top, off = (torch.zeros(-(-want.numel() // 256) * 256, dtype=torch.float64, device="cuda") for _ in range(2))
            top[:want.numel()], off[:want.numel()] = want.abs(), err
            # a maximum is off by no more than its elements are (where the two terms of m cancel, that is many times its
            # own rounding), and is divided by 448
            top, off = (t.view(-1, 256).max(1).values for t in (top, off))
            assert ((s[name + "_scale"].double() * 448 - top).abs() <= off + top * 4 * U + 2.0 ** -100).all()
            q = s[name].double().reshape(-1)
            tol = half_step(q) * per * (1 + 1e-5) + err + want.abs() * 32 * U
            if name == "exp_rms":  # what is not zero keeps at least the smallest value
                tol = torch.where(q == 2.0 ** -9, 2.0 ** -9 * per * (1 + 1e-5) + err, tol)
                assert ((q > 0) | (want <= 2.0 ** -100)).all()
            assert ((got - want).abs() <= tol).all(), (name, ((got - want).abs() / tol).max())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, True), (torch.float16, True), (torch.bfloat16, True),
                                          (torch.float16, False), (torch.bfloat16, False)])
def test_steps(dtype, master, bits):
    """Three steps over odd sizes, parameters at odd places of one buffer, one parameter without a gradient."""
    from fast_jtnn_hip import AdamW

    for flat in (None, 1):
        ps = params_of(SHAPES, dtype, 3, flat)
        opt = AdamW(ps, lr=1e-2, betas=(0.9, 0.95), eps=1e-6, weight_decay=0.1, state_bits=bits, master=master)
        for step in range(3):
            if step == 1:
                ps[4].grad = None
            else:
                for i, q in enumerate(ps):
                    if q.grad is None or step:
                        q.grad = (torch.randn_like(q, dtype=torch.float32) * 0.01).to(dtype)
            grads = [None if p.grad is None else p.grad.clone() for p in ps]
            before = [snapshot(opt, p) for p in ps]
            lr = 1e-2 / (step + 1)
            opt.param_groups[0]["lr"] = lr
            opt.step()
            check_step(opt, ps, before, grads, lr, (0.9, 0.95), 1e-6, 0.1, bits)
            for p, g in zip(ps, grads):
                assert g is None or torch.equal(p.grad, g)  # gradients stay as they were
        assert int(opt.state[ps[4]]["step"]) == 2 and int(opt.state[ps[5]]["step"]) == 3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clip(dtype, bits):
    from fast_jtnn_hip import AdamW

    ps = params_of(SHAPES, dtype, 5)
    ps[7].grad = None
    total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps if p.grad is not None))
    for max_norm in (total / 3, total * 2):
        opt = AdamW(ps, lr=1e-3, weight_decay=0.0, state_bits=bits, max_norm=max_norm)
        grads = [None if p.grad is None else p.grad.clone() for p in ps]
        before = [snapshot(opt, p) for p in ps]
        opt.step()
        # squares summed in 32 bits over 4 elements, in 64 beyond
        assert abs(float(opt.grad_norm) - total) <= total * 8 * U
        factor = min(1.0, max_norm / (total + 1e-6))
        check_step(opt, ps, before, grads, 1e-3, (0.9, 0.999), 1e-8, 0.0, bits, factor, 0.0 if factor == 1 else 10 * U)


def test_groups_share_one_norm():
    from fast_jtnn_hip import AdamW

    a, b = params_of(SHAPES[:5], torch.float32, 1), params_of(SHAPES[5:], torch.bfloat16, 2)
    total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in a + b))
    opt = AdamW([{"params": a, "weight_decay": 0.0}, {"params": b, "state_bits": 8, "lr": 5e-3}], lr=1e-3,
                weight_decay=0.02, max_norm=total / 2)
    before = [snapshot(opt, p) for p in a + b]
    grads = [p.grad.clone() for p in a + b]
    opt.step()
    factor = 0.5 * total / (total + 1e-6)
    check_step(opt, a, before[:5], grads[:5], 1e-3, (0.9, 0.999), 1e-8, 0.0, 32, factor, 10 * U)
    check_step(opt, b, before[5:], grads[5:], 5e-3, (0.9, 0.999), 1e-8, 0.02, 8, factor, 10 * U)
    bufs = opt.state_buffers()
    assert len(bufs) == 2 and bufs[0]["exp_avg"].dtype == torch.float32
    assert bufs[1]["exp_avg"].dtype == torch.float8_e4m3fn and bufs[1]["master"].dtype == torch.float32


def test_many_tensors():
    """More tensors than one launch carries addresses for; every third without a gradient."""
    from fast_jtnn_hip import AdamW

    rs = np.random.RandomState(0)
    ps = params_of([(int(n),) for n in rs.randint(1, 700, size=1003)], torch.float32, 7)
    for p in ps[::3]:
        p.grad = None
    opt = AdamW(ps, lr=1e-2, max_norm=0.5)
    before = [snapshot(opt, p) for p in ps]
    grads = [None if p.grad is None else p.grad.clone() for p in ps]
    opt.step()
    total = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
    assert abs(float(opt.grad_norm) - total) <= total * 8 * U
    check_step(opt, ps, before, grads, 1e-2, (0.9, 0.999), 1e-8, 0.01, 32, 0.5 / (total + 1e-6), 10 * U)
    for p in ps[::3]:
        assert int(opt.state[p]["step"]) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(bits):
    """Zeros, values next to the type's limits, infinities and NaN: what is not finite spoils its own element only."""
    from fast_jtnn_hip import AdamW

    n = 1024
    p = torch.nn.Parameter(torch.ones(n, device="cuda"))
    p.grad = torch.full((n,), 1e-3, device="cuda")
    p.grad[:256] = 0
    p.grad[256:512] = 1e-30  # squares vanish in 32 bits
    p.grad[600] = float("inf")
    p.grad[601] = float("nan")
    p.grad[700] = 1e18
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
    for _ in range(2):
        opt.step()
    w = p.detach()
    assert (w[:256] == 1).all()
    assert torch.isfinite(w[:600]).all() and torch.isfinite(w[602:]).all()
    assert torch.isnan(w[[600, 601]]).all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[:512] = False
    rest[[600, 601]] = False
    if bits == 8:
        rest[512:768] = False  # 1e18 takes the whole range of its block
    assert ((w[rest] - 0.98).abs() < 1e-5).all()  # constant gradient: every step is the learning rate
    if bits == 8:
        st = opt.state[p]
        assert torch.isnan(st["exp_avg"][[600, 601]].float()).all()
        assert torch.isfinite(st["exp_avg_scale"]).all() and torch.isfinite(st["exp_rms_scale"]).all()
        assert (st["exp_rms"].float()[512:600] > 0).all()  # far below the maximum, not zero


def test_stochastic_rounding():
    """Either neighbour of the exact value, the right one on average, the same in every run; zeros stay zero, roots that
    are not zero stay above it, and what is not finite is marked."""
    from fast_jtnn_hip import AdamW

    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(3)
    grad = torch.randn(n, generator=g, device="cuda") * torch.exp(torch.randn(n, generator=g, device="cuda") * 3)
    grad[:300] = 0
    grad[5000] = float("nan")
    runs = []
    for _ in range(2):
        p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
        p.grad = grad
        opt = AdamW([p], betas=(0.5, 0.75), weight_decay=0.0, state_bits=8, rounding="stochastic")
        opt.step()
        runs.append({k: v.clone() for k, v in opt.state[p].items()})
    s = runs[0]
    for k in s:
        a, b = (r[k].view(torch.uint8) if r[k].dtype == torch.float8_e4m3fn else r[k] for r in runs)
        assert torch.equal(a, b), k
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[5000] = False
    for name, want in (("exp_avg", 0.5 * grad.double()), ("exp_rms", 0.5 * grad.double().abs())):
        got, per = deq(s, name)
        q = s[name].double()
        y = want / per.clamp(min=1e-300)  # exact value in units of the scale
        place = 2 * half_step(torch.minimum(q.abs(), y.abs()))
        err = (q - y)[fine]
        assert (err.abs() <= place[fine] * (1 + 1e-4) + y.abs()[fine] * 1e-6).all()
        assert (q[:256] == 0).all() and torch.isnan(q[5000])
        # mean error: below five standard deviations of n draws of at most half a place each way, element by element
        mid = fine & (y.abs() > 2.0 ** -5)  # the floor of the roots aside
        z = ((q - y) / place)[mid]
        assert abs(float(z.mean())) <= 5 * 0.5 / math.sqrt(z.numel())
        up = float((z > 0).double().mean())
        assert 0.4 < up < 0.6
    assert (s["exp_rms"].float()[300:5000] > 0).all()
    first = s["exp_avg"].view(torch.uint8)
    opt.step()  # another step, other bits
    assert float((opt.state[p]["exp_avg"].view(torch.uint8) != first).double().mean()) > 0.2


def test_stochastic_rounding_follows_gradients_that_nearest_rounding_loses():
    """Half of a block's elements stop receiving gradients, the others go on as before: after two thousand steps at beta2 =
    0.999 the exact root of those is their gradient.  Each stochastic root is a chain of steps of at most 1/8 of it, taken
    with probabilities below 0.005, whose stationary spread is some 15 %: over 8192 elements the mean is within 10 %, and
    nine in ten are within 50 %.  Rounded to nearest they sink with the scale of the block."""
    from fast_jtnn_hip import AdamW

    n = 1 << 14
    roots = {}
    for rounding in ("nearest", "stochastic"):
        p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
        opt = AdamW([p], lr=0.0, weight_decay=0.0, state_bits=8, rounding=rounding)
        even = torch.arange(n, device="cuda") % 2 == 0
        p.grad = torch.where(even, 3.0, 1.0)
        for _ in range(1000):
            opt.step()
        p.grad = torch.where(even, 0.0, 1.0)
        for _ in range(2000):
            opt.step()
        got, _ = deq(opt.state[p], "exp_rms")
        roots[rounding] = got[~even] / math.sqrt(1 - 0.999 ** 3000)
    r = roots["stochastic"]
    assert abs(float(r.mean()) - 1) < 0.1 and float(((r - 1).abs() < 0.5).double().mean()) > 0.9
    assert float(roots["nearest"].mean()) < 0.6


def test_state_dicts():
    """Round trip through a file (both kinds of state), continuing bit for bit; a dict of torch's own optimizer; refusals."""
    from fast_jtnn_hip import AdamW

    for dtype, bits in ((torch.float32, 32), (torch.bfloat16, 8), (torch.float16, 32)):
        a = params_of(SHAPES, dtype, 4)
        opt = AdamW(a, lr=1e-3, state_bits=bits)
        for _ in range(2):
            opt.step()
        f = io.BytesIO()
        torch.save(opt.state_dict(), f)
        f.seek(0)
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        other = AdamW(b, lr=7.0, state_bits=bits)
        other.load_state_dict(torch.load(f, weights_only=True))
        assert other.param_groups[0]["lr"] == 1e-3
        opt.step()
        other.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert int(other.state[q]["step"]) == (3 if q.numel() else int(opt.state[p]["step"]))
    ps = params_of(SHAPES[1:8], torch.float32, 6)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, twin):
        q.grad = p.grad.clone()
    ref = torch.optim.AdamW(twin, lr=1e-2)
    ref.step()
    opt = AdamW(ps, lr=1e-3)
    with torch.no_grad():
        for p, q in zip(ps, twin):
            p.copy_(q)
    opt.load_state_dict(copy.deepcopy(ref.state_dict()))
    opt.step()
    ref.step()
    for p, q in zip(ps, twin):
        assert ((p - q).abs() <= 1e-2 * 32 * U + p.abs() * 4 * U).all()
    with pytest.raises((KeyError, ValueError)):
        AdamW(ps, state_bits=8).load_state_dict(ref.state_dict())
    with pytest.raises(ValueError):
        AdamW(ps[:3]).load_state_dict(ref.state_dict())
    before = [opt.state[p]["exp_avg"].clone() for p in ps]
    bad = ref.state_dict()
    bad["state"][6] = {"step": 1}
    with pytest.raises(KeyError):
        opt.load_state_dict(bad)
    for p, m in zip(ps, before):
        assert torch.equal(opt.state[p]["exp_avg"], m)  # a refused dict changes nothing


def test_state_dicts_of_other_rules_refused():
    """Another optimizer's variants; a learning rate on the device takes a dict's value where it is."""
    from fast_jtnn_hip import AdamW

    for rule, kw, ok in ((torch.optim.AdamW, dict(amsgrad=True), False), (torch.optim.AdamW, dict(maximize=True), False),
                         (torch.optim.Adam, dict(weight_decay=0.1), False), (torch.optim.Adam, {}, True),
                         (torch.optim.AdamW, dict(weight_decay=0.1), True)):
        ps = params_of(SHAPES[1:4], torch.float32, 7)
        ref = rule(ps, lr=0.5, **kw)
        ref.step()
        lr = torch.tensor(0.25, device="cuda")
        opt = AdamW(ps, lr=lr)
        if ok:
            opt.load_state_dict(ref.state_dict())
            assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.5
            assert opt.param_groups[0]["weight_decay"] == kw.get("weight_decay", 0)
        else:
            with pytest.raises(ValueError):
                opt.load_state_dict(ref.state_dict())
            assert float(lr) == 0.25 and int(opt.state[ps[0]]["step"]) == 0
    other = AdamW(ps, lr=torch.tensor(1.0, device="cuda"))
    other.load_state_dict(opt.state_dict())
    lr.fill_(3.0)
    assert float(other.param_groups[0]["lr"]) == 0.5
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(opt)


def test_parameters_that_share_memory_refused():
    from fast_jtnn_hip import AdamW

    buf = torch.ones(512, device="cuda")
    for a, b, ok in ((buf[:256], buf[256:], True), (buf[:256], buf[255:], False), (buf, buf, False),
                     (buf[100:101], buf[:512], False), (buf[300:300], buf, True)):
        a, b = torch.nn.Parameter(a), torch.nn.Parameter(b)
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        opt = AdamW([a, b])
        if ok:
            opt.step()
        else:
            with pytest.raises(RuntimeError, match="share memory"):
                opt.step()


def test_works_with_schedulers_strided_gradients_and_closures():
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.ones(64, 32, device="cuda"))
    opt = AdamW([p], lr=0.5, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.ExponentialLR(opt, 0.5)

    def closure():
        opt.zero_grad()
        loss = (p.t() * torch.ones(32, 64, device="cuda")).sum()
        loss.backward()
        p.grad = torch.ones(32, 64, device="cuda").t()  # not contiguous
        return loss

    assert float(opt.step(closure)) == 64 * 32
    assert torch.allclose(p, torch.full_like(p, 0.5), atol=1e-6)
    sched.step()
    p.grad = torch.ones(1, 1, device="cuda").expand(64, 32)
    opt.step()
    assert torch.allclose(p, torch.full_like(p, 0.25), atol=1e-6)
    q = torch.nn.Parameter(torch.ones(4, 2, device="cuda"))
    q.grad = torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 2), device="cuda")
    with pytest.raises(RuntimeError):  # sparse gradients are not taken
        AdamW([q]).step()
    opt.zero_grad()
    before = p.detach().clone()
    opt.step()  # no gradients: nothing happens
    assert torch.equal(p, before) and int(opt.state[p]["step"]) == 2


def test_packed_weights_and_saved_tensors_see_the_step():
    """The step writes through raw addresses; autograd's version counters (which the packed-weight cache goes by) move."""
    from fast_jtnn_hip import AdamW
    from fast_jtnn_hip.linear import linear

    lin = torch.nn.Linear(40, 24).cuda()
    x = torch.randn(9, 40, device="cuda")
    opt = AdamW(lin.parameters(), lr=0.1)
    y0 = linear(x, lin)
    saved = (lin.weight * lin.weight).sum()
    linear(x, lin).sum().backward()
    opt.step()
    y1 = linear(x, lin)
    want = torch.nn.functional.linear(x.double(), lin.weight.double(), lin.bias.double())
    assert not torch.equal(y0, y1) and ((y1.double() - want).abs() <= 1e-4 * want.abs().max()).all()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        saved.backward()


def test_moved_parameters_and_master_refresh():
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.ones(600, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], lr=0.25, weight_decay=0.0)
    opt.step()
    p.data = torch.full((600,), 3.0, device="cuda", dtype=torch.bfloat16)  # new storage, new value
    opt.refresh_master()
    opt.step()
    assert torch.allclose(p.float(), torch.full_like(p.float(), 2.75), atol=1e-2)
    p.data = p.data.float()
    with pytest.raises(RuntimeError, match="changed its device, type, size or layout"):
        opt.step()


def test_gradients_of_another_type_or_size():
    """A gradient type of its own is converted; a parameter whose data was exchanged for another size is refused."""
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.ones(700, device="cuda", dtype=torch.bfloat16))
    if hasattr(p, "grad_dtype"):
        p.grad_dtype = None
        p.grad = torch.ones(700, device="cuda")
        opt = AdamW([p], lr=0.25, weight_decay=0.0)
        opt.step()
        assert (p.detach() == 0.75).all()
    for new in (torch.ones(9, device="cuda"), torch.ones(5000, device="cuda")):
        q = torch.nn.Parameter(torch.ones(300, device="cuda"))
        q.grad = torch.ones(300, device="cuda")
        opt = AdamW([q])
        opt.step()
        q.data = new
        with pytest.raises(RuntimeError, match="size"):  # the old gradient's size, the new parameter's address
            opt.step()
        q.grad = torch.ones_like(q)
        with pytest.raises(RuntimeError, match="size"):
            opt.step()
    q = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = AdamW([q])
    opt.step()
    q.data = q.data[:100]  # the same address
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="size"):
        opt.step()


def test_captured_and_replayed():
    """A captured step with the clip and a learning rate on the device, replayed with eager work in between, makes the
    steps that the eager optimizer makes; a capture before the first step is refused."""
    from fast_jtnn_hip import AdamW

    for bits in (32, 8):
        a, b = params_of(SHAPES, torch.float32, 9), params_of(SHAPES, torch.float32, 9)
        lr = torch.tensor(1e-2, device="cuda")
        first, second = AdamW(a, lr=lr, state_bits=bits, max_norm=0.3), AdamW(b, lr=lr, state_bits=bits, max_norm=0.3)
        graph = torch.cuda.CUDAGraph()
        first.step()
        second.step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            first.step()
        for k in range(4):
            for p, q in zip(a, b):
                g = torch.randn_like(p) * 0.01 * (k + 1)
                p.grad.copy_(g)
                q.grad.copy_(g)
            lr.fill_(1e-2 / (k + 1))
            graph.replay()
            second.step()
            torch.cuda.synchronize()
            for p, q in zip(a, b):
                assert torch.equal(p, q), k
            assert torch.equal(first.grad_norm, second.grad_norm)
        assert int(first.state[a[0]]["step"]) == 5


def test_captured_step_follows_moved_parameters():
    """The table that a captured step reads is written in its place: after an eager step has seen new storage, replays step
    that storage."""
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.ones(5000, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], lr=0.25, weight_decay=0.0)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    old = p.data
    p.data = torch.full_like(old, 8.0)
    opt.step()
    before = old.clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(old, before) and ((p.detach() - 7.0).abs() < 1e-5).all()


def test_capture_needs_a_step_first():
    """Refused on the host: nothing has been launched when the error comes."""
    from unittest import mock

    from fast_jtnn_hip import AdamW

    ps = params_of([(300,)], torch.float32, 9)
    opt = AdamW(ps)
    with mock.patch("torch.cuda.is_current_stream_capturing", return_value=True):
        with pytest.raises(RuntimeError, match="make one step first"):
            opt.step()
    opt.step()


def test_large_tensor():
    """A tensor of more than 2^31 elements, 16-bit without a copy: the far end is stepped like the near one."""
    from fast_jtnn_hip import AdamW

    n = (1 << 31) + 4099
    p = torch.nn.Parameter(torch.ones(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    opt = AdamW([p], lr=0.25, weight_decay=0.0, state_bits=8, master=False)
    opt.step()
    torch.cuda.synchronize()
    for at in (0, (1 << 31) - 300, n - 600):
        assert (p.detach()[at:at + 600] == 0.75).all()
    assert float(p.detach()[n - 4099:].float().sum()) == 0.75 * 4099


def test_a_step_of_the_losses_and_the_optimizer_together():
    """As a fine-tuning step uses them: products, preference and policy losses, backward, clipped step - against the
    same step written with torch's own operations."""
    from fast_jtnn_hip import AdamW, SequencePlan, policy_loss, preference_loss, sequence_log_probs
    from fast_jtnn_hip.linear import linear

    torch.manual_seed(3)
    n, h, v, s = 96, 45, 385, 8
    x = torch.randn(n, h, device="cuda")
    labels = torch.randint(0, v, (n,), device="cuda")
    row_seq = np.arange(n) % s
    pairs = np.arange(s).reshape(-1, 2)
    plan = SequencePlan(row_seq, s, "cuda", pairs=pairs)
    lin, twin = torch.nn.Linear(h, v).cuda(), torch.nn.Linear(h, v).cuda()
    twin.load_state_dict(lin.state_dict())
    with torch.no_grad():
        ref = sequence_log_probs(linear(x, lin) * 0.9, labels, plan)
        old = torch.log_softmax(linear(x, lin) * 0.95, 1)[torch.arange(n), labels]
    adv = torch.randn(n, device="cuda")
    opt = AdamW(lin.parameters(), lr=1e-2, max_norm=0.5)
    ref_opt = torch.optim.AdamW(twin.parameters(), lr=1e-2)
    member, pr = torch.from_numpy(row_seq).cuda(), torch.from_numpy(pairs).cuda()
    for _ in range(3):
        opt.zero_grad()
        logits = linear(x, lin)
        loss = preference_loss(logits, labels, plan, ref).loss + \
            policy_loss(logits, labels, old, adv, clip=(0.9, 9.0), scale=1.0 / n).loss
        loss.backward()
        opt.step()
        ref_opt.zero_grad()
        lp = torch.log_softmax(twin(x), 1)[torch.arange(n), labels]
        sums = torch.zeros(s, device="cuda").index_add(0, member, lp)
        margin = 0.1 * ((sums - ref)[pr[:, 0]] - (sums - ref)[pr[:, 1]])
        r = torch.exp(lp - old)
        want = -torch.nn.functional.logsigmoid(margin).mean() - torch.minimum(r * adv, r.clamp(0.1, 10.0) * adv).mean()
        want.backward()
        norm = torch.nn.utils.clip_grad_norm_(twin.parameters(), 0.5)
        ref_opt.step()
        assert abs(float(loss) - float(want)) <= 1e-4 * max(1.0, abs(float(want)))
        assert abs(float(opt.grad_norm) - float(norm)) <= 1e-4 * float(norm)
    # Adam divides by the gradient's own size: an element whose gradient is near zero may move by up to the learning
    # rate either way, so the weights are compared as a whole
    diff = torch.cat([(p - q).reshape(-1) for p, q in zip(lin.parameters(), twin.parameters())])
    assert float(diff.norm()) <= 1e-3 * 3e-2 * math.sqrt(diff.numel())
