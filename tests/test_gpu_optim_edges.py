"""GPU: the AdamW step at the edges of what it takes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.float32), (32, torch.bfloat16)])
@pytest.mark.parametrize("decay", [1e-5, 4e-5, 3e-3])
def test_small_decay_adds_up(decay, bits, dtype):
    """lr * decay of 1e-8 to 3e-6, around and above half the last place of one, over a thousand steps whose updates have no
    direction (beta1 = beta2 = 0, eps = 1: the update is lr g / (|g| + 1)).  A weight below one is rounded by at most 2^-25 a
    step, either way alike: the mean over 2^16 weights of a thousand roundings strays by sqrt(1000 / 2^16) 2^-25 / sqrt(3) =
    2e-9, tenfold allowed.  What leans one way: the update's 16 U in every step, 1000 * lr * 16 U = 1e-6, and the decay's
    own 4 U.  (8-bit states hold |g| and g to 2^-4 only after the update, which works on the gradient itself here.)"""
    from fast_jtnn_hip import AdamW

    n, lr = 1 << 16, float(np.float32(1e-3))
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.nn.Parameter((torch.rand(n, generator=g, device="cuda") * 0.4 + 0.55).to(dtype))
    opt = AdamW([p], lr=lr, weight_decay=decay, betas=(0.0, 0.0), eps=1.0, state_bits=bits)
    w = p.detach().double()
    for _ in range(1000):
        p.grad = torch.randn(n, generator=g, device="cuda").to(dtype)
        x = p.grad.double()
        opt.step()
        w = w - lr * decay * w - lr * x / (x.abs() + 1.0)
    now = (p.detach() if dtype == torch.float32 else opt.state[p]["master"]).double()
    assert abs(float((now - w).mean())) <= 2e-8 + 1000 * (lr * 16 * U + lr * decay * 4 * U)


def test_load_state_dict_hooks():
    """Hooks run around the load, a dict that one returns is the one that is taken, and what one changes is not the
    caller's; a refused dict runs none of those after it."""
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], lr=1e-3)
    opt.step()
    saved, seen = opt.state_dict(), []

    def slower(o, d):
        seen.append(float(d["param_groups"][0]["lr"]))
        return dict(d, param_groups=[dict(g, lr=5e-4) for g in d["param_groups"]])

    def changes(o, d):
        seen.append("changes")
        d["note"] = 1

    handles = [opt.register_load_state_dict_pre_hook(changes), opt.register_load_state_dict_pre_hook(slower),
               opt.register_load_state_dict_post_hook(lambda o: seen.append(o.param_groups[0]["lr"]))]
    opt.load_state_dict(saved)
    assert seen == ["changes", 1e-3, 5e-4] and "note" not in saved and saved["param_groups"][0]["lr"] == 1e-3
    del seen[:]
    handles[1].remove()
    with pytest.raises(ValueError):
        opt.load_state_dict({"state": {}, "param_groups": [{"params": [0, 1]}]})
    assert seen == ["changes"]
    handles[0].remove()
    handles[2].remove()
    opt.load_state_dict(saved)
    assert seen == ["changes"] and int(opt.state[p]["step"]) == 1


def test_a_parameter_turned_in_its_place_is_refused():
    """Transposed data keep address, size and type, and the old gradient keeps its order; turned back, steps go on."""
    from fast_jtnn_hip import AdamW

    p, q = (torch.nn.Parameter(torch.randn(40, 40, device="cuda")) for _ in range(2))
    for t in (p, q):
        t.grad = torch.randn(40, 40, device="cuda")
    opt = AdamW([p, q])
    opt.step()
    q.data = q.data.t()
    before = [t.detach().clone() for t in (p, q)]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="layout"):
            opt.step()
    assert all(torch.equal(t, b) for t, b in zip((p, q), before))
    q.data = q.data.t()
    opt.step()
    assert int(opt.state[q]["step"]) == 2 and not torch.equal(p, before[0])
    one = torch.nn.Parameter(torch.ones(1, 30, device="cuda"))  # a row turned into a column keeps its order
    opt = AdamW([one], lr=0.25, weight_decay=0.0)
    for shape in ((1, 30), (30, 1)):
        one.data = one.data.t() if one.shape != shape else one.data
        one.grad = torch.ones_like(one)
        opt.step()
    assert bool(((one.detach() - 0.5).abs() < 1e-6).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-42, 1e-36, 1e-28, 1e-20, 1e-13, 1.0, 1e15, 1e25, 1e37])
def test_norms_of_very_small_and_very_large_gradients(size, dtype):
    """Their squares vanish or overflow in 32 bits, the norm does not; a few ordinary ones among them, and zeros.  Large ones
    are clipped by it, not brought to nothing: with beta1 = beta2 = 0 and the clipped gradient c far above eps the update is
    lr c / (|c| + eps), the learning rate but for eps / |c|."""
    from fast_jtnn_hip import AdamW

    ps = [torch.nn.Parameter(torch.ones(n, device="cuda", dtype=dtype)) for n in (5000, 3, 4097)]
    gen = torch.Generator(device="cuda").manual_seed(2)
    for p in ps:
        p.grad = (torch.randn(p.numel(), generator=gen, device="cuda") * size).to(dtype)
        p.grad[1::7] = 0
    want = float(torch.cat([p.grad.double() for p in ps]).square().sum().sqrt())
    before = [p.detach().clone() for p in ps]
    opt = AdamW(ps, lr=0.25, betas=(0.0, 0.0), eps=1e-12, weight_decay=0.0, max_norm=1.0)
    opt.step()
    if want > torch.finfo(torch.float32).max:  # 1e37 sqrt(7800) = 9e38: no 32-bit number, while the factor is one
        assert float(opt.grad_norm) == float("inf")
    else:
        assert abs(float(opt.grad_norm) - want) <= want * 8 * U + 2.0 ** -149
    if size >= 1.0:
        for p, b in zip(ps, before):
            c = p.grad.double() / want
            sure = c.abs() > 1e-6  # eps moves these by at most 1e-6 of the update; bf16 parameters follow a 32-bit copy
            assert bool((((b - p.detach()).double() - 0.25 * c.sign()).abs()[sure] <= 1e-6 + torch.finfo(dtype).eps / 2).all())
    mixed = torch.nn.Parameter(torch.ones(4096, device="cuda", dtype=dtype))
    mixed.grad = torch.full_like(mixed, size)
    mixed.grad[::5] = 1.0
    opt = AdamW([mixed], max_norm=1.0)
    opt.step()
    want = float(mixed.grad.double().square().sum().sqrt())
    if want > torch.finfo(torch.float32).max:  # 1e37 * 57
        assert float(opt.grad_norm) == float("inf")
    else:
        assert abs(float(opt.grad_norm) - want) <= want * 8 * U


@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_of_weights_that_start_at_zero(bits):
    """Their first step is the update itself.  Relative to it: g 1 / (1 - beta1) by two roundings and the correction's one,
    the root 2^-23 and half of what its square (three roundings, the correction's one) is off by, the sum with eps by one, the
    reciprocal by two, the product with it, the learning rate times its correction and the last product by one each: 13 * 2^-24
    together where all lean one way."""
    from fast_jtnn_hip import AdamW

    p = torch.nn.Parameter(torch.zeros(100_000, device="cuda"))
    gen = torch.Generator(device="cuda").manual_seed(4)
    p.grad = torch.randn(p.numel(), generator=gen, device="cuda") * torch.exp(3 * torch.randn(p.numel(), generator=gen, device="cuda"))
    AdamW([p], lr=1e-3, eps=1e-3, weight_decay=0.5, state_bits=bits).step()
    g = p.grad.double()
    want = -float(np.float32(1e-3)) * g / (g.abs() + float(np.float32(1e-3)))
    assert float((p.detach().double() / want - 1).abs().max()) <= 13 * U


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, True), (torch.bfloat16, True), (torch.float16, False)])
def test_infinite_weights_stay(dtype, master, bits):
    """Masks kept among the parameters: an infinite weight is infinite after a step, with and without decay, for zero and
    other gradients, and leaves its neighbours alone; a weight that is NaN stays NaN."""
    from fast_jtnn_hip import AdamW

    inf = float("inf")
    for decay in (0.0, 0.125):
        p = torch.nn.Parameter(torch.ones(600, device="cuda", dtype=dtype))
        with torch.no_grad():
            p[3::10], p[4::10], p[5] = -inf, inf, float("nan")
        p.grad = torch.zeros_like(p)
        p.grad[300:] = 0.5
        opt = AdamW([p], lr=0.25, weight_decay=decay, state_bits=bits, master=master)
        opt.step()
        w = p.detach().float()
        assert bool((w[3::10] == -inf).all()) and bool((w[4::10] == inf).all()) and bool(torch.isnan(w[5]))
        kept = 1 - 0.25 * decay
        want = torch.where(torch.arange(600, device="cuda") < 300, kept, kept - 0.25)
        rest = torch.isfinite(w)
        assert int(rest.sum()) == 600 - 121 and bool(((w - want).abs()[rest] <= 1e-6 + torch.finfo(dtype).eps / 2).all())
