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
