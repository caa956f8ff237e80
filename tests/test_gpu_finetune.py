"""GPU: the callers of the fine-tuning operators - the tree decoder's log-likelihood and preference loss, the policy loss
on its word predictions, the trainer's AdamW."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from common import RTOL, fro_err, make_hip_model, make_oracle_vae
from test_gpu_training_side import _seeded_training_problem

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _problem(seed, B, atoms=20.0, V=60):
    g, x_batch = _seeded_training_problem(seed, B, atoms, V=V)
    z = torch.from_numpy(np.random.RandomState(seed).standard_normal((B, 28)).astype(np.float32))
    return g, x_batch, make_hip_model(g, "cuda"), z


def test_log_likelihood_is_minus_the_training_losses():
    """Summed over the batch it is what ``forward`` returns times -B, with the same gradient; tree by tree it is what the
    oracle's decoder gives for a batch of that tree alone."""
    B = 12
    g, x_batch, hip, z = _problem(61, B)
    x = x_batch()
    for holder in (None, x[1]):
        zt = z.cuda().requires_grad_()
        ll = hip.decoder.log_likelihood(x[0], zt, jtenc_holder=holder)
        word, stop, _, _ = hip.decoder(x[0], zt, jtenc_holder=holder)
        s = hip.decoder.trace_scores(x[0], zt, holder)
        rows = s.word_scores.shape[0] + s.stop_scores.shape[0]
        assert abs(float(ll.sum()) + B * float(word + stop)) <= rows * U * B * float(word + stop)
        hip.zero_grad(set_to_none=True)
        (ga,) = torch.autograd.grad(ll.sum(), zt)
        hip.zero_grad(set_to_none=True)
        (gb,) = torch.autograd.grad(-B * (word + stop), zt)
        assert fro_err(ga.cpu().numpy(), gb.cpu().numpy()) < 1e-5
    ora = make_oracle_vae(g)
    trees = x_batch()[0]
    for i, t in enumerate(trees):
        with torch.no_grad():
            w, st, _, _ = ora.decoder([t], z[i:i + 1])
        assert abs(float(ll[i]) + float(w + st)) <= RTOL * abs(float(w + st)), i


def test_log_likelihood_of_single_node_trees():
    from fast_jtnn_hip import synthetic

    g, _ = _seeded_training_problem(1, 2, 8.0, V=9)
    g.H, g.L = 32, 8
    hip = make_hip_model(g, "cuda")
    mol = synthetic.make_mol(np.random.RandomState(0), 6.0, 1.0, 4, 8)
    trees = [synthetic.Tree([synthetic.TreeNode(1, w)], mol) for w in (2, 5)]
    synthetic.set_batch_nodeID(trees)
    zt = torch.from_numpy(np.random.RandomState(1).standard_normal((2, 4)).astype(np.float32)).cuda().requires_grad_()
    ll = hip.decoder.log_likelihood(trees, zt)
    word, stop, _, _ = hip.decoder(trees, zt)
    assert ll.shape == (2,) and abs(float(ll.sum()) + 2 * float(word + stop)) <= 1e-5 * 2 * float(word + stop)
    r = hip.decoder.preference_loss(trees, zt, [[0, 1]], ll.detach())
    assert abs(float(r.loss) - math.log(2.0)) <= 1e-6
    r.loss.backward()
    assert torch.isfinite(zt.grad).all()


def test_preference_loss_of_the_decoder():
    """Against the same loss written with torch's operations on the log-likelihoods: value, margins, every gradient."""
    B = 10
    g, x_batch, hip, z = _problem(62, B)
    x = x_batch()
    pairs = np.array([[0, 1], [2, 3], [5, 4], [0, 6], [7, 8]])
    with torch.no_grad():
        ref = hip.decoder.log_likelihood(x[0], (z * 0.8).cuda(), x[1])
    zt = z.cuda().requires_grad_()
    r = hip.decoder.preference_loss(x[0], zt, pairs, ref, beta=0.3, label_smoothing=0.1, jtenc_holder=x[1])
    hip.zero_grad(set_to_none=True)
    r.loss.backward()
    got = {n: p.grad.clone() for n, p in hip.decoder.named_parameters() if p.grad is not None}
    gz = zt.grad.clone()
    zt.grad = None
    hip.zero_grad(set_to_none=True)
    ll = hip.decoder.log_likelihood(x[0], zt, x[1]).double()
    margin = 0.3 * ((ll - ref.double())[pairs[:, 0]] - (ll - ref.double())[pairs[:, 1]])
    ls = torch.nn.functional.logsigmoid
    want = -(0.9 * ls(margin) + 0.1 * ls(-margin)).mean()
    want.backward()
    # log-likelihoods of tens to hundreds are rounded to 32 bits on the torch side
    off = float(ll.abs().max()) * 2 * U
    assert ((r.log_probs.double() - ll).abs() <= off).all()
    assert ((r.margins.double() - margin).abs() <= 0.3 * 4 * off + margin.abs() * 4 * U).all()
    assert abs(float(r.loss) - float(want)) <= 0.3 * 4 * off + abs(float(want)) * 4 * U
    assert fro_err(gz.cpu().numpy(), zt.grad.cpu().numpy()) < 1e-4
    assert got
    for n, p in hip.decoder.named_parameters():
        if n in got:
            assert fro_err(got[n].cpu().numpy(), p.grad.cpu().numpy()) < 1e-4, n


def test_policy_loss_on_word_predictions():
    from fast_jtnn_hip import policy_loss

    g, x_batch, hip, z = _problem(63, 6)
    x = x_batch()
    zt = z.cuda().requires_grad_()
    s = hip.decoder.trace_scores(x[0], zt, x[1])
    n = s.word_scores.shape[0]
    rs = np.random.RandomState(0)
    adv = torch.from_numpy(rs.standard_normal(6).astype(np.float32)).cuda()[torch.from_numpy(s.plan.pred_ctx).cuda()]
    lp = torch.log_softmax(s.word_scores.double(), 1)[torch.arange(n), s.word_targets]
    old = (lp.detach() - torch.from_numpy(rs.uniform(-0.1, 0.1, n)).cuda()).float()  # every ratio inside the range
    out = policy_loss(s.word_scores, s.word_targets, old, adv, clip=0.3, scale=1.0 / n)
    (ga,) = torch.autograd.grad(out.loss, zt, retain_graph=True)
    want = -(torch.exp(lp - old.double()) * adv.double()).mean()
    (gb,) = torch.autograd.grad(want, zt)
    assert abs(float(out.loss) - float(want)) <= 1e-5 * float(adv.abs().mean())
    assert float(out.clipped) == 0 and float(out.kl) == 0
    assert fro_err(ga.cpu().numpy(), gb.cpu().numpy()) < 1e-4


@pytest.mark.parametrize("name", ["adamw", "adamw8"])
def test_trainer_steps_with_adamw(name):
    """One step: loss and gradients of the usual step, the weights moved by the formula from the gradients that are left
    in place, the clip included; the printed norm is the clipped one."""
    from fast_jtnn_hip import trainer

    g, x_batch = _seeded_training_problem(64, 8, 16.0, V=60)
    hip = make_hip_model(g, "cuda")
    lines = []
    sched = trainer.Schedule(lr=1e-3, clip_norm=0.25, print_iter=1)
    tr = trainer.Trainer(hip, sched, log=lines.append, optimizer=name, weight_decay=0.1)
    before = {n: p.detach().clone() for n, p in hip.named_parameters()}
    rs = np.random.RandomState(1)
    eps = [torch.from_numpy(rs.standard_normal((8, 28)).astype(np.float32)).cuda() for _ in range(2)]
    assert tr.step(x_batch(), epsilons=eps).ok
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in hip.parameters() if p.grad is not None))
    assert norm > 0.25 and abs(float(tr.optimizer.grad_norm) - norm) <= norm * 8 * U
    assert "GNorm: 0.25" in lines[0]
    factor = 0.25 / (norm + 1e-6)
    for n, p in hip.named_parameters():
        gr = p.grad.double() * factor
        m, v = 0.1 * gr / (1 - 0.9), 0.001 * gr * gr / (1 - 0.999)
        want = before[n].double() * (1 - 1e-4) - 1e-3 * m / (v.sqrt() + 1e-8)
        # the first update is at most the learning rate; squares below the normal range lose their digits
        tol = 1e-3 * 64 * U + before[n].double().abs() * 6 * U + torch.where(gr.abs() < 1e-15, 1e-3, 0.0)
        assert ((p.detach().double() - want).abs() <= tol).all(), n
    for k in range(2):  # the packed weights follow: further steps see the new weights
        hip_loss = tr.step(x_batch(), epsilons=eps)
        assert hip_loss.ok and np.isfinite(hip_loss.loss)
    fresh = make_hip_model(g, "cuda")
    fresh.load_state_dict(hip.state_dict())
    with torch.no_grad():
        a = hip(x_batch(), 0.0, epsilons=eps)[0]
        b = fresh(x_batch(), 0.0, epsilons=eps)[0]
    assert abs(float(a) - float(b)) <= 1e-5 * abs(float(b))


def test_training_cli_with_adamw8(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run(
        [sys.executable, os.path.join(root, "train.py"), "--train", "synthetic:64:3", "--vocab", "60", "--save_dir",
         str(tmp_path), "--batch_size", "32", "--epoch", "1", "--print_iter", "1", "--optimizer", "adamw8",
         "--weight_decay", "0.01"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "[2] Loss:" in out.stdout
    state = torch.load(os.path.join(tmp_path, "model.epoch-2"), map_location="cpu", weights_only=True)
    assert all(torch.isfinite(v).all() for v in state.values())
