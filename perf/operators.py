"""Timed cases of the training-end operators: log-probabilities of chosen words under a row of logits, the two
fine-tuning losses built on them (paired preferences, clipped policy with a KL term), and the AdamW step.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges; ``prepare`` makes what a program holds before
the call, ``run`` is one pass and ``exact`` the same outputs in 64 bits.  ``own`` selects between the plain form
(elementary torch operations in 32 bits) and the package's kernels.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jt-vae-tmcinvdes_amd")
_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 256  # elements of a parameter that share one scale of the 8-bit optimizer states
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.01


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from fast_jtnn_hip import losses, optim
    return losses, optim


# ---- cases ------------------------------------------------------------------------------------


def _rows_case(op, rows, vocab, dtype, **more):
    return dict({"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "skipped": 0.0, "seqs": 0, "layout": "none"},
                **more)


def listed():
    return [
        # word predictions of one junction tree of about 24 nodes at this model's vocabulary: latency
        _rows_case("tokens", 24, 385, "float32", name="tokens 24x385 fp32"),
        # a long padded batch of a text model with an odd vocabulary: rows are not aligned
        _rows_case("tokens", 1500, 50021, "float16", skipped=0.1, name="tokens 1500x50021 fp16"),
        # scoring one short answer: few rows over a long axis, no gradient
        _rows_case("score", 4, 128000, "bfloat16", seqs=1, layout="padded", name="score 4x128000 bf16"),
        # the frozen reference model's pass over a batch of answers, no gradient
        _rows_case("score", 4096, 32000, "bfloat16", skipped=0.2, seqs=32, layout="padded", name="score 4096x32000 bf16"),
        # 8 molecule pairs, 20 word predictions each, rows ordered by decoding step
        _rows_case("preference", 320, 385, "float32", seqs=16, layout="steps", name="preference 320x385 fp32"),
        # a training batch of 512 molecule pairs at a larger fragment vocabulary
        _rows_case("preference", 20480, 780, "float32", seqs=1024, layout="steps", name="preference 20480x780 fp32"),
        # 16 pairs of padded answers at a large text vocabulary
        _rows_case("preference", 4096, 128000, "bfloat16", skipped=0.2, seqs=32,
                   layout="padded", name="preference 4096x128000 bf16"),
        # sampled fragments of three molecules: latency
        _rows_case("policy", 64, 385, "float32", name="policy 64x385 fp32"),
        # a mini-batch of sampled tokens
        _rows_case("policy", 8192, 32000, "bfloat16", skipped=0.1, name="policy 8192x32000 bf16"),
        # the parameters of this package's model (hidden 450, vocabulary 385, latent 56) with the trainer's clip
        {"name": "adamw model fp32", "op": "adamw", "tensors": "model", "dtype": "float32", "bits": 32, "clip": 50.0},
        {"name": "adamw model fp32 8bit", "op": "adamw", "tensors": "model", "dtype": "float32", "bits": 8,
         "clip": 50.0},
        # eight blocks of a text model in bf16 with an fp32 copy of the weights and 8-bit states
        {"name": "adamw blocks bf16 8bit", "op": "adamw", "tensors": "blocks", "dtype": "bfloat16", "bits": 8,
         "clip": 1.0},
    ]


def _log_between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tokens", "score", "preference", "policy", "adamw"])
    if op == "adamw":
        return {"op": op, "tensors": "drawn", "count": _log_between(rng, 1, 200), "smallest": rng.choice([1, 7, 64, 450]),
                "largest": _log_between(rng, 2000, 4_000_000), "sizes": rng.randrange(1 << 30),
                "dtype": rng.choice(["float32", "bfloat16", "float16"]), "bits": rng.choice([32, 8]),
                "clip": rng.choice([0.0, 1.0, 50.0])}
    rows, vocab = _log_between(rng, 2, 20000), _log_between(rng, 64, 131072)
    while rows * vocab > 4096 * 128000:
        rows = max(2, rows // 2)
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if dtype == "float32" and rows * vocab > 2048 * 128000:
        rows = max(2, rows // 2)
    if op in ("tokens", "policy"):
        return _rows_case(op, rows, vocab, dtype, skipped=rng.choice([0.0, 0.1, 0.3]))
    seqs = 2 * _log_between(rng, 1, max(1, min(512, rows // 2)))
    return _rows_case(op, rows, vocab, dtype, skipped=rng.choice([0.0, 0.2]), seqs=seqs,
                      layout=rng.choice(["steps", "padded"]))


def _skipped_rows(case):
    """Number of rows that carry no label: fixed by the case, so that its work is known."""
    return int(case["rows"] * case["skipped"])


def work(case):
    """Every input read once, every output written once; rows without a label are not read."""
    if case["op"] == "adamw":
        n, size = sum(_numels(case)), _DTYPES[case["dtype"]].itemsize
        weights = 3 * size + (8 if size == 2 else 0)  # gradient in, weight in and out, or its fp32 copy in and out
        if size == 2:
            weights -= size  # the 16-bit weight itself is only written where the copy is kept
        states = 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK
        return {"bytes": n * (weights + states), "flops": 16 * n}
    rows, vocab, size = case["rows"], case["vocab"], _DTYPES[case["dtype"]].itemsize
    read = (rows - _skipped_rows(case)) * vocab
    grad = 0 if case["op"] == "score" else rows * vocab
    return {"bytes": (read + grad) * size + 32 * rows, "flops": 4 * read + 4 * grad}


# ---- inputs -----------------------------------------------------------------------------------


def _numels(case):
    """Element counts of the parameter tensors of an optimizer case."""
    if case["tensors"] == "drawn":
        rs = np.random.RandomState(case["sizes"] % (1 << 31))
        lo, hi = math.log(case["smallest"]), math.log(max(case["largest"], case["smallest"]))
        return [max(1, int(round(math.exp(v)))) for v in rs.uniform(lo, hi, case["count"])]
    if case["tensors"] == "blocks":
        d, f, vocab = 2048, 5632, 32000
        return [vocab * d] + [d * d, d * d, d * d, d * d, f * d, f * d, f * d, d, d] * 8 + [d]
    h, v, z, a, b = 450, 385, 28, 39, 12  # hidden, vocabulary, half of the latent, atom and bond features
    enc = [v * h, h * 2 * h, h, h * h, h * h, h, h * 2 * h, h, h * 2 * h, h]
    dec = [v * h, h * 2 * h, h, h * h, h * h, h, h * 2 * h, h, h * (h + z), h, h * (h + z), h, h * 2 * h, h, v * h, v, h, 1]
    graph = [h * (a + b), h * h, h * (a + h), h, h * 44, h * h, h * (38 + h), h]
    return enc + dec + graph + [h * z] + [z * h, z] * 4


def _row_sequences(case):
    """Sequence of every row, -1 where the row belongs to none: padded answers one after the other, or the words of
    all trees in the order of decoding steps (as the tree decoder lays them out)."""
    rows, seqs, skipped = case["rows"], case["seqs"], _skipped_rows(case)
    rs = np.random.RandomState(rows * 31 + seqs)
    if case["layout"] == "padded":
        of = np.minimum(np.arange(rows) * seqs // rows, seqs - 1)
        place = np.arange(rows) - np.searchsorted(of, of)  # position inside the sequence
        lost = np.lexsort((rs.rand(rows), -place))[:skipped]  # mostly the ends of the sequences
        of = of.copy()
        of[lost] = -1
        return of.astype(np.int32)
    spread = np.minimum(np.floor(rs.rand(rows - skipped) ** 1.3 * seqs), seqs - 1).astype(np.int32)
    steps = np.zeros(rows - skipped, dtype=np.int64)
    order = np.argsort(spread, kind="stable")
    first = np.searchsorted(spread[order], np.arange(seqs))
    steps[order] = np.arange(rows - skipped) - first[spread[order]]
    spread = spread[np.lexsort((spread, steps))]
    return np.concatenate([spread, np.full(skipped, -1, dtype=np.int32)])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"] == "adamw":
        return _prepare_adamw(case, normal)
    n, v, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    ld = -(-v // 4) * 4 if dtype == torch.float32 else v  # the package's fp32 products pad their rows to 16 bytes
    logits = normal(n, ld, dtype=dtype).mul_(2)[:, :v]
    labels = torch.randint(0, v, (n,), generator=gen, device="cuda")
    # a trained model: most labels stand well above the noise
    lift = normal(n).mul_(2).add_(9)
    at = torch.arange(n, device="cuda")
    logits[at, labels] = (logits[at, labels].float() + lift).to(dtype)
    s = {"case": case, "logits": logits.requires_grad_(case["op"] != "score"), "labels": labels}
    if case["layout"] == "none":
        lost = torch.randperm(n, generator=gen, device="cuda")[:_skipped_rows(case)]
        labels[lost] = -100
    else:
        row_seq = _row_sequences(case)
        pairs = None
        if case["op"] == "preference":
            order = np.random.RandomState(seed % (1 << 31)).permutation(case["seqs"]).astype(np.int32)
            pairs = order.reshape(-1, 2)  # (preferred, other) sequence of every pair
            s["pairs"] = torch.from_numpy(pairs.astype(np.int64)).cuda()
        s["row_seq"] = torch.from_numpy(row_seq.astype(np.int64)).cuda()
        labels[s["row_seq"] < 0] = -100
        if own:
            s["plan"] = _package()[0].SequencePlan(row_seq, case["seqs"], "cuda", pairs=pairs)
    if case["op"] == "tokens":
        s["dlogp"] = normal(n).div_(n)
        return s
    if case["op"] == "score":
        return s
    # log-probabilities that an earlier or a frozen copy of the model gave, a little away from the present ones
    parts = torch.split(logits.detach(), max(1, (1 << 27) // v))
    present = torch.cat([torch.log_softmax(x.float(), 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
                         for x, y in zip(parts, torch.split(labels, max(1, (1 << 27) // v)))])
    present = present.masked_fill(labels < 0, 0)
    if case["op"] == "policy":
        step = normal(n).mul_(0.15)
        # no ratio next to the border of the clipped range, where the gradient jumps
        for border in (math.log(1.2), math.log(0.8)):
            step = torch.where((step - border).abs() < 2e-3, step + 5e-3, step)
        s["old"] = present - step
        s["ref"] = present + normal(n).mul_(0.2)
        s["advantages"] = normal(n).add_(0.2)
        s["weights"] = torch.rand((n,), generator=gen, device="cuda").add_(0.5)
        return s
    per_seq = torch.zeros(case["seqs"], dtype=torch.float64, device="cuda")
    per_seq.index_add_(0, s["row_seq"].clamp(min=0), present.double())
    s["other"] = normal(case["seqs"]).sub_(4).requires_grad_()  # log-probability of the stop decisions
    s["ref"] = (per_seq + s["other"].detach() + 4 * normal(case["seqs"])).float()
    return s


def _prepare_adamw(case, normal):
    """Parameters as views of one flat buffer, each starting at a multiple of BLOCK elements; states of a run that
    has made 100 steps."""
    numels, dtype = _numels(case), _DTYPES[case["dtype"]]
    starts = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in numels])])
    total = int(starts[-1])
    gaps = torch.ones(total, dtype=torch.bool, device="cuda")
    for n, at in zip(numels, starts):
        gaps[at:at + n] = False
    s = {"case": case, "step": 100}
    scale = torch.exp(normal(total // BLOCK)).repeat_interleave(BLOCK).mul_(1e-3)  # gradients differ from block to block
    weights = normal(total).mul_(0.05).masked_fill_(gaps, 0)
    s["flat"] = weights.to(dtype)
    s["grad"] = (normal(total) * scale).masked_fill_(gaps, 0).to(dtype)
    m = (normal(total) * scale).mul_(0.3).masked_fill_(gaps, 0)
    v = (normal(total) * scale).square_().mul_(0.5).add_(scale.square().mul_(0.5)).masked_fill_(gaps, 0)
    del gaps, scale
    if dtype != torch.float32:
        s["master"] = weights
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = m, v
    else:
        s["exp_avg"], s["exp_avg_scale"] = _to_8bit(m, False)
        s["exp_rms"], s["exp_rms_scale"] = _to_8bit(v.sqrt(), True)
    if own:
        params = []
        for n, at in zip(numels, starts):
            p = torch.nn.Parameter(s["flat"][at:at + n])
            p.grad = s["grad"][at:at + n]
            params.append(p)
        opt = _package()[1].AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                  state_bits=case["bits"], max_norm=case["clip"] or None)
        names = [k for k in ("master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_rms", "exp_rms_scale") if k in s]
        loaded = {i: dict({k: s[k][at // BLOCK:at // BLOCK - (-n // BLOCK)] if k.endswith("scale") else s[k][at:at + n]
                           for k in names}, step=torch.tensor(100)) for i, (n, at) in enumerate(zip(numels, starts))}
        opt.load_state_dict({"state": loaded, "param_groups": opt.state_dict()["param_groups"]})
        s["opt"], s["params"] = opt, params
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    return _RUN[state["case"]["op"]](state)


def _log_probs(logits, labels):
    """Log-probability of every row's label (64 bits, 0 where there is none) and the row's softmax."""
    x = logits.detach().float()
    top = x.max(dim=1).values
    e = torch.exp(x - top[:, None])
    total = e.sum(dim=1)
    at = labels.clamp(min=0)[:, None]
    # one value per row in 64 bits: sums of thousands of them are compared with each other
    lp = x.gather(1, at)[:, 0].double() - top.double() - torch.log(total.double())
    return lp.masked_fill(labels < 0, 0), e.div_(total[:, None])


def _logits_grad(soft, labels, coef, dtype):
    """coef (onehot(label) - softmax) of every row with a label, zero elsewhere."""
    coef = coef.float().masked_fill(labels < 0, 0)
    g = soft.mul_(-coef[:, None])
    return g.scatter_add_(1, labels.clamp(min=0)[:, None], coef[:, None]).to(dtype)


def _per_sequence(lp, row_seq, seqs):
    total = torch.zeros(seqs, dtype=torch.float64, device=lp.device)
    return total.index_add_(0, row_seq.clamp(min=0), lp.masked_fill(row_seq < 0, 0))


def _run_tokens(s):
    if own:
        lp = _package()[0].token_log_probs(s["logits"], s["labels"])
        (d,) = torch.autograd.grad(lp, s["logits"], s["dlogp"])
        return {"log_probs": lp.detach(), "dlogits": d}
    lp, soft = _log_probs(s["logits"], s["labels"])
    return {"log_probs": lp.float(), "dlogits": _logits_grad(soft, s["labels"], s["dlogp"], s["logits"].dtype)}


def _run_score(s):
    if own:
        with torch.no_grad():
            return {"log_probs": _package()[0].sequence_log_probs(s["logits"], s["labels"], s["plan"])}
    lp, _ = _log_probs(s["logits"], s["labels"])
    return {"log_probs": _per_sequence(lp, s["row_seq"], s["case"]["seqs"]).float()}


def _run_preference(s):
    beta, smooth = 0.1, 0.05
    if own:
        r = _package()[0].preference_loss(s["logits"], s["labels"], s["plan"], s["ref"], beta=beta,
                                          label_smoothing=smooth, other_log_probs=s["other"])
        d, dother = torch.autograd.grad(r.loss, (s["logits"], s["other"]))
        return {"loss": r.loss.detach(), "log_probs": r.log_probs, "margins": r.margins, "dlogits": d, "dother": dother}
    seqs, pairs = s["case"]["seqs"], s["pairs"]
    lp, soft = _log_probs(s["logits"], s["labels"])
    per_seq = _per_sequence(lp, s["row_seq"], seqs) + s["other"].detach().double()
    gain = per_seq - s["ref"].double()
    margin = beta * (gain[pairs[:, 0]] - gain[pairs[:, 1]])
    # -log sigmoid(x) = max(-x, 0) + log(1 + exp(-|x|))
    log1 = torch.log1p(torch.exp(-margin.abs()))
    loss = ((1 - smooth) * ((-margin).clamp(min=0) + log1) + smooth * (margin.clamp(min=0) + log1)).mean()
    dmargin = beta * (1 / (1 + torch.exp(-margin)) - (1 - smooth)) / pairs.shape[0]
    coef = torch.zeros_like(per_seq).index_add_(0, pairs[:, 0], dmargin).index_add_(0, pairs[:, 1], -dmargin)
    d = _logits_grad(soft, s["labels"], coef[s["row_seq"].clamp(min=0)], s["logits"].dtype)
    return {"loss": loss.float(), "log_probs": per_seq.float(), "margins": margin.float(), "dlogits": d,
            "dother": coef.float()}


def _run_policy(s):
    clip, kl_coef, scale = 0.2, 0.05, 1.0 / s["case"]["rows"]
    if own:
        r = _package()[0].policy_loss(s["logits"], s["labels"], s["old"], s["advantages"], ref_log_probs=s["ref"],
                                      weights=s["weights"], clip=clip, kl_coef=kl_coef, scale=scale)
        (d,) = torch.autograd.grad(r.loss, s["logits"])
        return {"loss": r.loss.detach(), "log_probs": r.log_probs, "kl": r.kl, "clipped": r.clipped, "dlogits": d}
    lp, soft = _log_probs(s["logits"], s["labels"])
    w = (scale * s["weights"].double()).masked_fill(s["labels"] < 0, 0)
    a = s["advantages"].double()
    ratio, gap = torch.exp(lp - s["old"].double()), s["ref"].double() - lp
    plain, cut = ratio * a, ratio.clamp(1 - clip, 1 + clip) * a
    kl = torch.expm1(gap) - gap
    loss = (w * (kl_coef * kl - torch.minimum(plain, cut))).sum()
    coef = w * (kl_coef * (1 - torch.exp(gap)) - torch.where(plain <= cut, plain, torch.zeros_like(plain)))
    d = _logits_grad(soft, s["labels"], coef, s["logits"].dtype)
    return {"loss": loss.float(), "log_probs": lp.float(), "kl": (w * kl).sum().float(),
            "clipped": (w * (cut < plain)).sum().float(), "dlogits": d}


def _to_8bit(x, root):
    """e4m3 values and the scale of every BLOCK elements; a root of a second moment that is not zero keeps at least
    the smallest value, so that it never divides by eps alone."""
    x = x.view(-1, BLOCK)
    top = x.abs().max(dim=1).values
    inv = torch.where(top > 2.0 ** -100, 448 / top, torch.zeros_like(top))
    scaled = x * inv[:, None]
    if root:
        scaled = torch.where(scaled > 0, scaled.clamp(min=2.0 ** -9), scaled)
    scale = torch.where(top > 2.0 ** -100, top / 448, torch.zeros_like(top))
    return scaled.to(torch.float8_e4m3fn).view(-1), scale


def _from_8bit(q, scale):
    return (q.view(-1, BLOCK).float() * scale[:, None]).view(-1)


def _adamw_outputs(s, buffers):
    names = ("master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_rms", "exp_rms_scale")
    return dict({k: buffers[k] for k in names if k in buffers}, weights=s["flat"])


def _run_adamw(s):
    if own:
        s["opt"].step()
        return _adamw_outputs(s, s["opt"].state_buffers()[0])
    case = s["case"]
    s["step"] += 1
    g = s["grad"].float()
    if case["clip"]:
        norm = g.square().sum(dtype=torch.float64).sqrt()
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1).float()
    if case["bits"] == 8:
        m, v = _from_8bit(s["exp_avg"], s["exp_avg_scale"]), _from_8bit(s["exp_rms"], s["exp_rms_scale"]).square_()
    else:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    w = s["master"] if "master" in s else s["flat"]
    root = v.sqrt()
    denom = (root / math.sqrt(1 - BETA2 ** s["step"])).add_(EPS)
    w.mul_(1 - LR * DECAY).addcdiv_(m, denom, value=-LR / (1 - BETA1 ** s["step"]))
    if "master" in s:
        s["flat"].copy_(w)
    if case["bits"] == 8:
        s["exp_avg"], s["exp_avg_scale"] = _to_8bit(m, False)
        s["exp_rms"], s["exp_rms_scale"] = _to_8bit(root, True)
    return _adamw_outputs(s, s)


_RUN = {"tokens": _run_tokens, "score": _run_score, "preference": _run_preference, "policy": _run_policy,
        "adamw": _run_adamw}


# ---- the same outputs from the definitions, in 64 bits -----------------------------------------


def exact(case, seed):
    """Outputs of the first pass on these inputs, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    logits, labels = s["logits"].detach(), s["labels"]
    counted = labels >= 0
    piece = max(1, (1 << 26) // case["vocab"])
    at = torch.where(counted, labels, torch.zeros_like(labels))
    lp = torch.empty(case["rows"], dtype=torch.float64, device="cuda")
    for i in range(0, case["rows"], piece):
        x = logits[i:i + piece].double()
        lp[i:i + piece] = x[torch.arange(len(x)), at[i:i + piece]] - torch.logsumexp(x, dim=1)
    lp = torch.where(counted, lp, torch.zeros_like(lp)).requires_grad_()
    out, extra = {}, []
    if case["op"] == "tokens":
        target = (lp * s["dlogp"].double()).sum()
        out["log_probs"] = lp
    else:
        seqs = case["seqs"]
        if seqs:
            member = s["row_seq"]
            sums = torch.zeros(seqs + 1, dtype=torch.float64, device="cuda")
            sums = sums.index_add(0, torch.where(member < 0, torch.full_like(member, seqs), member), lp)[:seqs]
        if case["op"] == "score":
            return {"log_probs": sums.detach()}
        if case["op"] == "preference":
            other = s["other"].detach().double().requires_grad_()
            extra = [other]
            sums = sums + other
            delta = sums - s["ref"].double()
            margin = 0.1 * (delta[s["pairs"][:, 0]] - delta[s["pairs"][:, 1]])
            log_sigmoid = torch.nn.functional.logsigmoid
            target = -(0.95 * log_sigmoid(margin) + 0.05 * log_sigmoid(-margin)).sum() / margin.numel()
            out.update(loss=target, log_probs=sums, margins=margin)
        else:
            w = counted.double() * s["weights"].double() / case["rows"]
            a = s["advantages"].double()
            ratio = (lp - s["old"].double()).exp()
            bounded = torch.maximum(torch.minimum(ratio, torch.tensor(1.2, dtype=torch.float64, device="cuda")),
                                    torch.tensor(0.8, dtype=torch.float64, device="cuda"))
            kl = (s["ref"].double() - lp).exp() - (s["ref"].double() - lp) - 1
            unclipped = ratio * a <= bounded * a
            target = (w * (0.05 * kl - torch.where(unclipped, ratio * a, bounded * a))).sum()
            out.update(loss=target, log_probs=lp, kl=(w * kl).sum(), clipped=(w * (~unclipped).double()).sum())
    grads = torch.autograd.grad(target, [lp] + extra)
    coef = torch.where(counted, grads[0], torch.zeros_like(grads[0]))
    d = torch.empty(logits.shape, dtype=torch.float64, device="cuda")
    for i in range(0, case["rows"], piece):
        x = torch.softmax(logits[i:i + piece].double(), dim=1).neg_()
        x[torch.arange(len(x)), at[i:i + piece]] += 1
        d[i:i + piece] = x * coef[i:i + piece, None]
    out["dlogits"] = d
    if extra:
        out["dother"] = grads[1]
    return {k: t.detach() for k, t in out.items()}


def _exact_8bit(x, root):
    """Nearest e4m3 value (ties to even) of every element over its block's scale, by the format's definition."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(dim=1, keepdim=True)
    some = top > 2.0 ** -100
    scaled = torch.where(some, x * (448 / torch.where(some, top, torch.ones_like(top))), torch.zeros_like(x))
    grid = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.round(scaled / grid) * grid
    if root:
        q = torch.where((scaled > 0) & (q < 2.0 ** -9), torch.full_like(q, 2.0 ** -9), q)
    return q.view(-1), torch.where(some, top / 448, torch.zeros_like(top)).view(-1)


def _exact_adamw(s):
    case, t = s["case"], 101
    g = s["grad"].double()
    if case["clip"]:
        g = g * min(1.0, case["clip"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    eight = case["bits"] == 8
    if eight:
        spread = lambda k: s[k + "_scale"].double().repeat_interleave(BLOCK) * s[k].double()  # noqa: E731
        m, v = spread("exp_avg"), spread("exp_rms") ** 2
    else:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    del g
    start = (s["master"] if "master" in s else s["flat"]).double()
    w = start - LR * DECAY * start - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"weights": w}
    if "master" in s:
        out["master"] = w
    if not eight:
        return dict(out, exp_avg=m, exp_avg_sq=v)
    out["exp_avg"], out["exp_avg_scale"] = _exact_8bit(m, False)
    out["exp_rms"], out["exp_rms_scale"] = _exact_8bit(v.sqrt(), True)
    return out
