"""AdamW over many tensors at once on the package's kernels, states in 32 or in 8 bits.

``AdamW`` is a ``torch.optim.Optimizer`` (learning-rate schedulers, parameter groups and state dicts work as usual).  A
step is two launches per group whatever the number of tensors (step counts and bias corrections; the update), one more if
the gradients' global 2-norm is clipped (``max_norm``), the same again for every further 400 tensors, and nothing of it waits
on the host.

States live in one buffer per group and kind; ``optimizer.state[p]`` holds views of them.  With ``state_bits=8`` the
first moment and the square root of the second are kept as e4m3 values with one fp32 scale per 256 elements: 2.03 bytes
per parameter instead of 8.  Such a value has three bits behind the point, and a step with ``beta2 = 0.999`` moves a root by
less than half a place: rounded to nearest, an element's share in its block stands still until a gradient is eight to
eleven times its root, and only the block's scale follows the gradients.  ``rounding="stochastic"`` rounds to one of the
two neighbours with the right mean instead (by bits that are a function of element, tensor and step: runs repeat), so
that every element follows its own gradients, within some 15 % of the root, for 9 % more time where the step is bound by
memory (477 M bf16 elements: 1362 -> 1488 us; the trainer's 5.1 M: 25 -> 26 on the device).  16-bit parameters are stepped
on an fp32 copy (``master=True``), since a step is usually smaller than half their last place.
"""
from __future__ import annotations

import copy
import ctypes as C
import operator

import numpy as np
import torch

from . import _capi as K
from .losses import guard

_E4M3 = torch.float8_e4m3fn
_GRAD, _DTYPE = operator.attrgetter("grad"), operator.attrgetter("dtype")
_SCALED = ("exp_avg_scale", "exp_rms_scale")


def _up(n, to):
    return -(-n // to) * to


class _Group:
    """Buffers and tables of one parameter group."""

    def __init__(self, params, bits, master):
        self.params, self.bits = params, bits
        dev, dt = params[0].device, params[0].dtype
        self.device, self.dtype = dev, dt
        self.master = bool(master) and dt != torch.float32
        self.numels = [p.numel() for p in params]
        self.starts = np.concatenate([[0], np.cumsum([_up(n, K.ADAMW_BLOCK) for n in self.numels])]).astype(np.int64)
        self.n_elems = sum(self.numels)
        total = int(self.starts[-1])
        zeros = lambda n, t: torch.zeros(n, dtype=t, device=dev)  # noqa: E731
        self.buffers = {}
        if self.master:
            self.buffers["master"] = zeros(total, torch.float32)
        if bits == 32:
            self.buffers["exp_avg"] = zeros(total, torch.float32)
            self.buffers["exp_avg_sq"] = zeros(total, torch.float32)
        else:
            for k in ("exp_avg", "exp_rms"):
                self.buffers[k] = zeros(total, torch.uint8).view(_E4M3)
                self.buffers[k + "_scale"] = zeros(total // K.ADAMW_BLOCK, torch.float32)
        self.steps = zeros(len(params), torch.int32)
        self.bias = zeros(2 * len(params), torch.float32)
        n_chunks = [-(-n // K.ADAMW_CHUNK) for n in self.numels]
        self.chunk_ptr = np.concatenate([[0], np.cumsum(n_chunks)]).astype(np.int64)
        self.n_chunks = int(self.chunk_ptr[-1])
        of = np.repeat(np.arange(len(params)), n_chunks)
        chunks = np.stack([of, np.arange(self.n_chunks) - self.chunk_ptr[of]], axis=1).astype(np.int32)
        self.chunks = torch.from_numpy(chunks.reshape(-1) if chunks.size else np.zeros(2, np.int32)).to(dev)
        self.partials = zeros(max(self.n_chunks, 1), torch.float64)
        self.addresses = None
        self.table = zeros(C.sizeof(K.AdamwTensor) * len(params), torch.uint8)
        self.grads, self.grad_list = (C.c_void_p * len(params))(), None
        self.grads_at = C.addressof(self.grads)
        self.views = [self._views(i) for i in range(len(params))]
        if self.master:
            self.copy_master()

    def _views(self, i):
        """State tensors of parameter ``i``: views of the group's buffers."""
        at, n = int(self.starts[i]), self.numels[i]
        out = {"step": self.steps[i]}
        for k, buf in self.buffers.items():
            if k in _SCALED:
                out[k] = buf[at // K.ADAMW_BLOCK:at // K.ADAMW_BLOCK + _up(n, K.ADAMW_BLOCK) // K.ADAMW_BLOCK]
            else:
                out[k] = buf[at:at + n].view(self.params[i].shape)
        return out

    def copy_master(self, which=None):
        for i, p in enumerate(self.params):
            if which is None or i in which:
                self.views[i]["master"].copy_(p.detach())

    def bind(self):
        """The device table of addresses; written again, in its place, only when a parameter's storage has moved."""
        addresses = list(map(torch.Tensor.data_ptr, self.params))
        # a parameter may have been turned in its place (p.data = p.data.t()): the elements' order is part of the table
        if addresses == self.addresses and all(map(torch.Tensor.is_contiguous, self.params)):
            return
        for p, n in zip(self.params, self.numels):
            if p.device != self.device or p.dtype != self.dtype or p.numel() != n or not p.is_contiguous():
                raise RuntimeError("AdamW: a parameter changed its device, type, size or layout after the optimizer "
                                   "was built; build it again")
        spans = sorted((a, a + n * p.element_size()) for a, n, p in zip(addresses, self.numels, self.params) if n)
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise RuntimeError("AdamW: parameters of one group share memory; a step would work on it twice at once")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the parameters' addresses must be known before a capture; make one step first")
        items = (K.AdamwTensor * len(self.params))()
        second = "exp_avg_sq" if self.bits == 32 else "exp_rms"
        for i, (p, v) in enumerate(zip(self.params, self.views)):
            items[i] = K.AdamwTensor(addresses[i], K.ptr(v.get("master")), v["exp_avg"].data_ptr(), v[second].data_ptr(),
                                     K.ptr(v.get("exp_avg_scale")), K.ptr(v.get("exp_rms_scale")), self.numels[i])
        host = np.frombuffer(bytes(items), dtype=np.uint8).copy()
        self.table.copy_(torch.from_numpy(host))
        self.addresses = addresses

    def _name_grads(self, addresses):
        """The address list of the launches, written where it changed (gradients mostly stay where they are)."""
        if addresses != self.grad_list:
            self.grads[:] = self.grad_list = addresses

    def gather_grads(self):
        """Fills the address list; (parameters with a gradient, tensors to keep alive until the launches)."""
        grads, dt, T = list(map(_GRAD, self.params)), self.dtype, torch.Tensor
        try:  # the usual case in passes without Python code of their own: every parameter has a plain gradient
            plain = list(map(T.numel, grads)) == self.numels and all(map(T.is_contiguous, grads)) \
                and set(map(_DTYPE, grads)) == {dt}
        except TypeError:  # None among them
            plain = False
        if plain:
            self._name_grads(list(map(T.data_ptr, grads)))
            return self.params, grads
        if any(g is not None and g.numel() != n for g, n in zip(grads, self.numels)):
            raise RuntimeError("AdamW: a gradient has another size than its parameter had when the optimizer was built")
        grads = [None if g is None else g.detach().to(dt).contiguous() for g in grads]
        self._name_grads([None if g is None else g.data_ptr() for g in grads])
        return [p for p, g in zip(self.params, grads) if g is not None], grads

    def args(self, hyper):
        lr = hyper["lr"]
        lr_dev = None
        if isinstance(lr, torch.Tensor):
            if lr.device == self.device:
                if lr.dtype != torch.float32 or lr.numel() != 1:
                    raise ValueError("AdamW: a learning rate on the device is one float32 value")
                lr_dev, lr = lr.data_ptr(), 0.0
            else:
                lr = float(lr)
        b1, b2 = hyper["betas"]
        return K.AdamwGroup(self.table.data_ptr(), self.chunks.data_ptr(), self.chunk_ptr.ctypes.data,
                            self.grads_at, self.steps.data_ptr(), self.bias.data_ptr(),
                            len(self.params), self.n_chunks, K.DTYPE_CODE[self.dtype], self.bits, int(self.master),
                            int(hyper["rounding"] == "stochastic"), lr_dev, lr, b1, b2, hyper["eps"], hyper["weight_decay"])


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay: with g the gradient (times the clip factor), t the tensor's step count,

        m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2,
        w = w (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps).

    ``state_bits``: 32, or 8; ``rounding`` of 8-bit states: "nearest" or "stochastic" (see the module).  ``master``:
    16-bit parameters keep an fp32 copy that the step works on; it is the optimizer's, so a value written into such a
    parameter from outside needs ``refresh_master()``.  ``max_norm``: gradients are multiplied by
    ``min(1, max_norm / (norm + 1e-6))``, norm being the 2-norm over all parameters of all groups - inside the step,
    ``.grad`` keeps what backward left; ``grad_norm`` (a 0-d device tensor) holds the norm of the last step.  All
    parameters are contiguous and on one GPU, those of a group of one type and without memory in common; a parameter
    without a gradient is left alone.  A captured step replays with the gradients' addresses of the capture; a learning
    rate that changes between replays is a float32 tensor on the device."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master=True,
                 max_norm=None, rounding="nearest"):
        self._bound = []
        self._norm = None
        self.max_norm = self._check_norm(max_norm)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master=master, rounding=rounding))

    @staticmethod
    def _check_norm(max_norm):
        if max_norm is not None and not float(max_norm) > 0:
            raise ValueError("AdamW: max_norm must be positive, got %r" % (max_norm,))
        return max_norm

    @staticmethod
    def _check_hyper(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if not isinstance(lr, torch.Tensor) and not float(lr) >= 0:
            raise ValueError("AdamW: lr = %r" % (lr,))
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError("AdamW: betas = %r" % (g["betas"],))
        if not (g["eps"] >= 0 and g["weight_decay"] >= 0):
            raise ValueError("AdamW: eps = %r, weight_decay = %r" % (g["eps"], g["weight_decay"]))
        if g["rounding"] not in ("nearest", "stochastic"):
            raise ValueError("AdamW: rounding is nearest or stochastic, got %r" % (g["rounding"],))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            self._check_hyper(g)
            if g["state_bits"] not in (8, 32):
                raise ValueError("AdamW: state_bits is 32 or 8, got %r" % (g["state_bits"],))
            if len(set(g["params"])) != len(g["params"]):
                raise ValueError("AdamW: a parameter appears twice in a group")
            for p in g["params"]:
                if p.dtype not in K.DTYPE_CODE:
                    raise TypeError("AdamW: parameters are float32, float16 or bfloat16, got %s" % p.dtype)
                if p.dtype != g["params"][0].dtype:
                    raise TypeError("AdamW: a group holds parameters of one type, got %s and %s"
                                    % (g["params"][0].dtype, p.dtype))
                first = self._bound[0].device if self._bound else g["params"][0].device
                if p.device != first:
                    raise RuntimeError("AdamW: parameters on %s and %s" % (first, p.device))
                if not p.is_contiguous():
                    raise ValueError("AdamW: parameters must be contiguous")
            if not g["params"] or g["params"][0].device.type != "cuda":
                raise RuntimeError("fast_jtnn_hip.AdamW runs on an MI355X only (parameters are on %s); there is no CPU "
                                   "path" % (g["params"][0].device if g["params"] else "no device"))
        except Exception:
            self.param_groups.pop()
            raise
        with torch.no_grad(), torch.cuda.device(g["params"][0].device):
            group = _Group(g["params"], g["state_bits"], g["master"])
            if self._norm is None:
                self._norm = torch.zeros(2, dtype=torch.float32, device=group.device)
        self._bound.append(group)
        for p, v in zip(group.params, group.views):
            self.state[p] = v

    def __getstate__(self):
        raise TypeError("AdamW cannot be copied or pickled (its tables hold addresses): use state_dict()")

    @property
    def grad_norm(self):
        """2-norm of all gradients at the last step with ``max_norm``, before the clip (0-d, on the device)."""
        return self._norm[0]

    def state_buffers(self):
        """One dict per group: the buffers that hold its states, every tensor's part starting at a multiple of 256
        elements (scales: one per 256).  The buffers themselves, not copies."""
        return [dict(g.buffers) for g in self._bound]

    @torch.no_grad()
    def refresh_master(self):
        """Takes the fp32 copies of 16-bit parameters from the parameters' present values."""
        for g in self._bound:
            if g.master:
                g.copy_master()

    def step(self, closure=None):
        """One step of every parameter that has a gradient; returns what ``closure`` (which forms the gradients) does."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_norm = 0.0 if self.max_norm is None else float(self._check_norm(self.max_norm))
        with guard(self._bound[0].device):
            work, keep, args, changed = [], [], [], []
            for g, hyper in zip(self._bound, self.param_groups):
                self._check_hyper(hyper)
                g.bind()
                have, k = g.gather_grads()
                if have:
                    keep += k
                    changed += have
                    work.append(g)
                    args.append(g.args(hyper))
            if not work:
                return loss
            partials = None
            if max_norm:
                partials = work[0].partials if len(work) == 1 else \
                    torch.empty(sum(g.n_chunks for g in work), dtype=torch.float64, device=self._norm.device)
            K.adamw_step((K.AdamwGroup * len(args))(*args), len(args), max_norm, K.ptr(partials),
                         self._norm.data_ptr(), n_elems=[g.n_elems for g in work])
            # the kernels wrote through raw addresses: weights packed for the products, and autograd's check of saved
            # tensors, go by the version counter
            torch.autograd.graph.increment_version(changed)
        return loss

    def load_state_dict(self, state_dict):
        """Takes the states of a dict of the same parameter groups (this class's, or with ``state_bits=32`` that of
        ``torch.optim.AdamW`` / ``Adam`` without the variants that this class does not step by) into the buffers;
        hyperparameters follow the dict, ``state_bits`` and ``master`` do not.  A learning rate on the device takes its
        new value in its place.  A parameter without an entry starts afresh.  Registered hooks run around it."""
        state_dict = dict(state_dict)  # a hook may change it, not the caller's
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            new = hook(self, state_dict)
            state_dict = state_dict if new is None else new
        with torch.no_grad():
            self._load(state_dict)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def _load(self, state_dict):
        groups = state_dict["param_groups"]
        if len(groups) != len(self.param_groups):
            raise ValueError("AdamW: the state dict has %d parameter groups, the optimizer %d"
                             % (len(groups), len(self.param_groups)))
        for new, g in zip(groups, self._bound):
            if len(new["params"]) != len(g.params):
                raise ValueError("AdamW: a group of the state dict has %d parameters, the optimizer's %d"
                                 % (len(new["params"]), len(g.params)))
            for k in ("amsgrad", "maximize"):
                if new.get(k):
                    raise ValueError("AdamW: the state dict's %s is not offered" % k)
            if new.get("weight_decay") and not new.get("decoupled_weight_decay", True):
                raise ValueError("AdamW: the state dict's weight decay is part of its gradients, not decoupled")
        todo = []
        for new, g in zip(groups, self._bound):
            for i, key in enumerate(new["params"]):
                have = state_dict["state"].get(key, {})
                todo.append((g, i, have))
                if not have:
                    continue
                for k, dst in g.views[i].items():
                    if k == "master" and k not in have:
                        continue
                    if k not in have:
                        raise KeyError("AdamW: the state dict has no %s for a parameter (states of other bits?)" % k)
                    src = torch.as_tensor(have[k])
                    if src.numel() != dst.numel() or (dst.dtype == _E4M3) != (src.dtype == _E4M3):
                        raise ValueError("AdamW: %s is %s %s in the state dict, %s %s in the optimizer"
                                         % (k, src.dtype, tuple(src.shape), dst.dtype, tuple(dst.shape)))
        for g, i, have in todo:
            for k, dst in g.views[i].items():
                if k in have:
                    src = torch.as_tensor(have[k]).detach().reshape(dst.shape)
                    if dst.dtype == _E4M3:  # bytes: copies of the type itself are not needed
                        dst.view(torch.uint8).copy_(src.view(torch.uint8))
                    else:
                        dst.copy_(src)
                elif k == "master":
                    g.copy_master({i})
                elif dst.dtype == _E4M3:
                    dst.view(torch.uint8).zero_()
                else:
                    dst.zero_()
        for new, mine in zip(groups, self.param_groups):
            lr = mine["lr"]
            mine.update({k: copy.deepcopy(v) for k, v in new.items() if k not in ("params", "state_bits", "master")})
            if isinstance(lr, torch.Tensor):  # a captured step reads it where it is
                mine["lr"] = lr.fill_(float(mine["lr"]))
