"""Adam over one flat parameter buffer, one kernel launch per step.

``torch.optim.Adam`` (``rwgnn2/main.py:79``) issues ~45 small launches for the 10 parameter tensors of
``RW_NN``; at ~0.5 ms per training step that is a fifth of the step.  Here parameters, gradients and
both moment estimates are contiguous fp32 buffers and the update is ``rwk_adam_step``.  Same arithmetic
as ``torch.optim.Adam`` (no amsgrad, no maximize); the step count and the learning rate live on the
device, so the update can be captured in a HIP graph and a scheduler can change the rate between replays.
"""
from __future__ import annotations

from itertools import chain
from operator import is_

import numpy as np
import torch

from . import _lib
from .dp import FlatGradBucket

__all__ = ["FlatAdam", "StepTail", "Adam", "AdamW"]


class FlatAdam:
    def __init__(self, module: torch.nn.Module, bucket: FlatGradBucket = None, lr=1e-3, betas=(0.9, 0.999),
                 eps=1e-8, weight_decay=0.0):
        self.bucket = bucket if bucket is not None else FlatGradBucket(module)
        params = self.bucket.params
        dev = params[0].device
        if dev.type != "cuda":
            raise RuntimeError("FlatAdam runs on HIP devices only")
        self.flat_param = torch.cat([p.detach().reshape(-1) for p in params]).contiguous()
        off = 0
        for p in params:                      # parameters become views of the flat buffer
            n = p.numel()
            p.data = self.flat_param[off:off + n].view_as(p)
            off += n
        self.exp_avg = torch.zeros_like(self.flat_param)
        self.exp_avg_sq = torch.zeros_like(self.flat_param)
        self.lr = torch.tensor([float(lr)], dtype=torch.float32, device=dev)
        self.betas = (float(betas[0]), float(betas[1]))
        self.eps = float(eps)
        self.weight_decay = float(weight_decay)
        lib = _lib.load()
        self.step_counters = torch.zeros(lib.rwk_adam_n_counters(self.flat_param.numel()), dtype=torch.int64,
                                         device=dev)

    def set_lr(self, lr: float):
        self.lr.fill_(float(lr))

    def zero_grad(self):
        self.bucket.zero()

    @torch.no_grad()
    def step(self, gather: bool = False):
        """One Adam update from ``bucket.flat``.  ``gather=True``: take the gradients from the parameters'
        ``.grad`` tensors instead (after ``bucket.release()`` and a backward pass, without ``bucket.gather()``)
        and fill ``bucket.flat`` on the way: one launch for a single-process step."""
        lib = _lib.load()
        dev = self.flat_param.device
        params = self.bucket.params
        if gather and len(params) > 16:
            self.bucket.gather()
            gather = False
        if gather:
            import ctypes
            grads = [p.grad for p in params]
            grads = [g if g is None or (g.dtype is torch.float32 and g.is_contiguous())
                     else g.detach().contiguous().float() for g in grads]
            n = len(grads)
            srcs = (ctypes.c_void_p * n)(*[None if g is None else g.data_ptr() for g in grads])
            sizes = (ctypes.c_int64 * n)(*[p.numel() for p in params])
            with _lib.device_guard(dev):
                _lib.check(lib.rwk_adam_step_chunks(
                    self.flat_param.data_ptr(), srcs, sizes, n, self.bucket.flat.data_ptr(), self.exp_avg.data_ptr(),
                    self.exp_avg_sq.data_ptr(), self.flat_param.numel(), self.lr.data_ptr(), self.betas[0],
                    self.betas[1], self.eps, self.weight_decay, self.step_counters.data_ptr(),
                    _lib.current_stream(dev)), "rwk_adam_step_chunks")
            self._keep = grads                     # the launch reads them asynchronously
            return
        _lib.check(lib.rwk_adam_step(self.flat_param.data_ptr(), self.bucket.flat.data_ptr(),
                                     self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.flat_param.numel(),
                                     self.lr.data_ptr(), self.betas[0], self.betas[1], self.eps, self.weight_decay,
                                     self.step_counters.data_ptr(), _lib.current_stream(dev)), "rwk_adam_step")


class Adam(torch.optim.Optimizer):
    """``torch.optim.Adam`` for the reference's training loop (``rwgnn2/main.py:79``: ``optim.Adam(model.parameters(),
    lr=args.lr)``) with the whole update in ONE launch: ``optimizer = gnn_amd.Adam(model.parameters(), lr=args.lr)``.

    A ``torch.optim.Optimizer`` like any other - ``zero_grad()``, ``step()``, ``param_groups`` (a learning-rate
    scheduler such as ``StepLR``, ``main.py:80``, changes ``param_groups[0]["lr"]`` and the next step uses it),
    ``state_dict()`` / ``load_state_dict()`` in torch's layout (``main.py:133,146``).  Same arithmetic as
    ``torch.optim.Adam`` without amsgrad / maximize.  torch's own implementation spends 0.13-0.24 ms of host time per
    step on the ten small tensors of ``RW_NN`` (some forty launches); this one gathers the ``.grad`` tensors and
    updates the flat parameter buffer in one (:class:`FlatAdam`).  The parameters become views of one flat buffer
    (same values, same objects).  One parameter group, all parameters on one HIP device."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        if len(self.param_groups) != 1:
            raise ValueError("gnn_amd.Adam takes one parameter group")
        group = self.param_groups[0]
        bucket = FlatGradBucket([p for p in group["params"]], bind_grads=False)
        if len(bucket.params) != len(group["params"]):
            raise ValueError("every parameter must require a gradient")
        self._flat = FlatAdam(None, bucket, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                              weight_decay=group["weight_decay"])
        self._lr_on_device = float(group["lr"])
        off = 0
        for p in bucket.params:                   # torch's layout of the state, as views of the flat buffers
            n = p.numel()
            self.state[p] = {"step": torch.zeros((), dtype=torch.float32),
                             "exp_avg": self._flat.exp_avg[off:off + n].view_as(p),
                             "exp_avg_sq": self._flat.exp_avg_sq[off:off + n].view_as(p)}
            off += n

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        group = self.param_groups[0]
        lr = float(group["lr"])
        if lr != self._lr_on_device:              # a scheduler stepped: one fill, only then
            self._flat.set_lr(lr)
            self._lr_on_device = lr
        self._flat.betas = (float(group["betas"][0]), float(group["betas"][1]))
        self._flat.eps = float(group["eps"])
        self._flat.weight_decay = float(group["weight_decay"])
        self._flat.step(gather=True)
        return loss

    def state_dict(self):
        # the step count lives on the device (it is read here only: checkpoints, main.py:133)
        t = float(self._flat.step_counters[0].item())
        for st in self.state.values():
            st["step"] = torch.tensor(t, dtype=torch.float32)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)       # leaves freshly copied tensors in self.state: move them back
        off = 0
        steps = []
        for p in self._flat.bucket.params:
            n = p.numel()
            st = self.state.get(p, {})
            for name, flat in (("exp_avg", self._flat.exp_avg), ("exp_avg_sq", self._flat.exp_avg_sq)):
                view = flat[off:off + n].view_as(p)
                if name in st:
                    view.copy_(st[name])
                else:
                    view.zero_()
                st[name] = view
            steps.append(float(st.get("step", 0.0)))
            st.setdefault("step", torch.zeros((), dtype=torch.float32))
            self.state[p] = st
            off += n
        if len(set(steps)) > 1:
            raise ValueError("gnn_amd.Adam keeps one step count for all parameters")
        self._flat.step_counters.fill_(int(steps[0]) if steps else 0)
        self._lr_on_device = None                 # param_groups was replaced: push the rate at the next step


class StepTail:
    """The optimiser's update inside the backward pass's last launch (single-process training step).

    ``RW_NN``'s backward ends with one small launch (hidden-graph backward + the input projection's gradient sum) and
    the step with another (Adam over the flat buffer).  Adam is element-wise, so the threads of the former can apply
    it to the gradient elements they finish and a few more workgroups to the head's parameters, whose gradients are
    in memory by then (``rwk_hidden_backward_reduce_adam``): one launch less per step, the same arithmetic.

    ``Trainer`` hands an instance to the model (``model._step_tail``); the model passes it down with the hand-off
    dictionary, the head's backward leaves its gradient buffer there, and the layer's backward calls :meth:`launch`
    in place of ``rwk_hidden_backward_reduce``.  ``done`` then tells the trainer to skip ``optimizer.step()``.
    Requires the flat buffer to start with ``adj_hidden, features_hidden, fc.weight, fc.bias`` (``RW_NN``'s
    parameter order) followed by the head's six tensors.

    When the head's finishing launch is folded in as well (``head_fold``), the gradients of the head's six parameters
    do not travel through autograd at all: this launch computes them, and :meth:`launch` then points the parameters'
    ``.grad`` at them.  They are valid once that launch has run, i.e. for everything queued on the stream after the
    backward pass - not inside tensor hooks of the backward pass itself, which is why the fold is taken only when
    those parameters carry no hooks and no gradient to accumulate into (:meth:`fold_allowed`)."""

    def __init__(self, model, opt: FlatAdam, update: bool = True):
        self.opt = opt
        # update=False (data-parallel step): the launch only completes the flat gradient bucket - no gather launch,
        # no finishing launch of the head - and the all-reduce and the stand-alone Adam launch follow
        self.update = bool(update)
        self.done = False
        self.armed = False        # set by the trainer around its own forward + backward only
        self._shape = None
        self.head_folds = 0       # launches that also summed the head's parameter gradients (no finishing launch)
        params = opt.bucket.params
        want = [model.adj_hidden, model.features_hidden, model.fc.weight, model.fc.bias, model.bn.weight,
                model.bn.bias, model.fc1.weight, model.fc1.bias, model.fc2.weight, model.fc2.bias]
        if len(params) != len(want) or any(a is not b for a, b in zip(params, want)):
            raise ValueError("StepTail needs RW_NN's ten parameters, all trainable, in the module's order")
        sizes = [p.numel() for p in params]
        self.off_adj, self.off_feat, self.off_red = 0, sizes[0], sizes[0] + sizes[1]
        self.red_v = sizes[2] + sizes[3]
        self.rest_off = self.off_red + self.red_v
        self.n = sum(sizes)
        self.rest_sizes = sizes[4:]
        lib = _lib.load()
        n_hidden = model.adj_hidden.shape[0]
        n_counters = max(int(lib.rwk_step_tail_n_counters(n_hidden, self.n, self.rest_off)),
                         int(lib.rwk_step_tail_n_counters_head(n_hidden, self.n, self.rest_off)))
        dev = opt.flat_param.device
        # hand-over of Adam's bias corrections from one step's launch to the next (rwk.h: corr_slot);
        # RWK_NO_CORR_SLOT=1 switches it off (every workgroup then computes its own, as the stand-alone kernels do)
        import os
        self.corr_slot = None if os.environ.get("RWK_NO_CORR_SLOT") == "1" else torch.zeros(4, dtype=torch.int64,
                                                                                              device=dev)
        # one counter per workgroup of either launch shape, all at the optimiser's step count: the two shapes may
        # then alternate (the counters one shape does not touch are brought along by sync_counters)
        if not self.update:
            self.counters = None          # the stand-alone Adam launch keeps its own
            return
        self.counters = torch.zeros(max(n_counters, opt.step_counters.numel()), dtype=torch.int64, device=dev)
        self.counters.copy_(opt.step_counters[:1].expand_as(self.counters))
        opt.step_counters = self.counters

    def fold_allowed(self) -> bool:
        """The head's six parameters have nothing that would consume a gradient from autograd during the backward
        pass: no ``.grad`` to accumulate into, no tensor hooks, no post-accumulate hooks."""
        for p in self.opt.bucket.params[4:]:
            if p.grad is not None or getattr(p, "_backward_hooks", None) \
                    or getattr(p, "_post_accumulate_grad_hooks", None):
                return False
        return True

    def sync_counters(self):
        """After an update by the stand-alone Adam launch (which advances only its own workgroups' counters)."""
        if self.counters is not None:
            self.counters.copy_(self.counters[:1].expand_as(self.counters))

    def head_sources(self, head_grads: torch.Tensor, c: int, p: int, nc: int):
        """Device addresses of the gradients of bn.weight, bn.bias, fc1.weight, fc1.bias, fc2.weight, fc2.bias inside
        the head's gradient buffer ([w2 | b2 | w1 | b1 | gamma | beta])."""
        base, f = head_grads.data_ptr(), 4
        o_w2, o_b2 = 0, nc * p
        o_w1 = o_b2 + nc
        o_b1 = o_w1 + p * c
        o_ga = o_b1 + p
        o_be = o_ga + c
        if [c, c, p * c, p, nc * p, nc] != self.rest_sizes:
            raise ValueError("head gradient buffer does not match the optimiser's parameter sizes")
        return [base + f * o for o in (o_ga, o_be, o_w1, o_b1, o_w2, o_b2)]

    def head_columns(self, c: int, p: int, nc: int):
        """Columns of the head's partial rows (layout [w2 | b2 | w1 | b1 | gamma | beta]) at which the gradients of
        bn.weight, bn.bias, fc1.weight, fc1.bias, fc2.weight, fc2.bias start."""
        o_w2, o_b2 = 0, nc * p
        o_w1 = o_b2 + nc
        o_b1 = o_w1 + p * c
        o_ga = o_b1 + p
        o_be = o_ga + c
        if [c, c, p * c, p, nc * p, nc] != self.rest_sizes:
            raise ValueError("head gradient buffer does not match the optimiser's parameter sizes")
        return [o_ga, o_be, o_w1, o_b1, o_w2, o_b2]

    def before_launch(self, shape: str):
        """Bookkeeping in front of a launch of shape ``"head"`` (the head's parameter-gradient sums ride along) or
        ``"plain"``."""
        o = self.opt
        # the handed-over bias corrections are those of one (beta1, beta2) pair: other betas start a fresh slot
        if self.corr_slot is not None and getattr(self, "_slot_betas", o.betas) != o.betas:
            self.corr_slot.zero_()
        self._slot_betas = o.betas
        # the two launch shapes have different workgroup counts, each workgroup advancing its own counter: when the
        # shape changes, the counters the previous shape did not touch are brought along first
        if self.update and self._shape is not None and self._shape != shape:
            self.sync_counters()
        self._shape = shape

    def after_launch(self, head_fold: bool):
        """The launch was queued by someone else (``composite.TrainStep``)."""
        self.head_folds += int(head_fold)
        self.done = True

    def launch(self, lib, stream, head_srcs, adj_hidden, ah, z, dz, dz_rows, n_hidden, s, d, steps, d_adj, d_feat,
               partials, blocks, red_v, red_out, head_fold=None, n_graphs=0, head_columns=None):
        import ctypes
        if red_v != self.red_v:
            raise ValueError("projection gradient width does not match fc.weight and fc.bias")
        o = self.opt
        n = len(head_srcs)
        sizes = (ctypes.c_int64 * n)(*self.rest_sizes)
        upd = (lambda t: t.data_ptr()) if self.update else (lambda t: None)
        self.before_launch("head" if head_fold is not None else "plain")
        if head_fold is not None:
            # the head's finishing launch was left out: its parameter gradients are summed here from its partial rows
            hp_ = head_fold["partials"]
            cols = (ctypes.c_int64 * n)(*head_columns)
            _lib.check(lib.rwk_hidden_backward_reduce_adam_head(
                adj_hidden, ah, z, dz, dz_rows, n_hidden, s, d, steps, d_adj, d_feat, partials, blocks, red_v, red_out,
                upd(o.flat_param), upd(o.exp_avg), upd(o.exp_avg_sq), o.bucket.flat.data_ptr(),
                self.n, self.off_adj, self.off_feat, self.off_red, cols, sizes, n, self.rest_off, upd(o.lr),
                o.betas[0], o.betas[1], o.eps, o.weight_decay, upd(self.counters), _lib.ptr(self.corr_slot),
                hp_.data_ptr(), hp_.shape[0],
                hp_.shape[1], head_fold["d_loss"].data_ptr(), head_fold["grads"].data_ptr(),
                head_fold["loss_partials"].data_ptr(), head_fold["loss"].data_ptr(), int(n_graphs), stream),
                "rwk_hidden_backward_reduce_adam_head")
            # autograd handed these six parameters nothing (head.py): their gradients are what this launch writes
            for prm, view in zip(self.opt.bucket.params[4:], head_fold["views"]):
                prm.grad = view
            self.head_folds += 1
            self.done = True
            return
        srcs = (ctypes.c_void_p * n)(*head_srcs)
        _lib.check(lib.rwk_hidden_backward_reduce_adam(
            adj_hidden, ah, z, dz, dz_rows, n_hidden, s, d, steps, d_adj, d_feat, partials, blocks, red_v, red_out,
            upd(o.flat_param), upd(o.exp_avg), upd(o.exp_avg_sq), o.bucket.flat.data_ptr(), self.n,
            self.off_adj, self.off_feat, self.off_red, srcs, sizes, n, self.rest_off, upd(o.lr), o.betas[0],
            o.betas[1], o.eps, o.weight_decay, upd(self.counters), _lib.ptr(self.corr_slot), stream),
            "rwk_hidden_backward_reduce_adam")
        self.done = True


# looks at a tensor that map() takes at the interpreter's own speed: a step has one for every tensor it holds
_address, _contiguous = torch.Tensor.data_ptr, torch.Tensor.is_contiguous
_size, _version = torch.Tensor.numel, torch.Tensor._version.__get__


class _Snapshot:
    """What the tables of an optimiser were made from.  A caller may replace or clear any of it - parameters, states,
    groups - and the addresses in the tables would be those of memory given back.  Holds what launches write."""

    def __init__(self, opt: "AdamW"):
        self.groups = list(opt.param_groups)
        self.params = [p for g in self.groups for p in g["params"]]
        self.keys, self.states = list(opt.state.keys()), list(opt.state.values())
        own = [opt.state[p] for p in self.params]
        self.values = [st.values() for st in own]                 # these follow their states
        self.tensors = list(chain.from_iterable(self.values))
        self.steps = [st["step"] for st in own]
        self.written = self.params + [t for st in own for n, t in st.items() if n.startswith("exp_avg")]
        self.matrices = [p for p in self.params if p.dim() > 1]   # others of the same size and address lie the same way
        self.seen = self._seen()

    def _seen(self):
        """What may change in a tensor that stays the same object.  (A step count changes by what a caller does to it:
        the device counts by itself.)"""
        return list(map(_address, self.written)), list(map(_size, self.params)), list(map(_version, self.steps))

    def stands(self, opt: "AdamW"):
        params = list(chain.from_iterable([g["params"] for g in opt.param_groups]))
        pairs = ((opt.param_groups, self.groups), (params, self.params), (opt.state.keys(), self.keys),
                 (opt.state.values(), self.states), (list(chain.from_iterable(self.values)), self.tensors))
        return (all([len(now) == len(then) and all(map(is_, now, then)) for now, then in pairs])
                and self._seen() == self.seen and all(map(_contiguous, self.matrices)))


class _AdamWTable:
    """Device tables of one launch shape: the parameters of one group with one type on one device."""

    def __init__(self, opt: "AdamW", group: dict, params, ids):
        self.group, self.params = group, params
        self.dtype, self.device = params[0].dtype, params[0].device
        self.type = _lib.element_type(self.dtype)
        self.chunk_size = size = int(_lib.load().rwk_adamw_chunk_size(sum(p.numel() for p in params)))
        rows, steps = [], []
        for i, (p, pid) in enumerate(zip(params, ids)):
            st = opt.state[p]
            scales = (st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_scale"].data_ptr()) if opt.state_bits == 8 else (0, 0)
            rows.append((p.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), *scales, p.numel(), 0,
                         i | pid << 32))                                               # rwk_adamw_chunk
            steps.append(int(st["step"]))
        n_chunks = -(-np.array([p.numel() for p in params], dtype=np.int64) // size)
        ends = np.cumsum(n_chunks)
        self.first_chunk = [0] + ends.tolist()
        chunks = np.repeat(np.array(rows, dtype=np.int64), n_chunks, axis=0)
        chunks[:, 6] = (np.arange(len(chunks)) - np.repeat(ends - n_chunks, n_chunks)) * size
        packed = torch.from_numpy(np.concatenate([chunks.reshape(-1), np.repeat(steps, n_chunks)])).to(self.device)
        self.packed, self.stream = packed, _lib.current_stream(self.device)
        self.chunks, self.steps = packed.split([chunks.size, len(chunks)])             # one copy to the device
        self.lr = torch.tensor([float(group["lr"])], dtype=torch.float64, device=self.device)
        self.lr_on_device = float(group["lr"])
        self.states = [opt.state[p] for p in params]
        self.counts = [(st["step"], st["step"]._version) for st in self.states]
        self.sizes = [p.numel() for p in params]

    def push_lr(self):
        lr = float(self.group["lr"])
        if lr != self.lr_on_device:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the learning rate changed: call push_lr() before the capture (a captured step "
                                   "reads the rate from the device)")
            with _lib.device_guard(self.device):
                self.lr.fill_(lr)
            self.lr_on_device = lr

    def gather(self):
        """Addresses of the gradients, checked, and the copies among them.  Whoever launches on them holds the copies
        until then (memory given back is handed out again behind the launch, on its stream); the others are their
        owner's to free, at once if it likes."""
        copies, grads = [], []
        dtype, device, strided = self.dtype, self.device, torch.strided
        for p, size in zip(self.params, self.sizes):
            g = p.grad
            if g is not None:
                if g.layout is not strided:
                    raise RuntimeError("gnn_amd.AdamW does not take sparse gradients")
                if g.dtype is not dtype or g.device != device:
                    raise TypeError("a gradient must have its parameter's type and device")
                if g.numel() != size:
                    raise ValueError("a gradient must have its parameter's shape")
                if not g.is_contiguous():
                    g = g.contiguous()
                    copies.append(g)
                g = g.data_ptr()
            grads.append(g)
        return grads, copies

    def step(self, lib, opt: "AdamW", grads):
        import ctypes
        self.push_lr()
        group, stream = self.group, _lib.current_stream(self.device)
        if stream != self.stream:                         # the tables' memory waits for this stream, too
            for t in (self.packed, self.lr):
                t.record_stream(torch.cuda.current_stream(self.device))
        limit = 256                                       # RWK_ADAMW_TENSORS: gradient addresses of one launch
        with _lib.device_guard(self.device):
            for base in range(0, len(grads), limit):
                part = grads[base:base + limit]
                lo, hi = self.first_chunk[base], self.first_chunk[base + len(part)]
                if hi == lo or all(g is None for g in part):
                    continue
                _lib.check(lib.rwk_adamw_step(
                    self.chunks.data_ptr() + 64 * lo, hi - lo, self.chunk_size, base,
                    (ctypes.c_void_p * len(part))(*part), len(part), self.type, opt.state_bits, self.lr.data_ptr(),
                    float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                    float(group["weight_decay"]), opt.seed, self.steps.data_ptr() + 8 * lo, stream),
                    "rwk_adamw_step")

    def read_steps(self, opt: "AdamW"):
        steps = self.steps.tolist()
        for i, (p, lo, hi) in enumerate(zip(self.params, self.first_chunk, self.first_chunk[1:])):
            st, (count, version) = self.states[i], self.counts[i]
            # a tensor without elements has no chunk to count in; a count that a caller replaced is the caller's
            if hi > lo and opt.state.get(p) is st and st.get("step") is count and count._version == version:
                st["step"] = count = torch.tensor(float(steps[lo]), dtype=torch.float32)
                self.counts[i] = count, count._version


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over any number of tensors with one launch per 256 of them, their moment
    estimates held in 32 or in 8 bits: ``optimizer = gnn_amd.AdamW(model.parameters(), lr=1e-3, state_bits=8)``.

    A ``torch.optim.Optimizer``: parameter groups with their own rates, betas and decay, schedulers, closures,
    ``state_dict()`` / ``load_state_dict()``.  Parameters are contiguous float32, float16 or bfloat16 tensors on HIP
    devices and stay where they are (:class:`Adam` moves them into one flat fp32 buffer).  The update is computed in
    fp32 and rounded to the parameter's type once; a parameter whose ``.grad`` is ``None`` is skipped and does not
    age.  The step counts and the learning rate live on the device, so a captured step replays correctly;
    :meth:`push_lr` hands a changed rate to replays.  Replays go on with the states of the capture: after
    ``load_state_dict``, new groups or states of a caller's own, capture again.

    ``state_bits=32``: ``exp_avg`` and ``exp_avg_sq`` are float32, in torch's layout.  ``state_bits=8``: they are
    float8 (e4m3) tensors with one fp32 scale per 256 consecutive elements (``exp_avg_scale``, ``exp_avg_sq_scale``;
    a moment is value times scale), a quarter of the memory.  Values are rounded up or down at random in proportion to
    the distances - ``exp_avg_sq`` moves by a thousandth per step, far less than the spacing of 8-bit values - with
    bits that follow from ``seed``, the step, the tensor's place and the element, so runs repeat bit by bit.  A
    gradient that is not finite makes its whole block of 256 moments not finite."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not 0 <= int(seed) < 2 ** 64:
            raise ValueError("seed must be in 0 .. 2^64 - 1")
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._tables = self._made_from = None
        self._captured = []                               # what replays of captured steps read and write
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_options(group)
            for p in group["params"]:
                if not p.is_cuda:
                    raise RuntimeError("gnn_amd runs on HIP devices only (no CPU fallback)")
                _lib.element_type(p.dtype)
                if p.layout != torch.strided or not p.is_contiguous():
                    raise ValueError("gnn_amd.AdamW takes contiguous parameters")
        except Exception:
            self.param_groups.pop()
            raise
        for p in group["params"]:
            self.state[p] = self._new_state(p)
        self._drop_tables()

    @staticmethod
    def _check_options(group):
        if not float(group["lr"]) >= 0.0:
            raise ValueError("lr must not be negative")
        if not float(group["eps"]) >= 0.0:
            raise ValueError("eps must not be negative")
        if not float(group["weight_decay"]) >= 0.0:
            raise ValueError("weight_decay must not be negative")
        if not all(0.0 <= float(b) < 1.0 for b in group["betas"]):
            raise ValueError("betas must be in [0, 1)")
        for name in ("amsgrad", "maximize", "differentiable"):        # torch's, also out of its checkpoints
            if group.get(name):
                raise ValueError(f"gnn_amd.AdamW has no {name}")
        if not group.get("decoupled_weight_decay", True) and float(group["weight_decay"]):
            raise ValueError("gnn_amd.AdamW decouples the weight decay")

    def _new_state(self, p):
        st = {"step": torch.zeros((), dtype=torch.float32)}
        n = p.numel()
        for name in ("exp_avg", "exp_avg_sq"):
            if self.state_bits == 32:
                st[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                blocks = (n + 255) // 256
                flat = torch.zeros(blocks * 256, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                st[name] = flat[:n].view(p.shape)         # the kernel reads and writes whole blocks of 256
                st[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return st

    def _check_state(self, p):
        """The parameter's state as the kernels can use it: made anew if it was cleared, refused if it does not fit."""
        st = self.state.get(p)
        if not st:
            st = self.state[p] = self._new_state(p)
        if not isinstance(st.get("step"), torch.Tensor):
            st["step"] = torch.tensor(float(st.get("step", 0)), dtype=torch.float32)
        n, device = p.numel(), p.device
        blocks = (n + 255) // 256
        for name in ("exp_avg", "exp_avg_sq"):
            wanted = [(name, p.shape, torch.float32)]
            if self.state_bits == 8:
                wanted = [(name, p.shape, torch.float8_e4m3fn), (name + "_scale", (blocks,), torch.float32)]
            for key, shape, dtype in wanted:
                t = st.get(key)
                if t is None:
                    raise ValueError(f"the state of a parameter has no {key}")
                if t.device != device:
                    raise RuntimeError("a parameter or its state moved to another device after the optimiser was built")
                if t.dtype != dtype or t.shape != shape:
                    raise ValueError(f"{key} is {t.dtype} of shape {tuple(t.shape)} for a parameter of shape "
                                     f"{tuple(p.shape)}, not {dtype} of shape {tuple(shape)}")
                if not t.is_contiguous():
                    st[key] = t = t.contiguous()
                # the kernel reads and writes whole blocks, so the last one's rest has to be the tensor's own
                if dtype == torch.float8_e4m3fn and (t.storage_offset() or t.untyped_storage().nbytes() != 256 * blocks):
                    st[key] = self._new_state(p)[key].copy_(t)

    def _read_steps(self):
        """The step counts live on the device; the states get them when somebody looks."""
        if self._tables is not None:
            stood = self._made_from.stands(self)
            for t in self._tables:
                t.read_steps(self)
            if stood:
                self._made_from = _Snapshot(self)         # with the counts just written

    def _drop_tables(self):
        """The tables describe other tensors from here on: their step counts move to the state."""
        self._read_steps()
        self._tables = self._made_from = None

    def _build_tables(self):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gnn_amd.AdamW builds its tables at its first step and whenever a parameter moved: "
                               "take one step before the capture")
        self._drop_tables()
        tables, pid = [], 0
        for group in self.param_groups:
            kinds = {}
            for p in group["params"]:
                if not p.is_cuda or p.layout != torch.strided or not p.is_contiguous():
                    raise ValueError("gnn_amd.AdamW takes contiguous parameters on HIP devices")
                self._check_state(p)
                kinds.setdefault((p.dtype, p.device), ([], []))
                kinds[p.dtype, p.device][0].append(p)
                kinds[p.dtype, p.device][1].append(pid)
                pid += 1
            for params, ids in kinds.values():
                with _lib.device_guard(params[0].device):
                    tables.append(_AdamWTable(self, group, params, ids))
        self._tables, self._made_from = tables, _Snapshot(self)

    def push_lr(self):
        """Hand changed learning rates to the device (``step`` does it by itself; replays of a captured step do not)."""
        for t in self._tables or ():
            t.push_lr()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._tables is None or not self._made_from.stands(self):
            self._build_tables()
        lib = _lib.load()
        grads = [t.gather() for t in self._tables]        # all are checked before anything changes
        if torch.cuda.is_current_stream_capturing() and all(t is not self._tables for t, _ in self._captured):
            self._captured.append((self._tables, self._made_from))
        for t, (addresses, _) in zip(self._tables, grads):
            t.step(lib, self, addresses)
        return loss

    def __getstate__(self):                               # copy.deepcopy, pickle: tables are built anew
        self._read_steps()
        return super().__getstate__() | {"state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables = self._made_from = None
        self.__dict__.setdefault("_captured", [])

    def state_dict(self):
        self._read_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        names = ["exp_avg", "exp_avg_sq"]
        if self.state_bits == 8:
            names += ["exp_avg_scale", "exp_avg_sq_scale"]
        for group in state_dict["param_groups"]:
            self._check_options(group)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        new = {}
        for i, p in zip(saved, params):                   # checked whole before anything is changed
            st = self._new_state(p)
            src = state_dict["state"].get(i)
            if src:
                for name in names:
                    if name not in src:
                        raise ValueError(f"the saved state has no {name}: it was made with other state_bits")
                    dtype = torch.float8_e4m3fn if self.state_bits == 8 and not name.endswith("_scale") \
                        else torch.float32
                    if src[name].dtype != dtype or src[name].shape != st[name].shape:
                        raise ValueError(f"the saved {name} is {src[name].dtype} of shape {tuple(src[name].shape)}, "
                                         f"not {dtype} of shape {tuple(st[name].shape)}")
                    st[name].copy_(src[name])
                st["step"] = torch.tensor(float(src["step"]), dtype=torch.float32)
            new[p] = st
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        self._tables = self._made_from = None
        for p, st in new.items():
            self.state[p] = st
