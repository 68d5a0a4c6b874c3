"""``SparseGaussianAdam``: the reference's visibility-masked Adam (``fast_2d_gs/sparse_gaussian_adam.py:10-49``)
with every parameter group updated by ONE kernel launch instead of one launch per group; ``DenseAdam`` for dense
parameters through the same kernel; ``AdamW`` over many dense tensors with moments in 32 or in 8 bits, clipping by the
norm of all gradients (``grad_norm``) and a step count on the device."""
import ctypes

import numpy as np
import torch
from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from . import _lib
from ._lib import lib, check
from .ops import _need, _ptr, _stream


class SparseGaussianAdam(torch.optim.Adam):
    """Same constructor, ``set_before_step(visibility, N)`` and ``step()`` as the reference class; beta1 = 0.9 and
    beta2 = 0.999 are fixed and the bias correction is folded into the learning rate, as there.
    State layout (``step`` as a CPU float32 tensor, ``exp_avg``, ``exp_avg_sq``) is the reference's, so its
    checkpoints load."""

    def __init__(self, params, lr, eps):
        super().__init__(params=params, lr=lr, eps=eps)
        self.N = None
        self.visibility = None
        self._bias_cache = (None, None, None)

    def _bias_terms(self, step):
        """((1 - 0.999^t)^0.5, 1 - 0.9^t) as float32 tensors, computed once per distinct step count (all groups of a
        step share it) exactly as the reference's expression computes them."""
        t = float(step)
        if self._bias_cache[0] != t:
            self._bias_cache = (t, (1 - 0.999 ** step) ** 0.5, 1 - 0.9 ** step)
        return self._bias_cache[1], self._bias_cache[2]

    def set_before_step(self, visibility, N):
        self.visibility, self.N = visibility, N

    @torch.no_grad()
    def step(self, only=None):
        """``only``: an iterable of parameters; the step is then applied to those groups alone (each parameter keeps
        its own step count, so a step may be split to overlap with communication)."""
        self.step_visible(only)

    def step_visible(self, only=None):
        """The body of ``step`` as a plain method: ``torch.optim.Optimizer`` wraps ``step`` itself in profiling and
        hook layers that cost more host time than the launch; a training loop that has no use for them calls this."""
        batch = []
        only = None if only is None else {id(p) for p in only}
        for group in self.param_groups:
            assert len(group["params"]) == 1, "more than one tensor in group"
            param = group["params"][0]
            if only is not None and id(param) not in only:
                continue
            if param.grad is None or param.grad.numel() == 0:
                continue
            state = self.state[param]
            if len(state) == 0:
                state["step"] = torch.tensor(0.0, dtype=torch.float32)
                state["exp_avg"] = torch.zeros_like(param, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(param, memory_format=torch.preserve_format)
            state["step"] += 1
            s, b = self._bias_terms(state["step"])
            lr_eff = group["lr"] * s / b  # the reference's float32 tensor arithmetic, in its order
            batch.append((param, param.grad.detach(), state["exp_avg"], state["exp_avg_sq"], float(lr_eff),
                          group["eps"]))
        if not batch:
            return
        assert self.N is not None, "call set_before_step(visibility, N) before step()"
        masked_adam_step(batch, self.visibility, self.N)




class DenseAdam(torch.optim.Adam):
    """torch.optim.Adam for a few dense parameter tensors (the deformation network, the kernel weights), every tensor
    updated by the one launch that updates the Gaussians' tensors (``fsgs_adam_masked_multi``: each tensor is one
    "row" of its own length behind a one-element gate).  torch's fused Adam takes 0.08 ms for the 2 MB of the
    deformation network; this takes 0.005.  Same state layout as torch's (``step``, ``exp_avg``, ``exp_avg_sq``), same
    update -- ``p -= lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)`` -- written as the kernel's
    ``p -= lr' m / (sqrt(v) + eps')`` with ``lr' = lr sqrt(1 - b2^t) / (1 - b1^t)``, ``eps' = eps sqrt(1 - b2^t)``.
    The kernel forms ``1 - beta`` in float32, torch in double: second moments agree to 1.3e-5 relative, steps to 1e-5.
    ``step(gate=...)``: a one-element float32 device tensor; the step is applied where it is > 0 (default: applied)."""

    def __init__(self, params, lr, eps=1e-8, betas=(0.9, 0.999)):
        super().__init__(params=params, lr=lr, eps=eps, betas=betas)
        self._one = None

    @torch.no_grad()
    def step(self, gate=None):
        self.step_gated(gate)

    def step_gated(self, gate=None):
        for group in self.param_groups:
            b1, b2 = group["betas"]
            batch = []
            for param in group["params"]:
                if param.grad is None or param.numel() == 0:
                    continue
                state = self.state[param]
                if len(state) == 0:
                    state["step"] = torch.tensor(0.0, dtype=torch.float32)
                    state["exp_avg"] = torch.zeros_like(param, memory_format=torch.preserve_format)
                    state["exp_avg_sq"] = torch.zeros_like(param, memory_format=torch.preserve_format)
                state["step"] += 1
                t = float(state["step"])
                root = (1.0 - b2 ** t) ** 0.5
                batch.append((param, param.grad.detach(), state["exp_avg"], state["exp_avg_sq"],
                              group["lr"] * root / (1.0 - b1 ** t), group["eps"] * root))
            if not batch:
                continue
            if gate is None:
                if self._one is None or self._one.device != batch[0][0].device:
                    self._one = torch.ones(1, device=batch[0][0].device)
                gate = self._one
            masked_adam_step(batch, gate, 1, b1=b1, b2=b2)


def masked_adam_step(batch, visibility, N, b1=0.9, b2=0.999):
    """``batch``: list of (param, grad, exp_avg, exp_avg_sq, lr_eff, eps) with ``param.numel() % N == 0``.
    Launches ``fsgs_adam_masked_multi`` once per eight tensors."""
    vis = visibility.contiguous()
    # a float mask (visible where > 0) is the form in which the mask comes out of the gradient all-reduce
    launch = lib().fsgs_adam_masked_multi_fmask if vis.dtype == torch.float32 else lib().fsgs_adam_masked_multi
    if vis.dtype != torch.float32 and vis.dtype != torch.uint8:
        vis = vis.to(torch.uint8) if vis.dtype != torch.bool else vis
    for i in range(0, len(batch), 8):
        chunk = batch[i:i + 8]
        arr = (_lib.AdamTensor * len(chunk))()
        keep = []
        for k, (p, g, m, v, lr, eps) in enumerate(chunk):
            assert p.is_cuda and p.is_contiguous() and p.dtype == torch.float32
            g = g.contiguous()
            keep.append(g)
            arr[k].param, arr[k].grad, arr[k].exp_avg, arr[k].exp_avg_sq = p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr()
            arr[k].M, arr[k].lr, arr[k].eps = p.numel() // N, lr, eps
        check(launch(len(chunk), arr, _ptr(vis), int(N), b1, b2, _stream()), "fsgs_adam_masked_multi")


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # FSGS_F32, FSGS_BF16, FSGS_F16
_BLOCK = 256                                                        # FSGS_ADAMW_BLOCK
_STALE, _STRIDED = 1, 2                                             # answers of the host extension besides a status
_table_type = np.dtype([(n, np.float32 if t is ctypes.c_float else np.int64) for n, t in _lib.AdamWTensor._fields_])
assert _table_type.itemsize == ctypes.sizeof(_lib.AdamWTensor)


def grad_norm(tensors, max_norm=None):
    """``(norm, factor)``: the 2-norm of all elements of all ``tensors`` (float32, bfloat16 or float16, on one device)
    and ``min(1, max_norm / (norm + 1e-6))``, the factor that clips them to ``max_norm`` -- 1 without ``max_norm``, 0
    where the norm is not finite.  Two float32 device scalars, one pass (a launch per 256 tensors and one that closes the
    sum) and no synchronisation; the factor can be given to ``AdamW.step(grad_scale=...)``.  Summed in a fixed order: the
    same gradients give the same bits."""
    _need(max_norm is None or max_norm > 0, "grad_norm: max_norm must be positive")
    return _lib.host().norm(list(tensors), float("inf") if max_norm is None else float(max_norm))


def _number(v):
    """A setting as a number; a tensor on a device would make every step wait for it."""
    if v.__class__ is float:
        return v
    _need(not (torch.is_tensor(v) and v.is_cuda),
          "AdamW: lr, betas, eps and weight_decay are numbers on the host (a step would wait for the device to read them)")
    return float(v)


class _Plan:
    """The argument tables of a step for one list of parameters, and what the host extension compares them with: it reads
    every address, length and type of the parameters, gradients and states anew each step, and a plan is used only while
    they are what it was made from."""

    def __init__(self, opt):
        self.settings, self.form = self.current_settings(opt), (opt.state_bits, opt.master_weights)
        self.seen = self.plain_settings(opt)
        self.params, self.groups, found, kinds = [], [], [], {}
        for k, group in enumerate(opt.param_groups):
            tail = self.settings[k][2:]
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                _need(p.is_cuda and p.dtype in _TYPES and g.dtype in _TYPES, "AdamW: float32, bfloat16 or float16 CUDA parameters on one device")
                master = opt.master_weights and p.dtype != torch.float32
                kinds.setdefault((_TYPES[p.dtype], _TYPES[g.dtype], master) + tail, []).append(len(found))
                found.append((p, k, opt._state_of(p), master))
                self.params.append(p)
                self.groups.append(k)
        self.device = self.params[0].device
        self.launches, entries = [], [None] * len(found)
        for (param_type, grad_type, _, *numbers), rows in kinds.items():
            t = np.zeros(len(rows), _table_type)
            start = t.ctypes.data
            self.launches.append((rows, t, (len(rows), start, param_type, grad_type, opt.state_bits, *numbers)))
            for k, i in enumerate(rows):
                entries[i] = found[i] + (start + k * _table_type.itemsize,)
        self.rates()
        self.handle = _lib.host().plan(entries, [l[2] for l in self.launches], opt.state_bits)

    @staticmethod
    def current_settings(opt):
        """Learning rate, weight decay, both betas and eps of every group."""
        return [(_number(g["lr"]), _number(g["weight_decay"]), *map(_number, g["betas"]), _number(g["eps"]))
                for g in opt.param_groups]

    def plain_settings(self, opt):
        """The same as they stand there, None where one of them is no float (a tensor may change where it lies)."""
        found = [(g["lr"], g["weight_decay"], *g["betas"], g["eps"]) for g in opt.param_groups]
        return found if all(v.__class__ is float for t in found for v in t) else None

    def follow(self, opt):
        """Take over changed learning rates and weight decays; False where betas, eps or the form of the state changed."""
        if (opt.state_bits, opt.master_weights) != self.form:
            return False
        if self.seen is not None and self.seen == [(g["lr"], g["weight_decay"], *g["betas"], g["eps"]) for g in opt.param_groups]:
            return True
        self.seen = self.plain_settings(opt)
        now = self.current_settings(opt)
        if now != self.settings:
            if [s[2:] for s in now] != [s[2:] for s in self.settings]:
                return False
            self.settings = now
            self.rates()
        return True

    def rates(self):
        for rows, table, _ in self.launches:
            table["lr"], table["weight_decay"] = ([self.settings[self.groups[i]][k] for i in rows] for k in (0, 1))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over any number of dense tensors, one launch for all that share their types:

        ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
        ``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)``.

    Parameters are contiguous CUDA tensors of float32, bfloat16 or float16 on one device that share no memory, gradients
    of the parameter's type or (``param.grad_dtype``) float32.  ``lr``, ``betas``, ``eps`` and ``weight_decay`` are per group and may be
    changed between steps.

    * ``state_bits=32``: state ``step`` (float32 device scalar), ``exp_avg``, ``exp_avg_sq`` (float32): the layout of
      ``torch.optim.AdamW``, whose ``state_dict`` loads.
    * ``state_bits=8``: 2.03 bytes per element instead of 8.  ``exp_avg`` and ``exp_avg_sq_root`` = sqrt(v) are
      ``torch.float8_e4m3fn`` tensors, each with a float32 scale per 256 elements (``..._scale``): value = element *
      scale.  A gradient that is not finite spoils its block of 256.
      The rounding is to nearest, and with ``betas[1]`` = 0.999 a step moves an element's sqrt(v) by less than half a step
      of the format: it does not fall when its gradients do, rises only while they are over 8 to 11 times as large (35 at
      the format's smallest values), and in between follows the largest of its block.  So the steps are AdamW's while
      the gradients of a block keep their proportions.  Where they do not, an element's step is too small or too large
      by the change, up to those factors upwards: with normal gradients, 4500 steps after half of the elements' gradients
      fell to a fifth, these had a sqrt(v) 3.6 times the true one in the median (5.0 for a tenth of them) and a tenth of
      the others 0.32 of it; without a change 0.72 to 1.46 (98 % of the elements), with ``betas[1]`` = 0.95 0.83 to 1.22
      before and after a change.  Take 32 bits, or ``betas[1]`` <= 0.95, where proportions within blocks change.
    * ``master_weights=True``: 16-bit parameters are updated through a float32 copy in the state (``master``); without
      it an update below half a unit of the parameter's last place is lost.  The copy is then the parameter: who sets
      parameters from outside sets it too (or clears the state).
    * ``max_grad_norm``: every step is preceded by the norm of all its gradients and clips by it; ``self.grad_norm``
      is the last norm (a device scalar, overwritten by the next step).  A step whose norm is not finite is dropped.

    A dropped step -- that, or a closed ``gate`` -- leaves parameters, moments and step counts as they were; the decision
    is taken on the device.  Nothing synchronises.  A step can be captured into a CUDA graph once the state exists (after
    a step, or ``init_state()``): the step counts advance with every replay, while learning rates and the other numbers
    are those of the capture, and gradients are read where they lay then; the optimiser, whose states and workspaces a
    replay uses, has to live as long as the graph.  Steps of one optimiser have to follow one another, on one stream or on
    streams that wait for each other.  What a step writes counts as modified in place."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 master_weights=False, max_grad_norm=None):
        _need(state_bits in (8, 32), "AdamW: state_bits is 8 or 32")
        _need(max_grad_norm is None or max_grad_norm > 0, "AdamW: max_grad_norm must be positive")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.master_weights, self.max_grad_norm = state_bits, bool(master_weights), max_grad_norm
        self._plan = self._work = self._norm = None

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(g):
        _need(all(_number(g[k]) >= 0 for k in ("lr", "eps", "weight_decay")) and
              all(0 <= _number(b) < 1 for b in g["betas"]), "AdamW: lr, eps, weight_decay >= 0 and 0 <= beta < 1")
        for p in g["params"]:
            _need(p.dtype in _TYPES and p.layout == torch.strided, "AdamW: dense float32, bfloat16 or float16 parameters")

    @staticmethod
    def _on_host(g):
        number = lambda v: float(v) if torch.is_tensor(v) and v.is_cuda else v  # noqa: E731
        return dict(g, **{k: type(g[k])(map(number, g[k])) if k == "betas" else number(g[k])
                          for k in ("lr", "betas", "eps", "weight_decay") if k in g})

    @property
    def grad_norm(self):
        """Norm of all gradients of the last step (``max_grad_norm``), before clipping; a device scalar."""
        return None if self._norm is None else self._norm[0][0]

    # ---- state --------------------------------------------------------------------------------------------------
    def _names(self, param):
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else \
            ("exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale")
        return ("step",) + names + (("master",) if self.master_weights and param.dtype != torch.float32 else ())

    def _fresh(self, p, name):
        if name == "step":
            return torch.zeros((), dtype=torch.float32, device=p.device)
        if name == "master":
            return p.detach().float().contiguous()
        if name.endswith("_scale"):
            return torch.zeros((p.numel() + _BLOCK - 1) // _BLOCK, dtype=torch.float32, device=p.device)
        return torch.zeros(p.shape, dtype=torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn, device=p.device)

    @torch.no_grad()
    def init_state(self):
        """Create the state of every parameter that has none yet (a step does that for those with a gradient)."""
        for group in self.param_groups:
            for p in group["params"]:
                _need(p.is_cuda, "AdamW: CUDA parameters on one device")
                self._state_of(p)
                self._workspaces(p.device)

    def _state_of(self, p):
        st = self.state[p]
        if len(st) == 0:
            _need(not (p.is_cuda and torch.cuda.is_current_stream_capturing()),
                  "AdamW: the state has to exist before a step is captured (take a step, or call init_state())")
            for name in self._names(p):
                st[name] = self._fresh(p, name)
        return st

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As ``torch.optim.Optimizer.load_state_dict``, with every state tensor kept in its own type (the base class
        casts them to the parameter's) and copied to the parameter's device.  A state in another number of bits, or
        without the master copy that this optimiser keeps, is refused, and so are groups of another rule (``amsgrad``,
        ``maximize``, a weight decay that is added to the gradient) and settings that the constructor refuses; numbers
        that lie on a device are read."""
        loaded, before = {}, {p: st for p, st in self.state.items() if st}
        # after the user's hooks, which may give another dictionary, and before those that want the loaded state
        hooks = (self.register_load_state_dict_pre_hook(lambda _, sd: self._take_states(sd, loaded, before)),
                 self.register_load_state_dict_post_hook(lambda _: self._put_states(loaded, before), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _take_states(self, state_dict, loaded, before):
        """Checks a state dictionary, moves its states into ``loaded`` and returns what is left for the base class."""
        for g in state_dict["param_groups"]:
            _need(not g.get("amsgrad") and not g.get("maximize") and
                  (g.get("decoupled_weight_decay", True) or not g.get("weight_decay")),
                  "AdamW: the loaded state is of amsgrad, maximize or a weight decay that is not decoupled")
        groups = [self._on_host(g) for g in state_dict["param_groups"]]
        for g in groups:
            self._check_group(dict(self.defaults, **dict(g, params=())))
        ids = [i for g in groups for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        _need(len(ids) == len(own), "AdamW: the loaded state has another number of parameters")
        for i, p in zip(ids, own):
            st = state_dict["state"].get(i)
            if not st:
                continue
            for name in self._names(p):
                _need(name in st, f"AdamW: the loaded state has no {name} (state_bits={self.state_bits}, "
                                  f"master_weights={self.master_weights})")
                fresh, value = self._fresh(p, name), torch.as_tensor(st[name])
                _need(value.numel() == fresh.numel() and (value.dtype == fresh.dtype or name == "step"),
                      f"AdamW: the loaded {name} has another size or type")
                loaded.setdefault(p, {})[name] = fresh.copy_(value.reshape(fresh.shape))
        for p in own:
            if p in before and p not in loaded:      # no state: as before the first step
                loaded[p] = {n: self._fresh(p, n) for n in self._names(p)}
        return dict(state_dict, state={}, param_groups=groups)

    def _put_states(self, loaded, before):
        for p, new in loaded.items():
            st = before.get(p)
            if st is not None and set(st) == set(new) and all(st[n].shape == t.shape and st[n].dtype == t.dtype and
                                                              st[n].device == t.device for n, t in new.items()):
                for n, t in new.items():   # into the tensors that are there: a captured step goes on using them
                    st[n].copy_(t)
                new = st
            self.state[p] = new

    def __getstate__(self):
        return dict(super().__getstate__(), state_bits=self.state_bits, master_weights=self.master_weights,
                    max_grad_norm=self.max_grad_norm)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan = None
        self.__dict__.setdefault("_work", None)
        self.__dict__.setdefault("_norm", None)

    # ---- the step -----------------------------------------------------------------------------------------------
    def step(self, gate=None, grad_scale=None):
        """``gate``: a one-element float32 device tensor; the step is applied where it is > 0.  ``grad_scale``: a
        one-element float32 device tensor that multiplies every gradient; the step is dropped where it is not positive
        and finite (not together with ``max_grad_norm``, which makes its own)."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_optimizer_pre_hooks or \
                _global_optimizer_post_hooks or torch.autograd._profiler_enabled():
            return _hooked_step(self, gate, grad_scale)
        self.step_gated(gate, grad_scale)

    step.hooked = True   # the base class would wrap it: 10 us per step for hooks that are looked for above

    def step_gated(self, gate=None, grad_scale=None):
        """The body of ``step``, without hooks."""
        if gate is not None or grad_scale is not None:
            for t in (gate, grad_scale):
                _need(t is None or (torch.is_tensor(t) and t.is_cuda and t.numel() == 1 and t.dtype == torch.float32),
                      "AdamW: gate and grad_scale are one-element float32 tensors on the parameters' device")
            _need(grad_scale is None or self.max_grad_norm is None, "AdamW: grad_scale together with max_grad_norm")
        plan = self._plan
        if plan is None or not plan.follow(self):
            plan = self._new_plan()
            if plan is None:
                return
        rc = self._run(plan, gate, grad_scale)
        if rc == _STALE:   # other parameters have gradients, or something lies elsewhere
            plan = self._new_plan()
            if plan is None:
                return
            rc = self._run(plan, gate, grad_scale)
        if rc == _STRIDED:
            kept = [p.grad for p in plan.params]
            for p, g in zip(plan.params, kept):
                p.grad = g.contiguous()
            try:
                rc = self._run(plan, gate, grad_scale)
            finally:
                for p, g in zip(plan.params, kept):
                    p.grad = g
        check(rc, "fsgs_adamw_multi")

    def _new_plan(self):
        self._plan = None
        if any(p.grad is not None for g in self.param_groups for p in g["params"]):
            self._plan = _Plan(self)
        return self._plan

    def _run(self, plan, gate, grad_scale):
        device, clip = plan.device, self.max_grad_norm
        if self._work is None or self._work[0] != device or (clip is not None and self._norm is None):
            self._workspaces(device)
        scale = where = 0
        if grad_scale is not None:
            _need(grad_scale.device == device, "AdamW: gate and grad_scale are on the parameters' device")
            scale = grad_scale.data_ptr()
        if gate is not None:
            _need(gate.device == device, "AdamW: gate and grad_scale are on the parameters' device")
            where = gate.data_ptr()
        return _lib.host().step(plan.handle, self.param_groups, self.state, clip, self._words, self._own, scale, where)

    def _workspaces(self, device):
        """Created once and never replaced on the same device: a captured step goes on using them."""
        _need(not torch.cuda.is_current_stream_capturing(),
              "AdamW: take a step, or call init_state(), before a step is captured")
        space = lambda n: torch.empty(int(n), dtype=torch.uint8, device=device)  # noqa: E731
        stream = torch.cuda.current_stream(device).cuda_stream
        if self._work is None or self._work[0] != device:
            self._work, self._norm = (device, space(lib().fsgs_adamw_workspace_bytes())), None
            self._own = ((self._work[1], stream),)
        if self.max_grad_norm is not None and self._norm is None:
            self._norm = (torch.zeros(2, device=device), space(lib().fsgs_grad_norm_workspace_bytes()))
            self._own += tuple((t, stream) for t in self._norm)
        work, norm = self._work[1], self._norm
        self._words = (norm[1].data_ptr(), norm[1].numel(), norm[0].data_ptr()) if norm is not None else (0, 0, 0)
        self._words += (work.data_ptr(), work.numel())


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW.step_gated)
