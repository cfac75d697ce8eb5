"""AdamW over the tensors where they lie, and the norm its clipping needs (csrc/prl_optim.hip).

The reference steps with torch's clip_grad_norm_ + AdamW (PPO/PPO.py:247-250).  The update engines
here do that inside their kernels, or on one flat float32 vector (prl_flat_adamw).  This module is
the same step for every other case: any list of parameters, float32 or 16-bit, with or without
float32 masters, moments in 32 or in 8 bits, in a few launches for the whole list.  It is a
torch.optim.Optimizer, so it goes where one goes:

    ppo.optimizer = AdamW(ppo.policy.parameters(), lr=1e-3, state_bits=8)

PPO.learn() and RND.update_pred() then step through it.
"""
from __future__ import annotations

import struct
from array import array
from importlib import import_module
from itertools import chain, repeat
from operator import attrgetter, is_

import torch
from torch import nn

import prl_native

_BLOCK, _WORDS, _DTYPES = prl_native.LIST_BLOCK, prl_native.LIST_ENTRY_WORDS, prl_native.LIST_DTYPES
# state keys of the two forms of the moments: (first, second, first's scales, second's scales)
_MOMENTS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_rms", "exp_avg_scale", "exp_rms_scale")}
# one attribute of every tensor of a list by map(): some 40 ns a tensor, a loop's body costs several times that
_ptr, _numel, _contiguous, _device = (torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous,
                                      torch.Tensor.get_device)
_dtype, _layout = attrgetter("dtype"), attrgetter("layout")
_GLOBAL_HOOKS = [getattr(import_module("torch.optim.optimizer"), f"_global_optimizer_{k}_hooks", (True,))
                 for k in ("pre", "post")]


def _dense(tensors, device, name):
    """The tensors, contiguous (those that are not: copies), after checking that they are dense
    device tensors of a known type on one device."""
    if (set(map(_layout, tensors)) != {torch.strided} or set(map(_device, tensors)) != {device} or device < 0
            or not _DTYPES.keys() >= set(map(_dtype, tensors))):
        for t in tensors:
            if t.layout is not torch.strided or not t.is_cuda:
                raise ValueError(f"{name} must be a dense device tensor (got {t.layout} on {t.device})")
            if t.dtype not in _DTYPES:
                raise ValueError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
        raise ValueError(f"{name}: all must be on one device (got {sorted({str(t.device) for t in tensors})})")
    return tensors if all(map(_contiguous, tensors)) else [t.detach().contiguous() for t in tensors]


def _refuse_shared(written):
    """Refuses (kind, tensor) pairs of which two share memory: a value written by two workgroups would
    be either's."""
    spans = sorted((str(t.device), t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), kind)
                   for kind, t in written if t.numel())
    for a, b in zip(spans, spans[1:]):
        if a[0] == b[0] and b[1] < a[2]:
            if a[3] == b[3] == "a parameter":
                raise ValueError("two parameters share memory (or one is listed twice)")
            raise ValueError(f"{a[3]} and {b[3]} are (in part) the same memory: each needs its own")


def grad_norm(tensors) -> torch.Tensor:
    """The global 2-norm of a list of device tensors (float32, bfloat16, float16, mixed as they
    are), as a 0-dim float32 tensor: sqrt of the sum of all squares, summed in float64 in a fixed
    order.  What torch.nn.utils.clip_grad_norm_ returns for them."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError("grad_norm needs at least one tensor")
    tensors = _dense(tensors, tensors[0].get_device(), "a tensor of the list")
    table = array("q", bytes(8 * _WORDS * len(tensors)))
    table[1::_WORDS] = array("q", map(_ptr, tensors))
    table[8::_WORDS] = array("q", map(_numel, tensors))
    table[9::_WORDS] = array("q", map(_DTYPES.__getitem__, map(_dtype, tensors)))
    return prl_native.list_norm(table, tensors[0].device)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (decoupled weight decay; no amsgrad, no maximize) on device
    parameters, and clipping by the global norm in the same call: step(max_norm=2.0) does what
    nn.utils.clip_grad_norm_(params, 2.0) and step() do, except that p.grad is left unclipped;
    the norm is then in `total_norm` (a 0-dim float32 device tensor).  `params` are all parameters of
    this optimizer that have a gradient: see clip_and_step for any others.

    state_bits=32: exp_avg and exp_avg_sq in float32 whatever the parameter's type (state_dict() is
    torch's AdamW's for float32 parameters).  state_bits=8: 2 bytes of state per value instead of 8:
    blocks of 256 consecutive values share a float32 scale A, the largest magnitude in the block, and
    hold exp_avg, and exp_rms = sqrt(exp_avg_sq), as float8_e4m3fn of value / A * 256 with
    stochastic rounding (bits hashed from the index and the step count: the same run gives the same
    bits; past 2^24 steps, where a float32 count of 32-bit moments stays, theirs goes on by the next
    float32).  A gradient that is not finite, or so large that its square is not, makes its whole
    block's moments NaN.

    master=True: a float32 copy (`master` in the state) behind every 16-bit parameter takes the
    step, the parameter receives its rounding.  It is made from the parameter at its first step;
    weights that are loaded into the parameter later have to be copied into it too, or the next step
    brings the old ones back.  Without masters a 16-bit parameter is read, stepped in float32 and
    rounded back.

    Parameters, state tensors and masters share no memory with each other (a step refuses it) or
    with gradients; parameters may share a gradient.  A step raises the parameters' autograd versions
    as any in-place operation does (a graph's replay does not, as with torch's optimizers).

    lr may be a float32 device tensor: a captured step then reads it at every replay.  The step
    count of every parameter lives on the device, so a step can be captured into a HIP graph once
    every parameter has taken one step outside it (which lays out the state).  A graph goes on with the
    tensors it was captured with: load_state_dict() installs new ones, so capture again after it."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits: int = 32, master: bool = False):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                        state_bits=state_bits, master=master, capturable=True)
        self._plan = None       # the last step's list, laid out (_Plan)
        self.total_norm = None
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, group):
        beta1, beta2 = group["betas"]
        if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
            raise ValueError(f"betas must be in [0, 1) (got {group['betas']})")
        if not (torch.is_tensor(group["lr"]) or group["lr"] >= 0.0):
            raise ValueError(f"lr must not be negative (got {group['lr']})")
        if not (group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
            raise ValueError("eps and weight_decay must not be negative")
        if group["state_bits"] not in _MOMENTS:
            raise ValueError(f"state_bits must be 32 or 8 (got {group['state_bits']})")
        for p in group["params"]:
            if p.dtype not in prl_native.LIST_DTYPES:
                raise ValueError(f"parameters must be float32, bfloat16 or float16 (got {p.dtype})")
            if p.is_sparse or not p.is_contiguous():
                raise ValueError("parameters must be dense and contiguous")
        _refuse_shared(("a parameter", p) for g in self.param_groups for p in g["params"])

    # ------------------------------------------------------------------ state
    def _init_state(self, p, group, st):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter without state in a captured step: take one step outside it first")
        st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        if group["state_bits"] == 32:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            scales = -(-p.numel() // _BLOCK)
            for k in ("exp_avg", "exp_rms"):
                st[k] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
                st[k + "_scale"] = torch.zeros(scales, dtype=torch.float32, device=p.device)
        if group["master"] and p.dtype != torch.float32:
            st["master"] = p.detach().float()

    def _check_state(self, p, group, st):
        """p's state tensors by the entry's columns (2 .. 7); None: a null pointer."""
        bits, numel = group["state_bits"], p.numel()
        half_master = group["master"] and p.dtype != torch.float32
        columns = [None] * 6
        for k, column in zip(_MOMENTS[bits] + ("step",) + (("master",) if half_master else ()),
                             ((1, 2) if bits == 32 else (1, 2, 3, 4)) + (5, 0)):
            t = st.get(k)
            if not torch.is_tensor(t):
                raise ValueError(f"the state of a parameter has no {k} (state_bits={bits}, master={group['master']})")
            want = torch.float8_e4m3fn if bits == 8 and k in ("exp_avg", "exp_rms") else torch.float32
            size = 1 if k == "step" else -(-numel // _BLOCK) if k.endswith("_scale") else numel
            if t.dtype != want or t.numel() != size or t.device != p.device or not t.is_contiguous():
                raise ValueError(f"{k} must be {size} contiguous {want} values on {p.device} "
                                 f"(got {t.numel()} {t.dtype} on {t.device})")
            columns[column] = t
        return columns

    def load_state_dict(self, state_dict):
        """torch's, except that the state keeps its own types (torch casts every state tensor to the
        parameter's), and that this optimizer's state_bits / master stay: state of the other form
        is refused by the next step."""
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise ValueError("the state is of an AdamW with amsgrad or maximize")
        own = [(g["state_bits"], g["master"]) for g in self.param_groups]
        super().load_state_dict(state_dict)
        for g, (bits, master) in zip(self.param_groups, own):
            g.update(state_bits=bits, master=master, capturable=True)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for k, v in state_dict["state"].get(i, {}).items():
                if k == "step":
                    v = torch.as_tensor(v, dtype=torch.float32).reshape(())
                if torch.is_tensor(v):
                    want = v.dtype if v.dtype == torch.float8_e4m3fn else torch.float32
                    self.state[p][k] = v.detach().to(device=p.device, dtype=want, copy=True)
        self._plan = None

    def flat_state(self, params) -> bool:
        """Whether this optimizer's step is one AdamW step of exactly these parameters in float32, with
        float32 moments (those in the state too, if there are any) and one set of hyper-parameters:
        what the update engine runs inside its kernels."""
        group, params = self.param_groups[0], list(params)
        if not (len(self.param_groups) == 1 and group["state_bits"] == 32
                and not torch.is_tensor(group["lr"]) and len(params) == len(group["params"])
                and all(map(is_, params, group["params"]))
                and all(p.dtype == torch.float32 for p in params)):
            return False
        try:
            for p in params:
                if self.state.get(p):
                    self._check_state(p, group, self.state[p])
        except ValueError:       # the per-step path's first step refuses it by name
            return False
        return True

    def steps_exactly(self, params) -> bool:
        """Whether the parameters with gradients are the same here and in params: step(max_norm=..) then
        clips by the norm of params' gradients."""
        own = [p for group in self.param_groups for p in group["params"]]
        if len(own) == len(params) and all(map(is_, own, params)):
            return True
        return {id(p) for p in own if p.grad is not None} == {id(p) for p in params if p.grad is not None}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan, self.total_norm = None, None

    # ------------------------------------------------------------------ step
    def step(self, closure=None, *, max_norm=None):
        """One step of every parameter that has a gradient; with max_norm (>= 0) the gradients of
        all groups are clipped together by their global norm first (p.grad stays as it is)."""
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or any(_GLOBAL_HOOKS)
                or torch.autograd._profiler_enabled()):
            return self._traced_step(closure, max_norm=max_norm)
        return self._step(closure, max_norm)

    # torch wraps an optimizer's step() to run its hooks and mark it for the profiler, some 5 us; this
    # one goes through that wrapper when there is a hook to run or a profiler to see the mark
    step.hooked = True

    @torch.optim.Optimizer.profile_hook_step
    def _traced_step(self, closure=None, *, max_norm=None):
        return self._step(closure, max_norm)

    def _step(self, closure, max_norm):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative (got {max_norm})")
        groups = self.param_groups
        params = [p for group in groups for p in group["params"]]
        grads = [p.grad for p in params]
        plan, filled = self._plan, None
        if plan is not None and plan.holds(groups, params, grads, self.state):
            filled = plan.fill(grads)
        if filled is None:
            self._plan = None     # (dropped first: laying out may refuse)
            plan = _Plan(self, groups, params, grads)
            if not plan.params:
                self.total_norm = None if max_norm is None else torch.zeros(
                    (), dtype=torch.float32, device=params[0].device if params else None)
                return loss
            filled, self._plan = plan.fill(grads), plan
        words = b"".join(map(self._group_words, groups))
        table, keep = filled
        self.total_norm = prl_native.list_adamw(table, array("q", words), plan.device,
                                                None if max_norm is None else float(max_norm), plan.workspace)
        # the kernels write through addresses: autograd is told, so that backward() on a graph from before
        # this step is refused (some 60 ns a parameter)
        torch.autograd.graph.increment_version(plan.params)
        return loss

    @staticmethod
    def _group_words(group):
        lr, (beta1, beta2), on_device = group["lr"], group["betas"], 0
        if torch.is_tensor(lr):
            if lr.is_cuda:
                if lr.dtype != torch.float32 or lr.numel() != 1 or any(p.device != lr.device for p in group["params"][:1]):
                    raise ValueError("a device lr must be one float32 value on the parameters' device")
                lr, on_device = 0.0, lr.data_ptr()
            else:
                lr = float(lr)
        return struct.pack("5dq", lr, beta1, beta2, group["eps"], group["weight_decay"], on_device)


class _Plan:
    """A step's list as prl_list_entry words, and what to compare before it serves the next step:
    which parameters step, with which state tensors, and where those lie.  Gradients are looked up
    anew by every step; a list of which anything else differs is laid out, and checked, again."""

    def __init__(self, opt, groups, params, grads):
        self.every, self.without = params, list(map(is_, grads, repeat(None)))
        self.settings = self._settings(groups)
        index = [(i, g) for i, g in enumerate(groups) for _ in g["params"]]
        chosen = [(p, g, *ig) for p, g, ig in zip(params, grads, index) if g is not None]
        self.params = [c[0] for c in chosen]
        if not chosen:
            return
        self.device = self.params[0].device
        _dense(self.params, self.params[0].get_device(), "a parameter")
        columns = []
        for p, g, _, group in chosen:
            if not p.is_contiguous():
                raise ValueError("a parameter must be contiguous")
            if g.dtype != p.dtype or g.numel() != p.numel():
                raise ValueError(f"a gradient must be of its parameter's type and size (got {g.numel()} {g.dtype} "
                                 f"for {p.numel()} {p.dtype})")
            st = opt.state[p]
            if not st:
                opt._init_state(p, group, st)
            columns.append(opt._check_state(p, group, st))
        _refuse_shared(("a parameter" if k == 0 else "a state tensor", t)
                       for p, c in zip(self.params, columns) for k, t in enumerate([p, *c]) if t is not None)
        self.values = list(chain.from_iterable(map(dict.values, opt.state.values())))
        self.dtypes, self.numels = list(map(_dtype, self.params)), list(map(_numel, self.params))
        self.tensors = self.params + [t for c in columns for t in c if t is not None]
        self.at, self.grads_at = list(map(_ptr, self.tensors)), None
        self.table = array("q", bytes(8 * _WORDS * len(chosen)))
        for k, (p, c) in enumerate(zip(self.params, columns)):
            self.table[k * _WORDS] = p.data_ptr()
            for column, t in enumerate(c):
                self.table[k * _WORDS + 2 + column] = 0 if t is None else t.data_ptr()
        self.table[8::_WORDS] = array("q", self.numels)
        self.table[9::_WORDS] = array("q", [_DTYPES[p.dtype] | group["state_bits"] << 32 for p, _, _, group in chosen])
        self.table[10::_WORDS] = array("q", [i for _, _, i, _ in chosen])
        self.workspace = prl_native.list_workspace_bytes(self.table, len(groups))

    @staticmethod
    def _settings(groups):
        return [(g["state_bits"], g["master"], len(g["params"])) for g in groups]

    def holds(self, groups, params, grads, state):
        """Whether this step takes the same parameters with the same state tensors in the same places."""
        if (len(params) != len(self.every) or not all(map(is_, params, self.every))
                or list(map(is_, grads, repeat(None))) != self.without or self._settings(groups) != self.settings):
            return False
        values = list(chain.from_iterable(map(dict.values, state.values())))
        return (len(values) == len(self.values) and all(map(is_, values, self.values))
                and list(map(_numel, self.params)) == self.numels and all(map(_contiguous, self.params))
                and list(map(_ptr, self.tensors)) == self.at)     # (the types: by the gradients, in fill())

    def fill(self, grads):
        """The table with the gradients' addresses, and the tensors that these are of; None if their types
        or sizes are not the parameters' (any more: the list is to be laid out, and checked, again)."""
        if len(grads) != len(self.params):
            grads = [g for g in grads if g is not None]
        if list(map(_dtype, grads)) != self.dtypes or list(map(_numel, grads)) != self.numels:
            return None
        try:
            contiguous = all(map(_contiguous, grads))
        except RuntimeError:      # a sparse one: _dense says so
            contiguous = False
        if not contiguous:
            grads = _dense(grads, self.device.index, "a gradient")
        at = list(map(_ptr, grads))
        if at != self.grads_at:
            _dense(grads, self.device.index, "a gradient")
            self.grads_at, self.table[1::_WORDS] = at, array("q", at)
        return self.table, grads


def clip_and_step(optimizer, params, max_norm: float) -> None:
    """nn.utils.clip_grad_norm_(params, max_norm) + optimizer.step() (PPO.py:248-250); in one call (the
    gradients stay unclipped) for this module's AdamW if it steps exactly the gradients of params."""
    params = [params] if isinstance(params, torch.Tensor) else list(params)
    if isinstance(optimizer, AdamW) and optimizer.steps_exactly(params):
        optimizer.step(max_norm=max_norm)
    else:
        nn.utils.clip_grad_norm_(params, max_norm)
        optimizer.step()
