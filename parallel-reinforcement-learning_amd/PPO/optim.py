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

import torch
from torch import nn

import prl_native

_entry = prl_native.list_entry
_BLOCK = prl_native.LIST_BLOCK
# state keys of the two forms of the moments: (first, second, first's scales, second's scales)
_MOMENTS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_rms", "exp_avg_scale", "exp_rms_scale")}


def grad_norm(tensors) -> torch.Tensor:
    """The global 2-norm of a list of device tensors (float32, bfloat16, float16, mixed as they
    are), as a 0-dim float32 tensor: sqrt of the sum of all squares, summed in float64 in a fixed
    order.  What torch.nn.utils.clip_grad_norm_ returns for them."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError("grad_norm needs at least one tensor")
    device, table, keep = tensors[0].device, array("q"), []
    for i, t in enumerate(tensors):
        _check_tensor(t, device, f"tensor {i}")
        if not t.is_contiguous():
            t = t.contiguous()
            keep.append(t)
        table.extend(_entry(grad=t.data_ptr(), numel=t.numel(), dtype=prl_native.LIST_DTYPES[t.dtype]))
    return prl_native.list_norm(table, device)


def _check_tensor(t, device, name):
    if t.is_sparse or not t.is_cuda:
        raise ValueError(f"{name} must be a dense device tensor (got {t.layout} on {t.device})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others on {device}")
    if t.dtype not in prl_native.LIST_DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (decoupled weight decay; no amsgrad, no maximize) on device
    parameters, and clipping by the global norm in the same call: step(max_norm=2.0) does what
    nn.utils.clip_grad_norm_(params, 2.0) and step() do, except that p.grad is left unclipped;
    the norm is then in `total_norm` (a 0-dim float32 device tensor).

    state_bits=32: exp_avg and exp_avg_sq in float32 whatever the parameter's type (state_dict() is
    torch's AdamW's for float32 parameters).  state_bits=8: 2 bytes of state per value instead of 8:
    blocks of 256 consecutive values share a float32 scale A, the largest magnitude in the block, and
    hold exp_avg, and exp_rms = sqrt(exp_avg_sq), as float8_e4m3fn of value / A * 256 with
    stochastic rounding (bits hashed from the index and the step count: the same run gives the same
    bits).  A gradient that is not finite makes its whole block's moments NaN.

    master=True: a float32 copy (`master` in the state) behind every 16-bit parameter takes the
    step, the parameter receives its rounding.  Without it a 16-bit parameter is read, stepped in
    float32 and rounded back.

    lr may be a float32 device tensor: a captured step then reads it at every replay.  The step
    count of every parameter lives on the device, so a step can be captured into a HIP graph once
    every parameter has taken one step outside it (which lays out the state)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits: int = 32, master: bool = False):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                        state_bits=state_bits, master=master, capturable=True)
        self._checked = {}      # parameter -> the state tensors found right the last time
        self._last_rows = self._last_table = None
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
        # a value stepped by two entries of a list would race
        spans = sorted((str(p.device), p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                       for g in self.param_groups for p in g["params"] if p.numel())
        for a, b in zip(spans, spans[1:]):
            if a[0] == b[0] and b[1] < a[2]:
                raise ValueError("two parameters share memory (or one is listed twice)")

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
        """The state tensors of p, in the order of the entry's pointers."""
        bits, numel = group["state_bits"], p.numel()
        half_master = group["master"] and p.dtype != torch.float32
        names = _MOMENTS[bits] + ("step",) + (("master",) if half_master else ())
        found = []
        for k in names:
            t = st.get(k)
            if not torch.is_tensor(t):
                raise ValueError(f"the state of a parameter has no {k} (state_bits={bits}, master={group['master']})")
            want = torch.float8_e4m3fn if bits == 8 and k in ("exp_avg", "exp_rms") else torch.float32
            size = 1 if k == "step" else -(-numel // _BLOCK) if k.endswith("_scale") else numel
            if t.dtype != want or t.numel() != size or t.device != p.device or not t.is_contiguous():
                raise ValueError(f"{k} must be {size} contiguous {want} values on {p.device} "
                                 f"(got {t.numel()} {t.dtype} on {t.device})")
            found.append(t)
        self._checked[p] = (bits, numel, tuple(names), found)
        return self._checked[p]

    def load_state_dict(self, state_dict):
        """torch's, except that the state keeps its own types (torch casts every state tensor to the
        parameter's) and that this optimizer's state_bits / master stay."""
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
                    self.state[p][k] = v.detach().to(device=p.device, copy=True)
        self._checked.clear()
        self._last_rows = None

    def flat_state(self) -> bool:
        """Whether this optimizer's step is one AdamW step of float32 parameters with float32 moments
        and one set of hyper-parameters: what the update engine runs inside its kernels."""
        group = self.param_groups[0]
        return (len(self.param_groups) == 1 and group["state_bits"] == 32
                and not torch.is_tensor(group["lr"])
                and all(p.dtype == torch.float32 for p in group["params"]))

    def __setstate__(self, state):
        super().__setstate__(state)
        self._checked, self._last_rows, self._last_table = {}, None, None

    def __getstate__(self):
        return {**super().__getstate__(), "total_norm": self.total_norm}

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None, *, max_norm=None):
        """One step of every parameter that has a gradient; with max_norm (>= 0) the gradients of
        all groups are clipped together by their global norm first (p.grad stays as it is)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative (got {max_norm})")
        rows, groups, keep, device = [], bytearray(), [], None
        dtypes, state, checked = prl_native.LIST_DTYPES, self.state, self._checked
        for index, group in enumerate(self.param_groups):
            groups += self._group_words(group)
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if device is None:
                    device = p.device
                if p.device != device or g.dtype != p.dtype or not p.is_contiguous() or not p.is_cuda:
                    _check_tensor(p, device, "a parameter")
                    raise ValueError("a parameter must be contiguous and its gradient of its type")
                if not g.is_contiguous() or g.is_sparse:
                    _check_tensor(g, device, "a gradient")
                    g = g.contiguous()
                    keep.append(g)
                st = state[p]
                if not st:
                    self._init_state(p, group, st)
                known = checked.get(p)
                if (known is None or known[0] != group["state_bits"] or known[1] != p.numel()
                        or any(st.get(k) is not t for k, t in zip(known[2], known[3]))):
                    known = self._check_state(p, group, st)
                bits, numel, names, t = known
                rows.extend(_entry(p.data_ptr(), g.data_ptr(),
                                   t[-1].data_ptr() if names[-1] == "master" else 0,
                                   t[0].data_ptr(), t[1].data_ptr(),
                                   t[2].data_ptr() if bits == 8 else 0,
                                   t[3].data_ptr() if bits == 8 else 0,
                                   t[4 if bits == 8 else 2].data_ptr(), numel, dtypes[p.dtype], bits, index))
        if not rows:
            self.total_norm = None if max_norm is None else torch.zeros((), device=self.param_groups[0]["params"][0].device)
            return loss
        if rows != self._last_rows:     # the arguments' table; the tensors' values are never kept
            steps = rows[7::prl_native.LIST_ENTRY_WORDS]
            if len(set(steps)) < len(steps):
                raise ValueError("two parameters share a step count tensor: each needs its own")
            self._last_rows, self._last_table = rows, array("q", rows)
        self.total_norm = prl_native.list_adamw(self._last_table, array("q", bytes(groups)), device,
                                                None if max_norm is None else float(max_norm))
        return loss

    @staticmethod
    def _group_words(group):
        lr, (beta1, beta2), on_device = group["lr"], group["betas"], 0
        if torch.is_tensor(lr):
            if lr.is_cuda:
                if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != group["params"][0].device:
                    raise ValueError("a device lr must be one float32 value on the parameters' device")
                lr, on_device = 0.0, lr.data_ptr()
            else:
                lr = float(lr)
        return struct.pack("5dq", lr, beta1, beta2, group["eps"], group["weight_decay"], on_device)


def clip_and_step(optimizer, params, max_norm: float) -> None:
    """nn.utils.clip_grad_norm_(params, max_norm) + optimizer.step() (PPO.py:248-250); in one call
    for this module's AdamW."""
    if isinstance(optimizer, AdamW):
        optimizer.step(max_norm=max_norm)
    else:
        nn.utils.clip_grad_norm_(params, max_norm)
        optimizer.step()
