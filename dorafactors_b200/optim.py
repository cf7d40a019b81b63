"""AdamW over many tensors at once, native, with moments in 32 or in 8 bits.

An adapted model has hundreds of small trainable tensors (A, B and the magnitude
of each projection); ``AdamW`` updates all of a parameter group in one or two kernel
launches.  It computes what ``torch.optim.AdamW`` does, in fp32 whatever the
parameters' type.

``state_bits=8`` holds both moments as 8-bit floating-point codes with an fp32 scale for
each 256 elements (2.03 bytes a parameter in place of 8).  ``master_weights`` keeps
an fp32 copy of 16-bit parameters, on which the step is taken: updates smaller than
the parameter's own rounding then add up instead of vanishing.

The state of a group lies in flat buffers, in the parameters' order, each
parameter at a multiple of 256 elements; ``state[p]`` has views of them.
"""

from __future__ import annotations

import array
import math

import numpy as np
import torch
from torch.optim import optimizer as _base

from . import _native

BLOCK = 256  # elements that share a scale, and the granule of the flat buffers

_data_ptr, _contiguous = torch.Tensor.data_ptr, torch.Tensor.is_contiguous
_numel, _device = torch.Tensor.numel, torch.Tensor.get_device


class _Group:
    """The flat state of one parameter group, and its table for the native call."""

    def __init__(self, group: dict, state: dict, first: int):
        params = group["params"]
        self.params = params
        self.bits, self.has_master = group["state_bits"], group["master_weights"]
        p0 = params[0]
        self.dtype, self.device = p0.dtype, p0.device
        for p in params:
            if not p.is_cuda:
                raise RuntimeError(f"AdamW: parameters must be on a CUDA device (got {p.device})")
            if p.dtype is not self.dtype or p.device != self.device:
                raise ValueError("AdamW: a parameter group must have one dtype and one device; split it")
            if not p.is_contiguous():
                raise ValueError(f"AdamW: parameters must be contiguous (got strides {tuple(p.stride())})")
        _native.dtype_code(p0)
        self.has_master = self.has_master and self.dtype is not torch.float32
        sizes = [p.numel() for p in params]
        self.blocks = [-(-n // BLOCK) for n in sizes]
        starts = np.concatenate(([0], np.cumsum(self.blocks, dtype=np.int64)))
        nblocks = int(starts[-1])
        self.numel = nblocks * BLOCK
        dev = self.device

        def zeros(n, dtype):
            return torch.zeros(n, dtype=dtype, device=dev)

        if self.bits == 32:
            self.flat = {"exp_avg": zeros(self.numel, torch.float32), "exp_avg_sq": zeros(self.numel, torch.float32)}
        else:
            self.flat = {}
            for name in ("exp_avg", "exp_avg_sq"):
                self.flat[name + "_codes"] = zeros(self.numel, torch.uint8)
                self.flat[name + "_scale"] = zeros(nblocks, torch.float32)
        if self.has_master:
            self.flat["master"] = zeros(self.numel, torch.float32)

        self.table = np.zeros(len(params), dtype=_native.ADAMW_TENSOR)
        self.address = self.table.ctypes.data
        self.table["numel"] = sizes
        column = {"exp_avg_codes": "exp_avg", "exp_avg_sq_codes": "exp_avg_sq"}
        for name, buf in self.flat.items():
            per = 1 if name.endswith("_scale") else BLOCK
            self.table[column.get(name, name)] = buf.data_ptr() + starts[:-1] * (per * buf.element_size())
        self.index = np.arange(first, first + len(params), dtype=np.uint64)
        # What every step holds the tensors to, as lists that compare in one pass.
        self.sizes, self.dtypes = sizes, [self.dtype] * len(params)
        self.devices = [dev.index] * len(params)
        self.states = [state[p] for p in params]
        for i, p in enumerate(params):
            st = state[p]
            st["step"] = 0
            for name, buf in self.flat.items():
                if name.endswith("_scale"):
                    st[name] = buf[starts[i]: starts[i] + self.blocks[i]]
                else:
                    st[name] = buf[starts[i] * BLOCK: starts[i] * BLOCK + sizes[i]].view(p.shape)
            if self.has_master:
                st["master"].copy_(p.detach())


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay (``torch.optim.AdamW``'s arguments and formulas).

    ``state_bits`` (32 or 8) and ``master_weights`` may differ from group to group, like
    ``lr``, ``betas``, ``eps`` and ``weight_decay``; the parameters of a group are contiguous CUDA
    tensors of one dtype (fp32, fp16 or bf16).  ``seed`` feeds the rounding of 8-bit second
    moments, which is a function of (seed, step, parameter, element).

    A step cannot be captured in a CUDA graph: its bias corrections are host numbers.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, master_weights: bool = False, seed: int = 0):
        self.seed = int(seed)
        self._groups: list[_Group] = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=bool(master_weights)))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check(group)
            if not group["params"]:
                raise ValueError("AdamW: a parameter group is empty")
            first = sum(len(g.params) for g in self._groups)
            self._groups.append(_Group(group, self.state, first))
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> None:
        b1, b2 = group["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {group['betas']}")
        for name in ("lr", "eps", "weight_decay"):
            if not 0.0 <= float(group[name]) < math.inf:
                raise ValueError(f"AdamW: {name} must be finite and not negative, got {group[name]}")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {group['state_bits']}")

    def step(self, closure=None):
        # The base class wraps ``step`` for its hooks and a profiler range, which takes the host
        # longer than a step of few tensors does; without hooks there is nothing to wrap.
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks
                or getattr(_base, "_global_optimizer_pre_hooks", None)
                or getattr(_base, "_global_optimizer_post_hooks", None)):
            return _step_with_hooks(self, closure)
        return self._step_all(closure)

    step.hooked = True  # the base class wraps it otherwise

    def _step_all(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a step cannot be captured in a CUDA graph (its bias corrections are host numbers)")
        for group, g in zip(self.param_groups, self._groups):
            self._check(group)
            self._step(group, g)
        return loss

    def _step(self, group: dict, g: _Group) -> None:
        params = g.params
        grads = [p.grad for p in params]
        table, index, states = g.table, g.index, g.states
        sizes, dtypes, devices = g.sizes, g.dtypes, g.devices
        try:
            grad_ptrs = list(map(_data_ptr, grads))
        except TypeError:  # parameters without a gradient stay as they are
            at = [i for i, x in enumerate(grads) if x is not None]
            if not at:
                return
            table, index = table[at], index[at]
            params, grads, states, sizes, dtypes, devices = ([of[i] for i in at] for of in (
                params, grads, states, sizes, dtypes, devices))
            grad_ptrs = None
        if not all(map(_contiguous, grads)):
            if any(x.layout is not torch.strided for x in grads):
                raise ValueError("AdamW: gradients must be dense")
            grads, grad_ptrs = [x.contiguous() for x in grads], None
        if grad_ptrs is None:
            grad_ptrs = list(map(_data_ptr, grads))
        for of, what in ((params, "parameters"), (grads, "gradients")):
            if list(map(_device, of)) != devices:
                raise RuntimeError(f"AdamW: {what} must stay on {g.device}")
            if [x.dtype for x in of] != dtypes or list(map(_numel, of)) != sizes:
                raise ValueError(f"AdamW: {what} must keep their type ({g.dtype}) and size")
        if not all(map(_contiguous, params)):
            raise ValueError("AdamW: parameters must stay contiguous")
        table["param"] = array.array("Q", map(_data_ptr, params))
        table["grad"] = array.array("Q", grad_ptrs)
        steps = [st["step"] for st in states]
        if steps.count(steps[0]) == len(steps):
            self._launch(group, g, table, index, steps[0] + 1)
        else:  # parameters that have seen different numbers of steps have their own corrections
            of = np.array(steps)
            for t in sorted(set(steps)):
                self._launch(group, g, table[of == t], index[of == t], t + 1)
        for st, t in zip(states, steps):
            st["step"] = t + 1

    def _launch(self, group: dict, g: _Group, table, index, step: int) -> None:
        if g.bits == 8:
            key = (self.seed + step * 0x9E3779B1) & 0xFFFFFFFF
            table["key"] = (np.uint64(key) + index * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
        address = g.address if table is g.table else table.ctypes.data
        _native.adamw_step(address, len(table), g.dtype, g.bits, float(group["lr"]), group["betas"], group["eps"],
                           group["weight_decay"], step, g.device)

    def moments(self, group: int = 0):
        """``(exp_avg, exp_avg_sq)`` of a group as flat fp32 tensors, each parameter at a multiple
        of 256 elements.  With 32-bit state these are the state itself, else decoded copies."""
        g = self._groups[group]
        if g.bits == 32:
            return g.flat["exp_avg"], g.flat["exp_avg_sq"]
        m = torch.empty(g.numel, dtype=torch.float32, device=g.device)
        v = torch.empty(g.numel, dtype=torch.float32, device=g.device)
        f = g.flat
        if g.numel:
            _native.adamw_decode(f["exp_avg_codes"], f["exp_avg_scale"], f["exp_avg_sq_codes"], f["exp_avg_sq_scale"],
                                 m, v)
        return m, v

    def masters(self, group: int = 0):
        """The flat fp32 masters of a group (laid out as ``moments``), None where it has none."""
        return self._groups[group].flat.get("master")

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Load what ``state_dict`` gave, of an optimizer with the same groups and the same kind of state."""
        groups, saved = state_dict["param_groups"], state_dict["state"]
        if len(groups) != len(self.param_groups):
            raise ValueError("AdamW: the state dict has another number of parameter groups")
        plan = []
        for mine, theirs in zip(self.param_groups, groups):
            if len(mine["params"]) != len(theirs["params"]):
                raise ValueError("AdamW: the state dict has a parameter group of another size")
            for name in ("state_bits", "master_weights"):
                if name in theirs and theirs[name] != mine[name]:
                    raise ValueError(f"AdamW: the state dict has {name}={theirs[name]}, this optimizer {mine[name]}")
            self._check({**mine, **{k: v for k, v in theirs.items() if k != "params"}})
            for p, key in zip(mine["params"], theirs["params"]):
                if key not in saved:
                    continue
                for name, to in self.state[p].items():
                    value = saved[key].get(name)
                    if value is None:
                        raise ValueError(f"AdamW: the state dict lacks {name} of parameter {key}")
                    if name != "step" and value.shape != to.shape:
                        raise ValueError(f"AdamW: {name} of parameter {key} is {tuple(value.shape)}, not {tuple(to.shape)}")
                    if name.endswith("_codes") and value.dtype is not torch.uint8:
                        raise ValueError(f"AdamW: {name} of parameter {key} is {value.dtype}, not uint8")
                plan.append((self.state[p], saved[key]))
        for st, value in plan:  # nothing has changed until all of it is known to fit
            for name, to in st.items():
                if name == "step":
                    st["step"] = int(value["step"])
                else:
                    to.copy_(value[name])
        for mine, theirs in zip(self.param_groups, groups):
            mine.update({k: v for k, v in theirs.items() if k != "params"})

    def __setstate__(self, state: dict) -> None:
        raise NotImplementedError("AdamW: pickle its state_dict(), not the optimizer")


_step_with_hooks = torch.optim.Optimizer.profile_hook_step(AdamW._step_all)
