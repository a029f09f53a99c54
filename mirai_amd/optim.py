"""The optimiser step of adapter training: AdamW over every factor in a few launches.

``AdapterAdamW`` is a ``torch.optim.Optimizer`` over the LoRA factors of
``attach_expert_lora`` (or any bf16 / fp32 parameters on one GPU). One HIP kernel
(mx_adamw_step) takes up to 88 tensors per launch, in one pass over parameters,
gradients and moments. The moments of a parameter group lie in one flat buffer
(``flat_moments``), each parameter from a multiple of 128 positions on; the entries
of ``state`` are views of it. ``state_bits=8`` holds them in blocks of 128 elements
with one exponent (a byte per element and moment instead of four), rounded
stochastically, so that the small steps of a slow average are not lost: m with a
sign, 4 exponent and 3 fraction bits, v with 5 exponent and 3 fraction bits. The
noise is a function of (seed, step, group, position): a run is repeatable bit for
bit.
"""

from __future__ import annotations

import ctypes
from itertools import chain, islice
from operator import is_

import numpy as np
import torch

from . import _native as nat

STATE_BLOCK = 128
_NAMES = {32: ("exp_avg", "exp_avg_sq"),
          8: ("exp_avg_q", "exp_avg_sq_q", "exp_avg_e", "exp_avg_sq_e")}


def _blocks(n: int) -> int:
    return -(-n // STATE_BLOCK)


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill its storage span without gaps or overlaps."""
    if t.is_contiguous():
        return True
    span = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s != 1),
                               key=lambda v: v[1]):
        if stride != span:
            return False
        span *= size
    return True


def _check_lr(lr, capturable) -> None:
    if not isinstance(lr, torch.Tensor):
        if not float(lr) >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
    elif not capturable:
        raise ValueError("a tensor lr needs capturable=True.")
    elif lr.numel() != 1 or lr.dtype != torch.float32 or lr.device.type != "cuda":
        raise ValueError("a tensor lr must hold one fp32 value on the GPU.")


class _Group:
    """The flat moments of one parameter group and where each parameter lies."""

    def __init__(self, params, bits, capturable):
        devices = {p.device for p in params}
        if len(devices) > 1:
            raise ValueError("the parameters of one group must live on one device, got "
                             f"{sorted(map(str, devices))}.")
        self.device = devices.pop()
        nat.require_gpu(*params)
        self.at, total = [], 0
        for p in params:
            self.at.append(total)
            total += _blocks(p.numel()) * STATE_BLOCK
        self.total = total
        self.bits = bits
        self.numel = [p.numel() for p in params]
        # Rows of mx_adamw_tensor: addresses (filled per step), length, place, index.
        self.table = np.zeros((len(params), 5), dtype=np.int64)
        self.table[:, 2] = self.numel
        self.table[:, 3] = self.at
        self.table[:, 4] = range(len(params))

        def empty(n, dtype):
            return torch.empty((n,), dtype=dtype, device=self.device)

        if bits == 32:
            self.flats = (empty(total, torch.float32), empty(total, torch.float32))
        else:
            self.flats = (empty(total, torch.uint8), empty(total, torch.uint8),
                          empty(total // STATE_BLOCK, torch.uint8),
                          empty(total // STATE_BLOCK, torch.uint8))
        self.steps = empty(len(params), torch.int64) if capturable else None
        self.scalars = empty(32 * len(params), torch.uint8) if capturable else None
        self.clear()

    def clear(self):
        """No steps taken: moments of zero (codes 0 under the smallest exponent)."""
        # What the optimiser's state holds of each parameter; None: not begun.
        self.entries = [None] * len(self.at)
        for name, flat in zip(_NAMES[self.bits], self.flats):
            flat.fill_(1 if name.endswith("_e") else 0)
        if self.steps is not None:
            self.steps.zero_()

    def begin(self, i, p, entry):
        """Parameter i's state without a step taken."""
        views = self.views(i, p)
        if self.entries[i] is not None:  # its place holds the moments of an entry taken away
            for name, view in views.items():
                view.fill_(1 if name.endswith("_e") else 0)
            if self.steps is not None:
                self.steps[i] = 0
        entry.update(views)
        entry["step"] = 0 if self.steps is None else self.steps[i]
        self.entries[i] = entry

    def views(self, i, p):
        """The state entries of parameter i."""
        at, n = self.at[i], p.numel()
        out = {}
        for name, flat in zip(_NAMES[self.bits], self.flats):
            if name.endswith("_e"):
                out[name] = flat[at // STATE_BLOCK:at // STATE_BLOCK + _blocks(n)]
            else:  # in the parameter's storage order
                out[name] = flat.as_strided(p.shape, p.stride(), at)
        return out


class AdapterAdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay (the defaults of torch.optim.AdamW):
    m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr wd) - lr / (1 - b1^t) *
    m / (sqrt(v) / sqrt(1 - b2^t) + eps), in fp32 whatever the parameters' type.

    state_bits: 32 (fp32 moments) or 8. seed: of the 8-bit moments' rounding noise.
    capturable: the step counts (and, where ``lr`` is a CUDA tensor of one fp32
    value, the learning rate) live on the GPU, so that ``step()`` can be captured
    into a HIP graph and replayed; without it a captured step is refused. Parameters
    without a gradient are left alone, their step not counted. state_dict() /
    load_state_dict() hold the moments as stored.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits: int = 32, seed: int = 0, capturable: bool = False):
        _check_lr(lr, capturable)
        if not float(eps) >= 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i, beta in enumerate(betas):
            if not 0.0 <= float(beta) < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {beta}")
        if len(betas) != 2:
            raise ValueError("betas holds two values.")
        if not float(weight_decay) >= 0.0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32.")
        defaults = {"lr": lr, "betas": (float(betas[0]), float(betas[1])), "eps": float(eps),
                    "weight_decay": float(weight_decay), "state_bits": int(state_bits),
                    "seed": int(seed) & 0xFFFFFFFF, "capturable": bool(capturable)}
        self._groups: dict[int, _Group] = {}
        super().__init__(params, defaults)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._groups = {}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            if group["state_bits"] not in (8, 32):
                raise ValueError("state_bits must be 8 or 32.")
            _check_lr(group["lr"], group["capturable"])
            if len({id(p) for p in group["params"]}) != len(group["params"]):
                raise ValueError("a parameter appears twice in one group.")
            for p in group["params"]:
                if p.dtype not in (torch.bfloat16, torch.float32):
                    raise ValueError(f"parameters must be bf16 or fp32, got {p.dtype}.")
                if not _dense(p):
                    raise ValueError("parameters must fill their storage without gaps or overlaps.")
        except ValueError:
            self.param_groups.pop()
            raise

    # ----------------------------------------------------------------- state
    def _group(self, gi: int) -> _Group:
        """Group gi's flat moments, taking over what state holds for its parameters."""
        group = self.param_groups[gi]
        held = self._groups.get(gi)
        if held is not None and len(held.at) == len(group["params"]):
            return held
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the optimiser's state must exist before its step is captured: take "
                               "one step, or call flat_moments(), beforehand.")
        held = _Group(group["params"], group["state_bits"], group["capturable"])
        for i, p in enumerate(group["params"]):
            given = self.state.get(p)
            if given:
                self._adopt(held, i, p, given)
        self._groups[gi] = held
        return held

    def _adopt(self, held: _Group, i: int, p: torch.Tensor, given: dict) -> None:
        views = held.views(i, p)
        missing = [name for name in ("step", *views) if name not in given]
        if missing:
            raise ValueError(f"the state of parameter {i} lacks {', '.join(missing)}; moments of "
                             f"state_bits={held.bits} hold {', '.join(views)}.")
        for name, view in views.items():
            t = given[name]
            if tuple(t.shape) != tuple(view.shape) or (held.bits == 8 and t.dtype != torch.uint8):
                raise ValueError(f"{name} of parameter {i} must have shape {tuple(view.shape)} and "
                                 f"type {view.dtype}, got {tuple(t.shape)} {t.dtype}.")
            view.copy_(t)
        entry = dict(views)
        step = int(given["step"])
        if held.steps is not None:
            held.steps[i] = step
            entry["step"] = held.steps[i]
        else:
            entry["step"] = step
        self.state[p] = held.entries[i] = entry

    def load_state_dict(self, state_dict) -> None:
        """The moments are taken as stored (type and layout of this optimiser's)."""
        given = state_dict["state"]
        saved_groups = state_dict["param_groups"]
        if len(saved_groups) == len(self.param_groups):
            for saved, group in zip(saved_groups, self.param_groups):
                if saved.get("state_bits", group["state_bits"]) != group["state_bits"]:
                    raise ValueError(f"the saved moments have state_bits={saved['state_bits']}, this "
                                     f"optimiser {group['state_bits']}.")
                for what in ("amsgrad", "maximize"):
                    if saved.get(what):
                        raise ValueError(f"the saved state is of a run with {what}, which AdapterAdamW "
                                         "does not offer.")
        keep = [(g["capturable"], g["state_bits"], g["lr"]) for g in self.param_groups]
        groups = self._groups
        super().load_state_dict({"state": {}, "param_groups": saved_groups})
        self._groups = groups
        # The flat buffers and a learning rate on the GPU stay where they are: a captured
        # step goes on with them.
        for group, (capturable, bits, lr) in zip(self.param_groups, keep):
            group["capturable"], group["state_bits"] = capturable, bits
            group.setdefault("seed", self.defaults["seed"])
            if isinstance(lr, torch.Tensor):
                group["lr"] = lr.fill_(float(group["lr"]))
            elif isinstance(group["lr"], torch.Tensor):
                group["lr"] = float(group["lr"])
        for gi, (saved, group) in enumerate(zip(saved_groups, self.param_groups)):
            held = self._group(gi)
            own = {t.untyped_storage().data_ptr() for t in (*held.flats, held.steps) if t is not None}
            rows = []
            for i, (key, p) in enumerate(zip(saved["params"], group["params"])):
                entry = given.get(key)
                if entry:
                    rows.append((i, p, {
                        k: v.clone() if isinstance(v, torch.Tensor)
                        and v.untyped_storage().data_ptr() in own else v for k, v in entry.items()}))
            held.clear()
            for row in rows:
                self._adopt(held, *row)

    def flat_moments(self, group: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
        """fp32 (exp_avg, exp_avg_sq) of a parameter group as flat tensors, each
        parameter from the next multiple of 128 on, in its storage order, zeros
        between: the buffers themselves with 32-bit moments, their values with
        8-bit ones."""
        held = self._group(group)
        if held.bits == 32:
            return held.flats
        out = []
        with nat.on_device(held.device):
            for i, is_signed in ((0, 1), (1, 0)):
                t = torch.empty(held.total, dtype=torch.float32, device=held.device)
                nat.call("mx_adamw_moments", held.flats[i].data_ptr(), held.flats[i + 2].data_ptr(),
                         held.total, is_signed, t.data_ptr(), nat.stream(held.device))
                out.append(t)
        return out[0], out[1]

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi in range(len(self.param_groups)):
            self._step_group(gi)
        return loss

    def _step_group(self, gi: int) -> None:
        group = self.param_groups[gi]
        params = group["params"]
        grads = [p.grad for p in params]
        if all(g is None for g in grads):
            return
        held = self._group(gi)
        if held.total == 0:  # no parameter holds an element
            return
        _check_lr(group["lr"], group["capturable"])
        device, host_steps = held.device, held.steps is None
        if host_steps and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdapterAdamW.step() is captured into a graph only with capturable=True: "
                               "its step counts live on the host otherwise.")
        addresses = self._plain_case(gi, held, params, grads)
        if addresses is not None:
            entries, touched = held.entries, params
            step = int(entries[0]["step"]) + 1 if host_steps else 0
            held.table[:, 0], held.table[:, 1] = addresses
            calls = [(step, params[0].dtype, held.table)]
        else:
            calls, keep, entries, touched = self._any_case(held, params, grads)
        lr = group["lr"]
        lr_ptr = None
        if isinstance(lr, torch.Tensor):
            if lr.device != device:
                raise ValueError(f"lr lives on {lr.device}, the parameters on {device}.")
            lr_ptr, lr = lr.data_ptr(), 0.0
        flats = held.flats
        config = nat.MxAdamwConfig(
            lr=float(lr), beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"],
            weight_decay=group["weight_decay"], seed=group["seed"], group=gi, state_bits=held.bits,
            exp_avg=flats[0].data_ptr(), exp_avg_sq=flats[1].data_ptr(),
            exp_avg_e=flats[2].data_ptr() if held.bits == 8 else None,
            exp_avg_sq_e=flats[3].data_ptr() if held.bits == 8 else None,
            steps=nat.ptr(held.steps), scalars=nat.ptr(held.scalars), lr_ptr=lr_ptr)
        with nat.on_device(device):
            for step, dtype, table in calls:
                config.step, config.dtype = step, nat.dtype_code(dtype)
                nat.call("mx_adamw_step", table.ctypes.data, len(table), ctypes.byref(config),
                         nat.stream(device))
        # Counted once the step is queued: a refused one leaves the state as it was.
        if host_steps:
            for entry in entries:
                entry["step"] += 1
        # The kernel writes through raw pointers: what caches by version has to see it.
        torch.autograd.graph.increment_version(touched)
        del addresses, calls

    def _plain_case(self, gi, held, params, grads):
        """Addresses of the parameters and gradients where every parameter has a
        contiguous gradient of its own length, one type and one step count, and state
        is as the steps before left it; else None. Everything is looked at anew, in few
        calls per tensor: a step of 72 small tensors 51 us, of which 20 are fixed, and 111
        with _any_case for all."""
        numel, contiguous = torch.Tensor.numel, torch.Tensor.is_contiguous
        try:
            if not (list(map(numel, grads)) == held.numel == list(map(numel, params))
                    and all(map(contiguous, params)) and all(map(contiguous, grads))):
                return None
        except (TypeError, RuntimeError):  # no gradient, or a sparse one
            return None
        if (set(map(torch.Tensor.get_device, chain(params, grads))) != {held.device.index}
                or len(set(map(torch.Tensor.dtype.__get__, chain(params, grads)))) != 1):
            return None
        first = sum(len(g["params"]) for g in self.param_groups[:gi])
        last = first + len(params)
        if (len(self.state) < last or not all(map(is_, islice(self.state, first, last), params))
                or not all(map(is_, islice(self.state.values(), first, last), held.entries))):
            return None
        if held.steps is None and len({entry["step"] for entry in held.entries}) != 1:
            return None
        return list(map(torch.Tensor.data_ptr, params)), list(map(torch.Tensor.data_ptr, grads))

    def _any_case(self, held, params, grads):
        """(step, type, mx_adamw_tensor rows) per (step, type) among the tensors that
        have gradients, what must outlive the launches, and the entries and parameters
        stepped."""
        device, host_steps = held.device, held.steps is None
        found: dict = {}
        keep, entries, touched = [], [], []
        for i, (p, g) in enumerate(zip(params, grads)):
            if g is None:
                continue
            if p.device != device:
                raise ValueError(f"a parameter moved from {device} to {p.device} under its optimiser.")
            if g.layout is not torch.strided:
                raise ValueError("AdapterAdamW takes dense gradients.")
            if g.dtype is not p.dtype or g.device != device or g.shape != p.shape:
                raise ValueError(f"a gradient must have its parameter's shape, type and device, got "
                                 f"{tuple(g.shape)} {g.dtype} {g.device}.")
            if p.numel() != held.numel[i] or not _dense(p):
                raise ValueError("a parameter's storage changed under its optimiser.")
            if g.stride() != p.stride() and not (g.is_contiguous() and p.is_contiguous()):
                g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
                keep.append(g)
            entry = self.state[p]
            if entry is not held.entries[i]:  # the first step, or state was changed from outside
                if held.entries[i] is not None and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the state was replaced: take one step before capturing.")
                if entry:
                    self._adopt(held, i, p, entry)
                    entry = self.state[p]
                else:
                    held.begin(i, p, entry)
            step = int(entry["step"]) + 1 if host_steps else 0
            at = found.setdefault((step, p.dtype), ([], [], []))
            at[0].append(i)
            at[1].append(p.data_ptr())
            at[2].append(g.data_ptr())
            entries.append(entry)
            touched.append(p)
        calls = []
        for (step, dtype), (index, p_ptrs, g_ptrs) in found.items():
            table = held.table[index]
            table[:, 0], table[:, 1] = p_ptrs, g_ptrs
            calls.append((step, dtype, table))
        return calls, keep, entries, touched
