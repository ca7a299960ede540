"""AdamW over many tensors at once, with moments in 32 or in 8 bits and, for bf16 parameters, optional fp32 masters.

The reference trains with `mlx.optimizers.AdamW`, and its planner books two fp32 moments a parameter
(plan/estimate.py:57-135).  Here a step is one launch over all tensors of a dtype (csrc/optim.cu):

    m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

`adamw_step` is that step on lists of tensors, in place or into other buffers; `AdamW` is the `torch.optim.Optimizer` a trainer
holds.  8-bit moments take 2 bytes a parameter and 8 for every 256: e4m3 codes of m and of sqrt(v) times a scale for each
block of 256 elements; sqrt(v), and m wherever rounding to nearest could hold a value that no gradient feeds (small codes; with
beta1 above 0.9 all of them), is rounded up or down by a dither fixed by position and step, so every rank of a data-parallel run gets
the same codes.  They hold m up to 1e-30 and sqrt(v) up to 4e-19 as zero, and an element with a moment that is not finite gets NaN for
both and for its parameter.  Moments, scales and codes are bit for bit those of fp32 operations rounded one by one, in the order written
here.  beta1 above 0.9 takes a third more time.
"""
from __future__ import annotations

import ctypes as C
from operator import attrgetter
from typing import Any, Sequence

import numpy as np
import torch
from torch.autograd.graph import increment_version

from mlx_train_perf_b200 import _lib
from mlx_train_perf_b200.errors import OptimizerInputError

BLOCK = 256
_DTYPES = (torch.float32, torch.bfloat16)


def _padded(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK * BLOCK


class AdamWState:
    """Moments (and masters) of a list of tensors, flat: each buffer holds the tensors' elements one behind the other, every
    tensor starting at a multiple of 256 with zeros behind it (`view` gives tensor i's share).  `exp_avg`, `exp_avg_sq`: fp32, or float8_e4m3fn
    codes with `scales` (blocks, 2) fp32; `master`: fp32 or None; `steps`: steps taken, one count for each tensor."""

    __slots__ = ("numels", "exp_avg", "exp_avg_sq", "scales", "master", "steps", "rows")

    def __init__(self, numels: Sequence[int], exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, *,
                 scales: torch.Tensor | None = None, master: torch.Tensor | None = None, steps: Sequence[int] | None = None):
        self.numels = tuple(numels)
        # rows of the library's table: parameter, gradient, output, elements, place in the states
        self.rows = rows = np.zeros((len(self.numels), 5), dtype=np.int64)
        rows[:, 3] = self.numels
        ends = (rows[:, 3] + (BLOCK - 1) & -BLOCK).cumsum()
        rows[1:, 4] = ends[:-1]
        total = int(ends[-1]) if self.numels else 0
        self.exp_avg, self.exp_avg_sq, self.scales, self.master = exp_avg, exp_avg_sq, scales, master
        self.steps = [0] * len(self.numels) if steps is None else list(steps)
        if len(self.steps) != len(self.numels):
            raise OptimizerInputError(f"{len(self.steps)} step counts for {len(self.numels)} tensors")
        moments = torch.float32 if scales is None else torch.float8_e4m3fn
        for name, t, dtype, size in (("exp_avg", exp_avg, moments, total), ("exp_avg_sq", exp_avg_sq, moments, total),
                                     ("scales", scales, torch.float32, 2 * (total // BLOCK)), ("master", master, torch.float32, total)):
            if t is None:
                continue
            if t.dtype != dtype or t.numel() != size or not t.is_contiguous() or not t.is_cuda or t.device != exp_avg.device:
                raise OptimizerInputError(f"{name} must be a contiguous {dtype} CUDA tensor of {size} elements beside exp_avg; got "
                                          f"{t.dtype}, {t.numel()} on {t.device}")

    @classmethod
    def zeros(cls, params: Sequence[torch.Tensor], *, bits: int = 32, master: bool = False) -> "AdamWState":
        """States of step 0 for `params`; `master` copies them in fp32."""
        params = list(params)
        if bits not in (8, 32):
            raise OptimizerInputError(f"moments are kept in 8 or 32 bits, got {bits}")
        if not params:
            raise OptimizerInputError("no parameters")
        dev = params[0].device
        if not params[0].is_cuda:
            raise OptimizerInputError(f"parameters must be CUDA tensors (the operator has no CPU path); got {dev}")
        numels = [p.numel() for p in params]
        total = sum(_padded(n) for n in numels)
        dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
        state = cls(numels, torch.zeros(total, dtype=dtype, device=dev), torch.zeros(total, dtype=dtype, device=dev),
                    scales=torch.zeros(total // BLOCK, 2, dtype=torch.float32, device=dev) if bits == 8 else None,
                    master=torch.zeros(total, dtype=torch.float32, device=dev) if master else None)
        if master:
            for i, p in enumerate(params):
                state.view("master", i).copy_(p.detach().reshape(-1))
        return state

    @property
    def bits(self) -> int:
        return 32 if self.scales is None else 8

    def view(self, name: str, i: int) -> torch.Tensor:
        """Tensor i's share of a buffer: (numel,), or its blocks' scales (blocks, 2)."""
        flat, o, n = getattr(self, name), int(self.rows[i, 4]), self.numels[i]
        return flat[o // BLOCK:(o + _padded(n)) // BLOCK] if name == "scales" else flat[o:o + n]

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Tensor i's m and v as fp32 values, (numel,) each."""
        if self.scales is None:
            return self.view("exp_avg", i), self.view("exp_avg_sq", i)
        o, n = int(self.rows[i, 4]), self.numels[i]
        scales = self.view("scales", i)
        m, r = ((t[o:o + _padded(n)].float().reshape(-1, BLOCK) * scales[:, k:k + 1]).reshape(-1)[:n]
                for k, t in enumerate((self.exp_avg, self.exp_avg_sq)))
        return m, r.square()


_T = torch.Tensor
_dtype_of = attrgetter("dtype")


_PLAIN = {torch.Tensor, torch.nn.Parameter}


def _fast_rows(rows: np.ndarray, column: int, tensors: Sequence[torch.Tensor], dtype: torch.dtype, device: torch.device) -> bool:
    """Checks the tensors and puts their addresses into the table's column, all in one call; False: not done, ask one by one."""
    fn = _lib.tensor_rows()
    if fn is None or not _PLAIN.issuperset(map(type, tensors)):
        return False
    objects = np.fromiter(map(id, tensors), np.int64, len(tensors))
    try:
        return fn(objects.ctypes.data, len(tensors), dtype is torch.bfloat16, device.index, rows.ctypes.data, column) == -1
    except Exception:                                    # a tensor without memory (sparse, fake): the checks below name it
        return False


def _rows_of(name: str, rows: np.ndarray, column: int, tensors: Sequence[torch.Tensor], dtype: torch.dtype, device: torch.device) -> None:
    """The tensors' addresses into the table's column, each tensor looked at before: `_fast_rows`, or a property of all of them at a
    time (128 tensors: 30 us)."""
    if _fast_rows(rows, column, tensors, dtype, device):
        return
    numels = rows[:, 3].tolist()
    if (set(map(_dtype_of, tensors)) != {dtype} or set(map(_T.get_device, tensors)) != {device.index}
            or not all(map(_T.is_contiguous, tensors)) or list(map(_T.numel, tensors)) != numels):
        t, n = next((t, n) for t, n in zip(tensors, numels)
                    if t.dtype != dtype or t.device != device or not t.is_contiguous() or t.numel() != n)
        raise OptimizerInputError(f"{name} must be contiguous {dtype} tensors on {device} with the elements their states were made "
                                  f"for; got {tuple(t.shape)} {t.dtype} on {t.device} for {n} elements")
    rows[:, column] = list(map(_T.data_ptr, tensors))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor | None], state: AdamWState, *, lr: float,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               grad_scale: float | torch.Tensor = 1.0, step: int | None = None,
               out: tuple[Sequence[torch.Tensor], AdamWState] | None = None) -> None:
    """One AdamW step on `params` (contiguous, one dtype) from `grads` (one dtype; strided ones are copied).

    A tensor whose gradient is None keeps its value, its moments and its step count.  Gradients are multiplied by `grad_scale`, a
    number or a one-element fp32 device tensor (a clipping coefficient, say).  `step`: the step's number for all tensors (bias
    correction and dither); default: each tensor's count in `state.steps`, plus one.  `out=(tensors, state)` takes the
    results in place of `params` and `state`, which are then only read; it must not overlap them.  With masters, `params` are only written.
    Not differentiable; launch arguments carry lr and step, so a captured step repeats that very step when it is replayed."""
    out_params, out_state = (params, state) if out is None else out
    if not len(params) == len(grads) == len(out_params) == len(state.numels) == len(out_state.numels):
        raise OptimizerInputError(f"{len(params)} parameters, {len(grads)} gradients and states of {len(state.numels)} tensors")
    if not params:
        return
    if out is not None and (state.numels != out_state.numels or state.bits != out_state.bits
                            or (state.master is None) != (out_state.master is None)
                            or state.exp_avg.device != out_state.exp_avg.device):
        raise OptimizerInputError("out's state must have the layout of `state`")
    dev, dtype = state.exp_avg.device, params[0].dtype
    if dtype not in _DTYPES:
        raise OptimizerInputError(f"parameters must be fp32 or bf16, got {dtype}")
    if state.master is not None and dtype != torch.bfloat16:
        raise OptimizerInputError("masters belong to bf16 parameters")
    rows = state.rows.copy()
    _rows_of("params", rows, 0, params, dtype, dev)
    if out is None:
        rows[:, 2] = rows[:, 0]
    else:
        _rows_of("out", rows, 2, out_params, dtype, dev)
    which = range(len(params))
    g_dtype = None if grads[0] is None else grads[0].dtype
    if g_dtype not in _DTYPES or not _fast_rows(rows, 1, grads, g_dtype, dev):
        which = [i for i, g in enumerate(grads) if g is not None]
        if len(which) < len(grads) and out is not None:
            raise OptimizerInputError("with out, every tensor needs a gradient")
        if not which:
            return
        rows = rows[which]
        if any(grads[i].layout is not torch.strided for i in which):
            raise OptimizerInputError("gradients must be dense")
        grads = [grads[i].contiguous() for i in which]
        g_dtype = grads[0].dtype
        if g_dtype not in _DTYPES:
            raise OptimizerInputError(f"gradients must be fp32 or bf16, got {g_dtype}")
        _rows_of("grads", rows, 1, grads, g_dtype, dev)
    scale_ptr = None
    if isinstance(grad_scale, torch.Tensor):
        if grad_scale.numel() != 1 or grad_scale.dtype != torch.float32 or grad_scale.device != dev:
            raise OptimizerInputError("grad_scale must be a number or one fp32 element on the parameters' device")
        scale_ptr, grad_scale = grad_scale.data_ptr(), 1.0
    steps = [state.steps[i] + 1 for i in which] if step is None else None
    a = _lib.AdamwArgs(
        state.exp_avg.data_ptr(), state.exp_avg_sq.data_ptr(), None if state.scales is None else state.scales.data_ptr(),
        None if state.master is None else state.master.data_ptr(), out_state.exp_avg.data_ptr(), out_state.exp_avg_sq.data_ptr(),
        None if state.scales is None else out_state.scales.data_ptr(), None if state.master is None else out_state.master.data_ptr(),
        float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay), float(grad_scale), scale_ptr, 0,
        dtype == torch.bfloat16, g_dtype == torch.bfloat16, state.bits, 0)
    lib = _lib.load()
    with _lib.on(dev):
        stream = _lib.stream(dev)
        numbers = {int(step)} if steps is None else set(steps)
        if len(numbers) > 1:                             # tensors that took different numbers of steps: a launch for each number ...
            a.step, a.check_only = 1, 1                  # ... but only if all tensors together pass
            _lib.check(lib.b200tp_adamw_step(C.byref(a), rows.ctypes.data, len(rows), stream))
            a.check_only = 0
        for number in sorted(numbers):
            part = rows if len(numbers) == 1 else np.ascontiguousarray(rows[[s == number for s in steps]])
            a.step = number
            _lib.check(lib.b200tp_adamw_step(C.byref(a), part.ctypes.data, len(part), stream))
    if out is not None or step is not None and len(which) == len(params):
        out_state.steps = steps if steps is not None else [int(step)] * len(which)
    else:
        for k, i in enumerate(which):
            out_state.steps[i] = int(step) if steps is None else steps[k]
    increment_version(out_params if len(which) == len(params) else [out_params[i] for i in which])    # autograd is told that saved copies are stale


class _Bucket:
    """The parameters of one group that share a dtype and a device, and their states."""

    def __init__(self, params: list[torch.Tensor], bits: int, master: bool):
        self.params = params
        self.state = AdamWState.zeros(params, bits=bits, master=master and params[0].dtype == torch.bfloat16)

    def names(self) -> list[str]:
        s = self.state
        return ["exp_avg", "exp_avg_sq"] + (["scales"] if s.scales is not None else []) + (["master"] if s.master is not None else [])


class AdamW(torch.optim.Optimizer):
    """AdamW as a `torch.optim.Optimizer` (parameter groups, schedulers, `state_dict`): one launch for each group and dtype.

    `bits`: 32 or 8, the moments'; `master=True` keeps fp32 masters of bf16 parameters, taken from them at the first step
    (weights loaded into the model later are overwritten by the next step unless the optimizer's state is loaded too)."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, bits: int = 32, master: bool = False):
        if bits not in (8, 32):
            raise OptimizerInputError(f"moments are kept in 8 or 32 bits, got {bits}")
        self._bits, self._master, self._buckets = bits, bool(master), {}
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay})

    def _of_group(self, k: int) -> list[_Bucket]:
        """The group's buckets, laid out at the first call with what `self.state` holds; kept only once all of it fits."""
        if k not in self._buckets:
            kinds: dict[Any, list[torch.Tensor]] = {}
            for p in self.param_groups[k]["params"]:
                kinds.setdefault((p.dtype, p.device), []).append(p)
            buckets, states = [_Bucket(ps, self._bits, self._master) for ps in kinds.values()], {}
            for b in buckets:
                for i, p in enumerate(b.params):
                    saved = self.state.get(p)
                    if saved:
                        self._check_saved(p, saved)
                        for name in b.names():
                            b.state.view(name, i).copy_(saved[name])
                        b.state.steps[i] = int(saved["step"])
                    states[p] = {"step": b.state.steps[i], **{name: b.state.view(name, i) for name in b.names()}}
            self.state.update(states)
            self._buckets[k] = buckets
        return self._buckets[k]

    def _check_saved(self, p: torch.Tensor, saved: dict) -> None:
        """Whether a saved state is one that this optimizer keeps for `p`."""
        n, moments = p.numel(), torch.float32 if self._bits == 32 else torch.float8_e4m3fn
        kept = {"exp_avg": ((n,), moments), "exp_avg_sq": ((n,), moments)}
        if self._bits == 8:
            kept["scales"] = ((_padded(n) // BLOCK, 2), torch.float32)
        if self._master and p.dtype == torch.bfloat16:
            kept["master"] = ((n,), torch.float32)
        if set(saved) != {"step", *kept}:
            raise OptimizerInputError(f"a saved state has {sorted(saved)}, this optimizer keeps {sorted(['step', *kept])}")
        for name, (shape, dtype) in kept.items():
            if tuple(saved[name].shape) != shape or saved[name].dtype != dtype:
                raise OptimizerInputError(f"{name} of a saved state is {tuple(saved[name].shape)} {saved[name].dtype}, not {shape} {dtype}")
        if int(saved["step"]) < 0:
            raise OptimizerInputError(f"a saved state has taken {int(saved['step'])} steps")

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: float | torch.Tensor = 1.0):
        """One step from the parameters' `.grad`; parameters without one are left alone."""
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise OptimizerInputError("AdamW.step cannot be captured: lr and the step's number are launch arguments, and a replay would "
                                      "repeat this step; capture the backward pass and call step() after it")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for k, group in enumerate(self.param_groups):
            for b in self._of_group(k):
                grads = [p.grad for p in b.params]
                adamw_step(b.params, grads, b.state, lr=float(group["lr"]), betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], grad_scale=grad_scale)
        return loss

    def state_dict(self):
        for buckets in self._buckets.values():
            for b in buckets:
                for i, p in enumerate(b.params):
                    self.state[p]["step"] = b.state.steps[i]
        return super().state_dict()

    def load_state_dict(self, state_dict: dict) -> None:
        """Hyperparameters and states as saved, in their own dtypes (the base class would cast moments to the parameters').  A saved
        state that does not fit is refused before anything is changed."""
        order = [p for group in self.param_groups for p in group["params"]]
        names = [i for group in state_dict["param_groups"] for i in group["params"]]
        saved = {p: state_dict["state"][name] for name, p in zip(names, order) if name in state_dict["state"]}
        for p, of_p in saved.items():
            self._check_saved(p, of_p)
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})     # refuses other groups than these
        self._buckets = {}
        for p, of_p in saved.items():
            self.state[p] = dict(of_p)
        for k in range(len(self.param_groups)):
            self._of_group(k)

    def __getstate__(self):
        self.state_dict()                                # brings the step counts in self.state up to date
        return {**super().__getstate__(), "_bits": self._bits, "_master": self._master}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        if "_bits" in state:                             # a copy: states are laid out anew from self.state at the next step
            self._buckets = {}
