"""AdamW (torch.optim.AdamW, the reference's tools/ldm/image.py:62) over many separately allocated tensors in a few launches, with the
moments in 32 or in 8 bits.  `train.FlatParams` + ddmi_train_adamw is the same step over ONE fp32 slab; this one takes tensors as they are:
fp32 or bf16 parameters and gradients, a learning rate and weight decay of their own, gradients that come and go.

8-bit moments (include/ddmi_hip.h, ddmi_adamw_tensor): e4m3 codes of the first moment and of the ROOT of the second, an fp32 power-of-two
scale for each 256 consecutive values of a tensor: 2.03 bytes a parameter instead of 8.  They and bf16 parameters are rounded
stochastically, from random bits that depend on (seed, step, the tensor's place in the list, the value's place in it) and nothing else: a
step gives the same bits on every run.
"""
from __future__ import annotations

import itertools
import operator
from typing import Dict, List, Optional, Sequence, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

BLOCK = 256
_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_ENTRY = np.dtype([("param", "u8"), ("grad", "u8"), ("exp_avg", "u8"), ("exp_avg_sq", "u8"), ("exp_avg_scale", "u8"), ("exp_avg_sq_scale", "u8"),
                   ("numel", "i8"), ("step", "i8"), ("lr", "f8"), ("weight_decay", "f8"), ("index", "i8")])


_NUMEL, _CONTIGUOUS, _POINTER, _DEVICE = torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.data_ptr, torch.Tensor.get_device
_DTYPE, _SHAPE = operator.attrgetter("dtype"), operator.attrgetter("shape")


def blocks_of(n: int) -> int:
    """Scales of a tensor of n values."""
    return -(-n // BLOCK)


def _overlap(ptrs, nbytes, written) -> bool:
    """Whether a range that is written meets any other."""
    at = np.argsort(ptrs, kind="stable")
    start, w = ptrs[at].astype(np.int64), written[at]
    end = start + nbytes[at]
    before = np.maximum.accumulate(end)[:-1]                                     # where the ranges so far end
    before_written = np.maximum.accumulate(np.where(w, end, 0))[:-1]
    return bool(np.any(before_written > start[1:]) or np.any(w[1:] & (before > start[1:])))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor],
               step: Union[int, Sequence[int]], lr: Union[float, Sequence[float]], betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: Union[float, Sequence[float]] = 0.0, grad_scale: float = 1.0, exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, seed: int = 0) -> None:
    """One AdamW step in place over lists of contiguous tensors on one GPU, on its current stream.

    params, grads: fp32 or bf16 (each its own type), any shapes; a gradient has its parameter's.  Moments: all fp32 of the parameters' sizes,
    or all float8_e4m3fn (exp_avg: codes of the first moment; exp_avg_sq: codes of the second one's root) with fp32 scales of
    ceil(numel / 256) values each.  step (this step's number, from 1), lr and weight_decay: one for all tensors, or one a tensor.  Gradients
    are multiplied by grad_scale first (1 / world_size after a sum, 1 / accumulated micro-steps).  The step number is an argument, so the
    call is refused inside a graph capture, where it would be frozen."""
    who = "adamw_step"
    lists = [list(v) for v in (params, grads, exp_avgs, exp_avg_sqs)]
    params, grads, exp_avgs, exp_avg_sqs = lists
    n = len(params)
    if any(len(v) != n for v in lists):
        raise ValueError(f"{who}: params, grads, exp_avgs and exp_avg_sqs have {[len(v) for v in lists]} tensors")
    if n == 0:
        return
    kinds = set(map(_DTYPE, exp_avgs)) | set(map(_DTYPE, exp_avg_sqs))
    if kinds == {torch.float32}:
        bits = 32
        if exp_avg_scales is not None or exp_avg_sq_scales is not None:
            raise ValueError(f"{who}: fp32 moments have no scales")
    elif kinds == {torch.float8_e4m3fn}:
        bits = 8
        if exp_avg_scales is None or exp_avg_sq_scales is None:
            raise ValueError(f"{who}: 8-bit moments need exp_avg_scales and exp_avg_sq_scales")
        scales = [list(exp_avg_scales), list(exp_avg_sq_scales)]
        if any(len(v) != n for v in scales):
            raise ValueError(f"{who}: {n} parameters and {[len(v) for v in scales]} scales")
        lists = lists + scales
    else:
        raise ValueError(f"{who}: moments are all fp32 or all float8_e4m3fn, got {sorted(map(str, kinds))}")
    p_types, g_types = list(map(_DTYPE, params)), list(map(_DTYPE, grads))
    p_kinds, g_kinds = set(p_types), set(g_types)
    if not p_kinds | g_kinds <= set(_TYPES):
        raise ValueError(f"{who}: parameters and gradients are fp32 or bf16, got {sorted(map(str, p_kinds | g_kinds))}")
    flat = list(itertools.chain.from_iterable(lists))
    numels = np.fromiter(map(_NUMEL, flat), np.int64, len(flat)).reshape(-1, n)      # a row for each list
    numel = numels[0]
    for name, row in zip(("gradient", "exp_avg", "exp_avg_sq"), numels[1:4]):
        if not np.array_equal(row, numel):
            raise ValueError(f"{who}: a tensor's {name} has another number of values than the parameter")
    if list(map(_SHAPE, grads)) != list(map(_SHAPE, params)):
        raise ValueError(f"{who}: a gradient has another shape than its parameter")
    blocks = -(-numel // BLOCK)
    if bits == 8 and (np.any(numels[4:] != blocks) or any(set(map(_DTYPE, ts)) != {torch.float32} for ts in scales)):
        raise ValueError(f"{who}: scales are fp32, one for each {BLOCK} values of a tensor")
    if not all(map(_CONTIGUOUS, flat)):
        raise ValueError(f"{who}: tensors are contiguous")
    e = np.zeros(n, dtype=_ENTRY)
    e["numel"], e["step"], e["lr"], e["weight_decay"], e["index"] = numel, step, lr, weight_decay, np.arange(n)
    if e["step"].min() < 1:
        raise ValueError(f"{who}: step counts from 1")
    b1, b2 = float(betas[0]), float(betas[1])
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0):
        raise ValueError(f"{who}: betas in [0, 1) and eps >= 0, got {betas}, {eps}")
    if forward_ad._current_level >= 0:
        _lib.refuse_tangents(who, *flat)
    dev = params[0].get_device()
    if dev < 0 or not params[0].is_cuda or set(map(_DEVICE, flat)) != {dev}:
        raise ValueError(f"{who}: all tensors live on one GPU, got {sorted({str(t.device) for t in flat})}")
    ptrs = np.fromiter(map(_POINTER, flat), np.uint64, len(flat)).reshape(-1, n)
    for name, row in zip(("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"), ptrs):
        e[name] = row
    sizes = numels.copy()                                                                # bytes
    sizes[0] *= 4 if p_kinds == {torch.float32} else np.array([t.itemsize for t in p_types])
    sizes[1] *= 4 if g_kinds == {torch.float32} else np.array([t.itemsize for t in g_types])
    sizes[2:] *= 4
    if bits == 8:
        sizes[2:4] = numel
    written = np.ones(ptrs.shape, dtype=bool)
    written[1] = False
    some = (numels > 0).ravel()
    if _overlap(ptrs.ravel()[some], sizes.ravel()[some], written.ravel()[some]):
        raise ValueError(f"{who}: a tensor that is written shares memory with another (the same one twice?)")
    with _lib.on_device(dev):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{who}: not inside a graph capture: the step number is an argument and would be frozen")
        _lib.init_device(dev)
        of = list(zip(p_types, g_types)) if len(p_kinds) + len(g_kinds) > 2 else None
        for kind in dict.fromkeys(of) if of else [(p_types[0], g_types[0])]:
            part = np.ascontiguousarray(e[[k == kind for k in of]]) if of else e
            _lib.check(_lib.lib().ddmi_train_adamw_multi(part.ctypes.data, len(part), b1, b2, float(eps), float(grad_scale), int(seed) & 0xFFFFFFFF,
                                                         _TYPES[kind[0]], _TYPES[kind[1]], bits, _lib.raw_stream(dev)))
    torch.autograd.graph.increment_version(params)      # a backward through a graph that saved the old values raises, as after torch's own step


def encode_moment(x: torch.Tensor, root: bool):
    """fp32 moment -> (e4m3 codes, scales), rounded to nearest: how a checkpoint's 32-bit moments enter the 8-bit state.  root: the second
    moment, of which the root is stored, and of which only a zero becomes zero."""
    n = x.numel()
    rows = torch.zeros(blocks_of(n) * BLOCK, dtype=torch.float32, device=x.device)
    rows[:n] = x.detach().reshape(-1).float().sqrt() if root else x.detach().reshape(-1).float()
    rows = rows.view(-1, BLOCK)
    most = torch.where(rows.isfinite(), rows.abs(), torch.zeros_like(rows)).amax(1)
    mantissa, exponent = torch.frexp(most)                                   # most = mantissa 2^exponent, mantissa in [0.5, 1)
    k = (exponent - (mantissa == 0.5).int() - 8).clamp(-120, 120)             # most / 2^k in (128, 256]
    k = torch.where(most == 0, torch.full_like(k, -120), k)
    scale = torch.ldexp(torch.ones_like(most), k)
    code = (rows / scale[:, None]).to(torch.float8_e4m3fn)
    if root:
        code = torch.where((rows > 0) & (code.view(torch.uint8) == 0), torch.ones_like(code.view(torch.uint8)), code.view(torch.uint8)).view(code.dtype)
    return code.view(-1)[:n], scale


def decode_moment(codes: torch.Tensor, scales: torch.Tensor, root: bool) -> torch.Tensor:
    """(codes, scales) -> the fp32 moment they stand for."""
    n = codes.numel()
    rows = torch.zeros(blocks_of(n) * BLOCK, dtype=torch.float32, device=codes.device)
    rows[:n] = codes.reshape(-1).float()
    v = (rows.view(-1, BLOCK) * scales[:, None]).view(-1)[:n]
    return v * v if root else v


class AdamW:
    """The optimizer over parameters or parameter groups ({"params": [...], "lr": ..., "weight_decay": ...}), as torch.optim.AdamW is made;
    a parameter whose `.grad` is None sits the step out, its step count too.  `param_groups[i]["lr"]` and `["weight_decay"]` are read at every
    step.  state_bits: 32 or 8.  The moments of all parameters lie in one
    slab each, a parameter's from a multiple of 256 values on.

    It is not a torch.optim.Optimizer: a torch scheduler does not take it (set the groups' lr), betas and eps are those of all groups, zero_grad
    clears the gradients in place unless told otherwise, and bf16 parameters are rounded stochastically with either kind of moments.  The seed
    of the rounding is an argument and no part of the state: a resumed run gives the same bits with the same seed."""

    def __init__(self, params, lr: float = 1e-4, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, state_bits: int = 32, seed: int = 0):
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: state_bits is 32 or 8, got {state_bits}")
        params = list(params)
        groups = params if params and isinstance(params[0], dict) else [{"params": params}]
        self.params: List[torch.Tensor] = []
        self.param_groups: List[Dict] = []
        for g in groups:
            ps = list(g["params"])
            unknown = set(g) - {"params", "lr", "weight_decay"}
            if unknown:
                raise ValueError(f"AdamW: a parameter group sets lr and weight_decay, got {sorted(unknown)}")
            first = len(self.params)
            self.params += ps
            self.param_groups.append({"lr": float(g.get("lr", lr)), "weight_decay": float(g.get("weight_decay", weight_decay)),
                                      "params": list(range(first, len(self.params)))})
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if len({id(p) for p in self.params}) < len(self.params):
            raise ValueError("AdamW: a parameter is given twice")
        for p in self.params:
            if p.dtype not in _TYPES or not p.is_contiguous():
                raise ValueError(f"AdamW: parameters are contiguous fp32 or bf16 tensors, got {p.dtype} with strides {p.stride()}")
        self.betas, self.eps, self.state_bits, self.seed = (float(betas[0]), float(betas[1])), float(eps), int(state_bits), int(seed)
        self.steps = [0] * len(self.params)
        dev = self.params[0].device
        rows = [blocks_of(p.numel()) for p in self.params]
        total, dtype = sum(rows), torch.float32 if state_bits == 32 else torch.float8_e4m3fn

        def slab(values, unit, sizes, dtype):
            flat = torch.zeros(values * unit, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype, device=dev).view(dtype)
            at = np.concatenate([[0], np.cumsum(rows)]) * unit
            return [flat[int(a):int(a) + k] for a, k in zip(at, sizes)]

        sizes = [p.numel() for p in self.params]
        self.exp_avg, self.exp_avg_sq = slab(total, BLOCK, sizes, dtype), slab(total, BLOCK, sizes, dtype)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale, self.exp_avg_sq_scale = (slab(total, 1, rows, torch.float32) for _ in range(2))

    def step(self, grad_scale: float = 1.0) -> None:
        at = [i for i, p in enumerate(self.params) if p.grad is not None]
        take = (lambda v: v) if len(at) == len(self.params) else (lambda v: [v[i] for i in at])
        steps = [s + 1 for s in take(self.steps)]
        lr, weight_decay = (take([float(g[k]) for g in self.param_groups for _ in g["params"]]) for k in ("lr", "weight_decay"))
        with torch.no_grad():
            adamw_step(take(self.params), [self.params[i].grad for i in at], take(self.exp_avg), take(self.exp_avg_sq), steps,
                       lr=lr, betas=self.betas, eps=self.eps, weight_decay=weight_decay, grad_scale=grad_scale,
                       exp_avg_scales=None if self.state_bits == 32 else take(self.exp_avg_scale),
                       exp_avg_sq_scales=None if self.state_bits == 32 else take(self.exp_avg_sq_scale), seed=self.seed)
        for i, s in zip(at, steps):      # only a step that was taken counts
            self.steps[i] = s

    def zero_grad(self, set_to_none: bool = False) -> None:
        for p in self.params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.detach().zero_()

    # ---- moments as fp32 values: torch.optim.AdamW's state dict ------------------------------------------------------------------
    def moments(self, i: int):
        """(exp_avg, exp_avg_sq) of parameter i as fp32 tensors of its shape."""
        shape = self.params[i].shape
        if self.state_bits == 32:
            return self.exp_avg[i].clone().view(shape), self.exp_avg_sq[i].clone().view(shape)
        return (decode_moment(self.exp_avg[i], self.exp_avg_scale[i], False).view(shape),
                decode_moment(self.exp_avg_sq[i], self.exp_avg_sq_scale[i], True).view(shape))

    def _check_moments(self, i: int, exp_avg, exp_avg_sq, step: int) -> None:
        for name, new in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
            shape = tuple(torch.as_tensor(new).shape)
            if shape != tuple(self.params[i].shape):
                raise ValueError(f"AdamW: {name} of parameter {i} has shape {shape}, the parameter {tuple(self.params[i].shape)}")
        if step < 0:
            raise ValueError(f"AdamW: parameter {i} has taken {step} steps")

    def set_moments(self, i: int, exp_avg, exp_avg_sq, step: int) -> None:
        self._check_moments(i, exp_avg, exp_avg_sq, step)
        for name, new, root in (("exp_avg", exp_avg, False), ("exp_avg_sq", exp_avg_sq, True)):
            new = torch.as_tensor(new).to(self.params[i].device, torch.float32)
            if self.state_bits == 32:
                getattr(self, name)[i].copy_(new.reshape(-1))
            else:
                codes, scales = encode_moment(new, root)
                getattr(self, name)[i].view(torch.uint8).copy_(codes.view(torch.uint8))
                getattr(self, name + "_scale")[i].copy_(scales)
        self.steps[i] = int(step)

    def state_dict(self) -> Dict:
        state = {}
        for i, s in enumerate(self.steps):
            if s > 0:
                m, v = self.moments(i)
                state[i] = {"step": torch.tensor(float(s)), "exp_avg": m, "exp_avg_sq": v}
        rest = {"betas": self.betas, "eps": self.eps, "amsgrad": False, "maximize": False, "foreach": None, "capturable": False, "differentiable": False,
                "fused": None}
        return {"state": state, "param_groups": [dict(g, **rest) for g in self.param_groups]}

    def load_state_dict(self, sd: Dict) -> None:
        """torch.optim.AdamW's layout; 8-bit moments are rounded to the nearest code (exact for values that came out of an 8-bit state).  A
        state of another optimizer - amsgrad, maximize, weight decay that is not decoupled, betas or eps of a group's own - is refused, and a
        refused state changes nothing."""
        groups = sd["param_groups"]
        if [list(g["params"]) for g in groups] != [list(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the state dict has other parameter groups")
        for k in ("amsgrad", "maximize"):
            if any(g.get(k) for g in groups):
                raise ValueError(f"AdamW: the state dict is that of an optimizer with {k}")
        if any(float(g["weight_decay"]) != 0.0 and not g.get("decoupled_weight_decay", True) for g in groups):
            raise ValueError("AdamW: the state dict is that of an optimizer whose weight decay is a part of the gradient")
        rates = [(float(g["lr"]), float(g["weight_decay"])) for g in groups]
        shared = {(tuple(float(b) for b in g["betas"]), float(g["eps"])) for g in groups}
        if len(shared) > 1:
            raise ValueError(f"AdamW: all groups have the same betas and eps, the state dict has {sorted(shared)}")
        (betas, eps), = shared
        if len(betas) != 2 or not (all(0.0 <= b < 1.0 for b in betas) and eps >= 0.0):
            raise ValueError(f"AdamW: betas in [0, 1) and eps >= 0, the state dict has {betas}, {eps}")
        extra = [i for i in sd["state"] if not (isinstance(i, int) and 0 <= i < len(self.params))]
        if extra:
            raise ValueError(f"AdamW: state for parameters {extra[:5]}, of {len(self.params)}")
        state = {}
        for i, st in sd["state"].items():
            missing = {"step", "exp_avg", "exp_avg_sq"} - set(st)
            if missing:
                raise ValueError(f"AdamW: the state of parameter {i} has no {sorted(missing)}")
            state[i] = (st["exp_avg"], st["exp_avg_sq"], int(float(st["step"])))
            self._check_moments(i, *state[i])
        for (lr, weight_decay), mine in zip(rates, self.param_groups):
            mine["lr"], mine["weight_decay"] = lr, weight_decay
        self.betas, self.eps = betas, eps
        for i, p in enumerate(self.params):
            self.set_moments(i, *(state[i] if i in state else (torch.zeros(p.shape), torch.zeros(p.shape), 0)))
