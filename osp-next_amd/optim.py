"""AdamW over many tensors in few launches, with moments in fp32 or in 8 bits.

A step with t - 1 steps before it::

    m = b1 m + (1 - b1) g;    v = b2 v + (1 - b2) g^2
    p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

With 8-bit moments, m and sqrt(v) are e4m3 codes with a power-of-two scale for each 128 elements: 2 bytes a
parameter in place of 8.  sqrt(v) is rounded up or down at random (by numbers that the seed, the step and the
element decide, so that a run can be repeated): b2 near 1 moves it by less than half a step of its code,
and rounded to nearest it would never move.  A scale is finite: one gradient that is infinite or NaN makes its
block's 128 moments NaN, and with the next step their parameters, where fp32 moments lose its own alone; look
for such gradients before the step.  bf16 and fp16 parameters may have fp32 master weights, which
take the update, the parameter being their rounding.

The step count is on the GPU and every launch goes by it, so that a captured step counts on with each replay.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch import Tensor

from . import _lib

BLOCK = 128
MOST = 1 << 34                # elements of a tensor
Moment = Union[Tensor, Tuple[Tensor, Tensor]]


def pack_moment(t: Tensor) -> Tuple[Tensor, Tensor]:
    """A contiguous tensor as an 8-bit moment: (codes of its shape in float8_e4m3fn, scale bytes of each 128
    elements), rounded to nearest.  For the second moment pack its root."""
    if not t.is_contiguous():
        raise ValueError("pack_moment takes a contiguous tensor")
    from .fp8 import fp8_quantize
    n = t.numel()
    row = 64 * BLOCK              # 64 blocks a row, so that 2^34 elements stay within the rows that the quantiser takes
    flat = torch.zeros(max(1, (n + row - 1) // row) * row, dtype=torch.float32, device=t.device)
    flat[:n] = t.detach().reshape(-1)
    q = fp8_quantize(flat.view(-1, row))
    return q.codes.view(-1)[:n].clone().view(t.shape), q.scales.view(-1)[:(n + BLOCK - 1) // BLOCK].clone()


def unpack_moment(moment: Tuple[Tensor, Tensor]) -> Tensor:
    """The fp32 values of an 8-bit moment (m, or the root of v)."""
    codes, scales = moment
    s = (scales.to(torch.int32) << 23).view(torch.float32)
    return codes.to(torch.float32) * s.repeat_interleave(BLOCK)[:codes.numel()].view(codes.shape)


def _held(t: Tensor, dtype: torch.dtype, shape, device, name: str, i: int) -> int:
    """The address of a tensor that the step writes, of the given type and shape, contiguous on ``device``."""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} {i} is {t.dtype} {tuple(t.shape)}, not {dtype} {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} {i} must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} {i} lies on {t.device}, parameter 0 on {device}")
    return t.data_ptr()


def _rows(params, grads, exp_avgs, exp_avg_sqs, masters):
    """Refuses lists that do not fit; returns (whether the moments are in 8 bits, the tensors' rows for the entry
    point by dtype, what has to live until the call)."""
    n = len(params)
    if n == 0:
        raise ValueError("adamw_step of no tensors")
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n and (masters is None or len(masters) == n)):
        raise ValueError("adamw_step: the lists differ in length")
    bits8 = isinstance(exp_avgs[0], (tuple, list))
    dev = params[0].device
    by_dtype: dict = {}
    keep = []
    seen = set()
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs)):
        dt, shape, count = p.dtype, p.shape, p.numel()
        _lib.float_code(dt)
        if p.layout is not torch.strided or g.layout is not torch.strided:
            raise TypeError("adamw_step takes dense tensors and gradients")
        if g.dtype is not dt or g.shape != shape:
            raise ValueError(f"gradient {i} is {g.dtype} {tuple(g.shape)}, its parameter {dt} {tuple(shape)}")
        if bits8 != isinstance(m, (tuple, list)) or bits8 != isinstance(v, (tuple, list)):
            raise TypeError("adamw_step: moments in 8 bits and in fp32 mixed")
        pp = _held(p, dt, shape, dev, "parameter", i)
        if bits8:
            blocks = ((count + BLOCK - 1) // BLOCK,)
            mp, vp = (_held(t[0], torch.float8_e4m3fn, shape, dev, name, i) for t, name in ((m, "exp_avg"), (v, "exp_avg_sq")))
            ms, vs = (_held(t[1], torch.uint8, blocks, dev, name, i) for t, name in ((m, "exp_avg scales"), (v, "exp_avg_sq scales")))
        else:
            mp, vp = _held(m, torch.float32, shape, dev, "exp_avg", i), _held(v, torch.float32, shape, dev, "exp_avg_sq", i)
            ms = vs = 0
        wp = 0
        if masters is not None:
            if dt is torch.float32:
                raise TypeError("an fp32 parameter needs no master weight")
            wp = _held(masters[i], torch.float32, shape, dev, "master weight", i)
        if g.device != dev:
            raise ValueError(f"gradient {i} lies on {g.device}, parameter 0 on {dev}")
        if count == 0:
            continue
        if pp in seen:
            raise ValueError("adamw_step: a parameter appears twice")
        seen.add(pp)
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        by_dtype.setdefault(dt, []).append((pp, g.data_ptr(), mp, vp, ms, vs, wp, count, i))
    if len(by_dtype) > 1:
        _check_types(by_dtype, bits8)
    if dev.type != "cuda":
        raise ValueError(f"adamw_step takes GPU tensors (there is no CPU route), got {dev}")
    return bits8, by_dtype, keep


def _check_types(by_dtype: dict, bits8: bool) -> None:
    """What the entry point refuses, for a step of several types: it looks at one type's tensors, and none may be
    refused once another type's call has been made."""
    spans, grads = [], []
    for dt, rows in by_dtype.items():
        t = np.array(rows, dtype=np.int64)
        n, moment = t[:, 7], 1 if bits8 else 4
        if (n > MOST).any():
            raise ValueError(f"adamw_step: a tensor of {n.max()} elements (at most {MOST})")
        for at, size in ((0, dt.itemsize * n), (2, moment * n), (3, moment * n), (4, (n + BLOCK - 1) // BLOCK),
                         (5, (n + BLOCK - 1) // BLOCK), (6, 4 * n)):
            spans.append(np.stack((t[:, at], t[:, at] + size), 1)[t[:, at] != 0])
        grads.append(np.stack((t[:, 1], t[:, 1] + dt.itemsize * n), 1))
    s, g = np.concatenate(spans), np.concatenate(grads)
    s = s[np.argsort(s[:, 0])]
    if (s[1:, 0] < s[:-1, 1]).any():
        raise ValueError("adamw_step: two tensors that it writes share memory")
    before = np.searchsorted(s[:, 0], g[:, 1]) - 1          # the last written tensor that begins before the gradient's end
    if (s[before, 1] > g[:, 0])[before >= 0].any():
        raise ValueError("adamw_step: a gradient shares memory with a tensor that it writes")


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Moment],
               exp_avg_sqs: Sequence[Moment], step: Tensor, *, lr: float, betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, masters: Optional[Sequence[Tensor]] = None,
               seed: int = 0) -> None:
    """One AdamW step in place on contiguous bf16, fp16 or fp32 parameters, gradients of their types.  No two tensors that
    it writes may share memory, nor a gradient with one of them.

    ``exp_avgs`` and ``exp_avg_sqs`` are fp32 tensors, or (codes, scales) pairs in 8 bits, of m and of sqrt(v)
    (``pack_moment``).  ``masters``: fp32 master weights of 16-bit parameters.  ``step``: an int64 tensor of one
    element on the parameters' GPU, the number of steps done, which the call adds one to.  ``seed`` decides the
    rounding of 8-bit second moments."""
    bits8, by_dtype, keep = _rows(params, grads, exp_avgs, exp_avg_sqs, masters)
    dev = params[0].device
    if step.dtype != torch.int64 or step.numel() != 1 or step.device != dev:
        raise ValueError("step must be one int64 on the parameters' device")
    if isinstance(lr, Tensor):
        raise TypeError("lr is a number (a tensor's value would have to come from the GPU)")
    L = _lib.load()
    with _lib.on(dev):
        ws = torch.empty(L.hif8_adamw_workspace_bytes(), dtype=torch.uint8, device=dev)
        advance = 1
        for dt, rows in by_dtype.items():
            table = np.array(rows, dtype=np.uint64)
            _lib.check(L.hif8_adamw_step(table.ctypes.data, len(rows), _lib.float_code(dt), 8 if bits8 else 32,
                                         step.data_ptr(), advance, float(lr), float(betas[0]), float(betas[1]), float(eps),
                                         float(weight_decay), int(seed) & 0xFFFFFFFF, ws.data_ptr(), ws.numel(),
                                         _lib.stream_ptr(dev)), "hif8_adamw_step")
            advance = 0
        if advance:                       # nothing but empty parameters: the step counts all the same
            step.add_(1)
    del keep
    # the kernel wrote them by address: what goes by version counters (autograd, packed weights) has to see it
    torch.autograd.graph.increment_version([*params, *masters] if masters is not None else params)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s rule on ``adamw_step``.

    ``state_bits``: 32, or 8 for moments in 8 bits (2 bytes a parameter).  ``master``: keep fp32 master weights
    of bf16 and fp16 parameters (default: yes).  ``seed``: of the 8-bit rounding.  Parameters are contiguous GPU
    tensors.  A step can be captured into a graph after one eager step with the same parameters' gradients, which
    gives each its state and those that go together their count; the learning rate and the other numbers are those of
    the capture then, the step count goes on, and the graph keeps to the state's tensors as they were captured (an
    eager step of fewer parameters, or a loaded state, puts others in their place)."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, master: bool = True, seed: int = 0):
        self.seed = int(seed)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master=master))

    def add_param_group(self, param_group: dict) -> None:
        g = {**self.defaults, **param_group}
        if isinstance(g["lr"], Tensor):
            raise TypeError("lr is a number")
        if not g["lr"] >= 0 or not g["eps"] >= 0 or not g["weight_decay"] >= 0 or not all(0 <= b < 1 for b in g["betas"]):
            raise ValueError("AdamW: " + ", ".join(f"{k} {g[k]}" for k in ("lr", "betas", "eps", "weight_decay")))
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {g['state_bits']}")
        super().add_param_group(param_group)

    def _new_state(self, p: Tensor, group: dict, step: Tensor) -> dict:
        s = dict(step=step)
        if group["state_bits"] == 8:
            for k in ("exp_avg", "exp_avg_sq_root"):
                s[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                s[k + "_scales"] = torch.full(((p.numel() + BLOCK - 1) // BLOCK,), 127, dtype=torch.uint8, device=p.device)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master"] and p.dtype != torch.float32:
            s["master"] = p.detach().to(torch.float32)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # A step tensor is shared by the parameters that have always been stepped together.
        holders: dict = {}
        for s in self.state.values():
            if "step" in s:
                holders[id(s["step"])] = holders.get(id(s["step"]), 0) + 1
        for g_at, group in enumerate(self.param_groups):
            cohorts: dict = {}
            new = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not self.state[p]:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: a parameter without state in a captured step; run one eager step first")
                    if p.device not in new:
                        new[p.device] = torch.zeros(1, dtype=torch.int64, device=p.device)
                    self.state[p].update(self._new_state(p, group, new[p.device]))
                s = self.state[p]
                cohorts.setdefault((id(s["step"]), "master" in s), []).append(p)
            masters_of: dict = {}
            for step_id, with_master in cohorts:
                masters_of.setdefault(step_id, []).append(with_master)
            for step_id, kinds in masters_of.items():
                members = [p for k in kinds for p in cohorts[step_id, k]]
                step = self.state[members[0]]["step"]
                if holders.get(step_id, len(members)) > len(members):     # the others stay where they are
                    if step.is_cuda and torch.cuda.is_current_stream_capturing():
                        # each replay would copy the count that stays, and stand still
                        raise RuntimeError("AdamW: a captured step of some of the parameters that have been stepped "
                                           "together; run one eager step with these gradients first")
                    step = step.clone()
                    for p in members:
                        self.state[p]["step"] = step
                for at, k in enumerate(kinds):
                    ps = cohorts[step_id, k]
                    ss = [self.state[p] for p in ps]
                    if at:               # the second call of this step: it counts once
                        step.sub_(1)
                    if group["state_bits"] == 8:
                        m = [(s["exp_avg"], s["exp_avg_scales"]) for s in ss]
                        v = [(s["exp_avg_sq_root"], s["exp_avg_sq_root_scales"]) for s in ss]
                    else:
                        m, v = [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss]
                    adamw_step(ps, [p.grad for p in ps], m, v, step, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                               weight_decay=group["weight_decay"], masters=[s["master"] for s in ss] if k else None,
                               seed=self.seed + 7919 * (2 * g_at + at))
        return loss

    def load_state_dict(self, state_dict) -> None:
        """Loads a state as it was saved: fp32 and 8-bit tensors keep their types beside 16-bit parameters."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        shared: dict = {}
        for i, p in zip(ids, own):
            if i not in saved:
                continue
            s = {k: v.to(p.device, copy=True) if isinstance(v, Tensor) else v for k, v in saved[i].items()}
            if "step" in s:
                group = next(k for k, g in enumerate(self.param_groups) if any(q is p for q in g["params"]))
                s["step"] = shared.setdefault((group, p.device, int(s["step"])), s["step"])
            self.state[p] = s
