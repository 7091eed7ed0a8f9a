"""Muon for the convolution filters: momentum whose matrix is orthogonalised before it is applied.

    orthogonalize(matrices)      every matrix turned towards its nearest semi-orthogonal one (quintic Newton-Schulz steps)
    Muon(params, ...)            the optimiser; `training.configure_optimizers` builds it for `optimizer: muon`

A filter (out, in, kh, kw) is the matrix (out, in * kh * kw).  All filters of a step go through the phases of the iteration TOGETHER
(csrc/newton_schulz.hip): a network has many small ones, and one by one they would be bound by launches.

    v = momentum * v + g;   u = g + momentum * v  (nesterov) or v
    X = u / (|u| + eps);    steps times  A = X X^T,  X <- a X + (b A + c A^2) X
    p = p * (1 - lr * weight_decay) - lr * 0.2 * sqrt(max(out, in * kh * kw)) * X

The factor 0.2 sqrt(max) gives the update the root mean square of a usual AdamW update, so a learning rate and its schedule carry over.
The decay is part of the update's sum and rounded with it, so that it acts, on average, at lr * weight_decay below half a step of the weights (1e-8).
The reference trains with AdamW alone (modules/raft_spline.py:321-356).
"""
from __future__ import annotations

import math
from typing import Dict, List, Sequence, Tuple

import numpy as np
import torch

from . import hip

COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # a, b, c: singular values in (0.01, 1] end up near 1 (0.7 .. 1.2) after five steps
STEPS, EPS = 5, 1e-7


def _as_matrix(t: torch.Tensor, what: str) -> torch.Tensor:
    """(rows, cols) of a tensor with two dimensions or more, its elements next to each other inside a row."""
    if t.dim() < 2:
        raise hip.BflowHipError(f"{what}: a matrix or a filter has two dimensions or more, got {tuple(t.shape)}")
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t
    if t.dim() == 2:
        return t.contiguous()
    return t.contiguous().view(t.shape[0], math.prod(t.shape[1:]))


def _refused_size(shape: Sequence[int]) -> str:
    """Why a matrix or filter of this shape is too large for the kernels; empty where it is not."""
    rows, cols = shape[0], math.prod(shape[1:])
    if max(rows, cols) > hip.NS_MAX_SIDE or rows * cols > hip.NS_MAX_NUMBERS:
        return f"shape {tuple(shape)}: at most {hip.NS_MAX_SIDE} rows or columns and {hip.NS_MAX_NUMBERS} numbers are taken"
    return ""


def _table(entries: Sequence[Tuple[int, int, int, int, int, int, int]]) -> np.ndarray:
    return np.array(entries, dtype=hip.NS_MATRIX)


def _check_numbers(steps: int, coefficients: Sequence[float], eps: float):
    if len(coefficients) != 3:
        raise hip.BflowHipError(f"coefficients: three numbers a, b, c, got {coefficients!r}")
    if int(steps) != steps or not 1 <= steps <= 32:
        raise hip.BflowHipError(f"steps: a whole number in 1 .. 32, got {steps!r}")
    if not 1e-300 <= eps < 1.0:
        raise hip.BflowHipError(f"eps: a number in [1e-300, 1), got {eps!r}")


@torch.no_grad()
def orthogonalize(matrices: Sequence[torch.Tensor], steps: int = STEPS, coefficients: Sequence[float] = COEFFICIENTS, eps: float = EPS) -> List[torch.Tensor]:
    """Newton-Schulz steps on every matrix of a list: new tensors of the same shapes and types (float32, float16 or bfloat16, mixed as you like).

    Sums are held in 32 bits, products in fp16 pairs (fp32-class whatever the type; small matrices in 64 bits); a 16-bit result is rounded once.
    Tensors of more than two dimensions are taken as (shape[0], everything else).  An empty matrix stays empty, a zero matrix zero; one with a NaN or
    an infinity becomes all NaN.  The same list gives the same bits; a matrix in another list may be tiled another way and differ by roundings.  At
    most 2^20 rows or columns, 2^30 numbers.  Not differentiable: the results carry no graph."""
    _check_numbers(steps, coefficients, eps)
    if isinstance(matrices, torch.Tensor):
        raise hip.BflowHipError("orthogonalize takes a list of matrices")
    matrices = list(matrices)
    groups: Dict[Tuple[torch.dtype, torch.device], list] = {}
    for i, t in enumerate(matrices):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            hip._dev(t, None, f"matrix {i}", contiguous=False)                    # says why not
        if t.dim() > 1 and t.numel() > hip.NS_MAX_SIDE and _refused_size(t.shape):
            raise hip.BflowHipError(f"matrix {i}: {_refused_size(t.shape)}")
        key = (t.dtype, t.device)
        if key not in groups:
            if t.dtype not in hip.FLOAT_CODES:
                raise hip.BflowHipError(f"matrix {i}: dtype {t.dtype}, expected one of {sorted(str(d) for d in hip.FLOAT_CODES)}")
            groups[key] = []
        groups[key].append(i)
    results: List[torch.Tensor] = [None] * len(matrices)
    held = []                                             # contiguous copies live until the launches are enqueued
    for (dtype, device), members in groups.items():
        entries = []
        for i in members:
            t = matrices[i]
            x = _as_matrix(t, f"matrix {i}")
            y = results[i] = torch.empty_like(t, memory_format=torch.contiguous_format)
            rows, cols = x.shape
            if rows and cols:
                if x is not t:
                    held.append(x)
                entries.append((x.data_ptr(), y.data_ptr(), 0, x.stride(0) if rows > 1 else cols, cols, rows, cols))
        if entries:
            hip.ns_orthogonalize(_table(entries), dtype, device, int(steps), coefficients, eps)
    return results


class Muon(torch.optim.Optimizer):
    """Muon for matrices and filters; AdamW for the groups marked `adamw=True` (biases, the scales and shifts of norms).

    lr may be a float32 scalar tensor on the parameters' device: the kernels read it when they run, so a captured graph follows a schedule.
    Parameters, gradients and states are float32; a matrix has at most 2^20 rows or columns and 2^30 numbers.  capturable: a step may be captured,
    after a first one that creates the states; the AdamW step counters live on the device (torch.optim.AdamW)."""

    def __init__(self, params, lr=1e-3, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True, steps: int = STEPS,
                 coefficients: Sequence[float] = COEFFICIENTS, eps: float = EPS, betas: Tuple[float, float] = (0.9, 0.999), adamw_eps: float = 1e-8,
                 capturable: bool = False):
        defaults = dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps, coefficients=tuple(coefficients), eps=eps,
                        betas=betas, adamw_eps=adamw_eps, capturable=capturable, adamw=False)
        self._check_group(defaults)
        super().__init__(params, defaults)

    @staticmethod
    def _check_group(group):
        lr, momentum, decay = group["lr"], group["momentum"], group["weight_decay"]
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError(f"lr: {lr!r}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum: a number in [0, 1), got {momentum!r}")
        if not decay >= 0.0:
            raise ValueError(f"weight_decay: {decay!r}")
        _check_numbers(group["steps"], group["coefficients"], group["eps"])

    def add_param_group(self, group):
        self._check_group({**self.defaults, **group})
        super().add_param_group(group)
        group = self.param_groups[-1]
        for p in group["params"]:
            why = None
            if p.dtype != torch.float32:
                why = f"parameters are float32, got {p.dtype}"
            elif not group["adamw"] and (p.dim() < 2 or not p.is_contiguous()):
                why = f"a parameter of shape {tuple(p.shape)}, strides {p.stride()}: dense matrices or filters; put the others into a group with adamw=True"
            elif not group["adamw"] and _refused_size(p.shape):
                why = _refused_size(p.shape)
            if why is not None:
                self.param_groups.pop()
                raise hip.BflowHipError(f"Muon: {why}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None and p.numel()]
            if params and params[0].is_cuda and torch.cuda.is_current_stream_capturing():
                # a captured first step would clear the state at every replay; counters and rates on the host would stay as they were
                if not group["capturable"]:
                    raise hip.BflowHipError("Muon: a step is captured into a graph with capturable=True only")
                if any(not self.state.get(p) for p in params):
                    raise hip.BflowHipError("Muon: take a first step outside the capture, it creates the states")
            if params:
                (self._adamw if group["adamw"] else self._muon)(group, params)
        return loss

    def _muon(self, group, params):
        lr = group["lr"]
        if torch.is_tensor(lr) and (lr.numel() != 1 or lr.dtype != torch.float32):
            raise hip.BflowHipError(f"Muon: lr is a number or a float32 scalar, got {tuple(lr.shape)} {lr.dtype}")
        by_device: Dict[torch.device, list] = {}
        held = []
        for p in params:
            g = p.grad
            if g.layout is not torch.strided or g.dtype is not torch.float32 or g.device != p.device:
                raise hip.BflowHipError(f"Muon: gradients are dense float32 tensors on the parameter's device, got {g.dtype}, {g.layout}, {g.device}")
            hip._dev(p, torch.float32, "parameter")
            state = self.state[p]
            v = state.get("momentum_buffer")
            if v is None:
                v = state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            if v.shape != p.shape:
                raise hip.BflowHipError(f"Muon: momentum of shape {tuple(v.shape)} for a parameter of shape {tuple(p.shape)}")
            x = _as_matrix(g, "gradient")
            if x is not g:
                held.append(x)
            rows, cols = x.shape
            by_device.setdefault(p.device, []).append((x.data_ptr(), hip._dev(p, torch.float32, "parameter"), hip._dev(v, torch.float32, "momentum"),
                                                       x.stride(0) if rows > 1 else cols, cols, rows, cols))
        for device, entries in by_device.items():
            on_device = torch.is_tensor(lr) and lr.is_cuda
            hip.muon_step(_table(entries), device, int(group["steps"]), group["coefficients"], group["eps"], group["momentum"], group["nesterov"],
                          lr.to(device) if on_device else float(lr), group["weight_decay"])
        # the kernels wrote behind autograd's back: caches keyed on the version counters (packed filters, captured forwards) have to see it
        torch.autograd.graph.increment_version(params + [self.state[p]["momentum_buffer"] for p in params])

    def _adamw(self, group, params):
        from torch.optim.adamw import adamw
        for p in params:
            state = self.state[p]
            if not state:
                state["step"] = torch.zeros((), dtype=torch.float32, device=p.device if group["capturable"] else "cpu")
                state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        pick = lambda k: [self.state[p][k] for p in params]
        adamw(params, [p.grad for p in params], pick("exp_avg"), pick("exp_avg_sq"), [], pick("step"), capturable=group["capturable"], amsgrad=False,
              beta1=group["betas"][0], beta2=group["betas"][1], lr=group["lr"], weight_decay=group["weight_decay"], eps=group["adamw_eps"], maximize=False)
