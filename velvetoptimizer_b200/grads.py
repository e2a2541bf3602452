"""Global gradient norm and clipping over any number of tensors, in two kernel launches.

``clip_grad_norm_`` takes the place of ``torch.nn.utils.clip_grad_norm_`` in the reference's
training loop (python/train.py:465-480): a mixture layer has 14 E + 2 parameters, and reading
and scaling them one by one costs more launches than the step's own kernels.  Nothing waits for
the GPU unless ``error_if_nonfinite`` asks for it.
"""
from __future__ import annotations

import math

import torch

from .dense import _native

_NORMS = {math.inf: 0, 1.0: 1, 2.0: 2}  # VMOE_NORM_*


def _tensors(tensors):
    if type(tensors) in (list, tuple):
        return tensors
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type}")
    return code


def _run(items, use_grad: bool, max_norm: float, code: int) -> torch.Tensor:
    norm = _native().grad_norm(items, use_grad, max_norm, code)
    return torch.tensor(0.0) if norm is None else norm


def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``tensors`` (a tensor or an iterable of float32 and bfloat16
    CUDA tensors on one device) as a float32 scalar on their device.

    ``norm_type`` is 2, 1 or ``inf``.  A tensor given twice counts once.  Sums are held in fp64
    in a fixed order, so two calls give the same bits.  Without tensors the norm is 0.  The norm
    carries no gradient.
    """
    return _run(_tensors(tensors), False, -1.0, _norm_code(norm_type))


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by ``min(1, max_norm / (norm + 1e-6))`` and
    return their norm before the scaling, as ``torch.nn.utils.clip_grad_norm_`` does.

    Gradients are float32 or bfloat16 CUDA tensors on one device; parameters without one are
    skipped, and a gradient that several of them share is counted and scaled once.  A norm that
    is NaN makes every gradient NaN and an infinite one scales by 0, unless
    ``error_if_nonfinite``: then the call waits for the norm and raises before it scales.
    """
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, not {max_norm}")
    code = _norm_code(norm_type)
    items = _tensors(parameters)
    if error_if_nonfinite:
        norm = float(_run(items, True, -1.0, code))
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm of order {norm_type} is {norm}: not clipped")
    return _run(items, True, max_norm, code)
