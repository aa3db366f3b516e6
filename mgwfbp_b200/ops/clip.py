# -*- coding: utf-8 -*-
"""Global gradient norm over many tensors, and clipping (``csrc/grad_clip.cu``).

``clip_grad_norm_`` scales the gradients of all parameters in place so that their norm is at most ``max_norm``, as
``torch.nn.utils.clip_grad_norm_`` (the reference calls that between ``synchronize()`` and ``step()``,
``dist_trainer.py:89-94``), in two launches without a host round trip, for any mix of fp32, fp16 and bf16 gradients, with an
optional factor that is applied in the same pass (``grad_scale``: the inverse loss scale, the number of workers).
``grad_norm`` only measures.  ``DistributedOptimizer(norm_clip=...)`` uses it for every optimizer and type whose clip is
not part of the fused momentum-SGD update (``ops.sgd``).  On CPU tensors the same functions run plain PyTorch operations.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional, Union

import torch

from ._tokens import DTYPES, native

_NORMS = {2.0: 0, 1.0: 1, math.inf: 2}


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of ``t`` fill one stretch of memory, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def supported(grads: List[torch.Tensor]) -> bool:
    """Whether :func:`clip_grad_norm_` runs the kernels on these gradients."""
    return bool(grads) and grads[0].is_cuda and native().clip_supported(grads)


def _norm_code(norm_type: float) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError('norm_type must be 1, 2 or infinity, got %r' % (norm_type,))
    return code


def _check(grads: List[torch.Tensor]) -> None:
    first = grads[0].device
    for g in grads:
        if g.layout != torch.strided or not g.is_floating_point():
            raise TypeError('gradients must be dense floating-point tensors, got %s %s' % (g.dtype, g.layout))
        if g.device != first:
            raise ValueError('gradients are on %s and %s: clip the gradients of one device' % (first, g.device))
        if g.is_cuda and g.dtype not in DTYPES:
            raise TypeError('gradients must be float32, float16 or bfloat16, got %s' % g.dtype)
        if not _dense(g):
            raise ValueError('a gradient of shape %s has strides %s: its elements do not fill one stretch of memory'
                             % (tuple(g.shape), g.stride()))


def _kernels(tensors: List[torch.Tensor], parameters: bool, code: int, scale: float, max_norm: float, clip: bool) -> Optional[torch.Tensor]:
    """Norm (and scaling) by the kernels of ``tensors`` or of their gradients; ``None`` where those are not for them."""
    if not any(t.is_cuda for t in tensors):
        return None
    return native().clip_grads(tensors, parameters, code, scale, max_norm, clip)


def _reference_norm(grads: List[torch.Tensor], norm_type: float, scale: float) -> torch.Tensor:
    """The norm with plain tensor operations (any device); a tensor that is listed twice counts once."""
    each = {(g.data_ptr(), g.numel()): g for g in grads}.values()
    parts = torch.stack([torch.linalg.vector_norm(g.detach().double().reshape(-1), norm_type) if g.numel() else
                         torch.zeros((), dtype=torch.float64, device=g.device) for g in each])
    return torch.linalg.vector_norm(parts, norm_type) * abs(scale)


def _check_scale(grad_scale: float) -> float:
    scale = float(grad_scale)
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError('grad_scale must be positive, between 2^-100 and 2^100, got %r' % (grad_scale,))
    return scale


def grad_norm(grads: Iterable[torch.Tensor], norm_type: float = 2.0, grad_scale: float = 1.0) -> torch.Tensor:
    """Norm of all values of ``grads`` together, times ``grad_scale``, as an fp32 scalar on their device."""
    code, scale, grads = _norm_code(norm_type), _check_scale(grad_scale), list(grads)
    if not grads:
        return torch.zeros(())
    norm = _kernels(grads, False, code, scale, 0.0, False)
    if norm is None:
        _check(grads)
        norm = _reference_norm(grads, float(norm_type), scale).float()
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, grad_scale: float = 1.0) -> torch.Tensor:
    """Multiply the gradients of ``parameters`` by ``grad_scale`` and then by ``min(1, max_norm / (norm + 1e-6))``, in place
    and rounded once, and return the norm before clipping (of the scaled gradients) as an fp32 scalar.

    A gradient that is listed twice counts and is scaled once; gradients that share memory in part are refused.  A norm
    of NaN makes the gradients NaN, an infinite one makes the finite ones zero, as in PyTorch; ``error_if_nonfinite`` waits
    for the norm and raises before anything is changed."""
    code, scale, max_norm = _norm_code(norm_type), _check_scale(grad_scale), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError('max_norm must not be negative, got %r' % (max_norm,))
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if error_if_nonfinite:
        norm = grad_norm([p.grad for p in parameters if p.grad is not None], norm_type, scale)
        if not math.isfinite(float(norm)):
            raise RuntimeError('The total norm of order %s for the gradients is non-finite, so they cannot be clipped' % (norm_type,))
    norm = _kernels(parameters, True, code, scale, max_norm, True)
    if norm is not None:
        return norm
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros(())
    _check(grads)
    norm = _reference_norm(grads, float(norm_type), scale)
    factor = float(scale * torch.clamp(max_norm / (norm + 1e-6), max=1.0))
    for g in {(g.data_ptr(), g.numel()): g for g in grads}.values():
        g.detach().copy_((g.detach().double() * factor).to(g.dtype))
    return norm.float()
