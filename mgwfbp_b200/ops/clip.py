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

import ctypes as C
import math
from array import array
from typing import Iterable, List, Union

import torch

from . import _lib, counters
from ._tokens import DTYPE_CODES, device_guard, stream_of

_NORMS = {2.0: 0, 1.0: 1, math.inf: 2}
_ready = None


def _lib_ready():
    global _ready
    if _ready is None:
        lib = _lib.load(allow_build=False)
        lib.mgw_grad_clip_bytes.restype = C.c_size_t
        lib.mgw_grad_clip_bytes.argtypes = [C.c_int]
        lib.mgw_grad_clip.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_double, C.c_double, C.c_int, C.c_void_p,
                                      C.c_size_t, C.c_void_p, C.c_void_p]
        _ready = lib
    return _ready


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
    return bool(grads) and all(g.is_cuda and g.layout == torch.strided and g.dtype in DTYPE_CODES and g.device == grads[0].device
                               and _dense(g) for g in grads)


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
        if g.is_cuda and g.dtype not in DTYPE_CODES:
            raise TypeError('gradients must be float32, float16 or bfloat16, got %s' % g.dtype)
        if not _dense(g):
            raise ValueError('a gradient of shape %s has strides %s: its elements do not fill one stretch of memory'
                             % (tuple(g.shape), g.stride()))


_tensor = torch.Tensor


def _codes(grads: List[torch.Tensor]):
    """Type codes of the gradients when all of them are contiguous, on one GPU and of a type the kernels know, else None.
    (Models have hundreds of gradients: five C calls for each, no Python frame.)"""
    try:
        codes = bytes([DTYPE_CODES[g.dtype] for g in grads])
        if grads[0].is_cuda and len(set(map(_tensor.get_device, grads))) == 1 and all(map(_tensor.is_contiguous, grads)):
            return codes
    except (KeyError, RuntimeError):                      # another type; sparse
        pass
    return None


def _launch(grads: List[torch.Tensor], codes: bytes, code: int, scale: float, max_norm: float, clip: bool) -> torch.Tensor:
    lib, n, first = _lib_ready(), len(grads), grads[0]
    ptrs, numels = array('Q', map(_tensor.data_ptr, grads)), array('q', map(_tensor.numel, grads))
    with device_guard(first):
        out = torch.empty((), dtype=torch.float32, device=first.device)
        need = lib.mgw_grad_clip_bytes(n)
        work = torch.empty(need, dtype=torch.uint8, device=first.device)
        rc = lib.mgw_grad_clip(ptrs.buffer_info()[0], numels.buffer_info()[0], codes, n, code, scale, max_norm, clip, work.data_ptr(), need,
                               out.data_ptr(), stream_of(first))
        if rc == 2:
            raise ValueError('grad_clip: %s' % lib.mgw_last_error().decode(errors='replace'))
        _lib.check(rc, 'grad_clip')
        if clip:
            for g in [g for g in grads if g.requires_grad]:        # part of a graph (create_graph): it has changed in place
                torch.autograd.graph.increment_version(g)
        counters.bump('grad_norm', (n + 1023) // 1024)
        counters.bump('grad_scale' if clip else 'grad_norm_finish', (n + 1023) // 1024 if clip else 1)
    return out


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
    codes = _codes(grads)
    if codes is None:
        _check(grads)
        if not grads[0].is_cuda:
            return _reference_norm(grads, float(norm_type), scale).float()
        codes = bytes(DTYPE_CODES[g.dtype] for g in grads)
    return _launch(grads, codes, code, scale, 0.0, False)


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
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros(())
    codes = _codes(grads)
    if codes is None:
        _check(grads)
        if grads[0].is_cuda:
            codes = bytes(DTYPE_CODES[g.dtype] for g in grads)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type, scale)
        if not math.isfinite(float(norm)):
            raise RuntimeError('The total norm of order %s for the gradients is non-finite, so they cannot be clipped' % (norm_type,))
    if codes is not None:
        return _launch(grads, codes, code, scale, max_norm, True)
    norm = _reference_norm(grads, float(norm_type), scale)
    factor = float(scale * torch.clamp(max_norm / (norm + 1e-6), max=1.0))
    for g in {(g.data_ptr(), g.numel()): g for g in grads}.values():
        g.detach().copy_((g.detach().double() * factor).to(g.dtype))
    return norm.float()
