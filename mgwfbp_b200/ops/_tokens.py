# -*- coding: utf-8 -*-
"""What the operators on token lists share: type codes, the launch's device and stream, and the status words in which a
kernel records a token outside the vocabulary."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_OPS = {1: 'embedding', 2: 'embedding gradient', 3: 'token log probabilities'}
_same_device = contextlib.nullcontext()


class TokenIndexError(IndexError):
    """A kernel met a token outside the vocabulary."""


def device_guard(t: torch.Tensor):
    """Context in which ``t``'s device is the current one (nothing to do when it already is)."""
    return _same_device if t.get_device() == _current_device() else torch.cuda.device(t.device)


def stream_of(t: torch.Tensor) -> int:
    return _raw_stream(t.get_device())


# called with CUDA tensors only, so CUDA is up: no need for the lazy start of torch.cuda.current_device, and the stream's
# handle alone costs 0.1 us where a Stream object costs 2.2 us
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def once_differentiable(backward):
    """As ``torch.autograd.function.once_differentiable``, without its cost where no second derivative can be asked for."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


_words = None


def status_words() -> int:
    """Address of the process's status words: pinned host memory that every device can write."""
    global _words
    if _words is None:
        lib = _lib.load(allow_build=False)
        p = C.POINTER(C.c_int)()
        lib.mgw_token_status.argtypes = [C.POINTER(C.POINTER(C.c_int))]
        _lib.check(lib.mgw_token_status(C.byref(p)), 'token status')
        _words = (C.cast(p, C.c_void_p).value, p)
    return _words[0]


def check_status_nosync() -> None:
    """Raise :class:`TokenIndexError` if a launch that has already finished met a token outside the vocabulary."""
    if _words is None:
        return
    w = _words[1]
    if w[0] != 0:
        op, position, token = w[1], w[2], w[3]
        for i in range(8):
            w[i] = 0
        raise TokenIndexError('%s: token %d at position %d is outside the vocabulary' % (_OPS.get(op, '?'), token, position))


def check_status() -> None:
    """As :func:`check_status_nosync`, after waiting for every launch issued so far on the current device."""
    if _words is not None:
        torch.cuda.synchronize()
    check_status_nosync()


def check_tokens(tokens: torch.Tensor, name: str = 'tokens') -> None:
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError('%s must be int32 or int64, got %s' % (name, tokens.dtype))
