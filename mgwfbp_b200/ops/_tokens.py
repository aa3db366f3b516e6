# -*- coding: utf-8 -*-
"""What the operators on token lists share: the types, the bound native module, and the status words in which a kernel
records a token outside the vocabulary."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib, counters

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_OPS = {1: 'embedding', 2: 'embedding gradient', 3: 'token log probabilities'}
_FUNCTIONS = ('mgw_last_error', 'mgw_embedding_order_bytes', 'mgw_embedding_fwd', 'mgw_embedding_grad_bytes', 'mgw_embedding_grad', 'mgw_logprob_fwd',
              'mgw_logprob_bwd', 'mgw_cross_entropy_fwd', 'mgw_grad_clip_bytes', 'mgw_grad_clip')


class TokenIndexError(IndexError):
    """A kernel met a token outside the vocabulary."""


_native = None


def native():
    """The module that allocates, launches and records gradients for CUDA tensors (``csrc/torch_binding.cpp``)."""
    global _native
    if _native is None:
        lib, module = _lib.load(allow_build=False), _lib.load_binding(allow_build=False)
        module.bind({name: C.cast(getattr(lib, name), C.c_void_p).value for name in _FUNCTIONS}, status_words(), _lib.NativeLibraryError)
        counters.attach(module.launch_counts)
        _native = module
    return _native


_words = None


def status_words() -> int:
    """Address of the process's status words: pinned host memory that every device can write."""
    global _words
    if _words is None:
        p = C.POINTER(C.c_int)()
        _lib.check(_lib.load(allow_build=False).mgw_token_status(C.byref(p)), 'token status')
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
