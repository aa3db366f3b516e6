# -*- coding: utf-8 -*-
"""Embedding lookup with scaling, and the gradient of the table by sorted tokens (``csrc/embedding.cu``).

``embedding(tokens, weight, scale)`` returns ``scale * weight[tokens]``; its gradient is the dense sum over the rows'
gradients for each token, formed in fp32 in the order of the positions (the same result on every run) and rounded once.
``FusedEmbedding`` is a drop-in subclass of ``torch.nn.Embedding`` (same parameter and ``state_dict`` key) that runs it;
the PTB model's ``word_embeddings`` (reference ``models/lstm.py:13``) is one when the model is built with fused modules.

On CUDA the table may be fp32, fp16 or bf16.  A token outside the vocabulary gives a row of NaN, takes no part in
the gradient, and is reported by :func:`check_status` (``engine.TrainStep`` looks every step).  On CPU tensors the same
functions run plain PyTorch operations.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib, counters
from ._tokens import (DTYPE_CODES, TokenIndexError, check_status, check_status_nosync, check_tokens, device_guard,  # noqa: F401
                      once_differentiable, status_words, stream_of)

_ready = None


def _lib_ready():
    global _ready
    if _ready is None:
        lib = _lib.load(allow_build=False)
        lib.mgw_embedding_fwd.argtypes = [C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_longlong, C.c_longlong, C.c_int, C.c_int,
                                          C.c_float, C.c_void_p, C.c_void_p, C.c_void_p]
        lib.mgw_embedding_grad_bytes.restype = C.c_size_t
        lib.mgw_embedding_grad_bytes.argtypes = [C.c_longlong, C.c_longlong, C.c_int, C.c_int]
        lib.mgw_embedding_grad.argtypes = [C.c_void_p, C.c_longlong, C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_int, C.c_int,
                                           C.c_float, C.c_longlong, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p, C.c_void_p]
        _ready = lib
    return _ready


def _check(tokens: torch.Tensor, weight: torch.Tensor) -> None:
    check_tokens(tokens)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError('weight must be a non-empty [vocabulary, width] matrix, got shape %s' % (tuple(weight.shape),))
    if tokens.device != weight.device:
        raise ValueError('tokens are on %s, weight is on %s' % (tokens.device, weight.device))
    if weight.is_cuda:
        if weight.dtype not in DTYPE_CODES:
            raise TypeError('weight must be float32, float16 or bfloat16, got %s' % weight.dtype)
        _check_sizes(tokens.numel(), *weight.shape)


def _check_sizes(n: int, vocab: int, dim: int) -> None:
    if n > 0x7fffffff or vocab > 0x7ffffffe or dim > 1 << 30:
        raise ValueError('more than 2^31 - 1 tokens, 2^31 - 2 rows or 2^30 columns')


def _padding(padding_idx: Optional[int], vocab: int) -> int:
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError('padding_idx %d is outside a vocabulary of %d' % (padding_idx, vocab))
    return padding_idx % vocab


def _forward(tokens: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    vocab, dim = weight.shape
    if not weight.is_cuda:
        out = F.embedding(tokens, weight)
        return out if scale == 1.0 else (out.double() * scale).to(out.dtype)
    if weight.stride(1) != 1 or weight.stride(0) < dim:
        weight = weight.contiguous()
    tokens = tokens.contiguous()
    with device_guard(weight):
        out = torch.empty(*tokens.shape, dim, dtype=weight.dtype, device=weight.device)
        n = tokens.numel()
        if n:
            _lib.check(_lib_ready().mgw_embedding_fwd(tokens.data_ptr(), tokens.dtype == torch.int64, n, weight.data_ptr(),
                                                      weight.stride(0), vocab, dim, DTYPE_CODES[weight.dtype], scale, out.data_ptr(),
                                                      status_words(), stream_of(weight)), 'embedding_fwd')
            counters.bump('embedding_fwd')
    return out


def embedding_grad(grad: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                   padding_idx: Optional[int] = None) -> torch.Tensor:
    """``dW [num_embeddings, width]`` (in ``grad``'s type): row ``v`` is ``scale`` times the sum of ``grad`` over the
    positions whose token is ``v``; the row of ``padding_idx`` and rows without a token are zero."""
    check_tokens(tokens)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape or grad.shape[-1] < 1:
        raise ValueError('grad must have the shape of tokens and one more dimension: %s for tokens %s'
                         % (tuple(grad.shape), tuple(tokens.shape)))
    if num_embeddings < 1:
        raise ValueError('num_embeddings must be positive, got %d' % num_embeddings)
    if grad.device != tokens.device:
        raise ValueError('tokens are on %s, grad is on %s' % (tokens.device, grad.device))
    padding, scale, dim, n = _padding(padding_idx, num_embeddings), float(scale), grad.shape[-1], tokens.numel()
    if not grad.is_cuda:
        ids, rows = tokens.reshape(-1).long(), grad.reshape(-1, dim)
        dw = torch.zeros(num_embeddings, dim, dtype=torch.float64)
        keep = ids != padding
        dw.index_add_(0, ids[keep], rows[keep].double())
        return (dw * scale).to(grad.dtype)
    if grad.dtype not in DTYPE_CODES:
        raise TypeError('grad must be float32, float16 or bfloat16, got %s' % grad.dtype)
    _check_sizes(n, num_embeddings, dim)
    return _grad_cuda(grad, tokens, num_embeddings, scale, padding)


@functools.lru_cache(maxsize=256)
def _work_bytes(n: int, vocab: int, dim: int, code: int) -> int:
    return _lib_ready().mgw_embedding_grad_bytes(n, vocab, dim, code)


def _grad_cuda(grad: torch.Tensor, tokens: torch.Tensor, vocab: int, scale: float, padding: int) -> torch.Tensor:
    n, dim = tokens.numel(), grad.shape[-1]
    rows = grad.reshape(n, dim)
    if n and (rows.stride(1) != 1 or (n > 1 and rows.stride(0) < dim)):
        rows = rows.contiguous()
    tokens = tokens.contiguous()
    code = DTYPE_CODES[grad.dtype]
    with device_guard(grad):
        dw = torch.empty(vocab, dim, dtype=grad.dtype, device=grad.device)
        need = _work_bytes(n, vocab, dim, code)
        work = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
        _lib.check(_lib_ready().mgw_embedding_grad(rows.data_ptr(), rows.stride(0) if n > 1 else dim, tokens.data_ptr(),
                                                   tokens.dtype == torch.int64, n, vocab, dim, code, scale, padding, dw.data_ptr(),
                                                   None if work is None else work.data_ptr(), need, status_words(), stream_of(grad)), 'embedding_grad')
        counters.bump('embedding_grad')
    return dw


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.padding, ctx.vocab, ctx.dtype = scale, padding, weight.shape[0], weight.dtype
        return _forward(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return None, _grad_cuda(dy, tokens, ctx.vocab, ctx.scale, ctx.padding), None, None


class _EmbeddingCPU(_Embedding):
    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return None, embedding_grad(dy, tokens, ctx.vocab, ctx.scale, ctx.padding if ctx.padding >= 0 else None), None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, shape ``tokens.shape + [width]``, in ``weight``'s type (products in fp32, rounded once;
    ``scale == 1`` copies the rows).  ``tokens``: int32 or int64 of any shape; ``weight``: ``[vocabulary, width]``, rows may
    lie further apart than their width.  ``padding_idx`` only matters to the gradient: that row gets none."""
    _check(tokens, weight)
    padding, scale = _padding(padding_idx, weight.shape[0]), float(scale)
    if torch.is_grad_enabled() and weight.requires_grad:
        return (_Embedding if weight.is_cuda else _EmbeddingCPU).apply(tokens, weight, scale, padding)
    return _forward(tokens, weight, scale)


class FusedEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter and ``state_dict`` key) whose lookup and gradient run this package's kernels, with an
    optional factor on the rows (``scale``).  A table of a type that the kernels do not have (float64) runs the parent's
    lookup.  The options ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are refused."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, scale: float = 1.0, **kwargs):
        for option in ('max_norm', 'scale_grad_by_freq', 'sparse'):
            if kwargs.get(option):
                raise ValueError('FusedEmbedding does not support %s' % option)
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, **kwargs)
        self.scale = float(scale)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        if self.weight.is_cuda and self.weight.dtype not in DTYPE_CODES:
            return super().forward(tokens) * self.scale
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + ('' if self.scale == 1.0 else ', scale=%g' % self.scale)
