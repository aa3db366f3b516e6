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

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ._tokens import DTYPES, TokenIndexError, check_status, check_status_nosync, check_tokens, native  # noqa: F401


def _check(tokens: torch.Tensor, weight: torch.Tensor) -> None:
    check_tokens(tokens)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError('weight must be a non-empty [vocabulary, width] matrix, got shape %s' % (tuple(weight.shape),))
    if tokens.device != weight.device:
        raise ValueError('tokens are on %s, weight is on %s' % (tokens.device, weight.device))
    if weight.is_cuda:
        if weight.dtype not in DTYPES:
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
    if grad.dtype not in DTYPES:
        raise TypeError('grad must be float32, float16 or bfloat16, got %s' % grad.dtype)
    _check_sizes(n, num_embeddings, dim)
    return native().embedding_grad(grad, tokens, num_embeddings, scale, padding)


class _EmbeddingCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.padding, ctx.vocab = scale, padding, weight.shape[0]
        out = F.embedding(tokens, weight)
        return out if scale == 1.0 else (out.double() * scale).to(out.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return None, embedding_grad(dy, tokens, ctx.vocab, ctx.scale, ctx.padding if ctx.padding >= 0 else None), None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, shape ``tokens.shape + [width]``, in ``weight``'s type (products in fp32, rounded once;
    ``scale == 1`` copies the rows).  ``tokens``: int32 or int64 of any shape; ``weight``: ``[vocabulary, width]``, rows may
    lie further apart than their width.  ``padding_idx`` only matters to the gradient: that row gets none."""
    padding = -1 if padding_idx is None or weight.dim() != 2 else _padding(padding_idx, weight.shape[0])
    if weight.is_cuda:
        out = native().embedding(tokens, weight, scale, padding)
        if out is not None:                                    # else the check below says why
            return out
    _check(tokens, weight)
    return _EmbeddingCPU.apply(tokens, weight, float(scale), padding)


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
        if self.weight.is_cuda and self.weight.dtype not in DTYPES:
            return super().forward(tokens) * self.scale
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + ('' if self.scale == 1.0 else ', scale=%g' % self.scale)
