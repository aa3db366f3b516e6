# -*- coding: utf-8 -*-
"""Log probabilities of given tokens with entropy and top alternatives, and cross entropy (``csrc/logprob.cu``).

``token_log_probs(logits, tokens, top)`` reads every row of logits once and returns the log probability of the row's
token, the entropy of its distribution and the ``top`` likeliest tokens; log probability and entropy are differentiable.
``cross_entropy`` is the mean (or sum) of the negative log probabilities; ``FusedCrossEntropyLoss`` is the drop-in
subclass of ``torch.nn.CrossEntropyLoss`` that the PTB model trains with (reference ``dl_trainer.py:206``).

Logits: fp32, fp16 or bf16, ``[..., vocabulary]``; rows may lie further apart than the vocabulary.  Results are fp32, the
gradient has the logits' type.  A logit of minus infinity is a token that is not allowed.  A row without any finite
largest value (nothing allowed, a NaN, plus infinity) has no distribution: its results are NaN, as ``log_softmax``'s.
Rows whose token is ``ignore_index`` are padding: results and gradient are zero, ``top_tokens`` is -1, and their
logits are not read.  Any other token outside the vocabulary gives NaN and is reported by :func:`check_status`.
On CPU tensors the same functions run plain PyTorch operations.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from ._tokens import DTYPES, TokenIndexError, check_status, check_status_nosync, check_tokens, native  # noqa: F401

MAX_TOP = 32


class TokenLogProbs(NamedTuple):
    """Per row: log probability of the given token, entropy (natural logarithm), log probabilities and indices of the
    likeliest tokens (``[..., top]``, largest first, equal values by the lower index; ``None`` when ``top`` is 0)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _check(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> None:
    check_tokens(tokens)
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape or logits.shape[-1] < 1:
        raise ValueError('logits must have the shape of tokens and a vocabulary: %s for tokens %s'
                         % (tuple(logits.shape), tuple(tokens.shape)))
    if logits.device != tokens.device:
        raise ValueError('tokens are on %s, logits are on %s' % (tokens.device, logits.device))
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError('top must be between 0 and %d for a vocabulary of %d, got %d' % (MAX_TOP, logits.shape[-1], top))
    if logits.is_cuda:
        if logits.dtype not in DTYPES:
            raise TypeError('logits must be float32, float16 or bfloat16, got %s' % logits.dtype)
        if tokens.numel() > 0x7fffffff or logits.shape[-1] > 1 << 30:
            raise ValueError('more than 2^31 - 1 rows or 2^30 columns')
    elif not logits.is_floating_point():
        raise TypeError('logits must be floating point, got %s' % logits.dtype)


def _reference(logits: torch.Tensor, tokens: torch.Tensor, ignore: int, top: int):
    """The same results with plain tensor operations (any device, differentiable)."""
    v = logits.shape[-1]
    z = logits.reshape(-1, v)
    z = z if z.dtype == torch.float64 else z.float()
    ids = tokens.reshape(-1).long()
    pad = ids == ignore
    if bool(((ids < 0) | (ids >= v)).logical_and(~pad).any()):
        raise TokenIndexError('a token is outside the vocabulary of %d' % v)
    z = z.masked_fill(pad.unsqueeze(1), 0.0)
    logp = torch.log_softmax(z, 1)
    chosen = logp.gather(1, ids.masked_fill(pad, 0).unsqueeze(1)).squeeze(1)
    p = logp.exp()
    h = -(p * logp.masked_fill(p == 0, 0.0)).sum(1)
    logprob, h = chosen.masked_fill(pad, 0.0), h.masked_fill(pad, 0.0)
    s = tokens.shape
    if not top:
        return logprob.view(s), h.view(s), None, None
    order = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :top]
    tlp = logp.detach().gather(1, order).masked_fill(pad.unsqueeze(1), 0.0)
    tt = order.masked_fill(pad.unsqueeze(1), -1)
    return logprob.view(s), h.view(s), tlp.view(*s, top), tt.view(*s, top)


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, ignore_index: int = -100) -> TokenLogProbs:
    """Log probability of ``tokens`` (int32 or int64, any shape) under ``softmax(logits)``, entropy of every row, and its
    ``top`` (0 to 32) likeliest tokens.  See the module for masks, padding and what is refused."""
    if logits.is_cuda:
        found = native().token_log_probs(logits, tokens, int(ignore_index), top)
        if found is not None:                                  # else the check below says why
            return TokenLogProbs(*found)
    _check(logits, tokens, top)
    return TokenLogProbs(*_reference(logits, tokens, int(ignore_index), top))


def cross_entropy(logits: torch.Tensor, tokens: torch.Tensor, ignore_index: int = -100, reduction: str = 'mean',
                  expected_grad: float = 1.0) -> torch.Tensor:
    """Cross entropy of ``tokens`` under ``softmax(logits)`` in fp32: mean over the rows that are not padding (NaN when
    there is none, as ``torch.nn.functional.cross_entropy``), their ``'sum'``, or ``'none'``.

    The gradient of the logits is computed along with the loss, for the gradient that the loss itself is expected to get
    in backward: ``expected_grad`` is 1, or the loss scale of half-precision training.  Any other gradient is right too,
    at the cost of another pass over the logits."""
    if reduction not in ('mean', 'sum', 'none'):
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got %r" % (reduction,))
    if reduction == 'none':
        return -token_log_probs(logits, tokens, 0, ignore_index).logprob
    expected = float(expected_grad)
    if not math.isfinite(expected):
        raise ValueError('expected_grad must be finite, got %r' % (expected_grad,))
    if logits.is_cuda:
        loss = native().cross_entropy(logits, tokens, int(ignore_index), reduction == 'mean', expected)
        if loss is not None:                                   # else the check below says why
            return loss
    _check(logits, tokens)
    logprob = _reference(logits, tokens, int(ignore_index), 0)[0]
    total = -logprob.sum()
    return total / (tokens != ignore_index).sum() if reduction == 'mean' else total


class FusedCrossEntropyLoss(nn.CrossEntropyLoss):
    """``nn.CrossEntropyLoss`` over class indices that runs this package's kernels: logits ``[rows, vocabulary]`` (or one
    row), no class weights, no label smoothing.  Logits of a type that the kernels do not have (float64) run the parent's
    loss.  ``expected_grad``: see :func:`cross_entropy`."""

    def __init__(self, ignore_index: int = -100, reduction: str = 'mean', expected_grad: float = 1.0):
        super().__init__(ignore_index=ignore_index, reduction=reduction)
        self.expected_grad = float(expected_grad)

    def forward(self, logits: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        if logits.dim() > 2:
            raise ValueError('FusedCrossEntropyLoss takes [rows, vocabulary] logits, got shape %s' % (tuple(logits.shape),))
        if logits.is_cuda and logits.dtype not in DTYPES:
            return super().forward(logits, tokens)
        return cross_entropy(logits, tokens, self.ignore_index, self.reduction, self.expected_grad)
