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

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib, counters
from ._tokens import (DTYPE_CODES, TokenIndexError, check_status, check_status_nosync, check_tokens, device_guard,  # noqa: F401
                      once_differentiable, status_words, stream_of)

MAX_TOP = 32
_ready = None


def _lib_ready():
    global _ready
    if _ready is None:
        lib = _lib.load(allow_build=False)
        p, n, i = C.c_void_p, C.c_longlong, C.c_int
        lib.mgw_logprob_fwd.argtypes = [p, n, n, i, i, p, i, n, p, p, p, i, p, p, p, p]
        lib.mgw_logprob_bwd.argtypes = [p, n, n, i, i, p, i, n, p, p, p, p, p, p, i, C.c_float, p, n, p]
        lib.mgw_cross_entropy_fwd.argtypes = [p, n, n, i, i, p, i, n, i, C.c_float, p, p, p, p, n, p, p, p]
        _ready = lib
    return _ready


class TokenLogProbs(NamedTuple):
    """Per row: log probability of the given token, entropy (natural logarithm), log probabilities and indices of the
    likeliest tokens (``[..., top]``, largest first, equal values by the lower index; ``None`` when ``top`` is 0)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


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
        if logits.dtype not in DTYPE_CODES:
            raise TypeError('logits must be float32, float16 or bfloat16, got %s' % logits.dtype)
        if tokens.numel() > 0x7fffffff or logits.shape[-1] > 1 << 30:
            raise ValueError('more than 2^31 - 1 rows or 2^30 columns')
    elif not logits.is_floating_point():
        raise TypeError('logits must be floating point, got %s' % logits.dtype)


def _rows(logits: torch.Tensor):
    """The logits as ``[rows, vocabulary]`` with contiguous rows, and the distance between rows."""
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    n, v = z.shape
    ld, step = z.stride()
    if step != 1 and v > 1 or n > 1 and ld < v:
        z, ld = z.contiguous(), v
    return z, (ld if n > 1 else v)


def _grad_like(z: torch.Tensor, ld: int) -> torch.Tensor:
    """Gradient matrix for ``z``.  Rows keep the distance of a padded output layer (up to an eighth wider than the
    vocabulary), so that rows of logits and gradient start at the same place of a 16-byte block."""
    n, v = z.shape
    if v < ld <= v + v // 8:
        return torch.empty(n, ld, dtype=z.dtype, device=z.device)[:, :v]
    return torch.empty(n, v, dtype=z.dtype, device=z.device)


def _forward_cuda(logits, tokens, ignore, top, keep_stats):
    """Log probability, entropy, alternatives, and the rows' statistics for the backward pass."""
    shape, n, v, device = tokens.shape, tokens.numel(), logits.shape[-1], logits.device
    with device_guard(logits):
        z, ld = _rows(logits)
        tokens = tokens.contiguous()
        logprob = torch.empty(shape, dtype=torch.float32, device=device)
        h = torch.empty(shape, dtype=torch.float32, device=device)
        stats = torch.empty(n, 2, dtype=torch.float32, device=device) if keep_stats else None
        tlp = torch.empty(*shape, top, dtype=torch.float32, device=device) if top else None
        tt = torch.empty(*shape, top, dtype=torch.int64, device=device) if top else None
        if n:
            _lib.check(_lib_ready().mgw_logprob_fwd(z.data_ptr(), ld, n, v, DTYPE_CODES[z.dtype], tokens.data_ptr(),
                                                    tokens.dtype == torch.int64, ignore, logprob.data_ptr(), h.data_ptr(), _ptr(stats),
                                                    top, _ptr(tlp), _ptr(tt), status_words(), stream_of(z)), 'logprob_fwd')
            counters.bump('logprob_fwd')
    return logprob, h, tlp, tt, stats


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, ignore, top):
        logprob, h, tlp, tt, stats = _forward_cuda(logits, tokens, ignore, top, True)
        ctx.save_for_backward(logits, tokens, stats, h)
        ctx.ignore = ignore
        if top:
            ctx.mark_non_differentiable(tlp, tt)
        ctx.set_materialize_grads(False)
        return logprob, h, tlp, tt

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, _1, _2):
        logits, tokens, stats, h = ctx.saved_tensors
        if g_logprob is None and g_entropy is None:
            return None, None, None, None
        with device_guard(logits):
            z, ld = _rows(logits)
            dz = _grad_like(z, ld)
            n, v = z.shape
            g1 = None if g_logprob is None else g_logprob.contiguous()
            g2 = None if g_entropy is None else g_entropy.contiguous()
            tokens = tokens.contiguous()
            if n:
                _lib.check(_lib_ready().mgw_logprob_bwd(z.data_ptr(), ld, n, v, DTYPE_CODES[z.dtype], tokens.data_ptr(),
                                                        tokens.dtype == torch.int64, ctx.ignore, stats.data_ptr(), h.data_ptr(), _ptr(g1),
                                                        _ptr(g2), None, None, 0, 0.0, dz.data_ptr(), dz.stride(0) if n > 1 else v,
                                                        stream_of(z)), 'logprob_bwd')
                counters.bump('logprob_bwd')
            return dz if logits.dim() == 2 else dz.view(logits.shape), None, None, None


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
    _check(logits, tokens, top)
    if not logits.is_cuda:
        return TokenLogProbs(*_reference(logits, tokens, int(ignore_index), top))
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, int(ignore_index), top))
    return TokenLogProbs(*_forward_cuda(logits, tokens, int(ignore_index), top, False)[:4])


class _CrossEntropy(torch.autograd.Function):
    """The gradient of the logits is written by the forward launch, for the gradient that the loss is expected to get: the
    rows have just been read and come from L2.  The first backward pass hands it out (its launch looks at the actual
    gradient and recomputes the rows only where that differs); any further one computes its own."""

    @staticmethod
    def forward(ctx, logits, tokens, ignore, mean, expected):
        n, v = tokens.numel(), logits.shape[-1]
        with device_guard(logits):
            z, ld = _rows(logits)
            tokens = tokens.contiguous()
            train = ctx.needs_input_grad[0]
            loss = torch.empty((), dtype=torch.float32, device=z.device)
            # two words (the number of rows in the mean, a counter), {m, log2 s} of every row, log probability of every row
            work = torch.empty(2 + 3 * n, dtype=torch.float32, device=z.device)
            at = work.data_ptr()
            dz = _grad_like(z, ld) if train else None
            _lib.check(_lib_ready().mgw_cross_entropy_fwd(z.data_ptr(), ld, n, v, DTYPE_CODES[z.dtype], tokens.data_ptr(),
                                                          tokens.dtype == torch.int64, ignore, mean, expected, at + 8 + 8 * n,
                                                          at + 8 if train else None, loss.data_ptr(), _ptr(dz),
                                                          dz.stride(0) if train and n > 1 else v, at, status_words(), stream_of(z)),
                       'cross_entropy_fwd')
            counters.bump('cross_entropy_fwd')
        if train:
            ctx.save_for_backward(logits, tokens, work)
            ctx.ignore, ctx.expected, ctx.dz = ignore, expected, dz
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, tokens, work = ctx.saved_tensors
        dz, ctx.dz = ctx.dz, None
        written = dz is not None
        n, v = tokens.numel(), logits.shape[-1]
        with device_guard(logits):
            z, ld = _rows(logits)
            if not written:
                dz = _grad_like(z, ld)
            if n:
                _lib.check(_lib_ready().mgw_logprob_bwd(z.data_ptr(), ld, n, v, DTYPE_CODES[z.dtype], tokens.data_ptr(),
                                                        tokens.dtype == torch.int64, ctx.ignore, work.data_ptr() + 8, None, None, None,
                                                        g.data_ptr(), work.data_ptr(), written, ctx.expected, dz.data_ptr(),
                                                        dz.stride(0) if n > 1 else v, stream_of(z)), 'cross_entropy_bwd')
                counters.bump('cross_entropy_bwd')
            return dz if logits.dim() == 2 else dz.view(logits.shape), None, None, None, None


def cross_entropy(logits: torch.Tensor, tokens: torch.Tensor, ignore_index: int = -100, reduction: str = 'mean',
                  expected_grad: float = 1.0) -> torch.Tensor:
    """Cross entropy of ``tokens`` under ``softmax(logits)`` in fp32: mean over the rows that are not padding (NaN when
    there is none, as ``torch.nn.functional.cross_entropy``), their ``'sum'``, or ``'none'``.

    The gradient of the logits is computed along with the loss, for the gradient that the loss itself is expected to get
    in backward: ``expected_grad`` is 1, or the loss scale of half-precision training.  Any other gradient is right too,
    at the cost of another pass over the logits."""
    if reduction not in ('mean', 'sum', 'none'):
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got %r" % (reduction,))
    _check(logits, tokens)
    if reduction == 'none':
        return -token_log_probs(logits, tokens, 0, ignore_index).logprob
    if not logits.is_cuda:
        logprob = _reference(logits, tokens, int(ignore_index), 0)[0]
        total = -logprob.sum()
        return total / (tokens != ignore_index).sum() if reduction == 'mean' else total
    expected = float(expected_grad)
    if not math.isfinite(expected):
        raise ValueError('expected_grad must be finite, got %r' % (expected_grad,))
    return _CrossEntropy.apply(logits, tokens, int(ignore_index), reduction == 'mean', expected)


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
        if logits.is_cuda and logits.dtype not in DTYPE_CODES:
            return super().forward(logits, tokens)
        return cross_entropy(logits, tokens, self.ignore_index, self.reduction, self.expected_grad)
