"""Log probabilities of given tokens, with entropy and the top alternatives, as native kernels.

What a language model answers with, and what policy-gradient training differentiates:
``token_logprobs(logits, targets, top_k)`` reads the logits once and gives, per row, the target's log
probability, the distribution's entropy and the ``top_k`` likeliest tokens with theirs; the backward reads
the logits again and writes their gradient.  (``cross_entropy`` is the pretraining loss: the mean over
rows of ``-logp`` alone, bf16, aligned vocabularies.)  CUDA only, like every op here.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib
from .flash_born import _DTYPE_CODE, _stream_handle

__all__ = ["TokenLogprobs", "token_logprobs"]


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor  # (N,) fp32
    entropy: torch.Tensor  # (N,) fp32, in nats
    top_logp: torch.Tensor  # (N, top_k) fp32, falling
    top_index: torch.Tensor  # (N, top_k) int64


def _args(logits: torch.Tensor, targets: torch.Tensor, top_k: int) -> _lib.FbLogprobArgs:
    a = _lib.FbLogprobArgs()
    a.rows, a.vocab, a.ld = logits.shape[0], logits.shape[1], max(logits.stride(0), logits.shape[1])
    a.dtype, a.top_k = _DTYPE_CODE[logits.dtype], top_k
    a.logits, a.targets = logits.data_ptr(), targets.data_ptr()
    return a


def _forward(logits: torch.Tensor, targets: torch.Tensor, top_k: int) -> tuple[torch.Tensor, ...]:
    n, device = logits.shape[0], logits.device
    logp, entropy = torch.empty((2, n), dtype=torch.float32, device=device).unbind(0)
    stats = torch.empty((n, 2), dtype=torch.float32, device=device)
    top_logp = torch.empty((n, top_k), dtype=torch.float32, device=device)
    top_index = torch.empty((n, top_k), dtype=torch.int64, device=device)
    a = _args(logits, targets, top_k)
    a.logp, a.entropy, a.stats = logp.data_ptr(), entropy.data_ptr(), stats.data_ptr()
    a.top_logp, a.top_index = top_logp.data_ptr(), top_index.data_ptr()
    with torch.cuda.device(device):
        _lib.check(_lib.load().fb_logprob_fwd(ctypes.byref(a), _stream_handle(device)), "token log probabilities")
    return logp, entropy, stats, top_logp, top_index


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, targets: torch.Tensor, top_k: int):
        logp, entropy, stats, top_logp, top_index = _forward(logits, targets, top_k)
        ctx.save_for_backward(logits, targets, entropy, stats, top_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    def backward(ctx, g_logp: Optional[torch.Tensor], g_entropy: Optional[torch.Tensor],
                 g_top: Optional[torch.Tensor], _g_index):
        logits, targets, entropy, stats, top_index = ctx.saved_tensors
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        top_k = top_index.shape[1]
        a = _args(logits, targets, top_k)
        a.entropy, a.stats, a.top_index = entropy.data_ptr(), stats.data_ptr(), top_index.data_ptr()
        given = [g if g is None else g.to(torch.float32).contiguous() for g in (g_logp, g_entropy, g_top)]
        a.g_logp, a.g_entropy, a.g_top = (None if g is None else g.data_ptr() for g in given)
        a.grad, a.grad_ld = grad.data_ptr(), max(grad.stride(0), grad.shape[1])
        with torch.cuda.device(logits.device):
            _lib.check(_lib.load().fb_logprob_bwd(ctypes.byref(a), _stream_handle(logits.device)),
                       "token log probabilities backward")
        return grad, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Per row of ``logits (N, V)``: log probability of ``targets (N,)``, entropy, ``top_k`` alternatives.

    logits are float32 / float16 / bfloat16, any V and row stride (a column stride other than 1 is copied);
    targets any integer type.  All arithmetic is fp32 and all results are fp32.  The alternatives are the
    ``top_k`` (at most 64, and V) largest logits in falling order, equal ones by lowest index, a NaN above
    everything; ``-inf`` columns have no probability.  A target outside ``[0, V)`` gives a NaN logp, and a row
    of nothing but ``-inf``, or with a NaN or ``+inf``, is NaN.  ``logp``, ``entropy`` and ``top_logp`` are
    differentiable in the logits (the gradient has their dtype; a row whose incoming gradients are all 0 gets 0,
    whatever it holds).
    """
    if not (logits.is_cuda and targets.is_cuda):
        raise RuntimeError("token_logprobs (B200): CUDA tensors required; there is no CPU path")
    if logits.dim() != 2 or logits.shape[1] < 1 or logits.dtype not in _DTYPE_CODE:
        raise ValueError(f"token_logprobs takes (N, V) float32 / float16 / bfloat16 logits; got {tuple(logits.shape)} "
                         f"{logits.dtype}")
    N, V = logits.shape
    if targets.shape != (N,) or targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise ValueError(f"targets must be ({N},) integers; got {tuple(targets.shape)} {targets.dtype}")
    if not 0 <= top_k <= min(V, _lib.FB_MAX_TOP_K):
        raise ValueError(f"top_k must be in [0, {min(V, _lib.FB_MAX_TOP_K)}]; got {top_k}")
    if targets.device != logits.device:
        raise RuntimeError(f"token_logprobs: targets must be on {logits.device}; got {targets.device}")
    # rows closer than V elements (an expanded tensor's) are copied as well: the kernels need ld >= V
    x = logits if (V == 1 or logits.stride(1) == 1) and (N <= 1 or logits.stride(0) >= V) else logits.contiguous()
    t = targets.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(x, t, int(top_k)))
    logp, entropy, _, top_logp, top_index = _forward(x, t, int(top_k))
    return TokenLogprobs(logp, entropy, top_logp, top_index)
