"""Scores of given tokens: log probability, entropy and the most probable alternatives of every row of logits, and the gradient of the
first two (csrc/logprobs.cuh).  The reference's generation loop stops at the arg-max of the logits (generate.py:283, :305 of
Gu-J/TernaInfer); a program that scores texts, reports log probabilities or trains on them starts here."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .lib import load_library
from .linear import _on, _stream

MAX_TOP = 32
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                    # fp32 [...], of the targets
    entropy: torch.Tensor                    # fp32 [...]
    top_logprob: Optional[torch.Tensor]      # fp32 [..., top]
    top_token: Optional[torch.Tensor]        # int64 [..., top]


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """Logits as rows [N, V] with contiguous elements, any distance apart."""
    x = logits.reshape(-1, logits.shape[-1])
    return x if x.shape[0] <= 1 and x.stride(1) == 1 or (x.stride(1) == 1 and x.stride(0) >= x.shape[1]) else x.contiguous()


def _forward(logits, targets, top):
    x = _rows(logits)
    N, V = x.shape
    t = targets.reshape(-1).contiguous()
    stats = torch.empty((3, N), dtype=torch.float32, device=x.device)
    top_logprob = torch.empty((N, top), dtype=torch.float32, device=x.device) if top else None
    top_token = torch.empty((N, top), dtype=torch.int64, device=x.device) if top else None
    if N:
        with _on(x):
            status = load_library().ternaspmm_token_logprobs(
                x.data_ptr(), max(x.stride(0), V), _TYPES[x.dtype], t.data_ptr(), N, V, top, stats[0].data_ptr(), stats[1].data_ptr(),
                stats[2].data_ptr(), None if not top else top_logprob.data_ptr(), None if not top else top_token.data_ptr(), _stream())
        if status:
            raise RuntimeError(f"ternaspmm_token_logprobs: status {status}")
    return x, t, stats, top_logprob, top_token


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top):
        ctx.set_materialize_grads(False)
        x, t, stats, top_logprob, top_token = _forward(logits, targets, top)
        logprob, entropy = stats[0].clone(), stats[1].clone()
        ctx.save_for_backward(logits, t, stats)
        if top:
            ctx.mark_non_differentiable(top_logprob, top_token)
        return logprob, entropy, top_logprob, top_token

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, *_):
        if g_logprob is None and g_entropy is None:
            return None, None, None
        logits, t, stats = ctx.saved_tensors
        x = _rows(logits)
        N, V = x.shape
        grad = torch.empty((N, V), dtype=x.dtype, device=x.device)
        g_logprob, g_entropy = (None if g is None else g.contiguous() for g in (g_logprob, g_entropy))
        if N:
            with _on(x):
                status = load_library().ternaspmm_token_logprobs_grad(
                    x.data_ptr(), max(x.stride(0), V), _TYPES[x.dtype], t.data_ptr(), N, V, stats[2].data_ptr(), stats[1].data_ptr(),
                    None if g_logprob is None else g_logprob.data_ptr(), None if g_entropy is None else g_entropy.data_ptr(), grad.data_ptr(), _stream())
            if status:
                raise RuntimeError(f"ternaspmm_token_logprobs_grad: status {status}")
        return grad.reshape(logits.shape), None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits bf16, fp16 or fp32 [..., V], targets int64 [...]: log softmax at the target (0 for a negative target, which stands for no
    token), entropy in nats, and with ``top`` (up to 32) the log probabilities and ids of the most probable tokens, the lowest id first among equal
    logits.  Logits of -inf (banned tokens) have probability 0; a row without a finite logit gives NaN.  One pass over the logits; rows may
    be any distance apart.  Differentiable in the logits through ``logprob`` and ``entropy``.  A target of V or above gives NaN and status 1 of
    the library."""
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs needs CUDA tensors: the B200 library has no CPU path")
    if logits.dtype not in _TYPES or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits are bf16, fp16 or fp32 [..., V], not {logits.dtype} {list(logits.shape)}")
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:-1] or targets.device != logits.device:
        raise ValueError(f"targets are int64 {list(logits.shape[:-1])} on {logits.device}, not {targets.dtype} {list(targets.shape)} on {targets.device}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"top is at most {MAX_TOP} and the vocabulary {logits.shape[-1]}, not {top}")
    if logits.requires_grad and torch.is_grad_enabled():
        logprob, entropy, top_logprob, top_token = _TokenLogprobs.apply(logits, targets, top)
    else:
        _, _, stats, top_logprob, top_token = _forward(logits, targets, top)
        logprob, entropy = stats[0], stats[1]
    shape = logits.shape[:-1]
    return TokenLogprobs(logprob.reshape(shape), entropy.reshape(shape), None if not top else top_logprob.reshape(*shape, top),
                         None if not top else top_token.reshape(*shape, top))
