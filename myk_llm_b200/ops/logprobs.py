"""Log probabilities of given tokens, the entropy of their distributions and the most likely
alternatives, from logits.

``token_logprobs(logits, tokens, top=k)`` reads each row of logits once and keeps no fp32
copy of them.  Ties among the alternatives go to the lowest token id.  The log
probabilities, the entropy and the alternatives' log probabilities are differentiable with
respect to the logits (policy gradients, entropy bonuses, distillation onto the top tokens);
the backward pass reads the logits once more and writes their gradient.  On CUDA there is no
second derivative (asking for it raises).

A token equal to ``ignore_index`` gets log probability 0 and no gradient through it; one
outside the vocabulary gets NaN.  Logits of -inf (excluded tokens) have probability 0.  A row
that is -inf throughout has no distribution: log probabilities -inf, entropy 0, gradient 0.
A NaN or +inf anywhere in a row makes its numbers and its gradient NaN.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # (...) fp32
    entropy: torch.Tensor  # (...) fp32, natural units
    top_logprobs: torch.Tensor  # (..., top) fp32, largest first
    top_tokens: torch.Tensor  # (..., top) int64


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        lp, ent, stats, tl, tt = ext().logprobs_fwd(logits, tokens, top, ignore_index)
        ctx.save_for_backward(logits, tokens, stats, tt)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(tt)
        ctx.set_materialize_grads(False)
        return lp, ent, tl, tt

    @staticmethod
    def backward(ctx, g_lp, g_ent, g_top, _):
        logits, tokens, stats, tt = ctx.saved_tensors
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None, None
        return _Gradient.apply(logits, tokens, ctx.ignore_index, stats, tt, g_lp, g_ent, g_top), None, None, None


class _Gradient(torch.autograd.Function):
    """The gradient, as a function of its own so that differentiating it again is an error."""

    @staticmethod
    def forward(ctx, *args):
        return ext().logprobs_bwd(*args)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("token_logprobs has no second derivative on CUDA")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0,
                   ignore_index: int = ref.IGNORE_INDEX) -> TokenLogprobs:
    """logits (..., vocab) in bf16 or fp32, tokens (...) integer ids; ``top`` alternatives (at
    most 32).  See the module docstring."""
    vocab = logits.shape[-1]
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} must have the shape of the logits {tuple(logits.shape)} "
                         "without the vocabulary")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to min({MAX_TOP}, vocabulary); got {top}")
    if tokens.is_floating_point() or tokens.dtype == torch.bool:
        raise TypeError(f"tokens must be integers; got {tokens.dtype}")
    if not logits.is_cuda:
        return TokenLogprobs(*ref.token_logprobs_ref(logits, tokens, top, ignore_index))
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"token_logprobs needs bf16 or fp32 logits; got {logits.dtype}")
    x = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if vocab > 1 and x.stride(1) != 1:
        x = x.contiguous()
    t = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    t = t.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        lp, ent, tl, tt = _TokenLogprobs.apply(x, t, top, ignore_index)
    else:
        lp, ent, _, tl, tt = ext().logprobs_fwd(x, t, top, ignore_index)
    if tokens.dim() != 1:
        lp, ent = lp.view(tokens.shape), ent.view(tokens.shape)
        tl, tt = tl.view(*tokens.shape, top), tt.view(*tokens.shape, top)
    return TokenLogprobs(lp, ent, tl, tt)
