"""Log-probabilities of given tokens, the entropy of their distributions and the
best alternatives, and the mean loss: forward and backward in HIP kernels.

The reference's shell forms the mean cross entropy from an FP32 copy of the
logits (implementation/bdm/model.py:207-216); here the logits are read as they
are, once forward and once backward.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import ops
from .model import _differentiable, _dual, _torch_gradients

Tensor = torch.Tensor


class TokenLogProbs(NamedTuple):
    """Of each row of logits, in the tokens' shape."""
    log_probs: Tensor              # FP32: of the given token
    entropy: Tensor                # FP32: of the row's distribution
    top_log_probs: Tensor | None   # FP32 [..., alternatives], best first
    top_tokens: Tensor | None      # int64 [..., alternatives]


def _log_probs_ops(logits, tokens, top_tokens, ignore_index):
    """The results in torch ops of the logits: (log_probs, entropy, top_log_probs or None)."""
    x = logits.float()
    high = x.detach().amax(-1, keepdim=True)
    high = torch.where(high == -torch.inf, 0.0, high)
    d = x - high
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    empty = total == 0
    total = torch.where(empty, 1.0, total)
    offset = high + total.log()

    def at(index):
        return torch.where(empty, -torch.inf, x.gather(-1, index) - offset)

    ignored, outside = tokens == ignore_index, (tokens < 0) | (tokens >= x.shape[-1])
    given = at(tokens.masked_fill(ignored | outside, 0).unsqueeze(-1)).squeeze(-1)
    # an out-of-range token's NaN reaches its row's gradient, as the kernel's does
    given = torch.where(ignored, 0.0, given * torch.where(outside & ~ignored, torch.nan, 1.0))
    moment = (e * torch.where(e == 0, 0.0, d)).sum(-1)
    entropy = total.squeeze(-1).log() - moment / total.squeeze(-1)
    return given, entropy, None if top_tokens is None else at(top_tokens)


def _primal(dual):
    return forward_ad.unpack_dual(dual).primal.detach()


def _counted_rows(logits, tokens, ignore_index):
    """The logits with zeros in the ignored tokens' rows, whose NaN would reach their gradient."""
    return logits.masked_fill((tokens == ignore_index).unsqueeze(-1), 0)


def _loss_ops(logits, tokens, ignore_index):
    counted = tokens != ignore_index
    logits = _counted_rows(logits, tokens, ignore_index)
    return -_log_probs_ops(logits, tokens, None, ignore_index)[0].sum() / counted.sum()


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, alternatives, ignore_index):
        tokens = tokens.contiguous()
        log_probs, entropy, top, top_tokens, stats = ops.token_statistics(
            logits, tokens, alternatives=alternatives, ignore_index=ignore_index, stats=True)
        ctx.save_for_backward(logits, tokens, stats, entropy, top_tokens)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if top is None:
            return log_probs, entropy
        ctx.mark_non_differentiable(top_tokens)
        return log_probs, entropy, top, top_tokens

    @staticmethod
    def backward(ctx, *grads):
        logits, tokens, stats, entropy, top_tokens = ctx.saved_tensors
        grads = [*grads[:3], None][:3]
        present = [g for g in grads if g is not None]
        if not present:
            return None, None, None, None
        if _differentiable(present):
            def form(x):
                if grads[1] is None and grads[2] is None:
                    x = _counted_rows(x, tokens, ctx.ignore_index)
                results = _log_probs_ops(x, tokens, top_tokens, ctx.ignore_index)
                return [r for r, g in zip(results, grads) if g is not None]
            return (*_torch_gradients(form, (logits,), present), None, None, None)
        grad = ops.token_gradients(logits, tokens, stats, entropy, top_tokens, *grads, None, None, ctx.ignore_index)
        return grad, None, None, None


class _TokenLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, ignore_index):
        tokens = tokens.contiguous()
        log_probs, _, _, _, stats = ops.token_statistics(logits, tokens, ignore_index=ignore_index, entropy=False,
                                                         stats=True)
        loss, inverse_count = ops.token_loss_mean(log_probs, tokens, ignore_index=ignore_index)
        ctx.save_for_backward(logits, tokens, stats, inverse_count)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        logits, tokens, stats, inverse_count = ctx.saved_tensors
        if _differentiable([grad_loss]):
            form = functools.partial(_loss_ops, tokens=tokens, ignore_index=ctx.ignore_index)
            return (*_torch_gradients(form, (logits,), grad_loss), None, None)
        grad = ops.token_gradients(logits, tokens, stats, None, None, None, None, None, grad_loss, inverse_count,
                                   ctx.ignore_index)
        return grad, None, None


def token_log_probs(logits: Tensor, tokens: Tensor, *, alternatives: int = 0,
                    ignore_index: int = -100) -> TokenLogProbs:
    """Log-probabilities of given tokens under the logits' distributions, the
    entropies of these, and their ``alternatives`` best tokens with theirs.

    logits [..., vocab] BF16 or FP32 on a ROCm device, rows evenly spaced or not,
    vocabularies to 2^24 and fewer than 2^24 rows; tokens int64 [...].  All
    results are FP32 (statistics too), and all three take gradients; tangents of
    forward-mode differentiation go through torch ops.  Alternatives come best
    first, equal logits by the lower token; at most 32.

    A logit of -inf has the probability 0.  A row of nothing else has no
    distribution: log-probabilities -inf, entropy 0, gradient 0.  A NaN or +inf
    makes its row's results NaN (and a NaN comes first of the alternatives).  A
    token equal to ``ignore_index`` has the log-probability 0, which passes no
    gradient, whatever its row holds; one outside the vocabulary has the log-probability NaN, and its
    row's gradient is NaN where that of the log-probability arrives."""
    if _dual(logits):
        # the call's checks and the alternatives by the kernel, the results and their tangents in torch ops
        top_tokens = ops.token_statistics(_primal(logits), tokens, alternatives=alternatives, ignore_index=ignore_index)[3]
        return TokenLogProbs(*_log_probs_ops(logits, tokens, top_tokens, ignore_index), top_tokens)
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _TokenLogProbs.apply(logits, tokens, int(alternatives), int(ignore_index))
        return TokenLogProbs(*(*out, None, None)[:4])
    return TokenLogProbs(*ops.token_statistics(logits, tokens, alternatives=alternatives,
                                               ignore_index=ignore_index)[:4])


def token_loss(logits: Tensor, tokens: Tensor, *, ignore_index: int = -100) -> Tensor:
    """The mean of -``token_log_probs(logits, tokens).log_probs`` over the tokens
    that are not ``ignore_index``, an FP32 scalar (NaN where there is none): the
    cross entropy of the shell's training step.  The mean is formed in FP64 and in
    a fixed order."""
    if _dual(logits):
        ops.token_statistics(_primal(logits), tokens, ignore_index=ignore_index, entropy=False)  # the call's checks
        return _loss_ops(logits, tokens, ignore_index)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLoss.apply(logits, tokens, int(ignore_index))
    log_probs = ops.token_statistics(logits, tokens, ignore_index=ignore_index, entropy=False)[0]
    return ops.token_loss_mean(log_probs, tokens, ignore_index=ignore_index)[0]
