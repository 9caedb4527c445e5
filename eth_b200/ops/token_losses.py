"""Autograd ops over the vocabulary axis: log-probabilities of given tokens with entropy and top
alternatives, and the loss against a teacher's top logits.

Both stand beside `vocab_parallel_cross_entropy` and take the same `vocab_start` / `gather_fn` for
vocabulary-sharded logits: one exchange of per-token statistics per call. They leave the
logits as they are and allocate the gradient. Several of them, and that cross entropy, may share one set
of logits, built in any order (with `overwrite_logits` the cross entropy has to be built first).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import native, raw


class TokenScores(NamedTuple):
    logprob: torch.Tensor                  # [tokens] fp32
    entropy: torch.Tensor                  # [tokens] fp32, natural log
    top_logprob: Optional[torch.Tensor]    # [tokens, top_k] fp32, falling
    top_index: Optional[torch.Tensor]      # [tokens, top_k] int64 global ids


class _TokenScoresFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, vocab_start, gather_fn):
        logprob, entropy, top_logprob, top_index, stats = raw.token_scores_fwd(logits, tokens, top_k, temperature,
                                                                               vocab_start, gather_fn)
        ctx.temperature, ctx.vocab_start = temperature, vocab_start
        ctx.save_for_backward(logits, tokens.contiguous(), stats, entropy, top_index)
        ctx.set_materialize_grads(False)
        if top_index is not None:
            ctx.mark_non_differentiable(top_index)
        return logprob, entropy, top_logprob, top_index

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprob, d_entropy, d_top, _):
        logits, tokens, stats, entropy, top_index = ctx.saved_tensors
        dz = raw.token_scores_bwd(logits, tokens, stats, entropy, top_index, d_logprob, d_entropy, d_top,
                                  ctx.temperature, ctx.vocab_start)
        return dz, None, None, None, None, None


def token_logprobs(logits, tokens, top_k=0, temperature=1.0, vocab_start=0, gather_fn=None):
    """Scores of given tokens under softmax(logits / temperature): `TokenScores(logprob, entropy,
    top_logprob, top_index)`, all differentiable but the ids.

    logits: [tokens, vocab_local], fp32 / fp16 / bf16, any row pitch; tokens: [tokens] int64 global ids,
    a negative one marks a token that is not scored (log-probability 0, no gradient), one outside the
    vocabulary has NaN for both. `top_k` (up to 128) adds the most likely tokens, equal ones by rising id.
    `vocab_start` and `gather_fn` as in `vocab_parallel_cross_entropy` (`gather_fn` returns the `[tp,
    tokens, n]` stack of a `[tokens, n]` tensor over the tensor-parallel group)."""
    if gather_fn is None and native.use_native(logits):     # the autograd node is native too
        r = native.lib().token_logprobs(logits, tokens, top_k, temperature, vocab_start)
        return TokenScores(*r) if top_k else TokenScores(*r, None, None)
    return TokenScores(*_TokenScoresFn.apply(logits, tokens, int(top_k), float(temperature), int(vocab_start), gather_fn))


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_index, teacher_logit, temperature, vocab_start, gather_fn):
        loss, stats = raw.distill_fwd(logits, teacher_index, teacher_logit, temperature, vocab_start, gather_fn)
        ctx.temperature, ctx.vocab_start = temperature, vocab_start
        ctx.save_for_backward(logits, teacher_index, teacher_logit, stats)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        logits, index, logit, stats = ctx.saved_tensors
        dz = raw.distill_bwd(logits, index, logit, stats, dloss, ctx.temperature, ctx.vocab_start)
        return dz, None, None, None, None, None


def topk_distillation_loss(logits, teacher_index, teacher_logit, temperature=1.0, vocab_start=0, gather_fn=None):
    """Per-token Kullback-Leibler loss of a student against a teacher's listed logits.

    logits: [tokens, vocab_local]; teacher_index: [tokens, k] int64 global ids; teacher_logit:
    [tokens, k] fp32 logits or log-probabilities (what `token_logprobs(..., top_k=k)` reports), -inf for
    unused entries. The teacher is renormalised over its list at `temperature`, the student is its full
    softmax at the same temperature: loss = sum_k q_k (log q_k - log p_k). The customary factor
    temperature**2 is left to the caller. A row without entries has loss 0 and no gradient, one with a
    used entry outside the vocabulary NaN for both. No gradient flows to the teacher. `vocab_start` / `gather_fn`: see `token_logprobs`."""
    if gather_fn is None and native.use_native(logits):
        return native.lib().topk_distillation_loss(logits, teacher_index, teacher_logit, temperature, vocab_start)
    return _DistillFn.apply(logits, teacher_index, teacher_logit, float(temperature), int(vocab_start), gather_fn)
