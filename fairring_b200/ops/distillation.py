"""Distillation from a teacher's largest log probabilities
(``csrc/kernels/distillation.cu``): one sweep over the student's logits, and in
the backward one more that writes their gradient.
"""

from __future__ import annotations

import torch

from .. import _C
from ._plain import ordinary
from .token_log_probs import _check_logits, _check_tokens, _takes


def distillation_loss(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_log_probs: torch.Tensor, *,
                      temperature: float = 1.0, rest: bool = False, reduction: str = "mean") -> torch.Tensor:
    """Kullback-Leibler divergence of the student's ``softmax(logits / temperature)`` [..., vocab] (fp32, bf16 or
    fp16, computed in fp32) from a teacher of which ``k`` tokens a row are known: ``teacher_tokens`` [..., k] and
    ``teacher_log_probs`` [..., k], as ``token_log_probs(teacher_logits, top_k=k)`` gives them.

    ``rest=False``: the teacher is the softmax of the listed values, divided by the temperature, over the
    listed tokens; plain logits will do as well.  ``sum_k q_k (log q_k - log p_k)``

    ``rest=True``: the listed values are log probabilities over the whole vocabulary, taken at this temperature, and
    what they leave of 1 is the probability of "any other token", of the teacher as of the student:
    ``sum_k q_k (log q_k - log p_k) + q_rest (log q_rest - log p_rest)``.  Less than 2^-20 is what rounding leaves of
    values that sum to 1, and counts as nothing.  Where the teacher leaves more and the student nothing (every other token
    is masked or listed) the loss is infinite.

    A negative token is padding.  A row of padding (or, without the rest, of nothing but values of minus infinity) does
    not count: its loss and gradient are 0.  A token named twice is two terms of the sum, and one token of the
    student's.  A token past the vocabulary gives NaN.  ``reduction``: ``"mean"`` over the rows
    that count (0 if none does), ``"sum"``, or ``"none"`` for one value a row; fp32.  The loss is not multiplied by
    ``temperature ** 2``.  The teacher's values are constants: they must not require a gradient.

    On the GPU up to 256 tokens a row and, with the rest, 2^20 logits come from the kernel, with the leading
    dimensions in any order and strides; otherwise, and off the GPU, it is made of torch's own operations."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    if (_takes(logits) and ordinary(teacher_tokens) and ordinary(teacher_log_probs) and teacher_tokens.dim() > 0
            and teacher_tokens.shape[-1] <= _C.MOST_TEACHER_TOKENS and not (rest and logits.shape[-1] > _C.MOST_REST_VOCAB)):
        loss = _C.distillation(logits, teacher_tokens, teacher_log_probs, temperature, rest, reduction == "mean")  # checks them
        return loss.sum() if reduction == "sum" else loss
    _check_logits(logits, temperature)
    if teacher_tokens.dim() < 1 or teacher_tokens.shape[-1] < 1:
        raise ValueError("teacher_tokens must be [..., k] with at least one token a row")
    shape = (*logits.shape[:-1], teacher_tokens.shape[-1])
    teacher_tokens = _check_tokens(teacher_tokens, logits, shape, "teacher_tokens")
    if not teacher_log_probs.is_floating_point() or tuple(teacher_log_probs.shape) != shape or teacher_log_probs.device != logits.device:
        raise ValueError(f"teacher_log_probs must be floating-point {shape} on {logits.device}, not "
                         f"{teacher_log_probs.dtype} {tuple(teacher_log_probs.shape)} on {teacher_log_probs.device}")
    if teacher_log_probs.requires_grad and torch.is_grad_enabled():
        raise ValueError("teacher_log_probs are constants: detach them")
    loss, counts = _plain_distillation(logits, teacher_tokens, teacher_log_probs, temperature, rest)
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / counts.sum().clamp_min(1)


def _plain_distillation(logits, tokens, given, temperature, rest):
    """(loss, whether it counts) of every row."""
    low = float("-inf")
    there = tokens >= 0
    known = there & (tokens < logits.shape[-1])
    given = given.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    counts = there.any(-1) if rest else (there & (given != low)).any(-1)
    wide = torch.where(counts.unsqueeze(-1), logits if logits.dtype == torch.float64 else logits.float(), 0.0)
    logp = torch.log_softmax(wide / temperature, -1)
    at = tokens.where(known, 0)
    log_q = torch.where(known, given, low)
    if not rest:
        log_q = torch.log_softmax(torch.where(counts.unsqueeze(-1), log_q / temperature, 0.0), -1)
    q = torch.where(known, log_q.exp(), 0.0)
    terms = q * (log_q.masked_fill(q == 0, 0.0) - logp.gather(-1, at).masked_fill(q == 0, 0.0))
    loss = terms.sum(-1)
    if rest:
        left = 1 - q.double().sum(-1)
        left = torch.where(left >= _C.LEAST_REST, left, 0.0)
        listed = torch.zeros_like(logp).scatter_add_(-1, at, known.to(logp.dtype)) > 0
        # No other token, or none with any probability: the loss is infinite, and the gradient that of the row's own sum.
        gone = (listed | (logp == low)).all(-1, keepdim=True)
        others = torch.logsumexp(logp.masked_fill(listed & ~gone, low), -1)
        less_sum = (logp - wide / temperature).gather(-1, logp.detach().argmax(-1, keepdim=True)).squeeze(-1)
        others = torch.where(gone.squeeze(-1), low + (less_sum - less_sum.detach()), others)
        share = left * (left.clamp_min(1e-300).log() - others.double())
        loss = loss + torch.where(left > 0, share, 0.0).to(loss.dtype)
    loss = loss * torch.where((there & ~known).any(-1), float("nan"), 1.0)
    return torch.where(counts, loss, 0.0).float(), counts
