"""Log probabilities of given tokens under a language-model head's logits, with
the distribution's entropy and its largest entries
(``csrc/kernels/token_log_probs.cu``): one sweep over the logits, and in the
backward one more that writes their gradient.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _C
from ._plain import ordinary, plain_calls


_TYPES = (torch.bfloat16, torch.float32, torch.float16)


class TokenLogProbs(NamedTuple):
    """``None`` where it was not asked for; fp32, token numbers int64."""

    log_probs: torch.Tensor | None  # [...]
    entropy: torch.Tensor | None  # [...]
    top_log_probs: torch.Tensor | None  # [..., top_k], falling
    top_tokens: torch.Tensor | None  # [..., top_k]


def _check_logits(logits: torch.Tensor, temperature: float) -> None:
    if logits.dim() < 1 or logits.shape[-1] < 1 or not logits.is_floating_point():
        raise ValueError(f"logits must be floating-point [..., vocab], not {logits.dtype} {tuple(logits.shape)}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be positive and finite, from 1e-30 to 1e30, not {temperature}")


def _check_tokens(tokens: torch.Tensor, logits: torch.Tensor, shape, name: str) -> torch.Tensor:
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise ValueError(f"{name} must be integers, not {tokens.dtype}")
    if tuple(tokens.shape) != tuple(shape) or tokens.device != logits.device:
        raise ValueError(f"{name} must be {tuple(shape)} on {logits.device}, not {tuple(tokens.shape)} on {tokens.device}")
    return tokens.long()


def _takes(logits: torch.Tensor) -> bool:
    """Whether the kernels may be handed the logits."""
    return (ordinary(logits) and logits.is_cuda and plain_calls() and logits.dtype in _TYPES and logits.dim() > 0
            and 0 < logits.shape[-1] <= _C.MOST_VOCAB and logits.numel() < logits.shape[-1] * 2 ** 31
            and not (torch.is_inference_mode_enabled() and logits.requires_grad))


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, temperature: float = 1.0,
                    entropy: bool = False, top_k: int = 0) -> TokenLogProbs:
    """What the softmax of ``logits / temperature`` [..., vocab] (fp32, bf16 or fp16, computed in fp32) says:

    ``log_probs``   of ``tokens`` [...]; without ``tokens`` they are left out
    ``entropy``     of the distribution, in nats, if asked for
    ``top_log_probs``, ``top_tokens``   the ``top_k`` largest entries, the lower token first among equal logits

    A negative token (-100) marks a row that does not count: log probability and entropy 0, its
    ``top_tokens`` -1 at minus infinity, its gradient 0, and its logits are not looked at.  A token past the
    vocabulary has the log probability NaN, and the row's gradient is NaN, whichever output it is of.  Logits of
    minus infinity have probability 0; a row of nothing else, or with a NaN or infinite one, gives NaN as
    ``log_softmax`` does.  ``log_probs`` and
    ``entropy`` carry gradients to the logits, the largest entries are for reading.

    On the GPU the leading dimensions may have any order and strides (a batch without its last position,
    a vocabulary without its padding) as long as a row is contiguous; otherwise the logits are copied.  Up
    to 128 entries come from the kernel; off the GPU and for more it is made of torch's own operations."""
    if _takes(logits) and (tokens is None or ordinary(tokens)) and top_k <= _C.MOST_TOP_TOKENS:
        return TokenLogProbs(*_C.token_log_probs(logits, tokens, temperature, entropy, top_k))  # checks what it is given
    _check_logits(logits, temperature)
    if tokens is not None:
        tokens = _check_tokens(tokens, logits, logits.shape[:-1], "tokens")
    if not 0 <= top_k <= logits.shape[-1]:
        raise ValueError(f"top_k must be from 0 to the vocabulary, {logits.shape[-1]}, not {top_k}")
    if tokens is None and not entropy and not top_k:
        raise ValueError("nothing is asked for: give tokens, entropy=True or top_k")
    return _plain_token_log_probs(logits, tokens, temperature, entropy, top_k)


def _plain_token_log_probs(logits, tokens, temperature, entropy, top_k) -> TokenLogProbs:
    wide = logits if logits.dtype == torch.float64 else logits.float()
    counts = None if tokens is None else tokens >= 0
    if counts is not None:  # a row that does not count is not looked at, be it NaN
        wide = torch.where(counts.unsqueeze(-1), wide, 0.0)
    logp = torch.log_softmax(wide / temperature, -1)
    of = h = top = which = None
    if tokens is not None:
        known = counts & (tokens < logits.shape[-1])
        unknown = counts & ~known
        of = logp.gather(-1, tokens.where(known, 0).unsqueeze(-1)).squeeze(-1)
        of = torch.where(counts, of, 0.0) * torch.where(unknown, float("nan"), 1.0)
    if entropy:
        h = -(logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)).sum(-1)
        if counts is not None:
            h = torch.where(counts, h, 0.0)
            # The row's gradient is NaN though the entropy is not: 0 times the slope of a root at zero.
            h = h + 0.0 * torch.where(unknown, h - h.detach(), 1.0).sqrt()
    if top_k:
        order = wide.detach().sort(dim=-1, descending=True, stable=True).indices[..., :top_k]
        top, which = logp.detach().gather(-1, order), order
        if counts is not None:
            top = torch.where(counts.unsqueeze(-1), top, float("-inf"))
            which = torch.where(counts.unsqueeze(-1), which, -1)
    out = TokenLogProbs(of, h, top, which)
    return TokenLogProbs(*(x if x is None or not x.is_floating_point() else x.float() for x in out))
