"""Losses over token log-probabilities of packed sequences: a paired preference
loss and a clipped policy loss with a KL term, as functions and as modules beside
``SamplesLoss``.

Sequences are packed one behind the other: sequence i holds the tokens
``[offsets[i], offsets[i + 1])``.  The forward pass computes the gradient along
with the loss (as ``SamplesLoss`` does); the backward pass scales it.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import torch_ops


class PolicyLossResult(NamedTuple):
    """``policy_loss``'s return value.  ``loss`` is differentiable; ``kl`` (the
    mean KL estimate, averaged as the loss), ``clip_fraction`` (share of the
    counted tokens whose gradient the clip cuts) and ``logp`` (the token
    log-probabilities) are not."""
    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    logp: torch.Tensor


class PreferenceLossResult(NamedTuple):
    """``preference_loss``'s return value.  ``loss`` is differentiable; the
    rewards (beta times each sequence's log-ratio, one per pair) are not."""
    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


def policy_loss(logp: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                offsets: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, kl: str = "k3",
                average: str = "token") -> PolicyLossResult:
    """Clipped policy loss with a KL term over packed tokens.

    With r = exp(logp - old_logp) and A the advantage, a token's loss is
    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * KL``; with
    d = ref_logp - logp the KL estimate is ``-d`` ("k1"), ``d^2 / 2`` ("k2") or
    ``e^d - d - 1`` ("k3").  ``average="token"`` is the mean over the counted
    tokens, ``"sequence"`` the mean over the sequences of their tokens' means
    (sequences that count no token are left out).

    ``logp``, ``old_logp``, ``ref_logp``: float32, (tokens,).  ``advantages``:
    float32, one per token, else one per sequence (as many as there are tokens
    are one per token, whatever the sequences).  ``mask``: bool; False leaves a
    token out.  ``offsets``: int32 or int64, (sequences + 1,), non-decreasing;
    without it all tokens are one sequence.  Tokens outside the sequences are not
    counted and get a gradient of 0.  Differentiable in ``logp``.
    """
    loss, value, clipped = torch_ops().policy(logp, old_logp, advantages, ref_logp, mask, offsets,
                                              clip_low, clip_high, kl_coef, kl, average)
    return PolicyLossResult(loss, value, clipped, logp.detach())


def policy_loss_from_logits(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor,
                            advantages: torch.Tensor, *, temperature: float = 1.0,
                            ref_logp: Optional[torch.Tensor] = None,
                            mask: Optional[torch.Tensor] = None,
                            offsets: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                            clip_high: float = 0.2, kl_coef: float = 0.0, kl: str = "k3",
                            average: str = "token", grad_scale: float = 1.0) -> PolicyLossResult:
    """``policy_loss(token_logprobs(logits, tokens, temperature), ...)``, the
    logits' gradient computed along with the loss.

    ``logits``: (tokens, vocab), float32, float16 or bfloat16; the other
    arguments as in :func:`token_logprobs` and :func:`policy_loss`.  Rows with
    ``mask`` False are not read; their log-probability is given as 0.  Rows of
    tokens that get no gradient get zeros, whatever they hold.

    The gradient is held in the logits' type until the backward pass, which runs
    once.  It is made for a loss multiplied by ``grad_scale``: where the outer
    gradient is just that (1, or the factor of a loss scaler) the backward pass
    hands it over as it is; any other outer gradient costs a pass that scales it
    and rounds it a second time.  So pass ``grad_scale=1 / n`` for
    ``(loss / n).backward()``, and a loss scaler's factor with float16 logits,
    whose gradient's smallest elements are lost before a later factor could save
    them.  Saved-tensor hooks do not see this gradient.
    """
    return PolicyLossResult(*torch_ops().policy_from_logits(
        logits, tokens, old_logp, advantages, temperature, ref_logp, mask, offsets, clip_low,
        clip_high, kl_coef, kl, average, grad_scale))


def preference_loss(logp: torch.Tensor, offsets: torch.Tensor, *,
                    ref_logp: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                    beta: float = 0.1, label_smoothing: float = 0.0, kind: str = "sigmoid",
                    normalize: bool = False) -> PreferenceLossResult:
    """Loss of pairs of packed sequences, one preferred to the other.

    ``offsets`` (2 pairs + 1,) names the chosen sequences first, then the
    rejected ones in the same order.  R is the sum of ``logp - ref_logp`` over a
    sequence's counted tokens (``normalize``: their mean) and
    h = beta (R_chosen - R_rejected); a pair's loss is
    ``-(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)``
    ("sigmoid"), ``max(0, 1 - h)`` ("hinge") or ``(h / beta - 1 / (2 beta))^2``
    ("squared"), and the loss is the mean over the pairs.

    ``logp``, ``ref_logp``: float32, (tokens,); without ``ref_logp`` the
    log-probabilities themselves are compared.  ``mask``: bool; False leaves a
    token out.  A sequence that counts no token has R = 0.  Tokens outside the
    sequences get a gradient of 0.  Differentiable in ``logp``.
    """
    loss, rewards = torch_ops().preference(logp, offsets, ref_logp, mask, beta, label_smoothing,
                                           kind, normalize)
    pairs = rewards.numel() // 2
    return PreferenceLossResult(loss, rewards[:pairs], rewards[pairs:])


class PolicyLoss(torch.nn.Module):
    """:func:`policy_loss` (or, from logits, :func:`policy_loss_from_logits`) as a
    module holding its options."""

    def __init__(self, *, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                 kl: str = "k3", average: str = "token", temperature: float = 1.0):
        super().__init__()
        self.clip_low = clip_low
        self.clip_high = clip_high
        self.kl_coef = kl_coef
        self.kl = kl
        self.average = average
        self.temperature = temperature

    def _options(self):
        return {"clip_low": self.clip_low, "clip_high": self.clip_high, "kl_coef": self.kl_coef,
                "kl": self.kl, "average": self.average}

    def forward(self, logp, old_logp, advantages, *, ref_logp=None, mask=None, offsets=None):
        return policy_loss(logp, old_logp, advantages, ref_logp=ref_logp, mask=mask,
                           offsets=offsets, **self._options())

    def from_logits(self, logits, tokens, old_logp, advantages, *, ref_logp=None, mask=None,
                    offsets=None, grad_scale: float = 1.0):
        return policy_loss_from_logits(logits, tokens, old_logp, advantages,
                                       temperature=self.temperature, ref_logp=ref_logp, mask=mask,
                                       offsets=offsets, grad_scale=grad_scale, **self._options())


class PreferenceLoss(torch.nn.Module):
    """:func:`preference_loss` as a module holding its options."""

    def __init__(self, *, beta: float = 0.1, label_smoothing: float = 0.0, kind: str = "sigmoid",
                 normalize: bool = False):
        super().__init__()
        self.beta = beta
        self.label_smoothing = label_smoothing
        self.kind = kind
        self.normalize = normalize

    def forward(self, logp, offsets, *, ref_logp=None, mask=None):
        return preference_loss(logp, offsets, ref_logp=ref_logp, mask=mask, beta=self.beta,
                               label_smoothing=self.label_smoothing, kind=self.kind,
                               normalize=self.normalize)
