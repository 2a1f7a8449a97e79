"""Losses over token log-probabilities of packed sequences: a paired preference
loss and a clipped policy loss with a KL term, as functions and as modules beside
``SamplesLoss``.

Sequences are packed one behind the other: sequence i holds the tokens
``[offsets[i], offsets[i + 1])``.  The forward pass computes the gradient along
with the loss (as ``SamplesLoss`` does); the backward pass scales it.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, dtype_code, on_device, ptr, stream_of
from .logprobs import check_logits, grad_like

_KL = {"k1": 1, "k2": 2, "k3": 3}
_PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}


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


def _offset_bytes(offsets) -> int:
    return offsets.element_size() if offsets is not None else 8


def _policy_loss_impl(logp, old_logp, advantages, ref_logp, mask, offsets, adv_per_token, clip_low,
                      clip_high, kl_coef, kl, sequence_average, want_grad):
    """The body of the ``sinkslot_b200::policy_loss`` operator."""
    dev = logp.device
    t = logp.numel()
    s = offsets.numel() - 1 if offsets is not None else 1
    nb = _lib.out_i64()
    call("sinkslot_loss_workspace_bytes", s, ctypes.byref(nb))
    ws = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    values = torch.empty(4, dtype=torch.float32, device=dev)
    coef = torch.empty(t if want_grad else 0, dtype=torch.float32, device=dev)
    with on_device(dev):
        call("sinkslot_policy_loss", ptr(logp), ptr(old_logp), ptr(ref_logp), ptr(advantages),
             adv_per_token, ptr(mask), ptr(offsets), _offset_bytes(offsets), s, t, clip_low,
             clip_high, kl_coef, kl, sequence_average, ptr(values), ptr(coef), ptr(ws), ws.numel(),
             stream_of(dev))
    return values, coef


def _scale_tokens_impl(coef, values, g):
    """The body of the ``sinkslot_b200::scale_tokens`` operator."""
    dev = coef.device
    out = torch.empty_like(coef)
    with on_device(dev):
        call("sinkslot_scale_tokens", ptr(coef), coef.numel(), values.data_ptr() + 12, ptr(g),
             ptr(out), stream_of(dev))
    return out


def _policy_loss_logits_impl(z, tokens, old_logp, advantages, ref_logp, mask, offsets, temperature,
                             adv_per_token, clip_low, clip_high, kl_coef, kl, sequence_average,
                             grad_scale, want_grad):
    """The body of the ``sinkslot_b200::policy_loss_logits`` operator."""
    dev = z.device
    t, vocab = z.shape
    s = offsets.numel() - 1 if offsets is not None else 1
    nb = _lib.out_i64()
    call("sinkslot_policy_logits_workspace_bytes", t, s, ctypes.byref(nb))
    ws = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    values = torch.empty(4, dtype=torch.float32, device=dev)
    logp = torch.empty(t, dtype=torch.float32, device=dev)
    grad = grad_like(z) if want_grad else z.new_empty((0, vocab))
    with on_device(dev):
        call("sinkslot_policy_loss_logits", ptr(z), dtype_code(z), z.stride(0), t, vocab,
             ptr(tokens), tokens.element_size(), 1.0 / temperature, ptr(old_logp), ptr(ref_logp),
             ptr(advantages), adv_per_token, ptr(mask), ptr(offsets), _offset_bytes(offsets), s,
             clip_low, clip_high, kl_coef, kl, sequence_average, grad_scale, ptr(values),
             ptr(logp), ptr(grad), grad.stride(0), ptr(ws), ws.numel(), stream_of(dev))
    return values, logp, grad


def _scale_rows_impl(grad, g, grad_scale):
    """The body of the ``sinkslot_b200::scale_rows_`` operator (in place)."""
    dev = grad.device
    with on_device(dev):
        call("sinkslot_scale_rows", ptr(grad), dtype_code(grad), grad.stride(0), grad.shape[0],
             grad.shape[1], ptr(g), grad_scale, stream_of(dev))


def _preference_loss_impl(logp, offsets, ref_logp, mask, beta, smoothing, kind, normalize):
    """The body of the ``sinkslot_b200::preference_loss`` operator."""
    dev = logp.device
    s = offsets.numel() - 1
    nb = _lib.out_i64()
    call("sinkslot_loss_workspace_bytes", s, ctypes.byref(nb))
    ws = torch.empty(nb.value, dtype=torch.uint8, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rewards = torch.empty(s, dtype=torch.float32, device=dev)
    slope = torch.empty(s, dtype=torch.float32, device=dev)
    with on_device(dev):
        call("sinkslot_preference_loss", ptr(logp), ptr(ref_logp), ptr(mask), ptr(offsets),
             offsets.element_size(), s, logp.numel(), beta, smoothing, kind, normalize, ptr(loss),
             ptr(rewards), ptr(slope), ptr(ws), ws.numel(), stream_of(dev))
    return loss, rewards, slope


def _preference_grad_impl(slope, offsets, mask, g, tokens):
    """The body of the ``sinkslot_b200::preference_grad`` operator."""
    dev = slope.device
    out = torch.empty(tokens, dtype=torch.float32, device=dev)
    with on_device(dev):
        call("sinkslot_preference_grad", ptr(slope), ptr(mask), ptr(offsets),
             offsets.element_size(), slope.numel(), tokens, ptr(g), ptr(out), stream_of(dev))
    return out


class _PolicyLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, old_logp, advantages, ref_logp, mask, offsets, *args):
        values, coef = torch.ops.sinkslot_b200.policy_loss(
            logp, old_logp, advantages, ref_logp, mask, offsets, *args, ctx.needs_input_grad[0])
        ctx.save_for_backward(values, coef)
        loss, kl, clipped, _ = values.unbind()
        ctx.mark_non_differentiable(kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, kl, clipped

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 12
        values, coef = ctx.saved_tensors
        return (torch.ops.sinkslot_b200.scale_tokens(coef, values, g),) + (None,) * 11


class _PolicyLossLogitsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tokens, old_logp, advantages, ref_logp, mask, offsets, temperature, *args):
        *args, grad_scale = args
        values, logp, grad = torch.ops.sinkslot_b200.policy_loss_logits(
            z, tokens, old_logp, advantages, ref_logp, mask, offsets, temperature, *args,
            grad_scale, ctx.needs_input_grad[0])
        ctx.grad, ctx.grad_scale = grad, grad_scale
        loss, kl, clipped, _ = values.unbind()
        ctx.mark_non_differentiable(kl, clipped, logp)
        ctx.set_materialize_grads(False)
        return loss, kl, clipped, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 15
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            raise RuntimeError("policy_loss_from_logits: its backward pass runs once (the "
                               "gradient was handed over); use token_logprobs with policy_loss "
                               "for several")
        torch.ops.sinkslot_b200.scale_rows_(grad, g, ctx.grad_scale)
        return (grad,) + (None,) * 14


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, offsets, ref_logp, mask, beta, smoothing, kind, normalize):
        loss, rewards, slope = torch.ops.sinkslot_b200.preference_loss(
            logp, offsets, ref_logp, mask, beta, smoothing, kind, normalize)
        ctx.save_for_backward(slope, offsets, mask)
        ctx.tokens = logp.numel()
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 8
        slope, offsets, mask = ctx.saved_tensors
        return (torch.ops.sinkslot_b200.preference_grad(slope, offsets, mask, g, ctx.tokens),) \
            + (None,) * 7


def _tokens_f32(name: str, what: str, t, like: torch.Tensor):
    """``t`` as a contiguous float32 vector of one value per token, or an error."""
    if t.dtype != torch.float32:
        raise ValueError(f"{name}: {what} must be float32, got {t.dtype}")
    if t.shape != like.shape:
        raise ValueError(f"{name}: {what} must have the tokens' shape {tuple(like.shape)}, got "
                         f"{tuple(t.shape)}")
    return t.contiguous()


def _constants(name: str, **tensors) -> None:
    if torch.is_grad_enabled():
        for what, t in tensors.items():
            if t is not None and t.requires_grad:
                raise ValueError(f"{name}: no gradient is taken in {what}; detach it")


def _check_packing(name: str, like, mask, offsets):
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != like.shape:
            raise ValueError(f"{name}: mask must be bool of the tokens' shape {tuple(like.shape)}, "
                             f"got {mask.dtype} {tuple(mask.shape)}")
        mask = mask.contiguous()
    if offsets is not None:
        _lib.require_index(name, "offsets", offsets)
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError(f"{name}: offsets must hold (sequences + 1) values, got "
                             f"{tuple(offsets.shape)}")
        offsets = offsets.contiguous()
    return mask, offsets


def _check_policy(name, like, old_logp, advantages, ref_logp, mask, offsets, clip_low, clip_high,
                  kl_coef, kl, average):
    """Arguments behind logp, as both policy operators take them."""
    _lib.require_cuda(name, like, *(t for t in (old_logp, advantages, ref_logp, mask, offsets)
                                    if t is not None))
    _constants(name, old_logp=old_logp, advantages=advantages, ref_logp=ref_logp)
    old_logp = _tokens_f32(name, "old_logp", old_logp, like)
    if ref_logp is not None:
        ref_logp = _tokens_f32(name, "ref_logp", ref_logp, like)
    mask, offsets = _check_packing(name, like, mask, offsets)
    s = offsets.numel() - 1 if offsets is not None else 1
    if advantages.dtype != torch.float32:
        raise ValueError(f"{name}: advantages must be float32, got {advantages.dtype}")
    per_token = advantages.shape == like.shape
    if not per_token and advantages.shape != (s,):
        raise ValueError(f"{name}: advantages must be one per token {tuple(like.shape)} or per "
                         f"sequence {(s,)}, got {tuple(advantages.shape)}")
    if kl not in _KL:
        raise ValueError(f"{name}: kl must be one of {tuple(_KL)}, got {kl!r}")
    if average not in ("token", "sequence"):
        raise ValueError(f"{name}: average must be 'token' or 'sequence', got {average!r}")
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError(f"{name}: clip_low and clip_high must be >= 0, got {clip_low}, "
                         f"{clip_high}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"{name}: kl_coef must be finite, got {kl_coef}")
    if kl_coef != 0.0 and ref_logp is None:
        raise ValueError(f"{name}: kl_coef {kl_coef} needs ref_logp")
    return ((old_logp, advantages.contiguous(), ref_logp, mask, offsets),
            (per_token, float(clip_low), float(clip_high), float(kl_coef), _KL[kl],
             average == "sequence"))


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
    float32, one per token, else one per sequence.  ``mask``: bool; False leaves
    a token out.  ``offsets``: int32 or int64, (sequences + 1,), non-decreasing;
    without it all tokens are one sequence.  Tokens outside the sequences are not
    counted and get a gradient of 0.  Differentiable in ``logp``.
    """
    name = "policy_loss"
    if logp.dim() != 1:
        raise ValueError(f"{name}: logp must be (tokens,), got {tuple(logp.shape)}")
    tensors, args = _check_policy(name, logp, old_logp, advantages, ref_logp, mask, offsets,
                                  clip_low, clip_high, kl_coef, kl, average)
    flat = _tokens_f32(name, "logp", logp, logp)
    loss, value, clipped = _PolicyLossFn.apply(flat, *tensors, *args)
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
    ``mask`` False are not read; their log-probability is given as 0.

    The gradient is held in the logits' type until the backward pass, which runs
    once.  It is made for a loss multiplied by ``grad_scale``: where the outer
    gradient is just that (1, or the factor of a loss scaler) the backward pass
    hands it over as it is; any other outer gradient costs a pass that scales it
    and rounds it a second time.
    """
    name = "policy_loss_from_logits"
    if logits.dim() != 2:
        raise ValueError(f"{name}: logits must be (tokens, vocab), got {tuple(logits.shape)}")
    check_logits(name, logits, tokens, temperature)
    if not (math.isfinite(grad_scale) and grad_scale != 0.0):
        raise ValueError(f"{name}: grad_scale must be finite and not 0, got {grad_scale}")
    tensors, args = _check_policy(name, tokens, old_logp, advantages, ref_logp, mask, offsets,
                                  clip_low, clip_high, kl_coef, kl, average)
    z = logits
    if z.stride(1) != 1 and z.shape[1] > 1:
        z = z.contiguous()
    return PolicyLossResult(*_PolicyLossLogitsFn.apply(
        z, tokens.contiguous(), *tensors, float(temperature), *args, float(grad_scale)))


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
    name = "preference_loss"
    if logp.dim() != 1:
        raise ValueError(f"{name}: logp must be (tokens,), got {tuple(logp.shape)}")
    _lib.require_cuda(name, logp, offsets, *(t for t in (ref_logp, mask) if t is not None))
    _constants(name, ref_logp=ref_logp)
    if kind not in _PREFERENCE_KINDS:
        raise ValueError(f"{name}: kind must be one of {tuple(_PREFERENCE_KINDS)}, got {kind!r}")
    if not (0.0 < beta < math.inf):
        raise ValueError(f"{name}: beta must be positive and finite, got {beta}")
    if not 0.0 <= label_smoothing < 1.0 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"{name}: label_smoothing must be in [0, 1), and 0 unless kind is "
                         f"'sigmoid'; got {label_smoothing}")
    mask, offsets = _check_packing(name, logp, mask, offsets)
    if offsets.numel() % 2 == 0:
        raise ValueError(f"{name}: sequences come in pairs, got {offsets.numel() - 1}")
    if ref_logp is not None:
        ref_logp = _tokens_f32(name, "ref_logp", ref_logp, logp)
    flat = _tokens_f32(name, "logp", logp, logp)
    loss, rewards = _PreferenceLossFn.apply(flat, offsets, ref_logp, mask, float(beta),
                                            float(label_smoothing), _PREFERENCE_KINDS[kind],
                                            bool(normalize))
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
