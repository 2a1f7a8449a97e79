"""Log-probabilities and entropies of tokens under rows of logits.

The log-sum-exp over a row runs in one pass with a running maximum and sum; the
backward pass recomputes the softmax from the logits and the two row statistics,
so nothing of the logits' size is kept.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, dtype_code, on_device, ptr, stream_of


def grad_like(z: torch.Tensor) -> torch.Tensor:
    """An uninitialised (rows, vocab) tensor for the gradient of ``z``: laid out
    as ``z`` is (a view of a padded buffer gets rows as far apart, beginning on
    the same 16-byte phase), contiguous where the rows of ``z`` overlap."""
    rows, vocab = z.shape
    stride = z.stride(0)
    if stride < vocab or rows <= 1:
        stride = vocab
    phase = (z.data_ptr() % 16) // z.element_size()
    if stride == vocab and phase == 0:
        return torch.empty((rows, vocab), dtype=z.dtype, device=z.device)
    n = phase + max(rows - 1, 0) * stride + vocab
    flat = torch.empty(n, dtype=z.dtype, device=z.device)
    return flat.as_strided((rows, vocab), (stride, 1), phase)


def _token_logprobs_impl(z, tokens, temperature, ignore_index, entropy):
    """The body of the ``sinkslot_b200::token_logprobs`` operator."""
    dev = z.device
    rows, vocab = z.shape
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    ent = torch.empty(rows if entropy else 0, dtype=torch.float32, device=dev)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=dev)
    with on_device(dev):
        call("sinkslot_token_logprobs", ptr(z), dtype_code(z), z.stride(0), rows, vocab,
             ptr(tokens), tokens.element_size(), ignore_index, 1.0 / temperature, ptr(logp),
             ptr(ent), ptr(stats), stream_of(dev))
    return logp, ent, stats


def _token_logprobs_grad_impl(z, tokens, stats, entropy, g, g_entropy, temperature, ignore_index):
    """The body of the ``sinkslot_b200::token_logprobs_grad`` operator."""
    dev = z.device
    rows, vocab = z.shape
    out = grad_like(z)
    with on_device(dev):
        call("sinkslot_token_logprobs_grad", ptr(z), dtype_code(z), z.stride(0), rows, vocab,
             ptr(tokens), tokens.element_size(), ignore_index, 1.0 / temperature, ptr(stats),
             ptr(entropy), ptr(g), g.stride(0) if g is not None else 0, ptr(g_entropy),
             g_entropy.stride(0) if g_entropy is not None else 0, ptr(out), out.stride(0),
             stream_of(dev))
    return out


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tokens, temperature, ignore_index, entropy):
        ctx.set_materialize_grads(False)
        logp, ent, stats = torch.ops.sinkslot_b200.token_logprobs(z, tokens, temperature,
                                                                  ignore_index, entropy)
        ctx.save_for_backward(z, tokens, stats, ent)
        ctx.args = (temperature, ignore_index)
        return (logp, ent) if entropy else logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_entropy=None):
        if g is None and g_entropy is None:
            return None, None, None, None, None
        z, tokens, stats, ent = ctx.saved_tensors
        out = torch.ops.sinkslot_b200.token_logprobs_grad(z, tokens, stats, ent, g, g_entropy,
                                                          *ctx.args)
        return out, None, None, None, None


def check_logits(name: str, logits, tokens, temperature) -> None:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{name}: logits need a vocabulary axis, got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{name}: tokens must have the shape {tuple(logits.shape[:-1])} of the "
                         f"logits' rows, got {tuple(tokens.shape)}")
    _lib.require_cuda(name, logits, tokens)
    _lib.require_dtype(name, "logits", logits)
    _lib.require_index(name, "tokens", tokens)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{name}: temperature must be in [1e-30, 1e30], got {temperature}")
    if tokens.numel() > 1 << 27:
        raise ValueError(f"{name}: more than 2^27 rows are not supported")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0,
                   ignore_index: int = -100, entropy: bool = False):
    """``log_softmax(logits / temperature)`` at ``tokens``, in float32; with
    ``entropy`` the pair (log-probabilities, entropies of the rows).
    Differentiable in ``logits``.

    ``logits``: (..., vocab), float32, float16 or bfloat16 (rows may lie apart);
    ``tokens``: int32 or int64, the shape of the rows.  Rows whose token is
    ``ignore_index`` give 0, get a gradient of 0 and are not read.  Any other
    token outside the vocabulary gives NaN.  Logits of -inf are impossible
    tokens: probability 0, gradient 0; a row of nothing else gives -inf, entropy
    0 and gradient 0.
    """
    name = "token_logprobs"
    check_logits(name, logits, tokens, temperature)
    lead = tokens.shape
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if z.stride(1) != 1 and z.shape[1] > 1:
        z = z.contiguous()
    out = _TokenLogprobsFn.apply(z, tokens.reshape(-1).contiguous(), float(temperature),
                                 int(ignore_index), bool(entropy))
    if len(lead) == 1:
        return out
    return tuple(t.view(lead) for t in out) if entropy else out.view(lead)
