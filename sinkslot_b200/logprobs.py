"""Log-probabilities and entropies of tokens under rows of logits.

The log-sum-exp over a row runs in one pass with a running maximum and sum; the
backward pass recomputes the softmax from the logits and the two row statistics,
so nothing of the logits' size is kept.
"""

from __future__ import annotations

import torch

from ._lib import torch_ops


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
    0 and gradient 0.  A row whose outer gradients are 0 gets zeros, whatever it
    holds.
    """
    logp, ent = torch_ops().logprobs(logits, tokens, temperature, ignore_index, entropy)
    return (logp, ent) if entropy else logp
