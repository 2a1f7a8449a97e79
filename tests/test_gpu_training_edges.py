"""The training operators on the device where a bound of the usual size would hide a fault: extreme
temperatures, impossible sequences, exact sums, rows whose result is known in closed form, gradients
of views, and PyTorch's other ways of running a backward pass.

Tolerances are counted beside each test, in half steps of the result's type (EPS32 is float32's).
"""

from __future__ import annotations

import math

import pytest
import torch

import training_ref as ref
from test_gpu_training import _close, _gen, _grad_tolerance, _packed, _step, _step_state
from training_ref import EPS32, half_step, tiny

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def sk():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import sinkslot_b200
    sinkslot_b200.load_library()
    return sinkslot_b200


# ------------------------------------------------------------------ extreme temperatures
def _entropy_step(sk, z, tokens, temperature, g, gh):
    z = z.detach().requires_grad_()
    lp, h = sk.token_logprobs(z, tokens, temperature=temperature, entropy=True)
    grad, = torch.autograd.grad([lp, h], [z], [g, gh])
    want_lp, want_h, *_ = ref.logprobs64(z.detach(), tokens, temperature)
    want = ref.logprobs_grad64(z.detach(), tokens, g, gh, temperature)
    return lp.detach(), h.detach(), grad, want_lp, want_h, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 5003, 40000])
@pytest.mark.parametrize("temperature,outer", [(1e-30, 1e-30), (1e-12, 1e-12), (2e-9, 1e-9),
                                               (1e-4, 1e-4), (0.01, 1e-3)])
def test_entropy_gradient_at_low_temperatures(sk, temperature, outer, vocab, dtype):
    """Switched-off logits (-inf, or the type's lowest value) get a gradient of 0 at any temperature,
    in rows with and without an outer gradient of the entropy."""
    gen = _gen(vocab)
    z = torch.randint(-6, 1, (8, vocab), generator=gen, device="cuda").to(dtype)
    z[:, 0] = 0.0
    z[:4, 5:9] = -math.inf
    z[2:6, 9:14] = torch.finfo(dtype).min
    z[6, 1:] = -math.inf
    z[7, 1:] = torch.finfo(dtype).min
    tokens = torch.zeros(8, dtype=torch.int64, device="cuda")
    g = outer * torch.randn(8, generator=gen, device="cuda")
    gh = outer * torch.randn(8, generator=gen, device="cuda")
    gh[1] = 0.0
    lp, h, grad, want_lp, want_h, want = _entropy_step(sk, z, tokens, temperature, g, gh)
    _close(lp, want_lp, ref.logp_tolerance(z, tokens, temperature, vocab), "logp")
    _close(h, want_h, 4 * (ref.sum_error(vocab) + 8 * EPS32) * (math.log(vocab + 1.0) + 1.0),
           "entropy")
    _close(grad, want, _grad_tolerance(z, tokens, g, gh, temperature, want, dtype), "grad")
    off = z < -6
    assert off.any() and not grad[off].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entropy_gradient_under_a_loss_scale(sk, dtype):
    """Masked logits, T = 0.01 and an outer gradient of 2^17: the product of both scales and the mask
    must not reach infinity."""
    gen = _gen(5)
    z = torch.randn(6, 3001, generator=gen, device="cuda").to(dtype)
    z[:, 2000:] = -math.inf
    z[3:, 2000:] = torch.finfo(dtype).min
    tokens = torch.randint(0, 2000, (6,), generator=gen, device="cuda")
    g = torch.full((6,), 2.0 ** 17, device="cuda")
    *_, grad, _, _, want = _entropy_step(sk, z, tokens, 0.01, g, g)
    # a term under 2^-126 flushes to 0 before it is multiplied by at most (g + gh (|log p| + H)) / T
    # (its sum is 1 or more; log p is over -104 - ln 3001 there and H under ln 3001)
    flushed = 2.0 ** -126 * 2.0 ** 17 / 0.01 * (1 + 104 + 2 * math.log(3001))
    _close(grad, want, _grad_tolerance(z, tokens, g, g, 0.01, want, dtype) + flushed, "grad")
    assert not grad[:, 2000:].any()


def test_entropy_of_far_logits_at_a_high_temperature(sk):
    """Differences of many times 1e30 count as what they are where T is 1e30."""
    z = torch.tensor([[0.0, -2e30, -5e30, -1e31, -math.inf, -3e38]], device="cuda").repeat(3, 700)
    tokens = torch.tensor([1, 2, 6], device="cuda")
    g = torch.tensor([1e30, -1e30, 2e30], device="cuda")
    lp, h, grad, want_lp, want_h, want = _entropy_step(sk, z, tokens, 1e30, g, g)
    vocab = z.shape[1]
    _close(lp, want_lp, ref.logp_tolerance(z, tokens, 1e30, vocab), "logp")
    _close(h, want_h, 4 * (ref.sum_error(vocab) + 8 * EPS32) * (math.log(vocab + 1.0) + 1.0),
           "entropy")
    _close(grad, want, _grad_tolerance(z, tokens, g, g, 1e30, want, z.dtype), "grad")


# ------------------------------------------------------------------ preference
def test_preference_impossible_sequences(sk):
    """A rejected sequence of probability 0 costs its pair nothing; a chosen one costs everything,
    and with label smoothing either does."""
    inf = math.inf
    off = torch.arange(5, device="cuda")

    def run(values, **kw):
        logp = torch.tensor(values, device="cuda", requires_grad=True)
        r = sk.preference_loss(logp, off, beta=0.5, **kw)
        return r, torch.autograd.grad(r.loss, [logp])[0].tolist()

    r, grad = run([-1.0, -2.0, -inf, -2.0])  # pairs (0, 2) and (1, 3)
    # half of ln 2, rounded once from fp64
    assert abs(float(r.loss.detach()) - math.log(2) / 2) <= EPS32
    assert grad == [0.0, -0.125, 0.0, 0.125]
    assert r.rejected_rewards.tolist() == [-inf, -1.0]
    r, grad = run([-inf, -2.0, -1.0, -2.0])
    assert float(r.loss.detach()) == inf and grad == [-0.25, -0.125, 0.25, 0.125]
    r, _ = run([-1.0, -2.0, -inf, -2.0], label_smoothing=0.25)
    assert float(r.loss.detach()) == inf
    r, grad = run([-1.0, -2.0, -inf, -2.0], kind="hinge")
    assert float(r.loss.detach()) == 0.5 and grad == [0.0, -0.25, 0.0, 0.25]
    r, _ = run([-inf, -2.0, -inf, -2.0])
    assert r.loss.isnan()


# ------------------------------------------------------------------ gradients of views
def test_gradient_of_rows_far_apart_takes_its_own_size(sk):
    """The last position of each sequence, and every eighth row: the gradient is as large as the
    logits it belongs to, not as the buffer they are seen in."""
    gen = _gen(9)
    full = torch.randn(6, 64, 1003, generator=gen, device="cuda").bfloat16()
    tokens = torch.randint(0, 1003, (6,), generator=gen, device="cuda")
    old = torch.full((6,), -7.0, device="cuda")
    for z in (full[:, -1], full[:, 3, 1:1001], full[0, ::8][:6], full[:, 0, :5]):
        t = tokens % z.shape[1]
        want = None
        for leaf in (z.detach().clone(), z.detach()):
            leaf.requires_grad_()
            a, = torch.autograd.grad(sk.token_logprobs(leaf, t).sum(), [leaf])
            r = sk.policy_loss_from_logits(leaf, t, old, old)
            b, = torch.autograd.grad(r.loss, [leaf])
            if want is None:
                want = a, b
            # (rows on another phase are added up in another order: a few steps of float32 before
            # the rounding to 16 bits, so at most one step of those)
            torch.testing.assert_close(a, want[0], rtol=2 * half_step(a.dtype) * 2, atol=1e-6)
            torch.testing.assert_close(b, want[1], rtol=2 * half_step(a.dtype) * 2, atol=1e-6)
            for grad in (a, b):
                assert grad.shape == z.shape
                assert grad.untyped_storage().nbytes() <= 2 * (z.shape[0] * (z.shape[1] + 264))
                assert (grad.data_ptr() - leaf.data_ptr()) % 16 == 0
                if z.shape[0] > 1:
                    assert (grad.stride(0) - leaf.stride(0)) * 2 % 16 == 0
    padded = torch.randn(9, 1003 + 61, generator=gen, device="cuda")[:, :1003].requires_grad_()
    grad, = torch.autograd.grad(sk.token_logprobs(padded, tokens.repeat(2)[:9]).sum(), [padded])
    assert grad.stride() == padded.stride()  # a padded buffer keeps its rows' distance
