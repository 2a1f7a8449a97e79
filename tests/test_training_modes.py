"""The training operators under PyTorch's modes of differentiation, without a GPU (on fake CUDA
tensors, which no kernel sees)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

import sinkslot_b200 as sk


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def _cuda(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _calls():
    """(name, the function of one floating argument, that argument's shape), for every floating
    argument of every function."""
    ids, off = _cuda(8, dtype=torch.int64), _cuda(3, dtype=torch.int64)
    v, z = _cuda(8), _cuda(8, 30)
    return [
        ("table", lambda t: sk.embedding_lookup(t, ids), (20, 4)),
        ("logits", lambda t: sk.token_logprobs(t, ids), (8, 30)),
        ("logits, entropy", lambda t: sk.token_logprobs(t, ids, entropy=True)[1], (8, 30)),
        ("logp", lambda t: sk.policy_loss(t, v, v).loss, (8,)),
        ("old_logp", lambda t: sk.policy_loss(v, t, v).loss, (8,)),
        ("advantages", lambda t: sk.policy_loss(v, v, t).loss, (8,)),
        ("ref_logp", lambda t: sk.policy_loss(v, v, v, ref_logp=t, kl_coef=0.1).loss, (8,)),
        ("policy logits", lambda t: sk.policy_loss_from_logits(t, ids, v, v).loss, (8, 30)),
        ("policy old_logp", lambda t: sk.policy_loss_from_logits(z, ids, t, v).loss, (8,)),
        ("policy advantages", lambda t: sk.policy_loss_from_logits(z, ids, v, t).loss, (8,)),
        ("preference logp", lambda t: sk.preference_loss(t, off).loss, (8,)),
        ("preference ref_logp", lambda t: sk.preference_loss(v, off, ref_logp=t).loss, (8,)),
    ]


def test_forward_mode_is_refused(fake):
    """A tangent is never dropped, whether or not the call records a gradient."""
    for name, call, shape in _calls():
        with fwd.dual_level():
            dual = fwd.make_dual(_cuda(*shape), _cuda(*shape))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
            leaf = _cuda(*shape).requires_grad_()
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fwd.make_dual(leaf, _cuda(*shape)))
            call(fwd.unpack_dual(dual).primal)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (_cuda(*shape),), (_cuda(*shape),))
        call(_cuda(*shape))


def test_fake_gradients_lie_as_the_real_ones(fake):
    """Rows of a padded buffer keep their distance; rows far apart come together."""
    grad = torch.ops.sinkslot_b200.token_logprobs_grad.default
    ids, v = _cuda(8, dtype=torch.int64), _cuda(8)

    def stride(z):
        return grad(z, ids, _cuda(8, 2), v, v, None, 1.0, -100).stride()

    for dtype, lanes in ((torch.float32, 4), (torch.bfloat16, 8)):
        wide = _cuda(8, 8192, 1003, dtype=dtype)
        apart = 8192 * 1003 - 1003
        assert stride(wide[:, -1]) == (1003 + apart % lanes, 1)
        assert stride(_cuda(8, 1003 + 256, dtype=dtype)[:, :1003]) == (1003 + 256, 1)
        assert stride(_cuda(8, 1003 + 257, dtype=dtype)[:, :1003]) == (1003 + 257 % lanes, 1)
        assert stride(_cuda(8, 9000, dtype=dtype)[:, :8000]) == (9000, 1)
        assert stride(_cuda(1, 1003, dtype=dtype).expand(8, 1003)) == (1003, 1)
