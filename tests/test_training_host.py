"""The training operators' host side without a GPU: refusals of arguments (on fake CUDA tensors,
which no kernel sees), the operators' registration and fake shapes, and the C entries' checks."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import sinkslot_b200 as sk

OPS = ["lookup", "lookup_grad", "token_logprobs", "token_logprobs_grad", "policy_loss",
       "scale_tokens", "policy_loss_logits", "scale_rows_", "preference_loss", "preference_grad"]


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def _cuda(*shape, dtype=torch.float32, **kw):
    return torch.empty(shape, dtype=dtype, device="cuda", **kw)


def _ids(*shape, dtype=torch.int64):
    return _cuda(*shape, dtype=dtype)


@pytest.mark.parametrize("name", OPS)
def test_operator_is_registered(name):
    op = getattr(torch.ops.sinkslot_b200, name)
    assert op.default._schema.name == f"sinkslot_b200::{name}"


def test_cpu_tensors_are_refused():
    t, i = torch.randn(4, 3), torch.zeros(4, dtype=torch.int64)
    lp = torch.randn(4)
    for call in (lambda: sk.embedding_lookup(t, i), lambda: sk.token_logprobs(t, i),
                 lambda: sk.policy_loss(lp, lp, lp),
                 lambda: sk.policy_loss_from_logits(t, i, lp, lp),
                 lambda: sk.preference_loss(lp, torch.tensor([0, 2, 4]))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_lookup_refusals(fake):
    table, index = _cuda(10, 4), _ids(7)
    with pytest.raises(ValueError, match="table must be"):
        sk.embedding_lookup(_cuda(10), index)
    with pytest.raises(ValueError, match="table must be"):
        sk.embedding_lookup(_cuda(0, 4), index)
    with pytest.raises(ValueError, match="table must be float32"):
        sk.embedding_lookup(_cuda(10, 4, dtype=torch.float64), index)
    with pytest.raises(ValueError, match="index must be int32 or int64"):
        sk.embedding_lookup(table, _cuda(7))
    with pytest.raises(ValueError, match="padding_index"):
        sk.embedding_lookup(table, index, padding_index=10)
    with pytest.raises(ValueError, match="padding_index"):
        sk.embedding_lookup(table, index, padding_index=-11)


def test_logprob_refusals(fake):
    z, tok = _cuda(5, 30, dtype=torch.bfloat16), _ids(5)
    with pytest.raises(ValueError, match="tokens must have the shape"):
        sk.token_logprobs(z, _ids(4))
    with pytest.raises(ValueError, match="vocabulary axis"):
        sk.token_logprobs(_cuda(5, 0), tok)
    with pytest.raises(ValueError, match="logits must be float32"):
        sk.token_logprobs(_cuda(5, 30, dtype=torch.float64), tok)
    with pytest.raises(ValueError, match="tokens must be int32"):
        sk.token_logprobs(z, _cuda(5))
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            sk.token_logprobs(z, tok, temperature=t)


def test_policy_refusals(fake):
    lp, old, adv = _cuda(20), _cuda(20), _cuda(3)
    off, mask = _ids(4), _cuda(20, dtype=torch.bool)
    ok = dict(offsets=off, mask=mask)
    for bad, match in [
            (lambda: sk.policy_loss(_cuda(4, 5), old, adv, **ok), "logp must be"),
            (lambda: sk.policy_loss(lp, _cuda(19), adv, **ok), "old_logp must have"),
            (lambda: sk.policy_loss(lp, old.half(), adv, **ok), "old_logp must be float32"),
            (lambda: sk.policy_loss(lp.half(), old, adv, **ok), "logp must be float32"),
            (lambda: sk.policy_loss(lp, old, _cuda(4), **ok), "advantages must be one per"),
            (lambda: sk.policy_loss(lp, old, adv), "advantages must be one per"),
            (lambda: sk.policy_loss(lp, old, adv.bfloat16(), **ok), "advantages must be float32"),
            (lambda: sk.policy_loss(lp, old, adv, offsets=off, mask=_cuda(20)), "mask must be bool"),
            (lambda: sk.policy_loss(lp, old, adv, offsets=off, mask=mask[:5]), "mask must be bool"),
            (lambda: sk.policy_loss(lp, old, adv, offsets=_cuda(4)), "offsets must be int32"),
            (lambda: sk.policy_loss(lp, old, adv, offsets=off[:1]), "offsets must hold"),
            (lambda: sk.policy_loss(lp, old, adv, kl="k4", **ok), "kl must be"),
            (lambda: sk.policy_loss(lp, old, adv, average="batch", **ok), "average must be"),
            (lambda: sk.policy_loss(lp, old, adv, clip_low=-0.1, **ok), "clip_low"),
            (lambda: sk.policy_loss(lp, old, adv, clip_high=math.nan, **ok), "clip_low"),
            (lambda: sk.policy_loss(lp, old, adv, kl_coef=0.1, **ok), "needs ref_logp"),
            (lambda: sk.policy_loss(lp, old, adv, kl_coef=math.inf, ref_logp=old, **ok), "finite"),
            (lambda: sk.policy_loss(lp, _cuda(20, requires_grad=True), adv, **ok), "no gradient"),
            (lambda: sk.policy_loss_from_logits(_cuda(20), _ids(20), old, adv, **ok), "logits must"),
            (lambda: sk.policy_loss_from_logits(_cuda(20, 9), _ids(19), old, adv, **ok), "tokens"),
            (lambda: sk.policy_loss_from_logits(_cuda(20, 9), _ids(20), old, adv, grad_scale=0.0,
                                                **ok), "grad_scale"),
            (lambda: sk.policy_loss_from_logits(_cuda(20, 9), _ids(20), old, adv, grad_scale=1e200,
                                                **ok), "grad_scale"),
    ]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_preference_refusals(fake):
    lp, off = _cuda(20), _ids(5)
    for bad, match in [
            (lambda: sk.preference_loss(_cuda(2, 10), off), "logp must be"),
            (lambda: sk.preference_loss(lp, _ids(4)), "pairs"),
            (lambda: sk.preference_loss(lp, _cuda(5)), "offsets must be int32"),
            (lambda: sk.preference_loss(lp, off, kind="ranked"), "kind must be"),
            (lambda: sk.preference_loss(lp, off, beta=0.0), "beta"),
            (lambda: sk.preference_loss(lp, off, beta=math.inf), "beta"),
            (lambda: sk.preference_loss(lp, off, label_smoothing=1.0), "label_smoothing"),
            (lambda: sk.preference_loss(lp, off, label_smoothing=0.1, kind="hinge"), "smoothing"),
            (lambda: sk.preference_loss(lp, off, ref_logp=_cuda(19)), "ref_logp must have"),
            (lambda: sk.preference_loss(lp, off, ref_logp=_cuda(20, requires_grad=True)),
             "no gradient"),
            (lambda: sk.preference_loss(lp.half(), off), "logp must be float32")]:
        with pytest.raises(ValueError, match=match):
            bad()


def test_shapes_without_a_kernel(fake):
    z, tok, lp, off = _cuda(6, 50, dtype=torch.bfloat16), _ids(6), _cuda(6), _ids(5)
    assert sk.embedding_lookup(_cuda(10, 4), _ids(2, 3)).shape == (2, 3, 4)
    logp, ent = sk.token_logprobs(z.view(2, 3, 50), tok.view(2, 3), entropy=True)
    assert logp.shape == ent.shape == (2, 3) and logp.dtype == torch.float32
    r = sk.PolicyLoss(kl_coef=0.1)(lp, lp, _cuda(4), ref_logp=lp, offsets=off)
    assert r.loss.shape == r.kl.shape == r.clip_fraction.shape == ()
    r = sk.PolicyLoss(temperature=2.0).from_logits(z, tok, lp, _cuda(4), offsets=off)
    assert r.logp.shape == (6,) and r.loss.shape == ()
    p = sk.PreferenceLoss(normalize=True)(lp, off)
    assert p.loss.shape == () and p.chosen_rewards.shape == p.rejected_rewards.shape == (2,)


def test_c_entries_check_their_arguments():
    from sinkslot_b200 import _lib, build
    build.build()
    n = ctypes.c_int64(0)
    assert _lib.lib().sinkslot_abi_version() >= 102
    _lib.call("sinkslot_lookup_grad_workspace_bytes", 1000, 50, 8, ctypes.byref(n))
    assert n.value >= 16 * 1000
    _lib.call("sinkslot_loss_workspace_bytes", 10, ctypes.byref(n))
    assert n.value >= 320
    for name, args in [
            ("sinkslot_lookup", (None, 0, 4, 10, 4, None, 8, 3, 1.0, None, None)),
            ("sinkslot_lookup", (None, 7, 4, 10, 4, None, 8, 0, 1.0, None, None)),
            ("sinkslot_lookup_grad", (None, 0, 4, None, 8, 3, 10, 4, 1.0, -1, None, None, 0, None)),
            ("sinkslot_token_logprobs", (None, 2, 9, 3, 9, None, 8, -100, 1.0, None, None, None,
                                         None)),
            ("sinkslot_token_logprobs", (None, 2, 9, 3, 0, None, 8, -100, 1.0, None, None, None,
                                         None)),
            ("sinkslot_policy_loss", (None, None, None, None, 0, None, None, 8, 2, 5, 0.2, 0.2, 0.0,
                                      3, 0, None, None, None, 0, None)),
            ("sinkslot_policy_loss_logits", (None, 2, 9, 3, 9, None, 8, 1.0, None, None, None, 0,
                                             None, None, 8, 1, 0.2, 0.2, 0.0, 3, 0, 1.0, None, None,
                                             None, 0, None, 0, None)),
            ("sinkslot_policy_loss_logits", (None, 5, 9, 0, 9, None, 8, 1.0, None, None, None, 0,
                                             None, None, 8, 1, 0.2, 0.2, 0.0, 3, 0, 1.0, None, None,
                                             None, 0, None, 0, None)),
            ("sinkslot_preference_loss", (None, None, None, None, 8, 3, 5, 0.1, 0.0, 0, 0, None,
                                          None, None, None, 0, None))]:
        with pytest.raises(ValueError):
            _lib.call(name, *args)
