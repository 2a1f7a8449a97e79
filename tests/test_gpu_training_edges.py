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


# ------------------------------------------------------------------ sums that are exact
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,tokens", [
    (40, 20, 65), (40, 20, 1000), (40, 20, 16384), (3, 771, 4097), (9, 1032, 3000),
    (50, 24, 70000), (33, 40, 90112), (33, 40, 90113), (5, 5, 120001), (2000, 16, 200001),
    (30, 130, 100003), (256, 3, 10000), (9, 256, 256), (2, 1, 65536)])
def test_table_gradient_adds_every_token(sk, rows, dim, tokens, dtype):
    """Whole-numbered outer gradients, whose float32 sums are exact in any order (under 2^24): every
    element must be the exact sum, rounded once to the type."""
    gen = _gen(rows + dim + tokens)
    table = torch.zeros(rows, dim, device="cuda", dtype=dtype, requires_grad=True)
    g = torch.randint(-8, 9, (tokens, dim), generator=gen, device="cuda")
    g[:, 0] = 1
    spread = torch.randint(0, rows, (tokens,), generator=gen, device="cuda")
    one = torch.full_like(spread, rows - 1)
    mixed = torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.7, one // 2, spread)
    runs = (torch.arange(tokens, device="cuda") // 64) % rows  # a row for each window
    for index in (spread, one, mixed, runs):
        got, = torch.autograd.grad(sk.embedding_lookup(table, index), [table], g.to(dtype))
        want = torch.zeros(rows, dim, dtype=torch.float64, device="cuda")
        want.index_add_(0, index, g.double())
        assert float(want.abs().max()) < 2 ** 24
        assert torch.equal(got, want.float().to(dtype))


# ------------------------------------------------------------------ rows known in closed form
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [
    (5, 1), (7, 2), (9, 33), (300, 1000), (40, 2049), (1, 4103), (70, 4103), (1, 32768), (3, 32771),
    (40, 32771), (400, 32771), (2, 50021), (130, 50021), (4, 131072), (80, 130001), (3, 262144),
    (300, 262144)])
def test_equal_logits(sk, rows, vocab, dtype):
    """Every term of the sum is 1 and the sum, a whole number under 2^24, is exact: the logarithm is
    -ln(vocab), rounded once (and 2.7e-8, the mean error that is taken out of other sums).  One
    element more or less is 1 / vocab: five times that at the largest size."""
    exact = math.log(vocab)
    tol = EPS32 * exact + 2.8e-8
    for off in (0, 1, 3):
        buf = torch.full((rows, vocab + 5), 77.0, device="cuda", dtype=dtype)
        z = buf[:, off:off + vocab]
        z.copy_(torch.tensor([0.0, -5.5, 1024.0, torch.finfo(dtype).min], device="cuda")
                .repeat(rows)[:rows, None])
        tokens = torch.arange(rows, device="cuda") * 977 % vocab
        lp, h = sk.token_logprobs(z, tokens, entropy=True)
        plain = sk.token_logprobs(z, tokens)
        for got, want in ((lp, -exact), (plain, -exact), (h, exact)):
            assert float((got.double() - want).abs().max()) <= tol, (off, got[:3], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(5600, 13001), (2300, 32771), (1400, 50021), (1200, 131072),
                                        (600, 262144)])
def test_equal_logits_in_one_pass(sk, rows, vocab, dtype):
    exact = math.log(vocab)
    z = torch.full((rows, vocab + 3), 9.0, device="cuda", dtype=dtype)[:, 1:vocab + 1]
    z.fill_(-3.0)
    z.requires_grad_()
    tokens = torch.arange(rows, device="cuda") * 977 % vocab
    old = torch.full((rows,), -exact, device="cuda")
    r = sk.policy_loss_from_logits(z, tokens, old, torch.ones(rows, device="cuda"),
                                   grad_scale=float(rows))
    assert float((r.logp.double() + exact).abs().max()) <= EPS32 * exact + 2.8e-8
    grad, = torch.autograd.grad(r.loss, [z], torch.tensor(float(rows), device="cuda"))
    ratio = (r.logp.double() - old.double()).exp()
    want = (ratio / vocab)[:, None].expand(rows, vocab).clone()
    want[torch.arange(rows), tokens] -= ratio
    # ratio, norm, scale, 1 / s and their products: eight float32 roundings, then the type's
    _close(grad, want, (half_step(dtype) + 8 * EPS32) * want.abs() + tiny(dtype), "grad")


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 64), (torch.bfloat16, 1000),
                                         (torch.float16, 5001), (torch.bfloat16, 32768),
                                         (torch.float32, 50021), (torch.bfloat16, 131072),
                                         (torch.bfloat16, 262144)])
def test_log_probabilities_have_no_mean_error(sk, dtype, vocab):
    """Over 16384 rows the roundings average out: a result's step / sqrt(12) and about as much from
    the sum, over sqrt(16384), four times that as the bound.  What is left is a mean error, held
    under a quarter of float32's half step at 1, so that no sequence's sum shows it."""
    rows, total, steps = 16384, 0.0, 0.0
    gen = _gen(vocab)
    for part in range(4):
        z = torch.randn(rows // 4, vocab, generator=gen, device="cuda", dtype=dtype) * 2
        tokens = torch.randint(0, vocab, (rows // 4,), generator=gen, device="cuda")
        lp = sk.token_logprobs(z, tokens).double()
        for a in range(0, rows // 4, 128):
            want = ref.logprobs64(z[a:a + 128], tokens[a:a + 128])[0]
            total += float((lp[a:a + 128] - want).sum())
            steps += float(torch.exp2(torch.floor(torch.log2(want.abs())) - 23).sum())
    noise = 4 * math.sqrt(2 / 12) * (steps / rows) / math.sqrt(rows)
    assert abs(total / rows) <= EPS32 / 4 + noise, (total / rows, EPS32 / 4 + noise)


# ------------------------------------------------------------------ policy loss from logits
def _policy_case(sk, t, vocab, dtype, off, pad, *, kl, per_token, lo, hi, average, outer=1.0,
                 seed=0):
    """Loss, KL and gradient against 64 bits; `outer`: the outer gradient over grad_scale."""
    gen = _gen(t + vocab + seed)
    buf = (torch.randn(t, vocab + pad, generator=gen, device="cuda") * 2).to(dtype)
    z = buf[:, off:off + vocab].detach()
    tokens = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    lp, *_ = ref.logprobs64(z, tokens)
    step = 0.25 * torch.randn(t, generator=gen, device="cuda").double()
    for edge in (math.log1p(-lo), math.log1p(hi)):  # 1e-3 from the borders: far above logp's error
        step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
    old, refp = (lp - step).float(), (lp + 0.2).float()
    mask = torch.rand(t, generator=gen, device="cuda") > 0.25
    mask[0] = True
    count = 5
    offsets = _packed(t, count, t)
    adv = torch.randn(t if per_token else count, generator=gen, device="cuda")
    scale = 64.0 * t
    args = dict(ref_logp=refp, mask=mask, offsets=offsets, kl_coef=0.05, kl=kl, clip_low=lo,
                clip_high=hi, average=average)
    z.requires_grad_()
    r = sk.policy_loss_from_logits(z, tokens, old, adv, grad_scale=scale, **args)
    grad, = torch.autograd.grad(r.loss, [z], torch.tensor(scale * outer, device="cuda"))
    zd = z.detach()
    ltol = ref.logp_tolerance(zd, tokens, 1.0, vocab)
    leaf = lp.clone().requires_grad_()
    want, want_kl, share = ref.policy64(leaf, old, adv, refp, mask, offsets, lo, hi, 0.05, kl,
                                        average)
    big = 4 * float(adv.abs().max()) * float(ltol.max()) + 100 * EPS32
    _close(r.loss.detach(), want.detach(), big, "loss")
    _close(r.kl, torch.tensor(want_kl, device="cuda"), float(ltol.max()) + 100 * EPS32, "kl")
    _close(r.clip_fraction, torch.tensor(share, device="cuda"), 2 * EPS32, "clip fraction")
    coef, = torch.autograd.grad(want, [leaf])
    coef = coef * scale * outer
    made_of = ref.policy_coef_size(lp, old, adv, refp, mask, offsets, 0.05, average) * scale * outer
    wgrad = ref.logprobs_grad64(zd, tokens, coef) * mask[:, None]
    onto = ref.logprobs_grad64(zd, tokens, made_of).abs() * mask[:, None]
    tol = _grad_tolerance(zd, tokens, coef, None, 1.0, wgrad, dtype) \
        + onto * (4 * float(ltol.max()) + 32 * EPS32)
    if outer != 1.0:  # rounded to the type before it was scaled
        tol = tol + half_step(dtype) * (wgrad.abs() + tol) + outer * tiny(dtype) + 2 * EPS32 * wgrad.abs()
    _close(grad, wgrad, tol, "grad")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,vocab", [(60, 1003), (5600, 13001), (1400, 50021)])
@pytest.mark.parametrize("kl,per_token,lo,hi,average", [
    ("k1", True, 0.1, 0.3, "token"), ("k2", True, 0.3, 0.15, "sequence"),
    ("k1", False, 0.05, 0.4, "sequence"), ("k3", True, 0.2, 0.28, "sequence")])
def test_policy_from_logits_options(sk, t, vocab, dtype, kl, per_token, lo, hi, average):
    """Every KL estimate, advantages per token and unequal clip borders, in three passes and in one."""
    _policy_case(sk, t, vocab, dtype, 0, 0, kl=kl, per_token=per_token, lo=lo, hi=hi,
                 average=average)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,vocab,off,pad", [(30, 999, 0, 0), (30, 999, 1, 6), (17, 20, 3, 8),
                                             (300, 4096, 2, 70), (5600, 13001, 0, 0),
                                             (2300, 32771, 5, 64)])
def test_policy_from_logits_scales_its_gradient(sk, t, vocab, off, pad, dtype):
    """An outer gradient other than grad_scale: the finished gradient is scaled in place, on rows of
    any start and distance."""
    for outer in (3.0, 0.75):
        _policy_case(sk, t, vocab, dtype, off, pad, kl="k3", per_token=False, lo=0.2, hi=0.2,
                     average="token", outer=outer)


@pytest.mark.parametrize("t,vocab", [(40, 1003), (5600, 13001)])  # three passes; one pass
def test_tokens_without_advantage_count_nothing_at_any_ratio(sk, t, vocab):
    """A = 0 (a group of equal rewards): r A is 0 also where r = e^190 is past float32."""
    gen = _gen(t)
    z = torch.randn(t, vocab, generator=gen, device="cuda").half().requires_grad_()
    tokens = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    lp = sk.token_logprobs(z, tokens)
    adv = torch.ones(t, device="cuda")
    old = lp.detach().clone()
    adv[::3] = 0.0
    old[::3] -= 190.0
    want = -adv.double().mean()  # ratios of 1, rounded nowhere
    coef = (-adv / t).requires_grad_(False)
    wgrad, = torch.autograd.grad(lp, [z], coef, retain_graph=True)
    split = sk.policy_loss(lp, old, adv)
    fused = sk.policy_loss_from_logits(z, tokens, old, adv)
    for r in (split, fused):
        # (the fused pass may round a log-probability of 12 or less to the step beside old's)
        assert abs(float(r.loss.detach()) - float(want)) <= 16 * EPS32
        grad, = torch.autograd.grad(r.loss, [z], retain_graph=r is split)
        torch.testing.assert_close(grad, wgrad, rtol=2 * half_step(z.dtype) * 2, atol=2 * tiny(z.dtype) * 2)
        assert not grad[::3].any()


# ------------------------------------------------------------------ other ways through autograd
def test_saved_tensor_hooks(sk):
    """What is saved for the backward pass, moved to the host and back: the same gradients."""
    want = _step(sk, _step_state(71))
    with torch.autograd.graph.save_on_cpu():
        got = _step(sk, _step_state(71))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_compiled_steps(sk):
    """Each function with its backward pass under torch.compile (its own kernels, no generated
    ones): the eager results, bit for bit."""
    s = _step_state(72)

    def lookup(table):
        return sk.embedding_lookup(table, s["ids"], scale=2.0).square().sum()

    def entropies(z):
        lp, h = sk.token_logprobs(z, s["tokens"], temperature=0.7, entropy=True)
        return (lp + 0.1 * h).sum()

    def policy(lp):
        return sk.policy_loss(lp, s["old"], s["adv"], ref_logp=s["old"], kl_coef=0.1,
                              mask=s["mask"], offsets=s["offsets"]).loss

    def fused(z):
        return sk.policy_loss_from_logits(z, s["tokens"], s["old"], s["adv"], mask=s["mask"],
                                          offsets=s["offsets"]).loss * 3.0

    def preference(lp):
        return sk.preference_loss(lp, s["offsets"], mask=s["mask"]).loss

    lp = sk.token_logprobs(s["z"], s["tokens"]).detach()
    for fn, x in ((lookup, s["table"]), (entropies, s["z"]), (policy, lp), (fused, s["z"]),
                  (preference, lp)):
        results = []
        for run in (fn, torch.compile(fn, backend="aot_eager")):
            leaf = x.detach().clone().requires_grad_()
            value = run(leaf)
            value.backward()
            results.append((value.detach(), leaf.grad))
        for a, b in zip(*results):
            assert torch.equal(a, b), fn.__name__


def test_in_place_steps_on_the_loss(sk):
    """loss /= n and loss += other, as a training loop writes them, before the backward pass."""
    s = _step_state(73)
    lp = sk.token_logprobs(s["z"], s["tokens"])
    for make in (lambda: sk.policy_loss(lp, s["old"], s["adv"], offsets=s["offsets"]),
                 lambda: sk.preference_loss(lp, s["offsets"]),
                 lambda: sk.policy_loss_from_logits(s["z"], s["tokens"], s["old"], s["adv"],
                                                    offsets=s["offsets"])):
        want, = torch.autograd.grad(make().loss * 0.25 + 1.0, [s["z"]], retain_graph=True)
        loss = make().loss
        loss *= 0.25
        loss += torch.ones((), device="cuda")
        got, = torch.autograd.grad(loss, [s["z"]], retain_graph=True)
        assert torch.equal(got, want)


def test_batched_outer_gradients(sk):
    """Several outer gradients at once (vectorised over the backward pass): each as by itself, or an
    error where the gradient is handed over in place."""
    s = _step_state(74)
    lp = sk.token_logprobs(s["z"], s["tokens"])
    loss = sk.policy_loss(lp, s["old"], s["adv"], offsets=s["offsets"]).loss
    pref = sk.preference_loss(lp, s["offsets"]).loss
    x = sk.embedding_lookup(s["table"], s["ids"])
    outer = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    for out, leaf, g in ((loss, s["z"], outer), (pref, s["z"], outer),
                         (x, s["table"], torch.stack([k * s["outer"] for k in outer]))):
        got, = torch.autograd.grad(out, [leaf], g, retain_graph=True, is_grads_batched=True)
        for k in range(3):
            want, = torch.autograd.grad(out, [leaf], g[k], retain_graph=True)
            assert torch.equal(got[k], want)
    fused = sk.policy_loss_from_logits(s["z"], s["tokens"], s["old"], s["adv"],
                                       offsets=s["offsets"]).loss
    with pytest.raises(RuntimeError):
        torch.autograd.grad(fused, [s["z"]], outer, is_grads_batched=True)


# ------------------------------------------------------------------ sizes past 32 bits
@pytest.mark.parametrize("dim", [4096, 4099])
def test_lookup_of_more_than_2_to_the_32_elements(sk, dim):
    """Whole numbers: the rows are the table's own, the table's gradient an exact sum."""
    rows, tokens = 700, 1 << 20
    tokens += 77
    assert tokens * dim > 2 ** 32
    gen = _gen(dim)
    table = torch.randint(-99, 100, (rows, dim), generator=gen, device="cuda").bfloat16()
    table.requires_grad_()
    index = torch.randint(0, rows, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    out = sk.embedding_lookup(table, index)
    part = 1 << 16
    for a in range(0, tokens, part):
        assert torch.equal(out.detach()[a:a + part], table.detach()[index[a:a + part].long()])
    g = torch.empty_like(out)
    want = torch.zeros(rows, dim, device="cuda", dtype=torch.float64)
    for a in range(0, tokens, part):
        n = min(part, tokens - a)
        g[a:a + n] = torch.randint(-3, 4, (n, dim), generator=gen, device="cuda").bfloat16()
        want.index_add_(0, index[a:a + n].long(), g[a:a + n].double())
    got, = torch.autograd.grad(out, [table], g)
    assert torch.equal(got, want.bfloat16())
