"""The training operators on the device against plain 64-bit forms: table lookup, token
log-probabilities, policy and preference losses, each with its gradient, at the sizes, masks and
layouts where they can go wrong.

Tolerances follow from the arithmetic (tests/training_ref.py): half a step of the result's type,
plus the float32 roundings on the way.
"""

from __future__ import annotations

import math

import pytest
import torch

import training_ref as ref
from training_ref import EPS32, half_step, tiny

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def sk():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import sinkslot_b200
    sinkslot_b200.load_library()
    return sinkslot_b200


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _close(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN pattern"
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf]), f"{what}: inf"
    fine = ~(inf | want.isnan())
    tol = (tol if torch.is_tensor(tol) else torch.tensor(tol, device=got.device)).double()
    over = (got - want).abs() - tol
    over = over[fine]
    assert not over.numel() or float(over.max()) <= 0, \
        f"{what}: over its tolerance by {float(over.max()):.3e}, " \
        f"worst error {float((got - want)[fine].abs().max()):.3e}"


# ------------------------------------------------------------------ log-probabilities
def _grad_tolerance(z, tokens, g, gh, temperature, want, dtype):
    """Half a step of the type, the smallest subnormal, and the float32 roundings: of p
    relative to itself (its exponent's argument, at most 104 before p is 0 in float32, its sum
    and coefficient), and of the terms where they are added."""
    vocab = z.shape[1]
    _, h, p, _, logs, _ = ref.logprobs64(z, tokens, temperature)
    g = g.double().abs()[:, None] / temperature
    rel = ref.sum_error(vocab) + (4 * logs.abs().clamp_max(104) + 8) * EPS32
    size = g * p
    if gh is not None:
        gh = gh.double().abs()[:, None] / temperature
        ent = h.abs()[:, None] + logs.abs().clamp_max(104)
        size = size + gh * p * (ent + 1)
        # H itself: its float32 error times p
        size_h = gh * p * (math.log(vocab + 1.0) + 1.0) * (ref.sum_error(vocab) + 8 * EPS32) * 4
    else:
        size_h = 0.0
    # terms under 2^-126 flush to zero in the exponential
    return half_step(dtype) * want.abs() + tiny(dtype) + size * rel + size_h + 2 * EPS32 * want.abs() \
        + 2.0 ** -120


def _check_logprobs(sk, z, tokens, temperature=1.0, entropy=False, seed=0, ignore=-100):
    """z: a leaf (any layout), tokens: the rows' shape."""
    gen = _gen(seed + 1)
    z.requires_grad_()
    g = torch.randn(tokens.shape, generator=gen, device="cuda")
    gh = torch.randn(tokens.shape, generator=gen, device="cuda") if entropy else None
    out = sk.token_logprobs(z, tokens, temperature=temperature, entropy=entropy,
                            ignore_index=ignore)
    lp, ent = out if entropy else (out, None)
    assert lp.dtype == torch.float32 and lp.shape == tokens.shape
    grad, = torch.autograd.grad([lp, ent] if entropy else [lp], [z], [g, gh] if entropy else [g])
    z2, t2 = z.detach().reshape(-1, z.shape[-1]), tokens.reshape(-1)
    wlp, wh, *_ = ref.logprobs64(z2, t2, temperature, ignore)
    tol = ref.logp_tolerance(z2, t2, temperature, z.shape[-1])
    _close(lp.detach().reshape(-1), wlp, tol, "logp")
    if entropy:
        vocab = z.shape[-1]
        _close(ent.detach().reshape(-1), wh,
               4 * (ref.sum_error(vocab) + 8 * EPS32) * (math.log(vocab + 1.0) + 1.0), "entropy")
    want = ref.logprobs_grad64(z2, t2, g.reshape(-1), gh.reshape(-1) if entropy else None,
                               temperature, ignore)
    assert grad.dtype == z.dtype and grad.shape == z.shape
    _close(grad.reshape(-1, z.shape[-1]), want,
           _grad_tolerance(z2, t2, g.reshape(-1), gh.reshape(-1) if entropy else None, temperature,
                           want, z.dtype), "grad")
    return lp, grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (9, 33), (70, 1000), (17, 2049),
                                        (4, 4096), (33, 4103), (1, 32768), (8, 32771), (2, 50021),
                                        (400, 8200)])
def test_logprobs_sizes(sk, rows, vocab, dtype):
    gen = _gen(rows * 7 + vocab)
    z = (torch.randn(rows, vocab, generator=gen, device="cuda") * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    _check_logprobs(sk, z, tokens, entropy=vocab % 2 == 1, temperature=1.0 if rows % 2 else 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [61, 5001, 20000])
def test_logprobs_layouts(sk, vocab, dtype):
    gen = _gen(vocab)
    wide = (torch.randn(12, vocab + 37, generator=gen, device="cuda") * 2).to(dtype)
    tokens = torch.randint(0, vocab, (12,), generator=gen, device="cuda")
    for off in (0, 1, 3, 37):  # a view of a padded buffer, beginning on any element
        _check_logprobs(sk, wide[:, off:off + vocab].detach(), tokens.int(), entropy=True)
    _check_logprobs(sk, wide[::3, :vocab].detach(), tokens[:4])
    one = wide[2:3, :vocab].detach().expand(12, vocab)  # the same row for every token
    z = one.clone().requires_grad_()
    shared = sk.token_logprobs(one, tokens)
    # (rows that begin on different 16-byte phases are added up in different orders: each result is
    # within its tolerance of the same value, so the two are within twice that of each other)
    _close(shared, sk.token_logprobs(z, tokens).detach(),
           2 * ref.logp_tolerance(z.detach(), tokens, 1.0, vocab), "one row shared")
    leaf = wide[2:3, :vocab].detach().clone().requires_grad_()
    total, = torch.autograd.grad(sk.token_logprobs(leaf.expand(12, vocab), tokens).sum(), [leaf])
    each, = torch.autograd.grad(sk.token_logprobs(z, tokens).sum(), [z])
    torch.testing.assert_close(total, each.sum(0, keepdim=True))
    t = wide[:, :vocab].t().contiguous().t().detach()  # column-major
    _check_logprobs(sk, t, tokens)
    _check_logprobs(sk, wide[:, :vocab].detach().reshape(3, 4, vocab).clone(), tokens.view(3, 4),
                    entropy=True)
    scalar = sk.token_logprobs(wide[0, :vocab], tokens[0])
    assert scalar.shape == ()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [19, 700, 9001, 40000])
def test_logprobs_masked_and_extreme_rows(sk, vocab, dtype):
    gen = _gen(vocab)
    z = (torch.randn(16, vocab, generator=gen, device="cuda") * 4).to(dtype)
    tokens = torch.randint(0, vocab, (16,), generator=gen, device="cuda")
    low = torch.finfo(dtype).min
    z[0] = -math.inf                      # nothing left
    z[1] = low                            # uniform at the type's lowest value
    z[2] = -math.inf
    z[2, tokens[2]] = 1.5                 # one token left
    z[3, :] = low
    z[3, tokens[3]] = 0.0                 # all others masked by the lowest value
    z[4, tokens[4]] = -math.inf           # the chosen token is impossible
    z[5] = -math.inf
    z[5, vocab - 1] = 2.0
    z[6] = 30000.0                        # far from zero
    z[7, : vocab // 2] = low
    z[8, vocab // 2:] = -math.inf
    tokens[9] = -100                      # left out, with NaN in its row
    z[9] = math.nan
    tokens[10] = vocab                    # outside the vocabulary
    tokens[11] = -1
    for entropy in (False, True):
        lp, grad = _check_logprobs(sk, z.clone(), tokens, entropy=entropy)
        assert float(lp[9]) == 0.0 and not grad[9].any()
        assert float(lp[0]) == -math.inf and not grad[0].any()
        assert lp[10].isnan() and lp[11].isnan()
        lp, _ = _check_logprobs(sk, z.clone(), tokens, entropy=entropy, temperature=2.5)
    z[12, 3] = math.nan
    z[13, 5] = math.inf
    lp = sk.token_logprobs(z, tokens)
    assert lp[12].isnan() and lp[13].isnan() and lp[14].isfinite()


def test_logprobs_gradient_against_differences(sk):
    gen = _gen(3)
    z = torch.randn(4, 37, generator=gen, device="cuda", dtype=torch.float32).requires_grad_()
    tokens = torch.randint(0, 37, (4,), generator=gen, device="cuda")
    w = torch.randn(2, 4, generator=gen, device="cuda")
    lp, h = sk.token_logprobs(z, tokens, temperature=0.8, entropy=True)
    grad, = torch.autograd.grad((w[0] * lp + w[1] * h).sum(), [z])

    def value(x):
        a, b, *_ = ref.logprobs64(x, tokens, 0.8)
        return float((w[0].double() * a + w[1].double() * b).sum())
    for r, c in [(0, 0), (1, int(tokens[1])), (2, 36), (3, 5)]:
        step = torch.zeros_like(z, dtype=torch.float64)
        step[r, c] = 1e-5
        x = z.detach().double()
        diff = (value(x + step) - value(x - step)) / 2e-5
        # the difference itself is good to 1e-5^2 times a third derivative of a few units
        assert abs(diff - float(grad[r, c])) < 1e-6


def test_logprobs_gradient_for_one_output_only(sk):
    gen = _gen(4)
    z = torch.randn(6, 900, generator=gen, device="cuda").requires_grad_()
    tokens = torch.randint(0, 900, (6,), generator=gen, device="cuda")
    lp, h = sk.token_logprobs(z, tokens, entropy=True)
    a, = torch.autograd.grad(h.sum(), [z], retain_graph=True)
    b, = torch.autograd.grad(lp.sum(), [z], retain_graph=True)
    both, = torch.autograd.grad(lp.sum() + h.sum(), [z])
    one = torch.ones(6, device="cuda")
    want = ref.logprobs_grad64(z.detach(), tokens, 0 * one, one)
    _close(a, want, _grad_tolerance(z.detach(), tokens, 0 * one, one, 1.0, want, z.dtype), "entropy")
    torch.testing.assert_close(both, a + b, rtol=1e-5, atol=1e-7)
    again, = torch.autograd.grad(sk.token_logprobs(z, tokens).sum(), [z])
    want = ref.logprobs_grad64(z.detach(), tokens, one)
    _close(b, want, _grad_tolerance(z.detach(), tokens, one, None, 1.0, want, z.dtype), "logp")
    _close(again, want, _grad_tolerance(z.detach(), tokens, one, None, 1.0, want, z.dtype), "alone")


def test_logprobs_no_rows(sk):
    z = torch.empty(0, 50, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    tokens = torch.empty(0, dtype=torch.int64, device="cuda")
    lp = sk.token_logprobs(z, tokens)
    grad, = torch.autograd.grad(lp.sum(), [z])
    assert lp.shape == (0,) and grad.shape == (0, 50)


# ------------------------------------------------------------------ lookup
def _check_lookup(sk, table, index, scale, padding=None):
    table.requires_grad_()
    rows, dim = table.shape
    out = sk.embedding_lookup(table, index, scale=scale, padding_index=padding)
    assert out.shape == (*index.shape, dim) and out.dtype == table.dtype
    flat = index.reshape(-1)
    inside = (flat >= 0) & (flat < rows)
    want = table.detach().double()[flat.clamp(0, rows - 1).long()] * scale
    want = torch.where(inside[:, None], want, torch.full_like(want, math.nan))
    # scale is held in float32; its product is rounded in float32, then to the type
    _close(out.detach().reshape(-1, dim), want,
           (half_step(table.dtype) + 3 * EPS32) * want.abs().nan_to_num(0.0) + tiny(table.dtype),
           "lookup")
    g = torch.randn(out.shape, generator=_gen(11), device="cuda").to(table.dtype)
    grad, = torch.autograd.grad(out, [table], g)
    want, size, count = ref.lookup_grad64(g.reshape(-1, dim), flat, rows, scale, padding)
    assert grad.dtype == table.dtype and grad.shape == table.shape
    # one half step of float32 for each addition, of the sum of the absolute values
    _close(grad, want, half_step(table.dtype) * want.abs() + tiny(table.dtype)
           + (count[:, None] + 4) * EPS32 * size, "table gradient")
    again, = torch.autograd.grad(sk.embedding_lookup(table, index, scale=scale,
                                                     padding_index=padding), [table], g)
    assert torch.equal(grad, again), "the order of the sums changed"
    return grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,tokens", [(1, 1, 1), (3, 3, 50), (256, 3, 10000), (7, 16, 31),
                                             (5, 8, 32), (1000, 64, 33), (50, 771, 4097),
                                             (9000, 1032, 700), (2, 257, 20000), (70000, 24, 5000),
                                             (300, 4100, 64), (150000, 5, 90112),
                                             (600, 9, 90113), (30, 7, 1001), (9, 11, 515), (1 << 20, 2, 200001), (40, 40, 65000)])
def test_lookup_sizes(sk, rows, dim, tokens, dtype):
    gen = _gen(rows + dim + tokens)
    table = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    u = torch.rand(tokens, generator=gen, device="cuda")
    index = (torch.exp(u * math.log(rows + 1.0)) - 1).long().clamp(0, rows - 1)
    _check_lookup(sk, table, index, 1.0 if tokens % 2 else 13.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,tokens", [  # on both sides of where the sort begins
    (100, 3, 16384), (100, 3, 16385), (9, 256, 256), (9, 256, 257), (9, 300, 256), (4096, 5, 300),
    (4097, 5, 300), (1024, 4, 8192), (1024, 4, 8193), (2, 1, 65536), (1, 129, 255), (2048, 512, 7)])
def test_lookup_few_rows(sk, rows, dim, tokens, dtype):
    gen = _gen(rows * dim + tokens)
    table = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    index = torch.randint(-2, rows + 2, (tokens,), generator=gen, device="cuda")
    _check_lookup(sk, table.clone(), index, 3.3, padding=rows // 2)
    _check_lookup(sk, table.clone(), index.int(), 1.0)
    _check_lookup(sk, table.clone(), torch.full_like(index, rows - 1), 0.7)


def test_lookup_one_hot_row_and_runs_at_window_ends(sk):
    gen = _gen(5)
    table = torch.randn(40, 20, generator=gen, device="cuda")
    for n in (7, 8, 9, 16, 31, 32, 33, 64, 65, 96, 1000, 70000):
        _check_lookup(sk, table.clone(), torch.full((n,), 39, device="cuda"), 2.0)
        mixed = torch.zeros(n, dtype=torch.int64, device="cuda")
        mixed[n // 2:] = 7
        mixed[-1] = 39
        _check_lookup(sk, table.clone(), mixed[torch.randperm(n, generator=gen, device="cuda")],
                      0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_padding_and_indices_outside(sk, dtype):
    gen = _gen(6)
    table = torch.randn(50, 24, generator=gen, device="cuda").to(dtype)
    index = torch.randint(0, 50, (6, 70), generator=gen, device="cuda")
    grad = _check_lookup(sk, table.clone(), index, 1.5, padding=3)
    assert not grad[3].any()
    bad = index.clone()
    bad[0, :5] = torch.tensor([-1, 50, 2 ** 40, -2 ** 40, 51], device="cuda")
    _check_lookup(sk, table.clone(), bad, 1.5, padding=3)
    out = sk.embedding_lookup(table, index, padding_index=-1)  # counts from the end, as an index
    only = torch.full((4,), 49, device="cuda")
    leaf = table.clone().requires_grad_()
    grad, = torch.autograd.grad(sk.embedding_lookup(leaf, only, padding_index=-1).float().sum(),
                                [leaf])
    assert not grad.any() and torch.equal(out, table[index])
    grad = _check_lookup(sk, table.clone(), torch.full((40,), 60, device="cuda"), 1.0)
    assert not grad.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_layouts(sk, dtype):
    gen = _gen(7)
    wide = torch.randn(60, 53, generator=gen, device="cuda").to(dtype)
    index = torch.randint(0, 20, (90,), generator=gen, device="cuda")
    for t in (wide[:, 1:33], wide[:, :48], wide[::3], wide[::2, 5:6], wide[:40].t()):
        _check_lookup(sk, t.detach(), index.int(), 0.3)
    _check_lookup(sk, wide.detach(), index.view(9, 10).t(), 0.3)
    _check_lookup(sk, wide.detach(), index[3], 0.3)
    # an outer gradient that is one row for all tokens
    leaf = wide.clone().requires_grad_()
    out = sk.embedding_lookup(leaf, index)
    g = torch.randn(1, 53, generator=gen, device="cuda").to(dtype)
    a, = torch.autograd.grad(out, [leaf], g.expand(90, 53), retain_graph=True)
    b, = torch.autograd.grad(out, [leaf], g.expand(90, 53).contiguous())
    assert torch.equal(a, b)


def test_lookup_no_tokens(sk):
    table = torch.randn(5, 4, device="cuda", requires_grad=True)
    out = sk.embedding_lookup(table, torch.empty(0, 3, dtype=torch.int64, device="cuda"))
    grad, = torch.autograd.grad(out.sum(), [table])
    assert out.shape == (0, 3, 4) and not grad.any()


# ------------------------------------------------------------------ policy loss
def _packed(tokens, count, seed, outside=0):
    gen = torch.Generator().manual_seed(seed)
    inner = tokens - 2 * outside
    cuts = torch.randint(0, inner + 1, (count - 1,), generator=gen).sort().values
    o = torch.cat([torch.tensor([0]), cuts, torch.tensor([inner])]) + outside
    return o.cuda()


def _tokens_of(seed, t):
    gen = _gen(seed)
    logp = (-3 * torch.rand(t, generator=gen, device="cuda") ** 2).requires_grad_()
    old = logp.detach() + 0.2 * torch.randn(t, generator=gen, device="cuda")
    refp = logp.detach() + 0.3 * torch.randn(t, generator=gen, device="cuda")
    mask = torch.rand(t, generator=gen, device="cuda") > 0.3
    return logp, old, refp, mask, gen


POLICY = [  # tokens, sequences (0: no offsets), outside, per token, mask, kl, coefficient, average
    (1, 0, 0, True, False, "k3", 0.0, "token"),
    (1, 1, 0, False, False, "k3", 0.1, "sequence"),
    (77, 5, 0, False, True, "k3", 0.05, "token"),
    (77, 5, 0, False, True, "k3", 0.05, "sequence"),
    (300, 40, 11, False, True, "k1", 0.2, "sequence"),
    (300, 40, 11, True, True, "k2", 0.2, "token"),
    (5000, 0, 0, True, True, "k3", 0.05, "token"),
    (40000, 2, 100, False, True, "k3", 0.05, "sequence"),
    (9000, 700, 3, False, False, "k2", 0.01, "sequence"),
    (9000, 700, 3, False, True, "k3", 0.01, "token"),
    (100000, 0, 0, False, False, "k3", 0.02, "sequence"),
]


@pytest.mark.parametrize("t,count,outside,per_token,masked,kl,coef,average", POLICY)
def test_policy_loss(sk, t, count, outside, per_token, masked, kl, coef, average):
    logp, old, refp, mask, gen = _tokens_of(t + count, t)
    offsets = _packed(t, count, t, outside) if count else None
    adv = torch.randn(t if per_token else max(count, 1), generator=gen, device="cuda")
    use_ref = coef != 0.0
    args = dict(ref_logp=refp if use_ref else None, mask=mask if masked else None,
                offsets=offsets, clip_low=0.2, clip_high=0.28, kl_coef=coef, kl=kl, average=average)
    r = sk.policy_loss(logp, old, adv, **args)
    leaf = logp.detach().double().requires_grad_()
    want, want_kl, share = ref.policy64(
        leaf, old, adv, refp if use_ref else None, mask if masked else None,
        offsets, 0.2, 0.28, coef, kl, average)
    # sums are in 64 bits; a token's terms (exp, products, the fused KL) are good to 8 half steps
    # of their sizes: ratios up to e^2, |A| up to 5, KL terms of a few units
    _close(r.loss.detach(), want.detach(), 8 * EPS32 * 40, "loss")
    _close(r.kl, torch.tensor(want_kl, device="cuda"), 8 * EPS32 * (3 + abs(want_kl)), "kl")
    _close(r.clip_fraction, torch.tensor(share, device="cuda"), 2 * EPS32, "clip fraction")
    assert torch.equal(r.logp, logp.detach()) and not r.kl.requires_grad
    outer = torch.tensor(3.0, device="cuda")
    grad, = torch.autograd.grad(r.loss, [logp], outer, retain_graph=True)
    wgrad, = torch.autograd.grad(want, [leaf], torch.tensor(3.0, device="cuda").double())
    _close(grad, wgrad, 16 * EPS32 * wgrad.abs().amax().clamp_min(1e-30), "grad")
    twice, = torch.autograd.grad(r.loss, [logp], outer)
    assert torch.equal(grad, twice)


def test_policy_gradient_against_differences(sk):
    logp, old, refp, mask, gen = _tokens_of(9, 60)
    offsets = _packed(60, 4, 3)
    adv = torch.randn(4, generator=gen, device="cuda")
    r = sk.policy_loss(logp, old, adv, ref_logp=refp, mask=mask, offsets=offsets, kl_coef=0.1,
                       average="sequence")
    grad, = torch.autograd.grad(r.loss, [logp])
    for i in range(0, 60, 7):
        step = torch.zeros(60, dtype=torch.float64, device="cuda")
        step[i] = 1e-6
        a, b = (float(ref.policy64(logp.detach().double() + s * step, old, adv, refp, mask, offsets,
                                   kl_coef=0.1, average="sequence")[0]) for s in (1, -1))
        assert abs((a - b) / 2e-6 - float(grad[i])) < 1e-6


def test_policy_loss_counts_nothing(sk):
    for average in ("token", "sequence"):
        logp, old, refp, _, _ = _tokens_of(2, 50)
        r = sk.policy_loss(logp, old, torch.ones(5, device="cuda"), ref_logp=refp, kl_coef=0.1,
                           mask=torch.zeros(50, dtype=torch.bool, device="cuda"),
                           offsets=torch.arange(0, 51, 10, device="cuda"), average=average)
        grad, = torch.autograd.grad(r.loss, [logp])
        assert float(r.loss.detach()) == 0.0 and not grad.any() and float(r.clip_fraction) == 0.0
    e = torch.empty(0, device="cuda", requires_grad=True)
    r = sk.policy_loss(e, e.detach(), torch.ones(2, device="cuda"),
                       offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    grad, = torch.autograd.grad(r.loss, [e])
    assert float(r.loss.detach()) == 0.0 and grad.shape == (0,)


def test_policy_masked_tokens_may_hold_anything(sk):
    logp, old, refp, mask, gen = _tokens_of(8, 400)
    adv = torch.randn(3, generator=gen, device="cuda")
    offsets = torch.tensor([0, 100, 100, 400], device="cuda")
    args = dict(mask=mask, offsets=offsets, kl_coef=0.1)
    clean = sk.policy_loss(logp, old, adv, ref_logp=refp, **args)
    hole = torch.where(mask, 0.0, math.nan)
    with torch.no_grad():
        dirty_logp = (logp + hole)
    dirty_logp.requires_grad_()
    dirty = sk.policy_loss(dirty_logp, old.masked_fill(~mask, -math.inf), adv, ref_logp=refp + hole,
                           **args)
    assert torch.equal(clean.loss, dirty.loss) and torch.equal(clean.kl, dirty.kl)
    a, = torch.autograd.grad(clean.loss, [logp])
    b, = torch.autograd.grad(dirty.loss, [dirty_logp])
    assert torch.equal(a, b)


def test_policy_impossible_tokens(sk):
    """logp = -inf: the ratio is 0; only a KL term to a reference that allows the token is inf."""
    logp = torch.tensor([-math.inf, -1.0], device="cuda", requires_grad=True)
    old = torch.tensor([-2.0, -1.0], device="cuda")
    adv = torch.tensor([1.0, 1.0], device="cuda")
    r = sk.policy_loss(logp, old, adv)
    grad, = torch.autograd.grad(r.loss, [logp])
    assert float(r.loss.detach()) == -0.5 and grad.tolist() == [0.0, -0.5]
    r = sk.policy_loss(logp, old, adv, ref_logp=old, kl_coef=0.1)
    assert float(r.loss.detach()) == math.inf and float(r.kl) == math.inf


def test_clip_is_decided_at_its_border(sk):
    """Ratios one float32 step of the log-probability inside and outside of the range."""
    edge = torch.tensor(math.log1p(0.2), dtype=torch.float64)
    old = torch.zeros(4, device="cuda")
    near = edge.float()
    up = torch.nextafter(near, torch.tensor(1.0))
    down = torch.nextafter(near, torch.tensor(0.0))
    logp = torch.stack([down, near, up, up]).cuda().requires_grad_()
    adv = torch.tensor([1.0, 1.0, 1.0, -1.0], device="cuda")
    r = sk.policy_loss(logp, old, adv, clip_high=0.2)
    grad, = torch.autograd.grad(r.loss, [logp])
    assert (grad != 0).tolist() == [True, bool(near.double() <= edge), False, True]


# ------------------------------------------------------------------ policy loss from logits
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,vocab,count,average,pad", [
    (1, 17, 0, "token", 0), (40, 333, 3, "sequence", 5), (64, 50021, 3, "sequence", 0),
    (9, 32768, 2, "token", 64), (700, 4099, 12, "token", 1), (300, 130000, 4, "sequence", 0),
    (50, 262144, 1, "token", 0),
    # logits larger than L2: one pass over rows by 1, 2, 4 and 8 CTAs
    (5600, 13001, 40, "sequence", 0), (2300, 32768, 5, "token", 64), (1400, 50021, 9, "sequence", 3),
    (1200, 131072, 16, "token", 0)])
def test_policy_loss_from_logits(sk, t, vocab, count, average, pad, dtype):
    gen = _gen(t + vocab)
    buf = (torch.randn(t, vocab + pad, generator=gen, device="cuda") * 2).to(dtype)
    z = buf[:, :vocab].detach()
    z[:, vocab - vocab // 16:] = -math.inf
    tokens = torch.randint(0, vocab - vocab // 16, (t,), generator=gen, device="cuda")
    temperature = 0.9
    lp64, *_ = ref.logprobs64(z, tokens, temperature)
    step = 0.25 * torch.randn(t, generator=gen, device="cuda").double()
    for edge in (math.log(0.8), math.log(1.2)):  # 1e-3 from the borders: far above logp's error
        step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
    old, refp = (lp64 - step).float(), (lp64 + 0.2).float()
    mask = torch.rand(t, generator=gen, device="cuda") > 0.25
    mask[0] = True
    if t > 10:
        z[3] = math.nan
        mask[3] = False  # a row that is left out may hold anything
        z[4, :8] = torch.finfo(dtype).min
        tokens[4] = 9
        lp64, *_ = ref.logprobs64(z.nan_to_num(0.0) if z.isnan().any() else z, tokens, temperature)
        old[4] = lp64[4].float()
        refp[4] = lp64[4].float()
    adv = torch.randn(max(count, 1), generator=gen, device="cuda")
    offsets = _packed(t, count, t) if count else None
    scale = 64.0 * t
    args = dict(ref_logp=refp, mask=mask, offsets=offsets, kl_coef=0.05, average=average)
    z.requires_grad_()
    r = sk.policy_loss_from_logits(z, tokens, old, adv, temperature=temperature, grad_scale=scale,
                                   **args)
    grad, = torch.autograd.grad(r.loss, [z], torch.tensor(scale, device="cuda"))
    zd = z.detach().masked_fill(~mask[:, None], 0.0)
    lp, *_ = ref.logprobs64(zd, tokens, temperature)
    ltol = ref.logp_tolerance(zd, tokens, temperature, vocab)
    _close(r.logp, torch.where(mask, lp, torch.zeros_like(lp)), ltol, "logp")
    leaf = lp.clone().requires_grad_()
    want, want_kl, share = ref.policy64(leaf, old, adv, refp, mask, offsets, kl_coef=0.05,
                                        average=average)
    # logp's error goes into the loss times the ratio and the advantage
    big = 4 * float(adv.abs().max()) * float(ltol.max()) + 100 * EPS32
    _close(r.loss.detach(), want.detach(), big, "loss")
    _close(r.kl, torch.tensor(want_kl, device="cuda"), float(ltol.max()) + 100 * EPS32, "kl")
    _close(r.clip_fraction, torch.tensor(share, device="cuda"), 2 * EPS32, "clip fraction")
    coef, = torch.autograd.grad(want, [leaf])
    coef = coef * scale
    wgrad = ref.logprobs_grad64(zd, tokens, coef, None, temperature) * mask[:, None]
    # the coefficient is rA - 0.05 (e^gap - 1): where the two cancel (A = -0.0122 against a gap of 0.2
    # leaves one part in 160), its error is that of the two, not one relative to what is left
    made_of = ref.policy_coef_size(lp, old, adv, refp, mask, offsets, 0.05, average) * scale
    onto = ref.logprobs_grad64(zd, tokens, made_of, None, temperature).abs() * mask[:, None]
    tol = _grad_tolerance(zd, tokens, coef, None, temperature, wgrad, dtype) \
        + onto * (4 * float(ltol.max()) + 32 * EPS32)
    _close(grad, wgrad, tol, "grad")
    assert grad.stride() == z.stride() or t == 1


def test_policy_from_logits_outer_gradient_and_second_backward(sk):
    gen = _gen(21)
    z = torch.randn(30, 999, generator=gen, device="cuda").requires_grad_()
    tokens = torch.randint(0, 999, (30,), generator=gen, device="cuda")
    lp = sk.token_logprobs(z, tokens)
    old = lp.detach() + 0.01
    adv = torch.randn(30, generator=gen, device="cuda")
    plain = sk.policy_loss(lp, old, adv)
    want, = torch.autograd.grad(plain.loss, [z], torch.tensor(5.0, device="cuda"))
    for scale in (1.0, 5.0):
        r = sk.policy_loss_from_logits(z, tokens, old, adv, grad_scale=scale)
        got, = torch.autograd.grad(r.loss, [z], torch.tensor(5.0, device="cuda"),
                                   retain_graph=True)
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-7)
        with pytest.raises(RuntimeError, match="runs once"):
            torch.autograd.grad(r.loss, [z])
    with torch.no_grad():
        r = sk.policy_loss_from_logits(z, tokens, old, adv)
    assert not r.loss.requires_grad
    torch.testing.assert_close(r.loss, plain.loss.detach(), rtol=1e-5, atol=1e-6)


# ------------------------------------------------------------------ preference loss
PREFERENCE = [  # tokens, pairs, outside, masked, kind, smoothing, normalize, with a reference
    (8, 1, 0, False, "sigmoid", 0.0, False, True),
    (50, 4, 0, True, "sigmoid", 0.1, False, True),
    (50, 4, 3, True, "hinge", 0.0, False, True),
    (500, 30, 7, True, "squared", 0.0, True, True),
    (500, 200, 0, True, "sigmoid", 0.0, False, False),
    (30000, 1, 10, True, "sigmoid", 0.0, False, True),
    (70000, 300, 0, False, "sigmoid", 0.2, True, True),
    (9000, 2, 0, False, "hinge", 0.0, True, False),
]


@pytest.mark.parametrize("t,pairs,outside,masked,kind,smoothing,normalize,with_ref", PREFERENCE)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_preference_loss(sk, t, pairs, outside, masked, kind, smoothing, normalize, with_ref,
                         index):
    logp, _, refp, mask, _ = _tokens_of(t + pairs, t)
    offsets = _packed(t, 2 * pairs, t, outside).to(index)
    r = sk.preference_loss(logp, offsets, ref_logp=refp if with_ref else None,
                           mask=mask if masked else None, beta=0.2, label_smoothing=smoothing,
                           kind=kind, normalize=normalize)
    leaf = logp.detach().double().requires_grad_()
    want, rewards = ref.preference64(leaf, offsets, refp if with_ref else None,
                                     mask if masked else None, 0.2, smoothing, kind, normalize)
    # everything is summed in 64 bits from exact differences: each result is rounded once
    got = torch.cat([r.chosen_rewards, r.rejected_rewards])
    _close(got, rewards, 2 * EPS32 * rewards.abs() + 1e-12, "rewards")
    _close(r.loss.detach(), want.detach(), 2 * EPS32 * want.detach().abs() + 1e-12, "loss")
    grad, = torch.autograd.grad(r.loss, [logp], torch.tensor(0.5, device="cuda"))
    wgrad, = torch.autograd.grad(want, [leaf], torch.tensor(0.5, device="cuda").double())
    _close(grad, wgrad, 4 * EPS32 * wgrad.abs() + 1e-30, "grad")


def test_preference_far_apart_and_impossible(sk):
    """Differences of thousands of nats neither overflow nor lose the gradient; NaN stays NaN."""
    logp = torch.tensor([0.0, -5000.0, -5000.0, 0.0], device="cuda", requires_grad=True)
    offsets = torch.arange(5, device="cuda")
    r = sk.preference_loss(logp, offsets, beta=1.0)
    grad, = torch.autograd.grad(r.loss, [logp])
    assert float(r.loss.detach()) == 2500.0 and grad.tolist() == [0.0, -0.5, 0.0, 0.5]
    bad = torch.tensor([math.nan, 0.0], device="cuda")
    assert sk.preference_loss(bad, offsets[:3]).loss.isnan()


# ------------------------------------------------------------------ together
def test_training_steps_from_table_to_losses(sk):
    """Lookup, logits, log-probabilities and both losses in one step, with the transport loss on
    points of the same table beside them; the table's gradient against 64 bits."""
    gen = _gen(31)
    vocab, dim, t = 500, 12, 160
    table = (0.5 * torch.randn(vocab, dim, generator=gen, device="cuda")).requires_grad_()
    ids = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    tokens = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    offsets = torch.tensor([0, 30, 80, 100, t], device="cuda", dtype=torch.int32)
    adv = torch.randn(4, generator=gen, device="cuda")
    x = sk.embedding_lookup(table, ids, scale=2.0)
    logits = x @ table.t()
    lp, ent = sk.token_logprobs(logits, tokens, entropy=True)
    old = lp.detach() - 0.05
    pol = sk.policy_loss(lp, old, adv, ref_logp=old, kl_coef=0.1, offsets=offsets,
                         average="sequence")
    pre = sk.preference_loss(lp, offsets, ref_logp=old)
    total = pol.loss + pre.loss - 0.01 * ent.mean()
    grad, = torch.autograd.grad(total, [table])
    leaf = table.detach().double().requires_grad_()
    z = (2.0 * leaf[ids]) @ leaf.t()
    ls = torch.log_softmax(z, 1)
    lp64 = ls.gather(1, tokens[:, None])[:, 0]
    a, _, _ = ref.policy64(lp64, old, adv, old, None, offsets, kl_coef=0.1, average="sequence")
    b, _ = ref.preference64(lp64, offsets, old)
    want, = torch.autograd.grad(a + b + 0.01 * (ls.exp() * ls).sum(1).mean(), [leaf])
    # matrix products of 12 and 160 terms in float32 on both sides of the softmax
    torch.testing.assert_close(grad.double(), want, rtol=1e-4,
                               atol=1e-5 * float(want.abs().max()))
    points = sk.embedding_lookup(table, ids)
    goal = torch.randn(150, dim, generator=gen, device="cuda")
    loss = sk.SamplesLoss(eps=0.1, L=16, n_iters=20)(points, goal)
    grad, = torch.autograd.grad(loss, [table], retain_graph=True)
    outer, = torch.autograd.grad(loss, [points])
    want, size, count = ref.lookup_grad64(outer, ids, vocab, 1.0)
    _close(grad, want, EPS32 * want.abs() + (count[:, None] + 4) * EPS32 * size, "transport")


def _step(sk, s):
    x = sk.embedding_lookup(s["table"], s["ids"], scale=2.0)
    lp, ent = sk.token_logprobs(s["z"], s["tokens"], entropy=True)
    pol = sk.policy_loss(lp, s["old"], s["adv"], mask=s["mask"], offsets=s["offsets"],
                         average="sequence")
    pre = sk.preference_loss(lp, s["offsets"], mask=s["mask"])
    fused = sk.policy_loss_from_logits(s["z"], s["tokens"], s["old"], s["adv"], mask=s["mask"],
                                       offsets=s["offsets"])
    a = torch.autograd.grad([x, pol.loss + pre.loss + ent.sum()], [s["table"], s["z"]],
                            [s["outer"], torch.ones((), device="cuda")], retain_graph=True)
    b = torch.autograd.grad(fused.loss, [s["z"]])
    return [lp.detach(), pol.loss.detach(), pre.loss.detach(), fused.loss.detach(), fused.kl, *a,
            *b]


def _step_state(seed, t=200, vocab=40000, rows=3000, dim=40):
    gen = _gen(seed)
    s = {"table": torch.randn(rows, dim, generator=gen, device="cuda").requires_grad_(),
         "ids": torch.randint(0, rows, (t,), generator=gen, device="cuda"),
         "z": torch.randn(t, vocab, generator=gen, device="cuda").bfloat16().requires_grad_(),
         "tokens": torch.randint(0, vocab, (t,), generator=gen, device="cuda"),
         "adv": torch.randn(4, generator=gen, device="cuda"),
         "mask": torch.rand(t, generator=gen, device="cuda") > 0.2,
         "offsets": torch.tensor([0, 20, 90, 90, t], device="cuda"),
         "outer": torch.randn(t, dim, generator=gen, device="cuda")}
    lp, *_ = ref.logprobs64(s["z"].detach(), s["tokens"])
    s["old"] = (lp - 0.05).float()
    return s


def test_captured_steps_replay_on_new_inputs(sk):
    """Two captured graphs, replayed in turn on inputs other than the captured ones."""
    states, graphs, outs = [_step_state(41), _step_state(42, t=90)], [], []
    for s in states:
        s["offsets"].clamp_(max=s["tokens"].numel())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(sk, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(sk, s))
        graphs.append(g)
    fresh = [_step_state(51), _step_state(52, t=90)]
    for s, f in zip(states, fresh):
        f["offsets"].clamp_(max=f["tokens"].numel())
        with torch.no_grad():
            for k, v in s.items():
                v.copy_(f[k])
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for s, got in zip(states, outs):
        for a, b in zip(got, _step(sk, s)):
            assert torch.equal(a, b)


def test_streams_other_than_the_default(sk):
    want = _step(sk, _step_state(61))
    other = _step_state(62)
    want2 = _step(sk, other)
    s = _step_state(61)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st, state in zip(streams, (s, other)):
        with torch.cuda.stream(st):
            got.append([_step(sk, state) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for g, w in zip(got, (want, want2)):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


def test_two_threads_at_once(sk):
    """Each host thread on a stream of its own, at the same time: the results of one alone."""
    from concurrent.futures import ThreadPoolExecutor
    states = [_step_state(63), _step_state(64)]
    want = [_step(sk, s) for s in states]
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [_step(sk, states[k]) for _ in range(20)][-1]
            torch.cuda.current_stream().synchronize()
        return got

    with ThreadPoolExecutor(max_workers=2) as pool:
        got = list(pool.map(work, range(2)))
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


def test_offsets_that_lie_stay_in_bounds(sk):
    """Offsets beyond the tokens, negative or falling: no access outside the tensors."""
    logp, old, refp, mask, _ = _tokens_of(70, 1000)
    for o in ([0, 5000, 9000], [-50, 300, 1000], [0, 800, 200], [900, 100, 50]):
        offsets = torch.tensor(o, device="cuda")
        r = sk.policy_loss(logp, old, torch.ones(2, device="cuda"), offsets=offsets)
        torch.autograd.grad(r.loss, [logp])
        p = sk.preference_loss(logp, offsets)
        torch.autograd.grad(p.loss, [logp])
    torch.cuda.synchronize()


def test_without_recording(sk):
    """no_grad, inference mode and inputs that need no gradient: the same values, nothing recorded."""
    s = _step_state(65)

    def values():
        lp, h = sk.token_logprobs(s["z"], s["tokens"], entropy=True)
        pol = sk.policy_loss(lp, s["old"], s["adv"], mask=s["mask"], offsets=s["offsets"])
        pre = sk.preference_loss(lp, s["offsets"], mask=s["mask"])
        fused = sk.policy_loss_from_logits(s["z"], s["tokens"], s["old"], s["adv"], mask=s["mask"],
                                           offsets=s["offsets"])
        return [sk.embedding_lookup(s["table"], s["ids"]), lp, h, *pol, *pre, *fused]

    recorded = values()
    assert [t.requires_grad for t in recorded] == [True, True, True, True, False, False, False, True,
                                                   False, False, True, False, False, False]
    with torch.no_grad():
        plain = values()
    with torch.inference_mode():
        inferred = values()
    s["z"], s["table"] = s["z"].detach(), s["table"].detach()
    constant = values()
    for a, *others in zip(recorded, plain, inferred, constant):
        for b in others:
            assert torch.equal(a, b) and not b.requires_grad


@pytest.mark.parametrize("t,vocab", [(40, 1003), (5600, 13001)])  # three passes; one pass
def test_rows_without_gradient_may_hold_anything(sk, t, vocab):
    """Tokens outside the sequences, and tokens whose gradient is zero: NaN and infinities in their
    rows reach nothing, and the gradients of their rows are zeros."""
    gen = _gen(t)
    z = torch.randn(t, vocab, generator=gen, device="cuda").half()
    tokens = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    old = torch.full((t,), -7.0, device="cuda")
    adv = torch.ones(2, device="cuda")
    offsets = torch.tensor([3, 20, t - 5], device="cuda")
    inside = torch.zeros(t, dtype=torch.bool, device="cuda")
    inside[3:t - 5] = True
    z[0], z[1], z[t - 1] = math.nan, math.inf, -math.inf
    z[t - 2, 7] = math.nan
    z.requires_grad_()
    fused = sk.policy_loss_from_logits(z, tokens, old, adv, clip_high=9.0, offsets=offsets)
    grad, = torch.autograd.grad(fused.loss, [z])
    lp = sk.token_logprobs(z, tokens)
    loss = sk.policy_loss(lp, old, adv, clip_high=9.0, offsets=offsets).loss
    split, = torch.autograd.grad(loss, [z])
    assert fused.loss.isfinite()
    for g in (grad, split):
        assert not g[~inside].any() and g[inside].isfinite().all() and g[inside].any()
    lp, h = sk.token_logprobs(z, tokens, entropy=True)
    for part in (lp[inside].sum(), h[inside].sum(), (lp[inside] + h[inside]).sum()):
        g, = torch.autograd.grad(part, [z], retain_graph=True)
        assert not g[~inside].any() and g[inside].isfinite().all() and g[inside].any()


def test_second_derivatives_are_refused(sk):
    """create_graph gives the first derivative; differentiating it again is an error."""
    gen = _gen(71)
    table = torch.randn(20, 8, generator=gen, device="cuda", requires_grad=True)
    z = torch.randn(6, 300, generator=gen, device="cuda", requires_grad=True)
    lp = -torch.rand(12, generator=gen, device="cuda")
    lp.requires_grad_()
    ids = torch.randint(0, 20, (6,), generator=gen, device="cuda")
    old = torch.full((6,), -5.0, device="cuda")
    offsets = torch.tensor([0, 5, 12], device="cuda")
    for make, leaf in [
            (lambda: sk.embedding_lookup(table, ids).square().sum(), table),
            (lambda: sk.token_logprobs(z, ids).square().sum(), z),
            (lambda: sk.policy_loss(lp, lp.detach(), torch.ones(12, device="cuda")).loss.square(), lp),
            (lambda: sk.policy_loss_from_logits(z, ids, old, old).loss, z),
            (lambda: sk.preference_loss(lp, offsets).loss.square(), lp)]:
        plain, = torch.autograd.grad(make(), [leaf])
        first, = torch.autograd.grad(make(), [leaf], create_graph=True)
        assert torch.equal(plain, first) and first.requires_grad
        # (where the loss is linear, torch finds no way from the derivative back to the leaf)
        with pytest.raises(RuntimeError, match="second derivative|not have been used"):
            torch.autograd.grad(first.sum(), [leaf])


def test_policy_from_logits_without_rows(sk):
    z = torch.empty(0, 40, device="cuda", dtype=torch.float16, requires_grad=True)
    none = torch.empty(0, device="cuda")
    r = sk.policy_loss_from_logits(z, none.long(), none, torch.ones(2, device="cuda"),
                                   offsets=torch.zeros(3, dtype=torch.int64, device="cuda"))
    grad, = torch.autograd.grad(r.loss, [z])
    assert float(r.loss.detach()) == 0.0 and grad.shape == (0, 40) and r.logp.shape == (0,)


def test_captured_large_paths(sk):
    """What only large sizes take, captured and replayed on other inputs: zeros beside the sort, the
    tile sort, one pass over rows larger than L2."""
    gen = _gen(91)

    def inputs():
        return {
            "wide": torch.randn(9000, 2048, generator=gen, device="cuda").bfloat16(),
            "ids": torch.randint(0, 9000, (700,), generator=gen, device="cuda"),
            "narrow": torch.randn(3000, 5, generator=gen, device="cuda"),
            "many": torch.randint(0, 3000, (120000,), generator=gen, device="cuda"),
            "z": torch.randn(2200, 32768, generator=gen, device="cuda").bfloat16(),
            "tokens": torch.randint(0, 32768, (2200,), generator=gen, device="cuda"),
            "old": torch.full((2200,), -11.0, device="cuda"),
            "adv": torch.randn(2200, generator=gen, device="cuda"),
            "ga": torch.randn(700, 2048, generator=gen, device="cuda").bfloat16(),
            "gb": torch.randn(120000, 5, generator=gen, device="cuda")}

    def step(s):
        a = torch.autograd.grad(sk.embedding_lookup(s["wide"], s["ids"], 3.0), [s["wide"]], s["ga"])
        b = torch.autograd.grad(sk.embedding_lookup(s["narrow"], s["many"]), [s["narrow"]], s["gb"])
        r = sk.policy_loss_from_logits(s["z"], s["tokens"], s["old"], s["adv"])
        c = torch.autograd.grad(r.loss, [s["z"]])
        return [*a, *b, r.loss.detach(), r.logp, *c]

    s = inputs()
    for k in ("wide", "narrow", "z"):
        s[k].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(s)
    fresh = inputs()
    with torch.no_grad():
        for k, v in s.items():
            v.copy_(fresh[k])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step(s)):
        assert torch.equal(a, b)


def test_launching_operators_refuse_what_their_functions_never_pass(sk):
    """Called directly: wrong types, sizes and layouts are errors before any launch."""
    ops = torch.ops.sinkslot_b200
    f, i = torch.randn(6, 8, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    v, one = torch.zeros(6, device="cuda"), torch.ones((), device="cuda")
    off = torch.tensor([0, 3, 6], device="cuda")
    for call in [
            lambda: ops.lookup(f.double(), i, 1.0),
            lambda: ops.lookup(f.t(), i, 1.0),
            lambda: ops.lookup(f, v, 1.0),
            lambda: ops.lookup_grad(f, i[:5], 4, 1.0, -1),
            lambda: ops.lookup_grad(f, i, 0, 1.0, -1),
            lambda: ops.token_logprobs(f, i[:5], 1.0, -100, False),
            lambda: ops.token_logprobs_grad(f, i, v, v, v, None, 1.0, -100),
            lambda: ops.token_logprobs_grad(f, i, torch.zeros(6, 2, device="cuda"), v, v.half(), None,
                                            1.0, -100),
            lambda: ops.policy_loss(v, v[:5], v, None, None, off, True, 0.2, 0.2, 0.0, 3, False, True),
            lambda: ops.policy_loss(v, v, v, None, None, off, False, 0.2, 0.2, 0.0, 3, False, True),
            lambda: ops.policy_loss(v, v, v, None, v, off, True, 0.2, 0.2, 0.0, 3, False, True),
            lambda: ops.policy_loss(v, v, v, None, None, off, True, 0.2, 0.2, 0.0, 4, False, True),
            lambda: ops.scale_tokens(v, v, one),
            lambda: ops.policy_loss_logits(f, i, v, v, None, None, off[:1], 1.0, True, 0.2, 0.2, 0.0,
                                           3, False, 1.0, True),
            lambda: ops.scale_rows_(f, v, 1.0),
            lambda: ops.preference_loss(v.half(), off, None, None, 0.1, 0.0, 0, False),
            lambda: ops.preference_loss(v, off[:2], None, None, 0.1, 0.0, 0, False),
            lambda: ops.preference_grad(v, off, None, one, 6)]:
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ sizes past 32 bits
def test_logits_of_more_than_2_to_the_31_elements(sk):
    """The last rows of 16400 x 131072 logits, through the log-probabilities' own kernels and the
    policy loss's."""
    t, vocab = 16400, 131072
    assert t * vocab > 2 ** 31
    gen = _gen(81)
    z = torch.empty(t, vocab, device="cuda", dtype=torch.bfloat16)
    z.normal_(0.0, 2.0, generator=gen)
    tokens = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    z.requires_grad_()
    g = torch.randn(t, generator=gen, device="cuda")
    lp = sk.token_logprobs(z, tokens)
    grad, = torch.autograd.grad(lp, [z], g)
    for rows in (slice(0, 3), slice(t - 3, t)):
        zd, tk = z.detach()[rows], tokens[rows]
        want, *_ = ref.logprobs64(zd, tk)
        _close(lp.detach()[rows], want, ref.logp_tolerance(zd, tk, 1.0, vocab), "logp")
        wgrad = ref.logprobs_grad64(zd, tk, g[rows])
        _close(grad[rows], wgrad, _grad_tolerance(zd, tk, g[rows], None, 1.0, wgrad, z.dtype),
               "grad")
    del grad
    old = lp.detach() + 0.05
    r = sk.policy_loss_from_logits(z, tokens, old, g, grad_scale=float(t))
    grad, = torch.autograd.grad(r.loss, [z], torch.tensor(float(t), device="cuda"))
    # (the two ways of summing a row are each within the tolerance of the same value)
    _close(r.logp, lp.detach(), 2 * ref.logp_tolerance(z.detach()[:8], tokens[:8], 1.0, vocab).max()
           + 8 * EPS32 * lp.detach().double().abs(), "logp, two ways")
    for rows in (slice(0, 3), slice(t - 3, t)):
        zd, tk = z.detach()[rows], tokens[rows]
        ltol = float(ref.logp_tolerance(zd, tk, 1.0, vocab).max())
        coef = -torch.exp(lp.detach()[rows].double() - old[rows].double()) * g[rows].double()
        coef = torch.where((g[rows] < 0) & (lp.detach()[rows] - old[rows] < math.log(0.8)),
                           torch.zeros_like(coef), coef)
        wgrad = ref.logprobs_grad64(zd, tk, coef)
        _close(grad[rows], wgrad, _grad_tolerance(zd, tk, coef, None, 1.0, wgrad, z.dtype)
               + wgrad.abs() * (4 * ltol + 32 * EPS32), "policy grad")


def test_table_of_more_than_2_to_the_31_elements(sk):
    rows, dim = 600000, 4096
    assert rows * dim > 2 ** 31
    gen = _gen(82)
    table = torch.empty(rows, dim, device="cuda", dtype=torch.float16)
    table.normal_(0.0, 1.0, generator=gen)
    table.requires_grad_()
    index = torch.tensor([rows - 1, 0, rows - 1, 1, rows - 2, 555555], device="cuda")
    out = sk.embedding_lookup(table, index, scale=0.5)
    assert torch.equal(out, (table.detach()[index].float() * 0.5).half())
    g = torch.randn(6, dim, generator=gen, device="cuda").half()
    grad, = torch.autograd.grad(out, [table], g)
    want = torch.zeros(4, dim, dtype=torch.float64, device="cuda")
    for k, row in enumerate([rows - 1, 0, rows - 2, 555555]):
        want[k] = 0.5 * g[index == row].double().sum(0)
    got = grad[torch.tensor([rows - 1, 0, rows - 2, 555555], device="cuda")]
    # two addends at most, of a few units: one float32 addition, then the type's rounding
    _close(got, want, half_step(torch.float16) * want.abs() + 8 * EPS32 + tiny(torch.float16), "rows")
    assert int((grad != 0).any(1).sum()) == 5
