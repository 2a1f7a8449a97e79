"""Plain 64-bit forms of the training operators, and how far a correct kernel may be from them."""

from __future__ import annotations

import math

import torch

EPS32 = 2.0 ** -24  # half a step of float32


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half the smallest subnormal step (results under it may round to 0)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def logprobs64(z, tokens, temperature=1.0, ignore=-100):
    """(logp, entropy, softmax, counted) in 64 bits; z (rows, vocab), tokens (rows,)."""
    rows, vocab = z.shape
    keep = tokens != ignore
    z = torch.where(keep[:, None], z.double(), torch.zeros_like(z, dtype=torch.float64)) / temperature
    inside = (tokens >= 0) & (tokens < vocab)
    m = z.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    z = z - m  # first: rows at a type's lowest value would swallow the logarithm
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    empty = s[:, 0] == 0
    p = torch.where(empty[:, None], torch.zeros_like(e), e / s.clamp_min(1e-300))
    lse = torch.log(s)
    lp = z.gather(1, tokens.clamp(0, vocab - 1)[:, None].long()) - lse
    lp = torch.where(empty, torch.full_like(lp[:, 0], -math.inf), lp[:, 0])
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    logs = torch.where(p > 0, z - lse, torch.zeros_like(z))
    h = -(p * logs).sum(1)
    zero = torch.zeros_like(lp)
    return torch.where(keep, lp, zero), torch.where(keep, h, zero), p, keep, logs, empty


def logprobs_grad64(z, tokens, g, gh=None, temperature=1.0, ignore=-100):
    _, h, p, keep, logs, empty = logprobs64(z, tokens, temperature, ignore)
    vocab = z.shape[1]
    d = -p * g.double()[:, None]
    inside = (tokens >= 0) & (tokens < vocab) & ~empty
    hit = torch.zeros_like(p)
    hit.scatter_(1, tokens.clamp(0, vocab - 1)[:, None].long(),
                 torch.where(inside, g.double(), torch.zeros_like(g.double()))[:, None])
    d = d + hit
    if gh is not None:
        d = d - gh.double()[:, None] * p * (logs + h[:, None])
    return torch.where(keep[:, None], d, torch.zeros_like(d)) / temperature


def sum_error(vocab: int) -> float:
    """Relative error of a row's sum of exponentials in float32: each term's own (the exponential
    and the roundings of its argument, whose size the term's weight keeps under 1) and one half
    step for each addition that a thread makes (it reads at least 1/32 of the row, two sums at a
    time), 16 more to rescale and join."""
    return (vocab / 64 + 16 + 12) * EPS32


def logp_tolerance(z, tokens, temperature, vocab):
    """|z_tok - m| / T and ln s are rounded once each, their difference once."""
    zt = z.double().nan_to_num(0.0, math.inf, -math.inf) / temperature
    m = zt.amax(1)
    at = zt.gather(1, tokens.clamp(0, vocab - 1)[:, None].long())[:, 0]
    size = (m - at).abs().nan_to_num(0.0, 0.0, 0.0) + math.log(vocab + 1.0) + 1.0
    return 4 * EPS32 * size + sum_error(vocab)


def policy64(logp, old, adv, ref=None, mask=None, offsets=None, lo=0.2, hi=0.2, kl_coef=0.0,
             kl="k3", average="token"):
    """(loss, kl, clip fraction) in 64 bits, sequence by sequence; differentiable in logp."""
    t = logp.numel()
    o = [0, t] if offsets is None else [int(v) for v in offsets]
    keep = torch.ones(t, dtype=torch.bool, device=logp.device) if mask is None else mask
    logp = logp.double()
    spans = [(a, b, int(keep[a:b].sum())) for a, b in zip(o[:-1], o[1:])]
    total = sum(n for _, _, n in spans)
    used = sum(n > 0 for _, _, n in spans)
    loss, mean_kl, clipped = 0.0 * logp.nan_to_num(0.0, 0.0, 0.0).sum(), 0.0, 0
    for i, (a, b, n) in enumerate(spans):
        if n == 0:
            continue
        k = keep[a:b]
        lp = logp[a:b][k]
        av = adv.double()[a:b][k] if adv.numel() == t else adv.double()[i].expand(n)
        r = torch.exp(lp - old.double()[a:b][k])
        rc = r.clamp(1.0 - lo, 1.0 + hi)
        u, v = r * av, rc * av
        each = -torch.where(u <= v, u, v)
        clipped += int((v < u).sum())
        if ref is not None:
            d = ref.double()[a:b][k] - lp
            est = {"k1": -d, "k2": d * d / 2, "k3": torch.expm1(d) - d}[kl]
            each = each + kl_coef * est
        else:
            est = torch.zeros_like(lp)
        w = 1.0 / total if average == "token" else 1.0 / (n * used)
        loss = loss + w * each.sum()
        mean_kl = mean_kl + w * float(est.detach().sum())
    return loss, mean_kl, clipped / max(total, 1)


def policy_coef_size(logp, old, adv, ref, mask, offsets, kl_coef, average):
    """What a token's coefficient is made of: weight * (r |A| + kl_coef e^(ref - logp)).  An error
    of logp goes into r and into e^gap relative to themselves, so the coefficient's own error is
    that error (and the roundings) times this size, however much of it cancels."""
    t = logp.numel()
    o = [0, t] if offsets is None else [int(v) for v in offsets]
    keep = torch.ones(t, dtype=torch.bool, device=logp.device) if mask is None else mask
    size = torch.zeros(t, dtype=torch.float64, device=logp.device)
    spans = [(a, b, int(keep[a:b].sum())) for a, b in zip(o[:-1], o[1:])]
    total, used = sum(n for _, _, n in spans), sum(n > 0 for _, _, n in spans)
    for i, (a, b, n) in enumerate(spans):
        if n:
            av = adv.double()[a:b] if adv.numel() == t else adv.double()[i]
            part = torch.exp(logp[a:b] - old[a:b].double()) * av.abs() \
                + kl_coef * torch.exp(ref[a:b].double() - logp[a:b])
            size[a:b] = part * keep[a:b] / (total if average == "token" else n * used)
    return size


def preference64(logp, offsets, ref=None, mask=None, beta=0.1, smoothing=0.0, kind="sigmoid",
                 normalize=False):
    """(loss, rewards of all sequences) in 64 bits; differentiable in logp."""
    t = logp.numel()
    o = [int(v) for v in offsets]
    keep = torch.ones(t, dtype=torch.bool, device=logp.device) if mask is None else mask
    x = logp.double() - (ref.double() if ref is not None else 0.0)
    sums = []
    for a, b in zip(o[:-1], o[1:]):
        k = keep[a:b]
        v = x[a:b][k].sum()
        sums.append(v / max(1, int(k.sum())) if normalize else v)
    r = torch.stack(sums)
    n = r.numel() // 2
    h = beta * (r[:n] - r[n:])
    f = torch.nn.functional.logsigmoid
    if kind == "sigmoid":
        each = -(1 - smoothing) * f(h) - smoothing * f(-h)
    elif kind == "hinge":
        each = torch.relu(1 - h)
    else:
        each = (h / beta - 0.5 / beta) ** 2
    return each.mean(), beta * r.detach()


def lookup_grad64(g, index, rows, scale, padding=None):
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device)
    size = torch.zeros_like(out)
    ok = (index >= 0) & (index < rows)
    if padding is not None:
        ok &= index != padding
    at = index[ok].long()
    out.index_add_(0, at, g.double()[ok])
    size.index_add_(0, at, g.double()[ok].abs())
    count = torch.zeros(rows, dtype=torch.float64, device=g.device)
    count.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return out * scale, size * abs(scale), count
