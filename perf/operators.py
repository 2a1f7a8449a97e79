"""Training operators over tables, logits and token log-probabilities: the cases that are measured.

Four operators, each with its gradient:

* ``lookup``: rows of a table by index, times a scale; the table's gradient.
* ``logprob``: log-probability (and entropy) of chosen tokens under logits; the logits' gradient.
* ``preference``: the paired log-ratio loss over packed sequences; the gradient of the token
  log-probabilities, or of the logits that they come from.
* ``policy``: the clipped policy loss with a KL term; likewise.

``own`` says which side ``run`` computes: elementary torch operations, or this package's operators.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
IGNORE = -100


# ---------------------------------------------------------------------------- cases
def _lookup(name, rows, dim, tokens, dtype, scale, padding=False):
    return {"name": name, "op": "lookup", "rows": rows, "dim": dim, "tokens": tokens,
            "dtype": dtype, "scale": scale, "padding": padding}


def _logprob(name, tokens, vocab, dtype, temperature=1.0, entropy=False, prompt=0.0, pad=0):
    return {"name": name, "op": "logprob", "tokens": tokens, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "entropy": entropy, "prompt": prompt, "pad": pad}


def _preference(name, pairs, tokens, vocab=0, dtype="float32", kind="sigmoid", smoothing=0.0,
                normalize=False, prompt=0.0):
    return {"name": name, "op": "preference", "pairs": pairs, "tokens": tokens, "vocab": vocab,
            "dtype": dtype, "kind": kind, "smoothing": smoothing, "normalize": normalize,
            "prompt": prompt}


def _policy(name, sequences, tokens, vocab=0, dtype="float32", average="token", kl_coef=0.05,
            temperature=1.0, prompt=0.0, pad=0):
    return {"name": name, "op": "policy", "sequences": sequences, "tokens": tokens, "vocab": vocab,
            "dtype": dtype, "average": average, "kl_coef": kl_coef, "temperature": temperature,
            "prompt": prompt, "pad": pad}


def listed():
    return [
        # a learned palette of 256 colours looked up for a cloud of 10^4 points
        _lookup("lookup palette", 256, 3, 10000, "float32", 1.0),
        # an odd width, every row of a small table used many times
        _lookup("lookup odd width", 5003, 771, 40009, "float16", 0.125, padding=True),
        # the token table of a training step: most rows unused, a few very hot
        _lookup("lookup training step", 131072, 4096, 16384, "bfloat16", 64.0),
        # a few tokens being scored
        _logprob("logprob few rows", 8, 32768, "bfloat16"),
        # odd vocabulary (rows that begin on no vector boundary), entropy, a prompt left out
        _logprob("logprob odd entropy", 2049, 50021, "float16", 1.0, True, 0.25),
        # full-precision logits at a temperature, a view of a padded buffer
        _logprob("logprob float32", 4096, 32768, "float32", 0.7, False, 0.0, 64),
        # log-probabilities at hand, a small batch of pairs
        _preference("preference few pairs", 4, 1999),
        # log-probabilities at hand, a whole batch with its prompts masked
        _preference("preference batch", 256, 393216, smoothing=0.1, prompt=0.4),
        # the training step from the logits on
        _preference("preference from logits", 2, 8192, 131072, "bfloat16", prompt=0.25),
        # log-probabilities at hand, packed sequences averaged one by one
        _policy("policy packed", 32, 16384, average="sequence", prompt=0.25),
        # a small batch from the logits on, odd vocabulary
        _policy("policy small from logits", 3, 64, 50021, "float16", "sequence"),
        # the training step from the logits on
        _policy("policy from logits", 16, 8192, 131072, "bfloat16", "token", 0.05, 0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "logprob", "preference", "policy", "preference", "policy"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op == "lookup":
        dim = _log_int(rng, 1, 8192)
        tokens = _log_int(rng, 1, min(1 << 20, (1 << 26) // dim))
        rows = _log_int(rng, 2, min(1 << 18, (1 << 29) // (dim + 1)))
        return _lookup("", rows, dim, tokens, dtype, round(rng.uniform(0.05, 70.0), 3),
                       rng.random() < 0.5) | {"name": "lookup %d x %d, %d" % (rows, dim, tokens)}
    vocab = _log_int(rng, 16, 1 << 18)
    tokens = _log_int(rng, 1, min(1 << 17, (1 << 29) // vocab))
    prompt = rng.choice([0.0, rng.uniform(0.05, 0.7)]) if tokens >= 64 else 0.0
    pad = rng.choice([0, 0, rng.randint(1, 200)])
    temperature = rng.choice([1.0, round(rng.uniform(0.4, 1.6), 2)])
    if op == "logprob":
        return _logprob("logprob %d x %d" % (tokens, vocab), tokens, vocab, dtype, temperature,
                        rng.random() < 0.5, prompt, pad)
    if rng.random() < 0.4:  # log-probabilities at hand
        tokens, vocab, dtype, pad, temperature = _log_int(rng, 8, 1 << 20), 0, "float32", 0, 1.0
    if tokens < 64:
        prompt = 0.0
    count = _log_int(rng, 1, min(512, max(1, tokens // 2)))
    if op == "preference":
        return _preference("preference %d, %d x %d" % (count, tokens, vocab), count, tokens, vocab,
                           dtype, rng.choice(["sigmoid", "sigmoid", "squared"]),
                           rng.choice([0.0, 0.1]), rng.random() < 0.3, prompt)
    return _policy("policy %d, %d x %d" % (count, tokens, vocab), count, tokens, vocab, dtype,
                   rng.choice(["token", "sequence"]), rng.choice([0.0, 0.05]), temperature, prompt,
                   pad)


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    t = case["tokens"]
    if case["op"] == "lookup":
        v, d = case["rows"], case["dim"]
        # the rows that are used and the outer gradient in, the looked-up rows and the table's gradient out
        return {"bytes": size * d * (min(t, v) + 2 * t + v) + 16 * t, "flops": 3 * t * d}
    kept = t * (1.0 - case["prompt"])
    # logits of the counted tokens in, the gradient of all of them out; a few values for each token
    at_logits = size * case["vocab"] * (kept + t)
    return {"bytes": at_logits + 24 * t, "flops": 8 * kept * max(1, case["vocab"])}


# ---------------------------------------------------------------------------- inputs
def _offsets(count, tokens, gen, device):
    """Cuts of `tokens` into `count` sequences, of any length, a few of them perhaps empty."""
    cuts = torch.randint(0, tokens + 1, (max(0, count - 1),), generator=gen, device=device)
    ends = torch.tensor([0, tokens], device=device)
    return torch.cat([ends[:1], cuts.sort().values, ends[1:]]).to(torch.int32)


def _loss_scale(case):
    """What the loss is multiplied by before its backward pass: half-precision gradients of one
    over the number of tokens would vanish."""
    return 16.0 * 2.0 ** int(math.log2(case["tokens"])) if case["dtype"] == "float16" else 1.0


def _logits(case, gen, device):
    """Logits of a language model's shape: wide normal values, the chosen token among the likely
    ones, the last entries of the vocabulary switched off."""
    t, v, dtype = case["tokens"], case["vocab"], DTYPES[case["dtype"]]
    buf = torch.empty(t, v + case.get("pad", 0), dtype=dtype, device=device)
    buf.normal_(0.0, 2.5, generator=gen)
    tokens = torch.randint(0, v - v // 64, (t,), generator=gen, device=device)
    z = buf[:, :v]
    boost = 6.0 * torch.rand(t, 1, generator=gen, device=device)
    z.scatter_add_(1, tokens[:, None], boost.to(dtype))
    if v >= 64:
        z[:, v - v // 64:] = float("-inf")
    return z, tokens


def _true_logp(z, tokens, temperature):
    out = torch.empty(z.shape[0], dtype=torch.float64, device=z.device)
    for i in range(0, z.shape[0], 1024):
        c = z[i:i + 1024].to(torch.float32) / temperature
        out[i:i + 1024] = (c.gather(1, tokens[i:i + 1024, None])[:, 0]
                           - torch.logsumexp(c, 1)).to(torch.float64)
    return out


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    state = {"case": case}
    t = case["tokens"]
    if case["op"] == "lookup":
        v, d, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
        state["table"] = torch.randn(v, d, generator=gen, device=device, dtype=torch.float32) \
            .to(dtype).requires_grad_()
        # frequencies that fall off as one over the rank, the ranks spread over the table
        u = torch.rand(t, generator=gen, device=device, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        state["index"] = torch.randperm(v, generator=gen, device=device)[rank]
        state["padding"] = int(seed) % v if case["padding"] else None
        state["outer"] = torch.randn(t, d, generator=gen, device=device, dtype=torch.float32) \
            .to(dtype)
        return state
    state["mask"] = torch.rand(t, generator=gen, device=device) >= case["prompt"]
    if case["op"] == "logprob":
        z, tokens = _logits(case, gen, device)
        state["logits"] = z.detach().requires_grad_()
        state["tokens"] = torch.where(state["mask"], tokens, torch.full_like(tokens, IGNORE))
        state["outer"] = torch.randn(t, generator=gen, device=device)
        state["outer_entropy"] = 0.1 * torch.rand(t, generator=gen, device=device)
        return state
    count = 2 * case["pairs"] if case["op"] == "preference" else case["sequences"]
    state["offsets"] = _offsets(count, t, gen, device)
    if case["vocab"]:
        z, state["tokens"] = _logits(case, gen, device)
        state["logits"] = z.detach().requires_grad_()
        logp = _true_logp(z, state["tokens"], case.get("temperature", 1.0))
    else:
        logp = -2.0 * torch.rand(t, generator=gen, device=device, dtype=torch.float64) ** 2 - 1e-3
        state["logp"] = logp.to(torch.float32).requires_grad_()
        logp = state["logp"].detach().to(torch.float64)
    # the policy has moved from its reference, each sequence up or down: by a tenth or more for each
    # token, or where whole sequences are weighed against each other by ten nats or more for each
    side = 2.0 * torch.randint(0, 2, (count,), generator=gen, device=device) - 1.0
    if case["op"] == "preference":
        length = state["offsets"].diff().clamp_min(1)
        side = side * (48.0 + 72.0 * torch.rand(count, generator=gen, device=device)) / length
    drift = 0.1 + 0.2 * torch.rand(t, generator=gen, device=device, dtype=torch.float64)
    state["ref"] = (logp + drift * side[_owner(state["offsets"], t)]).to(torch.float32)
    state["outer"] = torch.full((), _loss_scale(case), device=device)
    if case["op"] == "policy":
        # log-ratios to the sampling policy, none of them next to a border of the clip range,
        # where one rounding of the logits would decide
        step = 0.15 * torch.randn(t, generator=gen, device=device, dtype=torch.float64)
        for edge in (math.log(0.8), math.log(1.2)):
            step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
        state["old"] = (logp - step).to(torch.float32)
        state["advantages"] = torch.randn(case["sequences"], generator=gen, device=device)
    return state


# ---------------------------------------------------------------------------- plain forms
def _owner(offsets, t):
    """The sequence of each token."""
    at = torch.arange(t, device=offsets.device)
    return torch.searchsorted(offsets[1:].contiguous().to(torch.int64), at, right=True)


def _plain_lookup(s):
    c, table, index = s["case"], s["table"].detach(), s["index"]
    out = (table[index].to(torch.float32) * c["scale"]).to(table.dtype)
    g = s["outer"].to(torch.float32) * c["scale"]
    if s["padding"] is not None:
        g = g * (index != s["padding"])[:, None]
    acc = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    acc.index_add_(0, index, g)
    return {"out": out, "grad": acc.to(table.dtype)}


def _softmax_parts(z, temperature):
    """(z - max) / temperature, its exponentials and their sums, in 32 bits."""
    z = z.to(torch.float32)
    z = (z - z.amax(1, keepdim=True)) / temperature
    e = torch.exp(z)
    return z, e, e.sum(1, keepdim=True)


def _rows_gradient(e, total, tokens, coef, temperature, dtype):
    """coef * (one-hot - softmax) / temperature."""
    coef = (coef / temperature).to(torch.float32)[:, None]
    d = e.mul_(-coef / total)
    d.scatter_add_(1, tokens[:, None], coef)
    return d.to(dtype)


def _plain_logprob(s):
    c, z, keep = s["case"], s["logits"].detach(), s["mask"]
    tokens = s["tokens"].clamp_min(0)
    x, e, total = _softmax_parts(z, c["temperature"])
    logp = (x.gather(1, tokens[:, None]) - torch.log(total))[:, 0] * keep
    if not c["entropy"]:
        coef = s["outer"] * keep
        return {"logp": logp,
                "grad": _rows_gradient(e, total, tokens, coef, c["temperature"], z.dtype)}
    x = x.clamp_min(-1e30)
    mean = (e * x).sum(1, keepdim=True) / total
    ent = (torch.log(total) - mean)[:, 0] * keep
    p = e / total
    d = -p * ((s["outer"] * keep)[:, None] + (s["outer_entropy"] * keep)[:, None] * (x - mean))
    d.scatter_add_(1, tokens[:, None], (s["outer"] * keep)[:, None])
    return {"logp": logp, "entropy": ent, "grad": (d / c["temperature"]).to(z.dtype)}


def _plain_preference(s):
    c, keep, beta = s["case"], s["mask"], 0.1
    pairs, t = c["pairs"], c["tokens"]
    if c["vocab"]:
        x, e, total = _softmax_parts(s["logits"].detach(), 1.0)
        logp = (x.gather(1, s["tokens"][:, None]) - torch.log(total))[:, 0]
    else:
        logp = s["logp"].detach()
    seq = _owner(s["offsets"], t)
    ratio = (logp.double() - s["ref"].double()) * keep  # long sums
    sums = torch.zeros(2 * pairs, dtype=torch.float64, device=logp.device).index_add_(0, seq, ratio)
    scale = torch.ones_like(sums)
    if c["normalize"]:
        n = torch.zeros_like(sums).index_add_(0, seq, keep.double())
        scale = 1.0 / n.clamp_min(1.0)
    r = beta * sums * scale
    h = r[:pairs] - r[pairs:]
    if c["kind"] == "squared":
        h = h / beta
        each, slope = (h - 0.5 / beta) ** 2, 2.0 * (h - 0.5 / beta) / beta
    else:
        ls = c["smoothing"]
        soft = torch.log1p(torch.exp(-h.abs()))
        each = (1 - ls) * (soft + (-h).clamp_min(0)) + ls * (soft + h.clamp_min(0))
        slope = ls * torch.sigmoid(h) - (1 - ls) * torch.sigmoid(-h)
    slope = slope * beta / pairs * _loss_scale(c)
    coef = (torch.cat([slope, -slope]) * scale)[seq] * keep
    out = {"loss": each.mean().float(), "chosen": r[:pairs].float(), "rejected": r[pairs:].float()}
    if c["vocab"]:
        out["grad"] = _rows_gradient(e, total, s["tokens"], coef, 1.0, s["logits"].dtype)
    else:
        out["grad"] = coef.float()
    return out


def _plain_policy(s):
    c, keep, t = s["case"], s["mask"], s["case"]["tokens"]
    if c["vocab"]:
        x, e, total = _softmax_parts(s["logits"].detach(), c["temperature"])
        logp = (x.gather(1, s["tokens"][:, None]) - torch.log(total))[:, 0]
    else:
        logp = s["logp"].detach()
    seq = _owner(s["offsets"], t)
    n = torch.zeros(c["sequences"], dtype=torch.float64, device=logp.device)
    n.index_add_(0, seq, keep.double())
    if c["average"] == "token":
        weight = keep.double() / n.sum().clamp_min(1.0)
    else:
        weight = keep.double() / (n.clamp_min(1.0) * (n > 0).sum().clamp_min(1))[seq]
    adv = s["advantages"].double()[seq]
    ratio = torch.exp(logp.double() - s["old"].double())  # next to the border of the clip range
    plain, clipped = ratio * adv, ratio.clamp(0.8, 1.2) * adv
    use = plain <= clipped
    gap = s["ref"].double() - logp.double()
    kl = torch.expm1(gap) - gap
    each = -torch.minimum(plain, clipped) + c["kl_coef"] * kl
    coef = weight * (torch.where(use, -plain, torch.zeros_like(plain))
                     - c["kl_coef"] * torch.expm1(gap)) * _loss_scale(c)
    share = 1.0 / keep.double().sum().clamp_min(1.0)
    out = {"loss": (each * weight).sum().float(), "kl": (kl * weight).sum().float(),
           "clipped": (((ratio < 0.8) & (adv < 0) | (ratio > 1.2) & (adv > 0)) & keep)
           .double().sum().mul(share).float()}
    if c["vocab"]:
        out["logp"] = logp * keep
        out["grad"] = _rows_gradient(e, total, s["tokens"], coef, c["temperature"],
                                     s["logits"].dtype)
    else:
        out["grad"] = coef.float()
    return out


# ---------------------------------------------------------------------------- the framework's calls
def _own_lookup(s):
    from sinkslot_b200 import embedding_lookup
    out = embedding_lookup(s["table"], s["index"], scale=s["case"]["scale"],
                           padding_index=s["padding"])
    grad, = torch.autograd.grad(out, [s["table"]], s["outer"])
    return {"out": out.detach(), "grad": grad}


def _own_logprob(s):
    from sinkslot_b200 import token_logprobs
    c = s["case"]
    if c["entropy"]:
        logp, ent = token_logprobs(s["logits"], s["tokens"], temperature=c["temperature"],
                                   ignore_index=IGNORE, entropy=True)
        grad, = torch.autograd.grad([logp, ent], [s["logits"]], [s["outer"], s["outer_entropy"]])
        return {"logp": logp.detach(), "entropy": ent.detach(), "grad": grad}
    logp = token_logprobs(s["logits"], s["tokens"], temperature=c["temperature"],
                          ignore_index=IGNORE)
    grad, = torch.autograd.grad(logp, [s["logits"]], s["outer"])
    return {"logp": logp.detach(), "grad": grad}


def _own_preference(s):
    from sinkslot_b200 import preference_loss, token_logprobs
    c = s["case"]
    leaf = s["logits"] if c["vocab"] else s["logp"]
    mask = s["mask"] if c["prompt"] else None
    logp = leaf
    if c["vocab"]:
        tokens = s["tokens"]
        if mask is not None:
            tokens = torch.where(mask, tokens, IGNORE)
        logp = token_logprobs(leaf, tokens, ignore_index=IGNORE)
    r = preference_loss(logp, s["offsets"], ref_logp=s["ref"], mask=mask, beta=0.1,
                        label_smoothing=c["smoothing"] if c["kind"] == "sigmoid" else 0.0,
                        kind=c["kind"], normalize=c["normalize"])
    grad, = torch.autograd.grad(r.loss, [leaf], s["outer"])
    return {"loss": r.loss.detach(), "chosen": r.chosen_rewards, "rejected": r.rejected_rewards,
            "grad": grad}


def _own_policy(s):
    from sinkslot_b200 import policy_loss, policy_loss_from_logits
    c = s["case"]
    args = {"ref_logp": s["ref"], "mask": s["mask"] if c["prompt"] else None,
            "offsets": s["offsets"], "clip_low": 0.2, "clip_high": 0.2, "kl_coef": c["kl_coef"],
            "average": c["average"]}
    if c["vocab"]:
        r = policy_loss_from_logits(s["logits"], s["tokens"], s["old"], s["advantages"],
                                    temperature=c["temperature"],
                                    grad_scale=_loss_scale(c), **args)
        leaf = s["logits"]
    else:
        r = policy_loss(s["logp"], s["old"], s["advantages"], **args)
        leaf = s["logp"]
    grad, = torch.autograd.grad(r.loss, [leaf], s["outer"])
    out = {"loss": r.loss.detach(), "kl": r.kl, "clipped": r.clip_fraction, "grad": grad}
    if c["vocab"]:
        out["logp"] = r.logp
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"lookup": _own_lookup, "logprob": _own_logprob, "preference": _own_preference,
                "policy": _own_policy}[op](state)
    return {"lookup": _plain_lookup, "logprob": _plain_logprob, "preference": _plain_preference,
            "policy": _plain_policy}[op](state)


# ---------------------------------------------------------------------------- 64 bits
def _exact_rows(z, tokens, temperature, outer, outer_entropy=None):
    """log softmax at the tokens, the entropies, and the logits' gradient for the outer gradients
    that ``outer(logp)`` gives, by automatic differentiation, some rows at a time."""
    step = max(1, (1 << 27) // z.shape[1])
    parts = range(0, z.shape[0], step)
    logp = torch.cat([torch.log_softmax(z[i:i + step].double() / temperature, 1)
                      .gather(1, tokens[i:i + step, None])[:, 0] for i in parts])
    g = outer(logp)
    entropy = torch.zeros_like(logp)
    grad = torch.empty(z.shape, dtype=torch.float64, device=z.device)
    for i in parts:
        leaf = z[i:i + step].double().requires_grad_()
        ls = torch.log_softmax(leaf / temperature, 1)
        total = (ls.gather(1, tokens[i:i + step, None])[:, 0] * g[i:i + step]).sum()
        if outer_entropy is not None:
            h = -(ls.exp() * ls.masked_fill(leaf.isinf(), 0.0)).sum(1)
            entropy[i:i + step] = h.detach()
            total = total + (h * outer_entropy[i:i + step]).sum()
        grad[i:i + step], = torch.autograd.grad(total, [leaf])
    return logp, entropy, grad


def _spans(offsets):
    o = offsets.tolist()
    return list(zip(o[:-1], o[1:]))


def _exact_preference(c, s, logp):
    """The loss from the log-probabilities, sequence by sequence."""
    sums = []
    for lo, hi in _spans(s["offsets"]):
        m = s["mask"][lo:hi]
        v = ((logp[lo:hi] - s["ref"][lo:hi].double()) * m).sum()
        sums.append(v / max(1, int(m.sum())) if c["normalize"] else v)
    chosen, rejected = torch.stack(sums[:c["pairs"]]), torch.stack(sums[c["pairs"]:])
    if c["kind"] == "squared":
        loss = ((chosen - rejected - 5.0) ** 2).mean()
    else:
        h, ls = 0.1 * (chosen - rejected), c["smoothing"]
        f = torch.nn.functional.logsigmoid
        loss = -((1 - ls) * f(h) + ls * f(-h)).mean()
    return loss, {"loss": loss.detach(), "chosen": 0.1 * chosen.detach(),
                  "rejected": 0.1 * rejected.detach()}


def _exact_policy(c, s, logp):
    keep = s["mask"]
    spans = [(lo, hi, int(keep[lo:hi].sum())) for lo, hi in _spans(s["offsets"])]
    full, used = sum(n for _, _, n in spans), sum(n > 0 for _, _, n in spans)
    loss, kl, clipped = 0.0 * logp.sum(), 0.0, 0.0
    for i, (lo, hi, n) in enumerate(spans):
        if n == 0:
            continue
        m, a = keep[lo:hi], s["advantages"][i].double()
        w = 1.0 / full if c["average"] == "token" else 1.0 / (n * used)
        r = torch.exp(logp[lo:hi] - s["old"][lo:hi].double())
        d = s["ref"][lo:hi].double() - logp[lo:hi]
        k = torch.exp(d) - 1.0 - d
        gain = torch.minimum(r * a, torch.clamp(r, 0.8, 1.2) * a)
        loss = loss + w * ((c["kl_coef"] * k - gain) * m).sum()
        kl = kl + w * (k * m).sum().detach()
        over = (r > 1.2) if float(a) > 0 else (r < 0.8)
        clipped = clipped + (over & m).double().sum() / full
    zero = torch.zeros((), dtype=torch.float64, device=logp.device)
    return loss, {"loss": loss.detach(), "kl": kl + zero, "clipped": clipped + zero}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        scale = float(case["scale"])
        table, index = s["table"].detach(), s["index"]
        outer = s["outer"].double()
        if s["padding"] is not None:
            outer = outer.masked_fill((index == s["padding"])[:, None], 0.0)
        grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
        grad.index_put_((index,), outer, accumulate=True)
        return {"out": table.double()[index] * scale, "grad": grad * scale}
    keep = s["mask"].double()
    if case["op"] == "logprob":
        logp, h, grad = _exact_rows(s["logits"].detach(), s["tokens"].clamp_min(0),
                                    case["temperature"], lambda _: s["outer"].double() * keep,
                                    s["outer_entropy"].double() * keep if case["entropy"] else None)
        out = {"logp": logp * keep, "grad": grad}
        return out | {"entropy": h * keep} if case["entropy"] else out
    loss_of = _exact_preference if case["op"] == "preference" else _exact_policy
    said = {}

    def outer(logp):
        leaf = logp.detach().requires_grad_()
        loss, values = loss_of(case, s, leaf)
        said.update(values)
        return torch.autograd.grad(loss, [leaf])[0] * _loss_scale(case)

    if not case["vocab"]:
        grad = outer(s["logp"].detach().double())
        return said | {"grad": grad}
    logp, _, grad = _exact_rows(s["logits"].detach(), s["tokens"], case.get("temperature", 1.0),
                                outer)
    if case["op"] == "policy":
        said["logp"] = logp * keep
    return said | {"grad": grad}
