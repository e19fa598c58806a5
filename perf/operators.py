"""Cases of the operators over vocabulary rows that training on rollouts needs: the clipped policy loss, the
preference loss and the distillation loss with their gradients, and the teacher's top logits.

``run`` computes a case's operator in its plain form (elementary torch operations in 32 bits, sums of a row in 64)
or, with ``own`` set, through ``randomrepo_b200.losses``.  Rows are ``[batch, length, vocab]`` logits; the sizes are
the repository's own vocabularies (151 936 and 152 064 columns) and odd ones, the masks those of right-padded
rollouts (a masked prompt, then the completion, then padding).
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # A few GRPO rollouts of one group: the smallest optimiser step, where the launches' latency counts.
        dict(name="policy_small", op="policy", api="grad", batch=2, length=64, vocab=151936, dtype="bf16", fill=0.7,
             temperature=1.0, clip=0.2, kl=0.04, entropy=0.0, reduction="token_mean", scale=1.0),
        # One micro-batch of GRPO: 4 096 rows, about two thirds of them completion tokens.
        dict(name="policy_step", op="policy", api="grad", batch=8, length=512, vocab=151936, dtype="bf16", fill=0.7,
             temperature=1.0, clip=0.2, kl=0.04, entropy=0.0, reduction="token_mean", scale=1.0),
        # The largest: 8 192 rows of float32 logits at the larger model's vocabulary (5 GB), every token scored.
        dict(name="policy_wide", op="policy", api="grad", batch=16, length=512, vocab=152064, dtype="f32", fill=1.0,
             temperature=1.0, clip=0.2, kl=0.1, entropy=0.0, reduction="sequence_mean", scale=0.25),
        # Autograd with an entropy bonus and a sampling temperature, rows of an odd number of columns.
        dict(name="policy_entropy", op="policy", api="autograd", batch=4, length=301, vocab=50001, dtype="f16",
             fill=0.8, temperature=0.7, clip=0.2, kl=0.0, entropy=0.01, reduction="token_mean", scale=1024.0),
        # Two pairs of short answers.
        dict(name="preference_small", op="preference", api="grad", batch=4, length=48, vocab=151936, dtype="bf16",
             fill=0.7, beta=0.1, smoothing=0.0, normalised=False, scale=1.0),
        # A micro-batch of sixteen pairs.
        dict(name="preference_step", op="preference", api="grad", batch=32, length=256, vocab=151936, dtype="bf16",
             fill=0.8, beta=0.1, smoothing=0.0, normalised=False, scale=1.0),
        # Length-normalised and label-smoothed, float32, odd columns, through autograd.
        dict(name="preference_odd", op="preference", api="autograd", batch=6, length=333, vocab=32003, dtype="f32",
             fill=0.9, beta=2.0, smoothing=0.1, normalised=True, scale=1.0),
        # A draft model's update from one speculative round: four sequences of k + 1 = 5 rows.
        dict(name="distill_small", op="distill", api="grad", batch=4, length=5, vocab=151936, dtype="bf16", fill=1.0,
             temperature=1.0, k=32, with_lse=False, reduction="token_mean", scale=1.0),
        # A rollout's worth of teacher rows.
        dict(name="distill_step", op="distill", api="grad", batch=8, length=512, vocab=151936, dtype="bf16", fill=0.7,
             temperature=2.0, k=64, with_lse=False, reduction="token_mean", scale=1.0),
        # Teacher probabilities normalised over its whole row, an odd K and vocabulary, through autograd.
        dict(name="distill_odd", op="distill", api="autograd", batch=5, length=203, vocab=50001, dtype="f16",
             fill=0.8, temperature=1.5, k=17, with_lse=True, reduction="sequence_mean", scale=1024.0),
        # The teacher's rows of one speculative round (float32 logits, as the verify forward leaves them).
        dict(name="top_small", op="top", api="eval", batch=4, length=5, vocab=151936, dtype="f32", fill=1.0,
             temperature=1.0, k=32),
        # The teacher's rows of a rollout.
        dict(name="top_step", op="top", api="eval", batch=8, length=512, vocab=151936, dtype="bf16", fill=1.0,
             temperature=2.0, k=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["policy", "policy", "preference", "distill", "top"])
    vocab = rng.choice([151936, 152064]) if rng.random() < 0.4 else _spread(rng, 1000, 160000)
    batch, length = _spread(rng, 1, 32), _spread(rng, 1, 600)
    while batch * length * vocab > 4096 * 152064:
        batch, length = max(1, batch // 2), max(1, (2 * length) // 3)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    scale = 1024.0 if dtype == "f16" else rng.choice([1.0, 0.25])
    case = dict(op=op, api=rng.choice(["grad", "grad", "autograd"]), batch=batch, length=length, vocab=vocab,
                dtype=dtype, fill=round(rng.uniform(0.5, 1.0), 2))
    temperature = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 2)])
    reduction = rng.choice(["token_mean", "sequence_mean", "sum"])
    if op == "policy":
        case |= dict(temperature=temperature, clip=0.2, kl=rng.choice([0.0, 0.04, 0.1]),
                     entropy=rng.choice([0.0, 0.0, 0.01]), reduction=reduction, scale=scale)
    elif op == "preference":
        case |= dict(batch=2 * max(1, batch // 2), beta=round(rng.uniform(0.05, 0.5), 2),
                     smoothing=rng.choice([0.0, 0.1]), normalised=rng.random() < 0.3, scale=scale)
        if batch == 1:
            case |= dict(length=max(1, length // 2))
    elif op == "distill":
        case |= dict(temperature=temperature, k=_spread(rng, 1, 128), with_lse=rng.random() < 0.3,
                     reduction=reduction, scale=scale)
    else:
        case |= dict(api="eval", temperature=temperature, k=_spread(rng, 1, 128))
    return case


def _spans(case):
    """(first, last) scored position of each sequence: a masked prompt, the completion, then padding.  They go by the
    case alone, so that its work does; every sequence of more than one token has a scored one."""
    b, t = case["batch"], case["length"]
    r = random.Random(b * 1000003 + t)
    spans = []
    for _ in range(b):
        if case["fill"] >= 1.0 or t < 3:
            spans.append((0, t))
            continue
        n = max(1, min(t, round(t * min(1.0, case["fill"] * r.uniform(0.7, 1.3)))))
        first = r.randint(0, t - n) // 2
        spans.append((first, first + n))
    return spans


def _scored(case):
    return sum(b - a for a, b in _spans(case))


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    rows, vocab, scored = case["batch"] * case["length"], case["vocab"], _scored(case)
    if case["op"] == "top":
        return {"bytes": rows * (vocab * size + case["k"] * 12 + 4), "flops": 3.0 * rows * vocab}
    # A scored row is read once; a gradient row is written once, the masked ones' zeros among them.
    moved = scored * vocab * size + rows * vocab * size
    if case["op"] == "policy":
        moved += rows * (8 + 1 + 4 * 3 + 4 * 2)
    elif case["op"] == "preference":
        moved += rows * (8 + 1)
    else:
        moved += scored * case["k"] * 12 + rows * 5
    return {"bytes": moved, "flops": 7.0 * scored * vocab}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g, dev = _generator(seed), torch.device("cuda")
    b, t, v, dtype = case["batch"], case["length"], case["vocab"], DTYPES[case["dtype"]]
    state = dict(case=case)
    logits = torch.empty((b, t, v), dtype=dtype, device=dev)
    for row in logits:  # a sequence at a time: the largest case's float32 noise would be 5 GB more
        row.copy_(torch.randn((t, v), generator=g, device=dev) * 2.0)
    state["logits"] = logits
    if case["op"] == "top":
        return state
    mask = torch.zeros((b, t), dtype=torch.bool)
    for i, (first, last) in enumerate(_spans(case)):
        mask[i, first:last] = True
    state["mask"] = mask.to(dev)
    if case["op"] == "distill":
        k = min(case["k"], v)
        ids = torch.empty((b, t, k), dtype=torch.int64, device=dev)
        vals = torch.empty((b, t, k), dtype=torch.float32, device=dev)
        for i in range(b):  # the teacher agrees with the student about its likely tokens, and not wholly
            top = (logits[i].float() + torch.randn((t, v), generator=g, device=dev)).topk(k)
            ids[i], vals[i] = top.indices, 1.5 * top.values
        if k > 1:  # some rows' lists are short: a nucleus of fewer tokens
            short = torch.rand((b, t, 1), generator=g, device=dev) < 0.1
            ids = torch.where(short & (torch.arange(k, device=dev) >= (k + 1) // 2), -1, ids)
        state |= dict(ids=ids, teacher=vals)
        state["lse"] = None
        if case["with_lse"]:
            known = (vals / case["temperature"]).masked_fill(ids < 0, -math.inf).logsumexp(-1)
            state["lse"] = known + 0.3 * torch.rand((b, t), generator=g, device=dev)
        return state
    # Sampled tokens are mostly likely ones: the token's logit is raised by 6 to 13.
    tokens = torch.randint(0, v, (b, t), generator=g, device=dev)
    raised = logits.gather(-1, tokens.unsqueeze(-1)).float() + 6 + 7 * torch.rand((b, t, 1), generator=g, device=dev)
    logits.scatter_(-1, tokens.unsqueeze(-1), raised.to(dtype))
    logp = torch.empty((b, t), device=dev)
    temperature = case.get("temperature", 1.0)
    for i in range(b):
        z = logits[i].float() / temperature
        logp[i] = z.gather(-1, tokens[i].unsqueeze(-1)).squeeze(-1) - z.logsumexp(-1)
    state["tokens"] = tokens
    if case["op"] == "policy":
        # The policy has moved a little since the rollout.  A ratio within a thousandth of a clip border is moved off
        # it: on the border itself both one-sided gradients are right.
        moved = 0.15 * torch.randn((b, t), generator=g, device=dev)
        for border in (math.log(1 - case["clip"]), math.log(1 + case["clip"])):
            moved = torch.where((moved - border).abs() < 1e-3, moved + 4e-3, moved)
        state["old"] = logp - moved
        state["ref"] = logp + 0.3 * torch.randn((b, t), generator=g, device=dev) if case["kl"] else None
        state["advantages"] = 0.3 + torch.randn((b,), generator=g, device=dev)
    else:
        total = (logp * state["mask"]).sum(-1)
        count = state["mask"].sum(-1).clamp(min=1)
        drift = torch.randn((b,), generator=g, device=dev) * 0.2 * count.sqrt()
        state["ref"] = total + drift
        if case["normalised"]:
            state["ref"] = state["ref"] / count
    return state


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms: elementary operations, float32 columns, a row's sums and what is derived from them in 64 bits.


def _softmax(logits, temperature):
    """(x - max) / T, exp of it, its sum (float64) for rows [..., V]."""
    x = logits.float()
    y = (x - x.amax(-1, keepdim=True)) / temperature
    e = torch.exp(y)
    return y, e, e.sum(-1, keepdim=True, dtype=torch.float64)


def _token_logprobs(y, total, tokens):
    return (y.gather(-1, tokens.unsqueeze(-1)).double() - torch.log(total)).squeeze(-1)


def _weights(mask, reduction, scale):
    """What each scored token's loss counts in the mean, float64 [B, T]."""
    m = mask.double()
    if reduction == "sum":
        return m * scale
    if reduction == "token_mean":
        return m * (scale / m.sum().clamp(min=1))
    per = m.sum(-1, keepdim=True)
    return m * (scale / (per.clamp(min=1) * (per > 0).sum().clamp(min=1)))


def _policy(s, case):
    logits, mask, tokens = s["logits"], s["mask"], s["tokens"]
    t = case["temperature"]
    y, e, total = _softmax(logits, t)
    logp = _token_logprobs(y, total, tokens)
    p = e / total.float()
    w = _weights(mask, case["reduction"], case["scale"])
    adv = s["advantages"].double().unsqueeze(-1)
    ratio = torch.exp(logp - s["old"].double())
    low, high = 1.0 - case["clip"], 1.0 + case["clip"]
    per = -torch.minimum(ratio * adv, ratio.clamp(low, high) * adv)
    cut = ((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))
    slope = torch.where(cut, 0.0, -ratio * adv)
    out = {}
    if case["kl"]:
        delta = s["ref"].double() - logp
        kl = torch.exp(delta) - delta - 1.0
        per = per + case["kl"] * kl
        slope = slope + case["kl"] * (1.0 - torch.exp(delta))
        out["kl"] = torch.where(mask, kl, 0.0).float()
    one_less = -p
    one_less.scatter_add_(-1, tokens.unsqueeze(-1), torch.ones_like(tokens.unsqueeze(-1), dtype=p.dtype))
    grad = one_less * (w * slope / t).float().unsqueeze(-1)
    if case["entropy"]:
        logrow = y - torch.log(total).float()
        entropy = -(p * logrow).sum(-1, dtype=torch.float64)
        per = per - case["entropy"] * entropy
        grad += p * (logrow + entropy.float().unsqueeze(-1)) * (w * case["entropy"] / t).float().unsqueeze(-1)
        out["entropy"] = torch.where(mask, entropy, 0.0).float()
    out["loss"] = torch.where(mask, per * w, 0.0).sum().float()
    out["logprobs"] = torch.where(mask, logp, 0.0).float()
    out["dlogits"] = torch.where(mask.unsqueeze(-1), grad, 0.0).to(logits.dtype)
    return out


def _preference(s, case):
    logits, mask, tokens = s["logits"], s["mask"], s["tokens"]
    y, e, total = _softmax(logits, 1.0)
    logp = _token_logprobs(y, total, tokens)
    sums = torch.where(mask, logp, 0.0).sum(-1)
    count = mask.sum(-1).clamp(min=1).double()
    if case["normalised"]:
        sums = sums / count
    pairs = mask.shape[0] // 2
    gap = sums - s["ref"].double()
    margin = case["beta"] * (gap[:pairs] - gap[pairs:])
    eps = case["smoothing"]
    soft = torch.log1p(torch.exp(-margin.abs()))
    per = (1 - eps) * (soft + (-margin).clamp(min=0)) + eps * (soft + margin.clamp(min=0))
    slope = (eps - 1 + 1 / (1 + torch.exp(-margin))) * case["beta"] * case["scale"] / pairs
    slope = torch.cat([slope, -slope])
    if case["normalised"]:
        slope = slope / count
    p = e / total.float()
    grad = -p
    grad.scatter_add_(-1, tokens.unsqueeze(-1), torch.ones_like(tokens.unsqueeze(-1), dtype=p.dtype))
    grad *= torch.where(mask, slope.unsqueeze(-1), 0.0).float().unsqueeze(-1)
    return dict(loss=(per.mean() * case["scale"]).float(), logprobs=sums.float(), margins=margin.float(),
                dlogits=grad.to(logits.dtype))


def _distill(s, case):
    logits, mask, t = s["logits"], s["mask"], case["temperature"]
    y, e, total = _softmax(logits, t)
    known = s["ids"] >= 0
    ids = s["ids"].clamp(min=0)
    logq = (s["teacher"].double() / t).masked_fill(~known, -math.inf)
    if s["lse"] is None:
        top = logq.amax(-1, keepdim=True)
        logq = logq - top - torch.log(torch.exp(logq - top).sum(-1, keepdim=True))
    else:
        logq = logq - s["lse"].double().unsqueeze(-1)
    q = torch.exp(logq)
    logp = y.gather(-1, ids).double() - torch.log(total)
    per = t * t * torch.where(known, q * (logq - logp), 0.0).sum(-1)
    w = _weights(mask, case["reduction"], case["scale"])
    p = e / total.float()
    grad = p * q.sum(-1, keepdim=True).float()
    grad.scatter_add_(-1, ids, torch.where(known, -q, 0.0).float())
    grad *= (w * t).float().unsqueeze(-1)
    return dict(loss=torch.where(mask, per * w, 0.0).sum().float(), kl=torch.where(mask, per, 0.0).float(),
                dlogits=torch.where(mask.unsqueeze(-1), grad, 0.0).to(logits.dtype))


def _top(s, case):
    logits, t = s["logits"], case["temperature"]
    v = logits.shape[-1]
    k = min(case["k"], v)
    _, _, total = _softmax(logits, t)
    x = logits.float() + 0.0
    lse = x.amax(-1).double() / t + torch.log(total).squeeze(-1)
    # Larger values first, equal ones by their index: one 64-bit key for each column.
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2**32
    key += torch.arange(v - 1, -1, -1, device=x.device)
    ids = v - 1 - (key.topk(k, sorted=True).values & (2**32 - 1))
    return dict(values=x.gather(-1, ids), tokens=ids, lse=lse.float())


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"policy": _policy, "preference": _preference, "distill": _distill, "top": _top}[case["op"]](state, case)


def _own(s, case):
    from randomrepo_b200 import losses

    logits, op = s["logits"], case["op"]
    if op == "top":
        values, tokens, lse = losses.top_logits(logits, min(case["k"], case["vocab"]),
                                                temperature=case["temperature"])
        return dict(values=values, tokens=tokens, lse=lse)
    autograd = case["api"] == "autograd"
    if autograd:
        logits = logits.detach().requires_grad_()
    if op == "policy":
        fn = losses.policy_loss if autograd else losses.policy_loss_and_grad
        got = fn(logits, s["tokens"], s["advantages"], s["old"], s["mask"], ref_logprobs=s["ref"],
                 clip_low=case["clip"], clip_high=case["clip"], kl_coef=case["kl"], entropy_coef=case["entropy"],
                 temperature=case["temperature"], reduction=case["reduction"], scale=case["scale"])
    elif op == "preference":
        fn = losses.preference_loss if autograd else losses.preference_loss_and_grad
        got = fn(logits, s["tokens"], s["mask"], s["ref"], beta=case["beta"], label_smoothing=case["smoothing"],
                 length_normalised=case["normalised"], scale=case["scale"])
    else:
        fn = losses.distillation_loss if autograd else losses.distillation_loss_and_grad
        got = fn(logits, s["ids"], s["teacher"], s["mask"], teacher_lse=s["lse"], temperature=case["temperature"],
                 reduction=case["reduction"], scale=case["scale"])
    if autograd:
        got = got, torch.autograd.grad(got.loss, logits)[0]
    result, dlogits = got
    out = dict(loss=result.loss, dlogits=dlogits)
    if op == "policy":
        out["logprobs"] = result.logprobs
        if case["kl"]:
            out["kl"] = result.kl
        if case["entropy"]:
            out["entropy"] = result.entropy
    elif op == "preference":
        out |= dict(logprobs=result.logprobs, margins=result.margins)
    else:
        out["kl"] = result.kl
    return out


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits, a sequence at a time.


def exact(case, seed):
    s = prepare(case, seed)
    return {"policy": _exact_policy, "preference": _exact_preference, "distill": _exact_distill,
            "top": _exact_top}[case["op"]](s, case)


def _row_weights(case, mask):
    lengths = [int(n) for n in mask.sum(-1)]
    if case["reduction"] == "sum":
        return [case["scale"]] * len(lengths)
    if case["reduction"] == "token_mean":
        return [case["scale"] / max(1, sum(lengths))] * len(lengths)
    full = max(1, sum(n > 0 for n in lengths))
    return [case["scale"] / (max(1, n) * full) for n in lengths]


def _exact_policy(s, case):
    b, length, v = s["logits"].shape
    dev = s["logits"].device
    grads = torch.zeros((b, length, v), dtype=torch.float64 if b * length * v < 2**30 else torch.float32, device=dev)
    logprobs, kls, entropies = (torch.zeros((b, length), dtype=torch.float64, device=dev) for _ in range(3))
    loss = 0.0
    weights = _row_weights(case, s["mask"])
    for i in range(b):
        at = s["mask"][i].nonzero().squeeze(-1)
        if not len(at):
            continue
        logrow = torch.log_softmax(s["logits"][i, at].double() / case["temperature"], -1)
        pick = torch.arange(len(at), device=dev), s["tokens"][i, at]
        logp = logrow[pick]
        ratio = (logp - s["old"][i, at].double()).exp()
        a = float(s["advantages"][i])
        low, high = 1 - case["clip"], 1 + case["clip"]
        inside = ratio <= high if a > 0 else ratio >= low
        bounded = ratio.clamp(max=high) if a > 0 else ratio.clamp(min=low)
        per = -a * bounded
        d_logp = -a * ratio * inside
        if case["kl"]:
            gap = s["ref"][i, at].double() - logp
            kls[i, at] = torch.expm1(gap) - gap
            per = per + case["kl"] * kls[i, at]
            d_logp = d_logp - case["kl"] * torch.expm1(gap)
        prob = logrow.exp()
        d_row = -d_logp.unsqueeze(-1) * prob
        d_row[pick] += d_logp
        if case["entropy"]:
            h = -torch.special.xlogy(prob, prob).sum(-1)
            entropies[i, at] = h
            per = per - case["entropy"] * h
            d_row += case["entropy"] * prob * (logrow + h.unsqueeze(-1))
        grads[i, at] = (d_row * (weights[i] / case["temperature"])).to(grads.dtype)
        logprobs[i, at] = logp
        loss += weights[i] * float(per.sum())
    out = dict(loss=torch.tensor(loss, dtype=torch.float64), logprobs=logprobs, dlogits=grads)
    if case["kl"]:
        out["kl"] = kls
    if case["entropy"]:
        out["entropy"] = entropies
    return out


def _exact_preference(s, case):
    b, length, v = s["logits"].shape
    dev = s["logits"].device
    sums = []
    for i in range(b):
        row = torch.log_softmax(s["logits"][i].double(), -1).gather(-1, s["tokens"][i].unsqueeze(-1)).squeeze(-1)
        n = max(1, int(s["mask"][i].sum())) if case["normalised"] else 1
        sums.append(float(row[s["mask"][i]].sum()) / n)
    ref = [float(x) for x in s["ref"]]
    pairs, eps = b // 2, case["smoothing"]
    margins = [case["beta"] * ((sums[i] - ref[i]) - (sums[i + pairs] - ref[i + pairs])) for i in range(pairs)]

    def minus_log_sigmoid(x):
        return math.log1p(math.exp(-x)) if x > 0 else math.log1p(math.exp(x)) - x

    def sigmoid(x):
        return 1 / (1 + math.exp(-x)) if x > 0 else math.exp(x) / (1 + math.exp(x))

    loss = sum((1 - eps) * minus_log_sigmoid(x) + eps * minus_log_sigmoid(-x) for x in margins) / pairs
    grads = torch.zeros((b, length, v), dtype=torch.float64 if b * length * v < 2**30 else torch.float32, device=dev)
    for i in range(b):
        x = margins[i % pairs]
        slope = (eps * sigmoid(x) - (1 - eps) * sigmoid(-x)) * case["beta"] * case["scale"] / pairs
        slope *= 1 if i < pairs else -1
        if case["normalised"]:
            slope /= max(1, int(s["mask"][i].sum()))
        row = -torch.softmax(s["logits"][i].double(), -1)
        row[torch.arange(length, device=dev), s["tokens"][i]] += 1
        grads[i] = (row * (s["mask"][i].double() * slope).unsqueeze(-1)).to(grads.dtype)
    as64 = lambda x: torch.tensor(x, dtype=torch.float64)  # noqa: E731
    return dict(loss=as64(loss * case["scale"]), logprobs=as64(sums), margins=as64(margins), dlogits=grads)


def _exact_distill(s, case):
    b, length, v = s["logits"].shape
    dev, t = s["logits"].device, case["temperature"]
    grads = torch.zeros((b, length, v), dtype=torch.float64 if b * length * v < 2**30 else torch.float32, device=dev)
    kls = torch.zeros((b, length), dtype=torch.float64, device=dev)
    weights = _row_weights(case, s["mask"])
    for i in range(b):
        known = s["ids"][i] >= 0
        z = torch.where(known, s["teacher"][i].double() / t, -math.inf)
        norm = z.logsumexp(-1) if s["lse"] is None else s["lse"][i].double()
        q = (z - norm.unsqueeze(-1)).exp()
        whole = torch.zeros((length, v), dtype=torch.float64, device=dev)
        whole.scatter_add_(-1, s["ids"][i].clamp(min=0), q)
        logrow = torch.log_softmax(s["logits"][i].double() / t, -1)
        kls[i] = t * t * (torch.special.xlogy(whole, whole) - whole * logrow).sum(-1) * s["mask"][i]
        row = whole.sum(-1, keepdim=True) * logrow.exp() - whole
        grads[i] = (row * (t * weights[i]) * s["mask"][i].unsqueeze(-1)).to(grads.dtype)
    loss = sum(w * float(x.sum()) for w, x in zip(weights, kls))
    return dict(loss=torch.tensor(loss, dtype=torch.float64), kl=kls, dlogits=grads)


def _exact_top(s, case):
    b, _, v = s["logits"].shape
    values, tokens, lse = [], [], []
    for i in range(b):
        x = s["logits"][i].double()
        order = x.sort(dim=-1, descending=True, stable=True)
        values.append(order.values[:, : case["k"]])
        tokens.append(order.indices[:, : case["k"]])
        lse.append((x / case["temperature"]).logsumexp(-1))
    return dict(values=torch.stack(values), tokens=torch.stack(tokens), lse=torch.stack(lse))
