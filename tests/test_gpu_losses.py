"""The vocabulary-row losses, their gradients and the top logits on the GPU against definitions in 64 bits.

The definitions are torch double operations and the gradients their autograd.  Tolerances:

* a row's log-sum-exp: a column's 2^y is off by the rounding of y, at most 2^-24 |y| ln 2 relative (|y| <= 64 base-2
  units for the inputs here: 2.7e-6), and 2^-22 from the approximation of 2^y; a thread adds at most ~300 columns and
  then merges 2^5 + 2^4 partial sums, so the sum is off by at most ~350 x 2^-24 = 2.1e-5 relative, in practice by the
  root of that.  A log-probability in float32 adds half a step of its own (|lp| < 64: 2^-19 = 1.9e-6).  LP = 2.5e-5.
* a gradient entry c (p - q): p is off by LP relative, and p - 1 at the token by half a step of 1 (2^-24): c (LP p +
  2^-23), where c is the row's largest coefficient; rounded to the logits' type, eps / 2 relative and, for float16,
  half a subnormal step (2^-25).
* a loss: LP times the slope of each row's loss in lp, summed, and half a step.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LP = 2.5e-5
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(1, 1, 1), (1, 1, 7), (2, 3, 33), (3, 5, 1001), (2, 4, 8200), (1, 3, 50001), (2, 2, 151936), (5, 67, 519)]


def _logits(b, t, v, dtype, dev, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + 7 * b + 31 * t + v)
    return (torch.randn(b, t, v, generator=g) * spread).to(dtype).to(dev), g


def _mask(kind, b, t, g, dev):
    if kind == "none":
        return None
    if kind == "empty":
        return torch.zeros(b, t, dtype=torch.bool, device=dev)
    m = torch.rand(b, t, generator=g) < 0.6
    m[0, 0] = True
    if b > 1:
        m[-1] = False  # a sequence without a scored row
    return m.to(dev)


def _weights(mask, b, t, reduction, scale, dev):
    m = (torch.ones(b, t, dtype=torch.bool, device=dev) if mask is None else mask).double()
    if reduction == "sum":
        return m * scale
    if reduction == "token_mean":
        return m * scale / m.sum().clamp(min=1)
    per = m.sum(-1, keepdim=True)
    return m * scale / (per.clamp(min=1) * (per > 0).sum().clamp(min=1))


def _close_grad(got, want, coef, dtype):
    """``coef`` [..., 1]: the largest coefficient of each row's gradient."""
    want = want.double()
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tol = 2 * LP * want.abs() + coef.double().abs() * (LP * 1e-2 + 2.0**-23) + half * want.abs()
    if dtype == F16:
        tol = tol + 2.0**-25
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), ((got.double() - want).abs()[bad][:5], want[bad][:5], tol[bad][:5], int(bad.sum()))


def _policy_case(b, t, v, dtype, dev, mask_kind, seed=0):
    logits, g = _logits(b, t, v, dtype, dev, seed)
    tokens = torch.randint(0, v, (b, t), generator=g).to(dev)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    moved = torch.randn(b, t, generator=g).to(dev) * 0.3
    for border in (math.log(0.8), math.log(1.3)):  # both gradients are right on the border itself
        moved = torch.where((moved - border).abs() < 1e-2, moved + 4e-2, moved)
    old = (lp - moved).float()
    ref = (lp + torch.randn(b, t, generator=g).to(dev) * 0.4).float()
    adv = torch.randn(b, t, generator=g).to(dev)
    return logits, tokens, adv, old, ref, _mask(mask_kind, b, t, g, dev)


def _policy_definition(logits, tokens, adv, old, ref, mask, temperature, kl_coef, ent, reduction, scale):
    x = logits.double().requires_grad_()
    rows = torch.log_softmax(x / temperature, -1)
    lp = rows.gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    ratio = (lp - (lp.detach() if old is None else old.double())).exp()
    per = -torch.minimum(ratio * adv.double(), ratio.clamp(0.8, 1.3) * adv.double())
    kl = None
    if ref is not None:
        d = ref.double() - lp
        kl = d.exp() - d - 1
        per = per + kl_coef * kl
    p = rows.exp()
    entropy = -(p * rows).sum(-1)
    per = per - ent * entropy
    w = _weights(mask, *tokens.shape, reduction, scale, logits.device)
    loss = torch.where(w > 0, per * w, 0.0).sum()
    (grad,) = torch.autograd.grad(loss, x)
    seen = w > 0
    slope = (ratio * adv.double()).abs() + (0 if ref is None else kl_coef * (1 + d.exp())) + ent * 30
    return loss.detach(), torch.where(seen, lp, 0).detach(), kl, torch.where(seen, entropy, 0).detach(), grad, (
        w * slope / temperature).detach().unsqueeze(-1), seen


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("mask_kind,reduction", [("none", "sum"), ("some", "token_mean"), ("some", "sequence_mean"),
                                                 ("empty", "token_mean")])
def test_policy_loss_and_gradient(cuda_device, shape, dtype, mask_kind, reduction):
    from randomrepo_b200 import losses

    b, t, v = shape
    logits, tokens, adv, old, ref, mask = _policy_case(b, t, v, dtype, cuda_device, mask_kind)
    # Each shape meets another set of terms.
    ent, temperature, kl = ((0.0, 1.0, 0.05), (0.02, 0.7, 0.0), (0.01, 1.6, 0.1))[(b + t + v) % 3]
    use_ref, use_old = kl > 0, v % 2 == 1
    want = _policy_definition(logits, tokens, adv, old if use_old else None, ref if use_ref else None, mask,
                              temperature, kl, ent, reduction, 0.5)
    kw = dict(ref_logprobs=ref if use_ref else None, clip_low=0.2, clip_high=0.3, kl_coef=kl, entropy_coef=ent,
              temperature=temperature, reduction=reduction, scale=0.5)
    args = (tokens, adv, old if use_old else None, mask)
    got, grad = losses.policy_loss_and_grad(logits, *args, **kw)
    loss, lp, wkl, entropy, wgrad, coef, seen = want
    torch.testing.assert_close(got.logprobs.double(), lp, atol=LP, rtol=0)
    assert (got.logprobs[~seen] == 0).all()
    slack = float((coef * temperature).sum()) * LP + float(loss.abs()) * 2.0**-23 + 1e-12
    assert abs(float(got.loss) - float(loss)) <= slack
    if use_ref:
        torch.testing.assert_close(got.kl.double(), torch.where(seen, wkl, 0).detach(), atol=LP, rtol=1e-4)
    else:
        assert got.kl is None
    if ent:
        # H = ln s - sum e y / s: both sums are off by LP relative, the second is at most 64 ln 2 large.
        torch.testing.assert_close(got.entropy.double(), entropy, atol=LP, rtol=LP * 8)
    assert grad.dtype == dtype and grad.shape == logits.shape
    _close_grad(grad, wgrad, coef, dtype)
    assert (grad[~seen] == 0).all()
    # The differentiable form: the same loss, and the gradient times the upstream one.
    leaf = logits.detach().requires_grad_()
    out = losses.policy_loss(leaf, *args, **kw)
    # (its sums are made in another order: each form is within its bound of the definition)
    torch.testing.assert_close(out.logprobs.double(), lp, atol=LP, rtol=0)
    assert abs(out.loss.item() - float(loss)) <= slack
    (2.0 * out.loss).backward()
    _close_grad(leaf.grad, 2.0 * wgrad, 2 * coef, dtype)
    with torch.no_grad():
        assert torch.equal(losses.policy_loss(leaf, *args, **kw).loss, out.loss)


def _preference_definition(logits, tokens, mask, ref, beta, eps, normalised, scale):
    x = logits.double().requires_grad_()
    b, t = tokens.shape
    m = torch.ones(b, t, dtype=torch.bool, device=x.device) if mask is None else mask
    lp = torch.log_softmax(x, -1).gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    s = torch.where(m, lp, 0.0).sum(-1)
    n = m.sum(-1).clamp(min=1) if normalised else torch.ones(b, device=x.device)
    s = s / n
    gap = s - (0 if ref is None else ref.double())
    margin = beta * (gap[: b // 2] - gap[b // 2:])
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - eps) * ls(margin) - eps * ls(-margin)).mean() * scale
    (grad,) = torch.autograd.grad(loss, x)
    coef = (m.double() * (beta * scale / (b // 2) / n).unsqueeze(-1)).unsqueeze(-1)
    return loss.detach(), s.detach(), margin.detach(), grad, coef


@pytest.mark.parametrize("shape", [(2, 1, 7), (2, 3, 33), (4, 5, 1001), (6, 4, 8200), (2, 3, 50001), (4, 3, 151936),
                                   (8, 67, 519)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("mask_kind", ["none", "some", "empty"])
def test_preference_loss_and_gradient(cuda_device, shape, dtype, mask_kind):
    from randomrepo_b200 import losses

    b, t, v = shape
    logits, g = _logits(b, t, v, dtype, cuda_device, 3)
    tokens = torch.randint(0, v, (b, t), generator=g).to(cuda_device)
    mask = _mask(mask_kind, b, t, g, cuda_device)
    ref = None if v % 2 else (-8.0 * t + torch.randn(b, generator=g)).to(cuda_device)
    beta, eps, normalised = ((0.1, 0.0, False), (0.5, 0.2, True))[(t + v) % 2]
    loss, s, margin, wgrad, coef = _preference_definition(logits, tokens, mask, ref, beta, eps, normalised, 2.0)
    kw = dict(beta=beta, label_smoothing=eps, length_normalised=normalised, scale=2.0)
    got, grad = losses.preference_loss_and_grad(logits, tokens, mask, ref, **kw)
    torch.testing.assert_close(got.logprobs.double(), s, atol=LP * t, rtol=2.0**-23)
    torch.testing.assert_close(got.margins.double(), margin, atol=2 * beta * LP * t, rtol=2.0**-22)
    assert abs(float(got.loss) - float(loss)) <= 4 * beta * LP * t + float(loss.abs()) * 2.0**-23
    # The coefficient itself moves by beta times the margin's error.
    _close_grad(grad, wgrad, coef * (1 + 4 * beta * t), dtype)
    leaf = logits.detach().requires_grad_()
    out = losses.preference_loss(leaf, tokens, mask, ref, **kw)
    assert torch.equal(out.loss, got.loss) and torch.equal(out.margins, got.margins)
    (out.loss * 0.5).backward()
    _close_grad(leaf.grad, 0.5 * wgrad, coef * (1 + 4 * beta * t), dtype)


def _distill_case(b, t, v, k, dtype, dev, seed=5):
    logits, g = _logits(b, t, v, dtype, dev, seed)
    ids = torch.randint(0, v, (b, t, k), generator=g)
    if k > 2:
        ids[..., k // 2] = ids[..., 0]  # the same token twice
        ids[0, 0, k - 1] = -1
    teacher = torch.randn(b, t, k, generator=g) * 2
    if k > 1:
        teacher[0, 0, 1] = -math.inf
    if b * t > 1:
        ids[-1, -1] = -1  # nothing at all
    return logits, ids.to(dev), teacher.to(dev), g


def _distill_definition(logits, ids, teacher, mask, lse, temperature, reduction, scale):
    x = logits.double().requires_grad_()
    b, t = ids.shape[:2]
    known = (ids >= 0) & (teacher > -math.inf)
    z = torch.where(known, teacher.double() / temperature, -math.inf)
    norm = z.logsumexp(-1) if lse is None else lse.double()
    lq = torch.where(known, z - norm.unsqueeze(-1), 0.0)
    q = torch.where(known, lq.exp(), 0.0)
    lp = torch.log_softmax(x / temperature, -1).gather(-1, ids.clamp(min=0))
    per = temperature**2 * torch.where(known, q * (lq - lp), 0.0).sum(-1)
    w = _weights(mask, b, t, reduction, scale, x.device)
    loss = torch.where(w > 0, per * w, 0.0).sum()
    (grad,) = torch.autograd.grad(loss, x)
    coef = (w * temperature * q.sum(-1)).unsqueeze(-1)
    return loss.detach(), torch.where(w > 0, per, 0.0).detach(), grad, coef, q.sum(-1)


@pytest.mark.parametrize("shape,k", [((1, 1, 1), 1), ((1, 1, 7), 3), ((2, 3, 33), 33), ((3, 5, 1001), 17),
                                     ((2, 4, 8200), 256), ((1, 3, 50001), 40), ((2, 2, 151936), 64), ((5, 67, 519), 8)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("mask_kind,reduction", [("none", "sum"), ("some", "token_mean"), ("some", "sequence_mean"),
                                                 ("empty", "sum")])
def test_distillation_loss_and_gradient(cuda_device, shape, k, dtype, mask_kind, reduction):
    from randomrepo_b200 import losses

    b, t, v = shape
    logits, ids, teacher, g = _distill_case(b, t, v, k, dtype, cuda_device)
    mask = _mask(mask_kind, b, t, g, cuda_device)
    temperature = (1.0, 2.0, 0.6)[(b + v) % 3]
    lse = None if t % 2 else (teacher / temperature).logsumexp(-1) + 0.5
    loss, per, wgrad, coef, q = _distill_definition(logits, ids, teacher, mask, lse, temperature, reduction, 3.0)
    kw = dict(teacher_lse=lse, temperature=temperature, reduction=reduction, scale=3.0)
    got, grad = losses.distillation_loss_and_grad(logits, ids, teacher, mask, **kw)
    # T^2 Q LP for the student's log-probabilities; q and log q are off by ~2^-22.
    torch.testing.assert_close(got.kl.double(), per, atol=temperature**2 * LP * max(1.0, float(q.max())), rtol=2.0**-20)
    slack = float((coef * temperature).sum()) * LP + float(loss.abs()) * 2.0**-20 + 1e-12
    assert abs(float(got.loss) - float(loss)) <= slack
    # The list's entries are c (Q p - q) with q off by 2^-22 relative.
    _close_grad(grad, wgrad, coef * 2, dtype)
    leaf = logits.detach().requires_grad_()
    out = losses.distillation_loss(leaf, ids, teacher, mask, **kw)
    torch.testing.assert_close(out.kl.double(), per, atol=temperature**2 * LP * max(1.0, float(q.max())), rtol=2.0**-20)
    assert abs(out.loss.item() - float(loss)) <= slack
    (out.loss * 4.0).backward()
    _close_grad(leaf.grad, 4.0 * wgrad, coef * 8, dtype)


def _top_definition(x, k):
    """Stable descending order: equal values by their column; NaN first, as torch sorts it on the host (its CUDA sort
    goes by a NaN's sign bit)."""
    order = (x.cpu().double() + 0.0).sort(dim=-1, descending=True, stable=True)
    return order.values[..., :k].float().to(x.device), order.indices[..., :k].to(x.device)


@pytest.mark.parametrize("shape,k", [((1, 1, 1), 1), ((1, 1, 7), 7), ((2, 3, 33), 5), ((3, 5, 1001), 256),
                                     ((2, 4, 8200), 1), ((1, 3, 50001), 100), ((2, 2, 151936), 64),
                                     ((1, 2, 151936), 256), ((5, 67, 519), 8), ((1, 2, 2054), 256)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_top_logits(cuda_device, shape, k, dtype):
    from randomrepo_b200 import losses

    logits, _ = _logits(*shape, dtype, cuda_device, 11)
    values, tokens, lse = losses.top_logits(logits, k, temperature=0.8)
    wv, wt = _top_definition(logits, k)
    assert torch.equal(values, wv) and torch.equal(tokens, wt)
    torch.testing.assert_close(lse.double(), (logits.double() / 0.8).logsumexp(-1), atol=LP, rtol=2.0**-23)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [1, 64, 256])
def test_top_logits_of_hard_rows(cuda_device, dtype, k):
    """Ties, runs and special values: constant rows, rows of -inf with a few others, rows in order, rows whose large
    values lie together, few distinct values, signed zeros, infinities and NaN."""
    from randomrepo_b200 import losses

    v = 20011
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(v), torch.full((v,), -math.inf), torch.linspace(-5, 5, v), torch.linspace(5, -5, v),
            torch.randint(0, 3, (v,), generator=g).float(), torch.where(torch.rand(v, generator=g) < 0.5, 0.0, -0.0)]
    few = torch.full((v,), -math.inf)
    few[[5, 19999, 700, 20010, 0]] = torch.tensor([1.0, 2.0, 1.0, -3.0, 1.0])
    rows.append(few)
    run = torch.randn(v, generator=g)
    run[4096:8192] = 10 + torch.rand(4096, generator=g)
    rows.append(run)
    odd = torch.randn(v, generator=g)
    odd[[3, 9000]] = math.nan
    odd[[17, 12345]] = math.inf
    rows.append(odd)
    low = torch.full((v,), torch.finfo(dtype).min)
    low[100] = 0.5
    rows.append(low)
    rows.append(torch.full((v,), math.nan))
    x = torch.stack(rows).to(dtype).to(cuda_device)
    values, tokens, lse = losses.top_logits(x, k)
    wv, wt = _top_definition(x, k)
    assert torch.equal(torch.nan_to_num(values, nan=12345.0), torch.nan_to_num(wv, nan=12345.0))
    assert torch.equal(tokens, wt)
    want = x.double().logsumexp(-1)
    torch.testing.assert_close(lse[[0, 2, 3, 4, 5, 6, 7, 9]].double(), want[[0, 2, 3, 4, 5, 6, 7, 9]], atol=LP, rtol=2.0**-23)
    assert torch.isnan(lse[8]) and torch.isnan(lse[10])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_of_one_value_are_uniform(cuda_device, dtype):
    """The lowest and the largest finite value of the type everywhere: log p = -log V, as softmax has it."""
    from randomrepo_b200 import losses

    v = 517
    info = torch.finfo(dtype)
    x = torch.tensor([info.min, info.max, 0.0, -1.0, info.tiny]).to(dtype).unsqueeze(1).expand(5, v).contiguous().to(cuda_device)
    x[3, 7], x[3, 9] = info.min, info.max
    tokens = torch.tensor([3, 516, 0, 9, 100], device=cuda_device)
    got, grad = losses.policy_loss_and_grad(x, tokens, torch.ones(1, device=cuda_device), reduction="sum", entropy_coef=0.5)
    want = torch.full((5,), -math.log(v), dtype=torch.float64, device=cuda_device)
    want[3] = 0.0
    torch.testing.assert_close(got.logprobs.double(), want, atol=LP, rtol=0)
    torch.testing.assert_close(got.entropy.double(), -want, atol=LP, rtol=0)
    assert grad.isfinite().all()


@pytest.mark.parametrize("temperature", [0.7, 1.3, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_columns_count_nothing(cuda_device, dtype, temperature):
    """-inf columns at temperatures whose scale is two floats: the rows without them, and zeros in their gradient."""
    from randomrepo_b200 import losses

    logits, g = _logits(1, 3, 900, dtype, cuda_device)
    hole = torch.rand(3, 900, generator=g).to(cuda_device) < 0.5
    hole[:, :2] = False
    x = logits.masked_fill(hole, -math.inf)
    tokens = torch.tensor([[0, 1, 0]], device=cuda_device)
    adv = torch.ones(1, device=cuda_device)
    got, grad = losses.policy_loss_and_grad(x, tokens, adv, entropy_coef=0.1, temperature=temperature, reduction="sum")
    rows = torch.log_softmax(x.double() / temperature, -1)
    torch.testing.assert_close(got.logprobs.double(), rows.gather(-1, tokens.unsqueeze(-1)).squeeze(-1), atol=LP, rtol=0)
    assert grad.isfinite().all() and (grad[0][hole] == 0).all() and got.entropy.isfinite().all()
    values, ids, lse = losses.top_logits(x, 5, temperature=temperature)
    torch.testing.assert_close(lse.double(), (x.double() / temperature).logsumexp(-1), atol=LP, rtol=2.0**-23)


def test_special_values(cuda_device):
    """-inf columns count nothing, masked rows may hold anything, a bad token is loud and stays in its row."""
    from randomrepo_b200 import losses

    logits, g = _logits(2, 4, 1001, F32, cuda_device)
    logits[0, 0, 5:900] = -math.inf
    logits[0, 2] = math.nan
    logits[1, 3] = math.inf
    logits[0, 1, :] = torch.finfo(F32).min
    logits[0, 1, 3] = 1.0
    mask = torch.ones(2, 4, dtype=torch.bool, device=cuda_device)
    mask[0, 2] = mask[1, 3] = False
    tokens = torch.full((2, 4), 3, device=cuda_device)
    tokens[0, 2], tokens[1, 3] = -100, 1 << 40
    adv = torch.ones(2, device=cuda_device)
    got, grad = losses.policy_loss_and_grad(logits, tokens, adv, None, mask, entropy_coef=0.1)
    clean = logits.clone()
    clean[~mask] = 0.0
    clean = clean.clamp(min=-1e30)
    loss, lp, _, entropy, wgrad, coef, seen = _policy_definition(clean, tokens * mask, adv.unsqueeze(1).expand(2, 4), None,
                                                                 None, mask, 1.0, 0.0, 0.1, "token_mean", 1.0)
    torch.testing.assert_close(got.logprobs.double(), lp, atol=LP, rtol=0)
    torch.testing.assert_close(got.entropy.double(), entropy, atol=LP, rtol=LP * 8)
    assert abs(float(got.loss) - float(loss)) < 4e-4
    _close_grad(grad, wgrad, coef, F32)
    assert (grad[0, 0, 5:900] == 0).all() and (grad[~mask] == 0).all()
    # A token outside the vocabulary in a scored row.
    tokens[1, 0] = 1001
    got, grad = losses.policy_loss_and_grad(logits, tokens, adv, None, mask)
    assert torch.isnan(got.loss) and torch.isnan(got.logprobs[1, 0]) and torch.isnan(grad[1, 0]).all()
    assert torch.isfinite(grad[0]).all() and torch.isfinite(grad[1, 1:]).all()
    ids = torch.full((2, 4, 3), 7, device=cuda_device)
    ids[0, 0, 1] = 1001
    got, grad = losses.distillation_loss_and_grad(logits, ids, torch.zeros(2, 4, 3, device=cuda_device), mask)
    assert torch.isnan(got.loss) and torch.isnan(got.kl[0, 0]) and torch.isnan(grad[0, 0, 0])
    assert torch.isfinite(got.kl[1]).all() and torch.isfinite(grad[1]).all()
    # A row without a finite column has no distribution.
    logits[0, 3] = -math.inf
    got, grad = losses.policy_loss_and_grad(logits, tokens, adv, None, mask)
    assert torch.isnan(got.logprobs[0, 3])


@pytest.mark.parametrize("dtype,v", [(BF16, 1000), (BF16, 1001), (F32, 1003), (F16, 777)])
def test_strided_rows(cuda_device, dtype, v):
    """Shifted slices, padded rows, transposed batches and broadcast rows give what their copies give."""
    from randomrepo_b200 import losses

    full, g = _logits(3, 9, v + 5, dtype, cuda_device)
    views = [full[:, :-1, :v], full[:, 1:, 3:v + 3], full.transpose(0, 1)[2:7, :, :v], full[1:2, :, :v],
             full[:, :1, :v].expand(3, 6, v), full[::2, ::3, 1:v + 1]]
    for x in views:
        b, t = x.shape[:2]
        tokens = torch.randint(0, v, (b, t + 2), generator=g).to(cuda_device)[:, 1:-1]
        mask = (torch.rand(t, b, generator=g) < 0.7).to(cuda_device).t()
        adv = torch.randn(b, generator=g).to(cuda_device)
        old = -7 + torch.randn(t, b, generator=g).to(cuda_device).t()
        kw = dict(entropy_coef=0.01)
        got, grad = losses.policy_loss_and_grad(x, tokens, adv, old, mask, **kw)
        want, wgrad = losses.policy_loss_and_grad(x.contiguous(), tokens.contiguous(), adv.unsqueeze(1).expand(b, t).contiguous(),
                                                  old.contiguous(), mask.contiguous(), **kw)
        # (rows that start elsewhere in their 16 bytes are summed in another order)
        torch.testing.assert_close(got.loss, want.loss, atol=1e-4, rtol=1e-4)
        torch.testing.assert_close(got.logprobs, want.logprobs, atol=LP, rtol=0)
        torch.testing.assert_close(grad.float(), wgrad.float(), atol=1e-5, rtol=2 * torch.finfo(dtype).eps + 1e-4)
        assert (grad[~mask] == 0).all()
        values, tok, _ = losses.top_logits(x, 9)
        wv, wt = _top_definition(x, 9)
        assert torch.equal(values, wv) and torch.equal(tok, wt)
        leaf = x.detach().requires_grad_()
        losses.policy_loss(leaf, tokens, adv, old, mask, **kw).loss.backward()
        torch.testing.assert_close(leaf.grad.float(), grad.float(), atol=1e-6, rtol=torch.finfo(dtype).eps)


def test_gradients_are_the_losses_differences(cuda_device):
    """Central differences of the loss along random directions (float32 rows; a step of 1e-2 leaves an error of
    h^2 / 6 times the third derivative, under 1e-4 of the slope here, and 2^-23 |loss| / h of rounding)."""
    from randomrepo_b200 import losses

    logits, g = _logits(4, 6, 301, F32, cuda_device, spread=1.0)
    tokens = torch.randint(0, 301, (4, 6), generator=g).to(cuda_device)
    adv = torch.randn(4, generator=g).to(cuda_device)
    old = torch.log_softmax(logits, -1).gather(-1, tokens.unsqueeze(-1)).squeeze(-1) - 0.05
    ids = torch.randint(0, 301, (4, 6, 12), generator=g).to(cuda_device)
    teacher = torch.randn(4, 6, 12, generator=g).to(cuda_device)
    calls = [lambda x: losses.policy_loss_and_grad(x, tokens, adv, old, entropy_coef=0.1, temperature=0.9),
             lambda x: losses.preference_loss_and_grad(x, tokens, beta=0.3),
             lambda x: losses.distillation_loss_and_grad(x, ids, teacher, temperature=1.3)]
    for call in calls:
        base, grad = call(logits)
        for _ in range(3):
            d = torch.randn(logits.shape, generator=g).to(cuda_device)
            h = 1e-2
            slope = (float(call(logits + h * d)[0].loss) - float(call(logits - h * d)[0].loss)) / (2 * h)
            along = float((grad.double() * d.double()).sum())
            scale = float((grad.double().abs() * d.double().abs()).sum())
            assert abs(slope - along) <= 2e-3 * scale + 2.0**-22 * abs(float(base.loss)) / h, (slope, along)


def test_calls_repeat_bit_for_bit_and_leave_inputs_alone(cuda_device):
    from randomrepo_b200 import losses

    logits, ids, teacher, g = _distill_case(5, 40, 4099, 32, BF16, cuda_device)
    tokens = torch.randint(0, 4099, (5, 40), generator=g).to(cuda_device)
    mask = _mask("some", 5, 40, g, cuda_device)
    adv = torch.randn(5, generator=g).to(cuda_device)
    before = logits.clone()
    calls = [lambda: losses.policy_loss_and_grad(logits, tokens, adv, None, mask, entropy_coef=0.01),
             lambda: losses.preference_loss_and_grad(logits[:4], tokens[:4], mask[:4]),
             lambda: losses.distillation_loss_and_grad(logits, ids, teacher, mask)]
    for call in calls:
        first, grad = call()
        for _ in range(5):
            again, grad2 = call()
            assert torch.equal(first.loss, again.loss) and torch.equal(grad, grad2)
    assert torch.equal(logits, before)


@pytest.mark.parametrize("b,t", [(1, 1), (3, 700), (2000, 3), (1, 70000), (70000, 1), (37, 1901)])
def test_weights_of_many_rows(cuda_device, b, t):
    """The plan of the scored rows: every row in its place and every sequence's weight, for runs of rows of all lengths."""
    from randomrepo_b200 import losses

    g = torch.Generator().manual_seed(b + t)
    logits = torch.randn(b, t, 8, generator=g).to(cuda_device)
    mask = (torch.rand(b, t, generator=g) < 0.4).to(cuda_device)
    mask[0, 0] = True
    tokens = torch.randint(0, 8, (b, t), generator=g).to(cuda_device)
    adv = torch.randn(b, t, generator=g).to(cuda_device)
    for reduction in ("token_mean", "sequence_mean"):
        got, grad = losses.policy_loss_and_grad(logits, tokens, adv, None, mask, reduction=reduction, scale=float(b * t))
        w = _weights(mask, b, t, reduction, float(b * t), cuda_device)
        p = torch.softmax(logits.double(), -1)
        p.scatter_add_(-1, tokens.unsqueeze(-1), -torch.ones(b, t, 1, dtype=torch.float64, device=cuda_device))
        want = p * (w * adv.double()).unsqueeze(-1)
        torch.testing.assert_close(grad.double(), want, atol=1e-6 * float(w.max()) * 4, rtol=1e-5)
        assert abs(float(got.loss) + float((w * adv.double()).sum())) <= 1e-6 * float((w * adv.double()).abs().sum())


def test_capture_streams_and_two_calls_at_once(cuda_device):
    """A captured call replays on new inputs; two captured calls, and calls on two streams, do not share anything."""
    from randomrepo_b200 import losses

    def case(seed):
        logits, tokens, adv, old, ref, mask = _policy_case(3, 20, 5003, BF16, cuda_device, "some", seed)
        return dict(logits=logits, tokens=tokens, advantages=adv, old_logprobs=old, mask=mask, ref_logprobs=ref, kl_coef=0.1)

    a, b, new = case(1), case(2), case(3)
    want = [losses.policy_loss_and_grad(**c) for c in (a, b, new)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses.policy_loss_and_grad(**a)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in (a, b):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(losses.policy_loss_and_grad(**c))
        graphs.append(gr)
    for gr in graphs:
        gr.replay()
    for (got, grad), (w, wg) in zip(outs, want):
        assert torch.equal(got.loss, w.loss) and torch.equal(grad, wg)
    for key in ("logits", "tokens", "advantages", "old_logprobs", "mask", "ref_logprobs"):
        a[key].copy_(new[key])
    graphs[0].replay()
    graphs[1].replay()
    assert torch.equal(outs[0][0].loss, want[2][0].loss) and torch.equal(outs[0][1], want[2][1])
    assert torch.equal(outs[1][0].loss, want[1][0].loss) and torch.equal(outs[1][1], want[1][1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, c, into in zip(streams, (b, new), got):
            with torch.cuda.stream(s):
                into.append(losses.policy_loss_and_grad(**c))
    torch.cuda.synchronize()
    for into, (w, wg) in zip(got, want[1:]):
        for r, grad in into:
            assert torch.equal(r.loss, w.loss) and torch.equal(grad, wg)


def test_captured_backward(cuda_device):
    """Forward and backward of the differentiable form in one graph (its leaf in no other), replayed on new logits."""
    from randomrepo_b200 import losses

    logits, tokens, adv, old, ref, mask = _policy_case(2, 9, 4099, F16, cuda_device, "some", 8)
    other = _policy_case(2, 9, 4099, F16, cuda_device, "some", 9)[0]

    def step(x):
        leaf = x.detach().requires_grad_()
        out = losses.policy_loss(leaf, tokens, adv, old, mask, entropy_coef=0.01, scale=8.0)
        return out.loss.detach(), torch.autograd.grad(out.loss, leaf)[0]

    want = [step(logits), step(other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(logits)
    torch.cuda.current_stream().wait_stream(side)
    x = logits.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step(x)
    for data, (wl, wg) in zip((logits, other), want):
        x.copy_(data)
        graph.replay()
        assert torch.equal(loss, wl) and torch.equal(grad, wg)


def test_backward_twice_and_through_a_model(cuda_device):
    """retain_graph backward passes give the same gradient; a small head trains through the loss."""
    from randomrepo_b200 import losses

    g = torch.Generator().manual_seed(4)
    hidden = torch.randn(2, 5, 16, generator=g).to(cuda_device)
    head = torch.randn(301, 16, generator=g).to(cuda_device).requires_grad_()
    tokens = torch.randint(0, 301, (2, 5), generator=g).to(cuda_device)
    adv = torch.tensor([1.0, -0.5], device=cuda_device)
    out = losses.policy_loss((hidden @ head.t())[:, :-1], tokens[:, 1:], adv)
    (g1,) = torch.autograd.grad(out.loss, head, retain_graph=True)
    (g2,) = torch.autograd.grad(out.loss, head)
    assert torch.equal(g1, g2)
    x = hidden.double() @ head.detach().double().t()
    x.requires_grad_()
    lp = torch.log_softmax(x[:, :-1], -1).gather(-1, tokens[:, 1:].unsqueeze(-1)).squeeze(-1)
    ref = -((lp - lp.detach()).exp() * adv.double().unsqueeze(1)).mean()
    want = torch.autograd.grad(ref, x)[0].flatten(0, 1).t() @ hidden.double().flatten(0, 1)
    torch.testing.assert_close(g1.double(), want, atol=1e-5, rtol=1e-4)
    assert not out.logprobs.requires_grad


def test_empty_batches(cuda_device):
    from randomrepo_b200 import losses

    for b, t in ((0, 5), (2, 0), (0, 0)):
        x = torch.empty(b, t, 33, device=cuda_device)
        tok = torch.empty(b, t, dtype=torch.int64, device=cuda_device)
        got, grad = losses.policy_loss_and_grad(x, tok, torch.empty(b, t, device=cuda_device))
        assert float(got.loss) == 0.0 and grad.shape == x.shape and got.logprobs.shape == (b, t)
        got, grad = losses.distillation_loss_and_grad(x, tok.unsqueeze(-1).expand(b, t, 2), x[..., :2])
        assert float(got.loss) == 0.0 and grad.shape == x.shape
        got, grad = losses.preference_loss_and_grad(x, tok)
        want = math.log(2) if b else 0.0
        assert abs(float(got.loss) - want) < 1e-6 and grad.shape == x.shape and got.margins.shape == (b // 2,)
        values, ids, lse = losses.top_logits(x, 3)
        assert values.shape == (b, t, 3) and lse.shape == (b, t)


def test_a_rollouts_training_step(cuda_device):
    """The set as it is used: the teacher's top logits distil a student, and the policy loss of the same rows agrees
    with the sampler's own log-probabilities."""
    from randomrepo_b200 import losses
    from randomrepo_b200.sampling import DeviceSampler

    logits, tokens, adv, _, _, mask = _policy_case(4, 12, 8200, F32, cuda_device, "some")
    old = DeviceSampler(cuda_device).token_logprobs(logits, tokens)
    got, grad = losses.policy_loss_and_grad(logits, tokens, adv, old, mask)
    torch.testing.assert_close(got.logprobs, torch.where(mask, old, 0.0), atol=2 * LP, rtol=0)
    values, ids, lse = losses.top_logits(logits, 256, temperature=2.0)
    # A student that equals its teacher has nothing to learn but the list's missing tail.
    own, grad = losses.distillation_loss_and_grad(logits, ids, values, mask, teacher_lse=lse, temperature=2.0)
    assert own.kl.abs().max() <= 4 * 2 * LP
    student = torch.randn(logits.shape, generator=torch.Generator().manual_seed(9)).to(cuda_device).requires_grad_()
    first = None
    for _ in range(5):
        out = losses.distillation_loss(student, ids, values, mask, temperature=2.0, reduction="sum")
        first = out.loss.item() if first is None else first
        (step,) = torch.autograd.grad(out.loss, student)
        student = (student - step).detach().requires_grad_()
    assert step.isfinite().all() and out.loss.isfinite()


def test_operators_equal_the_functions(cuda_device):
    """``torch.ops.pkv`` losses are the same calls."""
    import randomrepo_b200.ops  # noqa: F401 - registers the operators
    from randomrepo_b200 import losses

    logits, ids, teacher, g = _distill_case(4, 6, 1001, 9, BF16, cuda_device)
    tokens = torch.randint(0, 1001, (4, 6), generator=g).to(cuda_device)
    mask = _mask("some", 4, 6, g, cuda_device)
    adv = torch.randn(4, generator=g).to(cuda_device)
    ref = -7 + torch.randn(4, 6, generator=g).to(cuda_device)
    want, grad = losses.policy_loss_and_grad(logits, tokens, adv, None, mask, ref_logprobs=ref, kl_coef=0.1)
    got = torch.ops.pkv.policy_loss(logits, tokens, adv, None, mask, ref, 0.2, 0.2, 0.1, 0.0, 1.0, "token_mean", 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, (*want[:3], torch.empty(0, device=cuda_device), grad)))
    want, grad = losses.preference_loss_and_grad(logits, tokens, mask, None, beta=0.3)
    got = torch.ops.pkv.preference_loss(logits, tokens, mask, None, 0.3, 0.0, False, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, (*want, grad)))
    want, grad = losses.distillation_loss_and_grad(logits, ids, teacher, mask, temperature=2.0)
    got = torch.ops.pkv.distillation_loss(logits, ids, teacher, mask, None, 2.0, "token_mean", 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, (*want, grad)))
    got = torch.ops.pkv.top_logits(logits, 5, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, losses.top_logits(logits, 5)))


def test_refusals_on_the_device(cuda_device):
    """What the host can see is refused before a launch; a second derivative and a changed input are errors."""
    from randomrepo_b200 import losses

    logits, g = _logits(2, 3, 33, F32, cuda_device)
    tokens = torch.randint(0, 33, (2, 3), generator=g).to(cuda_device)
    adv = torch.ones(2, device=cuda_device)
    with pytest.raises(ValueError):
        losses.policy_loss(logits, tokens.cpu(), adv)
    with pytest.raises(ValueError):
        losses.policy_loss(logits, tokens, adv, mask=torch.ones(2, 3))  # on the host
    with pytest.raises(ValueError):
        losses.top_logits(logits, 34)
    leaf = logits.detach().requires_grad_()
    out = losses.policy_loss(leaf, tokens, adv)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.loss, leaf, create_graph=True)
    out = losses.policy_loss(leaf, tokens, adv)
    tokens.add_(0)
    with pytest.raises(RuntimeError, match="modified"):
        out.loss.backward()


def test_int_masks_and_types_are_taken(cuda_device):
    """HF attention masks (int64), uint8 and float masks, int32 tokens, float64 inputs and [T, V] rows."""
    from randomrepo_b200 import losses

    logits, tokens, adv, old, ref, mask = _policy_case(3, 7, 301, F32, cuda_device, "some")
    want, grad = losses.policy_loss_and_grad(logits, tokens, adv, old, mask, ref_logprobs=ref, kl_coef=0.1)
    for m in (mask.long(), mask.byte() * 255, mask.float() * 0.5):
        got, g2 = losses.policy_loss_and_grad(logits, tokens.int(), adv.double(), old.double(), m, ref_logprobs=ref,
                                              kl_coef=0.1)
        assert torch.equal(got.loss, want.loss) and torch.equal(grad, g2)
    one, g1 = losses.policy_loss_and_grad(logits[0], tokens[0], adv[0], old[0], mask[0], reduction="sum")
    two, g2 = losses.policy_loss_and_grad(logits[:1], tokens[:1], adv[:1], old[:1], mask[:1], reduction="sum")
    assert one.logprobs.shape == (7,) and g1.shape == (7, 301)
    assert torch.equal(one.loss, two.loss) and torch.equal(g1, g2[0])
    leaf = logits[0].detach().requires_grad_()
    losses.policy_loss(leaf, tokens[0], adv[0], old[0], mask[0], reduction="sum").loss.backward()
    torch.testing.assert_close(leaf.grad, g1, atol=1e-6, rtol=1e-5)
    leaf = logits[0].detach().requires_grad_()  # [T, V] rows apart, at an odd place
    losses.policy_loss(leaf[1::2, 3:], tokens[0, 1::2] % 298, adv[0, 1::2], reduction="sum").loss.backward()
    _, g2 = losses.policy_loss_and_grad(logits[0, 1::2, 3:], tokens[0, 1::2] % 298, adv[0, 1::2], reduction="sum")
    torch.testing.assert_close(leaf.grad[1::2, 3:], g2, atol=1e-6, rtol=1e-5)


@pytest.mark.parametrize("dtype,chunk,slots", [(BF16, 20480, 5), (F32, 6144, 8), (F16, 4096, 5), (F32, 2048, 5)])
@pytest.mark.parametrize("chunks", [1, -1, 0, 2])
def test_rows_of_changing_chunk_counts(cuda_device, dtype, chunk, slots, chunks):
    """Odd rows start at every offset in their 16 bytes, so that some have a 16-byte vector, and here a chunk of the
    kernels' ring, less than others: around one chunk, and around as many as the ring holds (slots - 1, slots, + 2).
    Enough rows for several turns of every CTA."""
    from randomrepo_b200 import losses

    per = 16 // dtype.itemsize
    v = (1 if chunks == 1 else slots + chunks) * chunk + per + 1
    n = 330 if v > 60000 else 1500
    g = torch.Generator(device=cuda_device).manual_seed(v)
    logits = torch.randn(1, n, v, generator=g, device=cuda_device).to(dtype)
    assert len({logits[0, i].data_ptr() % 16 for i in range(16)}) == per
    tokens = torch.randint(0, v, (1, n), generator=g, device=cuda_device)
    adv = torch.randn(1, n, generator=g, device=cuda_device)
    got, grad = losses.policy_loss_and_grad(logits, tokens, adv, reduction="sum")
    ids = torch.randint(0, v, (1, n, 5), generator=g, device=cuda_device)
    teacher = torch.randn(1, n, 5, generator=g, device=cuda_device)
    dis, dgrad = losses.distillation_loss_and_grad(logits, ids, teacher, reduction="sum")
    for i in range(0, n, 150):
        at = slice(i, i + 150)
        rows = torch.log_softmax(logits[0, at].double(), -1)
        pick = rows.gather(-1, tokens[0, at].unsqueeze(-1)).squeeze(-1)
        torch.testing.assert_close(got.logprobs[0, at].double(), pick, atol=LP, rtol=0)
        want = rows.exp()
        want.scatter_add_(-1, tokens[0, at].unsqueeze(-1), -torch.ones_like(pick).unsqueeze(-1))
        coef = adv[0, at].double().unsqueeze(-1)
        _close_grad(grad[0, at], want * coef, coef, dtype)
        q = torch.softmax(teacher[0, at].double(), -1)
        want = rows.exp().scatter_add_(-1, ids[0, at], -q)
        _close_grad(dgrad[0, at], want, torch.ones_like(coef) * 2, dtype)


def test_rows_past_32_bits(cuda_device):
    """A tensor whose last rows start past 2^32 bytes and 2^31 elements."""
    from randomrepo_b200 import losses

    v = 151936
    flat = torch.zeros(16384, v, dtype=BF16, device=cuda_device)  # 2.5 G elements
    g = torch.Generator().manual_seed(3)
    small = (torch.randn(3, v, generator=g) * 3).to(BF16).to(cuda_device)
    flat[-3:] = small
    mask = torch.zeros(1, 16384, dtype=torch.bool, device=cuda_device)
    mask[0, -3:] = True
    tokens = torch.randint(0, v, (1, 16384), generator=g).to(cuda_device)
    adv = torch.ones(1, device=cuda_device)
    got, grad = losses.policy_loss_and_grad(flat.unsqueeze(0), tokens, adv, None, mask)
    want, wgrad = losses.policy_loss_and_grad(small.unsqueeze(0), tokens[:, -3:], adv)
    torch.testing.assert_close(got.logprobs[0, -3:], want.logprobs[0], atol=LP, rtol=0)
    torch.testing.assert_close(grad[0, -3:].float(), wgrad[0].float(), atol=1e-6, rtol=2.0**-7)
    assert not grad[0, :-3].any()
    del grad, wgrad
    values, ids, _ = losses.top_logits(flat, 4)
    assert torch.equal(ids[-3:], _top_definition(small, 4)[1]) and torch.equal(ids[0].cpu(), torch.arange(4))
