"""The vocabulary-row losses at their limits: certain tokens, large values, small divergences, what is left on the graph.

Definitions are torch operations in 64 bits; each tolerance is derived where it stands.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _half(dtype):
    """Half a step of a gradient of ``dtype``, relative."""
    return torch.finfo(dtype).eps / 2


def _float(x):
    """``x`` as the kernels have it."""
    return float(torch.tensor(x, dtype=F32))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature,top,gap", [(0.7, 24.0, 4.0), (0.7, 48.0, 6.0), (0.1, 30.0, 1.0), (0.01, 30.0, 0.125),
                                                 (2.0, 4096.0, 16.0)])
@pytest.mark.parametrize("entropy", [0.0, 0.5])
def test_a_certain_tokens_gradient(cuda_device, dtype, temperature, top, gap, entropy):
    """p near 1 at the token, and q near p in a teacher's list: terms of a large coefficient that nearly cancel.

    A term e a (a = -h / s) against h is off by 2^-22 each for the approximate 2^y of the column, of the sum's columns
    and for the factor that stands for the scale's low half, and by five roundings of 2^-24: 17 x 2^-24 < 2^-19 of h.
    The entropy's terms are p (log p + H), at most 1/e + H <= 1.1 of their coefficient here, of the same parts."""
    from randomrepo_b200 import losses

    v, t = 41, _float(temperature)
    x = torch.full((2, 3, v), top - 40.0 * temperature)
    x[..., 7], x[..., 19] = top, top - gap
    x = x.to(dtype)
    assert float(x[0, 0, 7] - x[0, 0, 19]) == gap
    x = x.to(cuda_device)
    tokens = torch.full((2, 3), 7, device=cuda_device)
    tokens[:, 1] = 19
    adv = torch.tensor([1.0, -0.5], device=cuda_device)

    def compare(grad, leaf, want, coef):
        # (the float32 coefficients are made of a few roundings of their own: 2^-22 of the value)
        tol = want.abs() * ((0 if dtype == F32 else _half(dtype)) + 2.0**-22) + coef.abs() * 2.0**-19
        if dtype == F16:
            tol = tol + 2.0**-25
        for got in (grad, leaf):
            off = (got.double() - want).abs()
            assert (off <= tol).all(), (off.max(), (off / tol).max(), got.double()[off > tol][:3], want[off > tol][:3])

    y = x.double().requires_grad_()
    rows = torch.log_softmax(y / t, -1)
    lp = rows.gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    h = -(rows.exp() * rows).sum(-1)
    want = torch.autograd.grad(-(lp * adv.double().unsqueeze(1)).sum() - _float(entropy) * h.sum(), y)[0]
    got, grad = losses.policy_loss_and_grad(x, tokens, adv, entropy_coef=entropy, temperature=temperature, reduction="sum")
    leaf = x.detach().requires_grad_()
    losses.policy_loss(leaf, tokens, adv, entropy_coef=entropy, temperature=temperature, reduction="sum").loss.backward()
    compare(grad, leaf.grad, want, ((adv.abs() + 1.1 * entropy) / t).double().view(2, 1, 1))
    if entropy:
        return
    ids = torch.tensor([7, 19], device=cuda_device).expand(2, 3, 2)
    teacher = x[..., [7, 19]].float() + torch.tensor([0.0, 0.02 * temperature], device=cuda_device)
    y = x.double().requires_grad_()
    q = torch.softmax(teacher.double() / t, -1)
    lp = torch.log_softmax(y / t, -1)[..., [7, 19]]
    want = torch.autograd.grad(t * t * (q * (q.log() - lp)).sum(), y)[0]
    got, grad = losses.distillation_loss_and_grad(x, ids, teacher, temperature=temperature, reduction="sum")
    leaf = x.detach().requires_grad_()
    losses.distillation_loss(leaf, ids, teacher, temperature=temperature, reduction="sum").loss.backward()
    # (q is an expf of a float32 argument of at most 12: 2^-20 of q)
    compare(grad, leaf.grad, want, torch.tensor(3 * t, device=cuda_device))
