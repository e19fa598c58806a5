"""The vocabulary-row losses at their limits: certain tokens, large values, small divergences, what is left on the graph.

Definitions are torch operations in 64 bits; each tolerance is derived where it stands.
"""

from __future__ import annotations

import ctypes
import math

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


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_of_large_values(cuda_device, dtype):
    """Rows whose values times the scale are far past what a float32 exponent's reference holds (a mask of -1e9 in every
    column, the largest float16 at a low temperature): uniform, and exact where neighbouring values differ.

    log p: a column's exponent is at most 40 where it counts, rounded three times (40 x 3 x 2^-24 ln 2 = 5e-6), its
    approximate 2^y is off by 2^-22 and a sum of up to 1000 columns in float32 by at most 16 additions a thread and
    their merges (32 x 2^-24 = 2e-6): below 1e-5.  Gradients: that of p."""
    from randomrepo_b200 import losses

    v = 1000
    values = {BF16: [-1e9, 1e9, 3e7, -1e30, 1e37], F16: [-65504.0, 65504.0, 30000.0], F32: [-1e9, 1e9, 123456789.0, -1e30, 1e37]}[dtype]
    for temperature in (1.0, 0.1, 1e-2, 1e-4, 1e-6):
        t = _float(temperature)
        x = torch.tensor(values).to(dtype).unsqueeze(1).repeat(1, v).unsqueeze(0)
        # Some columns a step of the type below the others.
        x[:, :, 100:900] = torch.nextafter(x[:, :, 100:900], torch.tensor(-math.inf, dtype=dtype)) if dtype != BF16 else x[:, :, 100:900]
        x = x.to(cuda_device)
        tokens = torch.full(x.shape[:2], 3, device=cuda_device)
        rows = torch.log_softmax(x.double() / t, -1)
        got, grad = losses.policy_loss_and_grad(x, tokens, torch.ones(1, device=cuda_device), temperature=temperature,
                                                reduction="sum", scale=t)
        want = rows.exp()
        want[..., 3] -= 1
        assert (got.logprobs.double() - rows[..., 3]).abs().max() <= 1e-5, (temperature, got.logprobs, rows[..., 3])
        off = (grad.double() - want).abs()
        tol = want.abs() * (_half(dtype) + 1e-5) + 1e-5 * rows.exp() + 2.0**-22 + (2.0**-25 if dtype == F16 else 0)
        assert (off <= tol).all(), (temperature, off.max())
        _, _, lse = losses.top_logits(x, 3, temperature=temperature)
        ref = (x.double() / t).logsumexp(-1)
        assert ((lse.double() - ref).abs() <= 1e-5 + 2.0**-23 * ref.abs()).logical_or(lse == ref.float()).all()
        ids = torch.tensor([5, 77], device=cuda_device).expand(*x.shape[:2], 2)
        q = torch.zeros(*x.shape[:2], 2, device=cuda_device)
        dis, _ = losses.distillation_loss_and_grad(x, ids, q, temperature=temperature, reduction="sum")
        per = t * t * (-math.log(2) - rows[..., [5, 77]].mean(-1))
        assert ((dis.kl.double() - per).abs() <= t * t * 1.2e-5 + 2.0**-22 * per.abs()).all()


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
def test_rows_across_the_far_border(cuda_device, temperature):
    """float32 values on both sides of where the kernels begin to subtract before they scale, in ascending and
    descending order (every warp's reference crosses it), 8 T apart at the least; bounds as above with more columns:
    50 001 of them in up to 80 additions a thread (1e-5 more)."""
    from randomrepo_b200 import losses

    v, t = 50001, _float(temperature)
    border = 1e8 * t / math.log2(math.e)
    g = torch.Generator().manual_seed(5)
    steps = torch.randint(-6, 7, (v,), generator=g).float() * 8
    for sign in (1.0, -1.0):
        base = torch.tensor(sign * border, dtype=F32)
        rows = torch.stack([base + steps, (base + steps).sort().values, (base + steps).sort(descending=True).values])
        x = rows.unsqueeze(0).to(cuda_device)
        tokens = x.argmax(-1)
        want = torch.log_softmax(x.double() / t, -1).gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
        got, grad = losses.policy_loss_and_grad(x, tokens, torch.ones(1, device=cuda_device), temperature=temperature,
                                                reduction="sum", scale=t)
        assert (got.logprobs.double() - want).abs().max() <= 2e-5, (got.logprobs, want)
        p = torch.softmax(x.double() / t, -1)
        p.scatter_add_(-1, tokens.unsqueeze(-1), -torch.ones_like(want).unsqueeze(-1))
        assert (grad.double() - p).abs().max() <= 2e-5
        _, _, lse = losses.top_logits(x, 3, temperature=temperature)
        ref = (x.double() / t).logsumexp(-1)
        assert ((lse.double() - ref).abs() <= 2e-5 + 2.0**-23 * ref.abs()).logical_or(lse == ref.float()).all()


def _header(call_ws):
    """The workspace's header as 32-bit words: scored rows, ticket, error."""
    return call_ws[:12].view(torch.int32)


class _Array(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64)]


class _Rows(ctypes.Structure):
    _fields_ = [("logits", _Array), ("grad", _Array), ("mask", _Array), ("batch", ctypes.c_int32),
                ("length", ctypes.c_int32), ("vocab", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("temperature", ctypes.c_float)]


class _Preference(ctypes.Structure):
    _fields_ = [("tokens", _Array), ("ref", ctypes.c_void_p), ("beta", ctypes.c_float), ("smoothing", ctypes.c_float),
                ("normalised", ctypes.c_int32), ("scale", ctypes.c_float)]


def _array2(t):
    return _Array(t.data_ptr(), t.stride(0), t.stride(1))


def test_an_error_of_the_forward_pass_makes_gradients_nan(cuda_device):
    """A wait that gave up in the forward launch leaves its mark in the workspace; a later backward pass is NaN."""
    from randomrepo_b200 import losses

    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 5, 301, generator=g).to(cuda_device)
    tokens = torch.randint(0, 301, (2, 5), generator=g).to(cuda_device)
    ids = torch.randint(0, 301, (2, 5, 4), generator=g).to(cuda_device)
    teacher = torch.randn(2, 5, 4, generator=g).to(cuda_device)
    mask = torch.ones(2, 5, dtype=torch.bool, device=cuda_device)
    mask[1, 3] = False
    for call in (lambda z: losses.policy_loss(z, tokens, torch.ones(2, device=cuda_device), None, mask),
                 lambda z: losses.policy_loss(z, tokens, torch.ones(2, device=cuda_device), None, mask, entropy_coef=0.1),
                 lambda z: losses.preference_loss(z, tokens, mask),
                 lambda z: losses.distillation_loss(z, ids, teacher, mask)):
        leaf = x.clone().requires_grad_()
        out = call(leaf)
        (grad,) = torch.autograd.grad(out.loss, leaf, retain_graph=True)
        assert grad.isfinite().all()
        ws = [s for s in out.loss.grad_fn.saved_tensors if s is not None and s.dtype == torch.uint8]
        assert len(ws) == 1
        _header(ws[0].data)[2] = 1  # (.data: not a change that the saved tensors' check should see)
        (grad,) = torch.autograd.grad(out.loss, leaf)
        assert grad[mask].isnan().all() and (grad[~mask] == 0).all()


def test_an_error_of_the_preference_sums_is_loud(cuda_device):
    """The mark of a wait that gave up in the sums' launch, set here by a copy while that launch runs (1.2 GB of rows:
    0.3 ms and more after the plan has cleared it): loss, margins, sums and the gradient are NaN.  The copy may come too
    late, so there are several trials; without a mark nothing is ever NaN."""
    from randomrepo_b200 import _lib
    from randomrepo_b200._lib import lib

    b, t, v = 2, 4096, 151936
    x = torch.zeros(b, t, v, dtype=BF16, device=cuda_device)
    grad = torch.empty_like(x)
    tokens = torch.zeros(b, t, dtype=torch.int64, device=cuda_device)
    rows = _Rows(logits=_array2(x), grad=_array2(grad), batch=b, length=t, vocab=v, dtype=_lib.PKV_BF16, temperature=1.0)
    terms = _Preference(tokens=_array2(tokens), beta=0.1, scale=1.0)
    n = lib.pkv_loss_workspace_bytes(b, t)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda_device)
    out = torch.empty(4, device=cuda_device)
    mark = torch.ones(1, dtype=torch.int32).pin_memory()
    side = torch.cuda.Stream()
    for _ in range(8):
        torch.cuda.synchronize()
        st = lib.pkv_preference_loss(ctypes.byref(rows), ctypes.byref(terms), out.data_ptr(), out.data_ptr() + 4,
                                     out.data_ptr() + 12, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert st == 0, _lib.last_error()
        with torch.cuda.stream(side):
            _header(ws)[2:3].copy_(mark, non_blocking=True)
        torch.cuda.synchronize()
        if out.isnan().any():
            break
    assert out.isnan().all()
    assert grad[0, 0].isnan().all() and grad[1, -1].isnan().all()


def _differentiable_calls(dev):
    """(name, call) of the three losses over rows [2, 4, 301], with inputs that need no conversion and some that do."""
    from randomrepo_b200 import losses

    g = torch.Generator().manual_seed(12)
    tokens = torch.randint(0, 301, (2, 4), generator=g).to(dev)
    old = (-6 + torch.randn(2, 4, generator=g)).to(dev)
    adv = torch.randn(2, generator=g).to(dev)
    mask = (torch.rand(4, 2, generator=g) < 0.8).to(dev).t()
    ids = torch.randint(0, 301, (2, 4, 6), generator=g).to(dev)
    teacher = torch.randn(2, 4, 12, generator=g).to(dev)[..., ::2]
    ref = torch.randn(2, generator=g).to(dev)
    return [lambda z: losses.policy_loss(z, tokens, adv, old, mask, ref_logprobs=old + 0.1, kl_coef=0.1, temperature=0.8),
            lambda z: losses.policy_loss(z, tokens.int(), adv.unsqueeze(1), old.double(), mask.long(), entropy_coef=0.1),
            lambda z: losses.preference_loss(z, tokens, mask, ref, beta=0.3, length_normalised=True),
            lambda z: losses.distillation_loss(z, ids, teacher, mask, temperature=2.0),
            lambda z: losses.distillation_loss(z, ids.int(), teacher, None, teacher_lse=old.abs())]


def test_the_backward_pass_frees_the_logits(cuda_device):
    """The loss may outlive its backward pass (a log keeps it); the logits and the workspace do not."""
    g = torch.Generator().manual_seed(1)
    head = torch.randn(2, 4, 301, generator=g).to(cuda_device).requires_grad_()
    for call in _differentiable_calls(cuda_device):
        call(head).loss.backward()  # (head.grad is there from now on)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        logits = head * 1.5
        size = torch.cuda.memory_allocated() - before
        out = call(logits)
        del logits
        out.loss.backward()
        # What is left: the loss and the rows' values, 512 bytes each at the least.
        assert torch.cuda.memory_allocated() - before <= 4 * 512 < size
        assert out.loss.isfinite()
        head.grad = torch.zeros_like(head)


def test_saved_tensor_hooks_are_heard(cuda_device):
    """Tensors that were offloaded to the host come back for the backward pass; recomputed ones likewise."""
    from torch.utils.checkpoint import checkpoint

    g = torch.Generator().manual_seed(6)
    data = torch.randn(2, 4, 301, generator=g).to(cuda_device)
    for call in _differentiable_calls(cuda_device):
        leaf = data.clone().requires_grad_()
        (want,) = torch.autograd.grad(call(leaf * 1.5).loss, leaf)
        before = torch.cuda.memory_allocated()
        with torch.autograd.graph.save_on_cpu():
            logits = leaf * 1.5
            out = call(logits)
        size = logits.numel() * 4
        del logits
        assert torch.cuda.memory_allocated() - before < size  # (the logits are on the host alone)
        (got,) = torch.autograd.grad(out.loss, leaf)
        assert torch.equal(got, want)
        (got,) = torch.autograd.grad(checkpoint(lambda z: call(z * 1.5).loss, leaf, use_reentrant=False), leaf)
        assert torch.equal(got, want)

        # What a hook hands back is what is read.
        def double(t):
            return t * 2 if t.shape == data.shape else t

        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), double):
            out = call(leaf)
        (got,) = torch.autograd.grad(out.loss, leaf)
        assert not torch.equal(got, torch.autograd.grad(call(leaf).loss, leaf)[0])

        # Another shape, type or device than was saved would be read out of bounds: refused before a launch.
        for wrong in (lambda t: t.cpu(), lambda t: t[:1] if t.dim() == 3 else t, lambda t: t.double()):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), wrong):
                out = call(leaf)
            with pytest.raises(RuntimeError, match="hook"):
                torch.autograd.grad(out.loss, leaf)
        # The same values in another order of memory are taken.
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t.mT.contiguous().mT if t.dim() > 1 else
                                                      t.repeat_interleave(2)[::2] if t.dtype != torch.uint8 else t):
            out = call(leaf)
        (got,) = torch.autograd.grad(out.loss, leaf)
        torch.testing.assert_close(got, torch.autograd.grad(call(leaf).loss, leaf)[0], atol=0, rtol=0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_without_a_teacher_entry(cuda_device, dtype):
    """A scored row whose entries are all absent (or have no share left) adds nothing and has a zero gradient, whatever
    its logits are: the lowest value, -inf, NaN in every column.  A NaN share and an id past the vocabulary stay loud."""
    from randomrepo_b200 import losses

    v, k = 300, 5
    g = torch.Generator().manual_seed(3)
    fills = [torch.finfo(dtype).min, -math.inf, math.nan, math.inf, torch.finfo(dtype).max, 0.0]
    x = torch.randn(len(fills) + 1, 2, v, generator=g)
    for i, f in enumerate(fills):
        x[i, 1] = f
    x = x.to(dtype).to(cuda_device)
    ids = torch.randint(0, v, (len(fills) + 1, 2, k), generator=g).to(cuda_device)
    teacher = torch.randn(len(fills) + 1, 2, k, generator=g).to(cuda_device)
    absent, low = ids.clone(), teacher.clone()
    absent[:, 1] = -1
    low[:, 1] = -math.inf
    far = torch.zeros(len(fills) + 1, 2, device=cuda_device)
    far[:, 1] = 1e30  # (the teacher's row has all its mass elsewhere: every share underflows)
    rows = x[:, 0].double()
    for i, t, lse in ((absent, teacher, None), (ids, low, None), (ids, teacher, far)):
        q = torch.softmax(t[:, 0].double(), -1) if lse is None else t[:, 0].double().exp()
        lq = q.log()
        per = (q * (lq - torch.log_softmax(rows, -1).gather(-1, i[:, 0]))).sum(-1)
        want = torch.softmax(rows, -1) * q.sum(-1, keepdim=True)
        want.scatter_add_(-1, i[:, 0], -q)
        got, grad = losses.distillation_loss_and_grad(x, i, t, teacher_lse=lse, reduction="sum")
        leaf = x.detach().requires_grad_()
        out = losses.distillation_loss(leaf, i, t, teacher_lse=lse, reduction="sum")
        (own,) = torch.autograd.grad(out.loss, leaf)
        for res, d in ((got, grad), (out, own)):
            empty = [r for r in range(len(fills) + 1) if lse is None or r != 2]  # (a share of 0 times NaN is NaN)
            assert (res.kl[empty, 1] == 0).all() and (d[empty, 1] == 0).all()
            if lse is not None:
                assert res.kl[2, 1].isnan() and res.loss.isnan() and d[2, 1].isnan().all()
                continue
            # (a share and a log-probability are off by at most 2e-5 of a term, as in the other tests of this loss)
            size = (q * (lq.abs() + 20)).sum(-1)
            assert ((res.kl[:, 0].double() - per).abs() <= 2.5e-5 * size).all()
            assert abs(float(res.loss.detach()) - float(per.sum())) <= 2.5e-5 * float(size.sum())
            assert ((d[:, 0].double() - want).abs() <= want.abs() * _half(dtype) + 2.5e-5 * q.sum(-1, keepdim=True)).all()
    ids[0, 1], teacher[1, 1, 2] = v, math.nan
    for f in (losses.distillation_loss_and_grad(x, ids, teacher)[0], losses.distillation_loss(x, ids, teacher)):
        assert f.loss.isnan() and f.kl[:2, 1].isnan().all()


def test_a_small_divergence_from_the_reference(cuda_device):
    """The KL estimate e^d - d - 1 near d = 0, on rows of one column: log p is 0 exactly and d is the reference's value.
    From 64 bits: 2^-52 |d| of cancellation against d^2 / 2, and the output's own half step: 2^-24 + 2^-51 / |d|."""
    from randomrepo_b200 import losses

    d = torch.tensor([1e-1, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 3.0, 0.0], dtype=torch.float64)
    d = torch.cat([d, -d]).float().to(cuda_device).unsqueeze(0)
    x = torch.zeros(1, 16, 1, device=cuda_device)
    tokens = torch.zeros(1, 16, dtype=torch.int64, device=cuda_device)
    exact = d.double()
    # e^d - d - 1 by its series where |d| is small (the terms fall by more than |d| / 3 each).
    small = sum(exact**i / math.factorial(i) for i in range(2, 8))
    want = torch.where(exact.abs() < 0.05, small, torch.expm1(exact) - exact)
    kw = dict(ref_logprobs=d, kl_coef=0.5, reduction="sum")
    adv = torch.zeros(1, device=cuda_device)
    for got in (losses.policy_loss_and_grad(x, tokens, adv, **kw)[0], losses.policy_loss(x, tokens, adv, **kw)):
        assert (got.kl >= 0).all()
        tol = want * (2.0**-24 + 2.0**-51 / exact.abs().clamp(min=1e-30))
        assert ((got.kl.double() - want).abs() <= tol).all(), (got.kl.double() / want - 1)


def test_forward_mode_is_refused(cuda_device):
    """A dual tensor's tangent is not dropped without a word."""
    import torch.autograd.forward_ad as fwad

    from randomrepo_b200 import losses

    x = torch.randn(2, 4, 33, device=cuda_device)
    tokens = torch.zeros(2, 4, dtype=torch.int64, device=cuda_device)
    with fwad.dual_level():
        assert losses.preference_loss(x, tokens).loss.isfinite()
        dual = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: losses.policy_loss(dual, tokens, x[:, 0, 0]), lambda: losses.preference_loss(dual, tokens),
                     lambda: losses.policy_loss_and_grad(dual, tokens, x[:, 0, 0]),
                     lambda: losses.distillation_loss(dual, tokens.unsqueeze(-1), x[..., :1]),
                     lambda: losses.preference_loss(dual.requires_grad_(), tokens)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
    assert losses.preference_loss(x, tokens).loss.isfinite()


def test_a_margin_without_bound(cuda_device):
    """A rejected answer of probability 0 (a masked token in it): nothing is left to learn, the loss is 0; a chosen one:
    the loss is infinite and the slope is beta.  With smoothing both are infinite."""
    from randomrepo_b200 import losses

    x = torch.zeros(4, 2, 9, device=cuda_device)
    x[2, 1, 5] = -math.inf  # rejected, of pair 0
    x[1, 0, 5] = -math.inf  # chosen, of pair 1
    tokens = torch.full((4, 2), 5, device=cuda_device)
    pair = torch.tensor([0, 2], device=cuda_device)
    got, grad = losses.preference_loss_and_grad(x[pair], tokens[pair], beta=0.5)
    assert float(got.loss) == 0.0 and float(got.margins[0]) == math.inf and (grad == 0).all()
    leaf = x[pair].requires_grad_()
    out = losses.preference_loss(leaf, tokens[pair], beta=0.5)
    out.loss.backward()
    assert out.loss.item() == 0.0 and (leaf.grad == 0).all()
    got, grad = losses.preference_loss_and_grad(x[[1, 3]], tokens[[1, 3]], beta=0.5)
    assert float(got.loss) == math.inf and float(got.margins[0]) == -math.inf
    p = torch.softmax(x[[1, 3]].double(), -1)
    p[..., 5] -= 1
    p[1] *= -1
    torch.testing.assert_close(grad.double(), 0.5 * p, atol=1e-7, rtol=1e-6)
    got, _ = losses.preference_loss_and_grad(x[pair], tokens[pair], beta=0.5, label_smoothing=0.1)
    assert float(got.loss) == math.inf


@pytest.mark.parametrize("dtype,v", [(F32, 130001), (BF16, 260009), (F16, 300007)])
def test_rows_of_a_pair_of_ctas(cuda_device, dtype, v):
    """Rows long enough for a pair of CTAs each, more of them than there are pairs, at every offset in their 16 bytes.

    A thread adds at most 600 columns and 2^5 x 2^4 x 2 sums are merged: 2.5e-5 of the sum at the most (rounding and the
    approximate 2^y); a gradient entry's coefficient is 1 or 2 here."""
    from randomrepo_b200 import losses

    n = 200
    g = torch.Generator(device=cuda_device).manual_seed(v)
    x = (torch.randn(1, n, v, generator=g, device=cuda_device) * 2).to(dtype)
    tokens = torch.randint(0, v, (1, n), generator=g, device=cuda_device)
    adv = torch.where(torch.rand(1, n, generator=g, device=cuda_device) < 0.5, 1.0, -1.0)
    ids = torch.randint(0, v, (1, n, 9), generator=g, device=cuda_device)
    teacher = torch.randn(1, n, 9, generator=g, device=cuda_device)
    mask = torch.rand(1, n, generator=g, device=cuda_device) < 0.9
    got, grad = losses.policy_loss_and_grad(x, tokens, adv, None, mask, reduction="sum")
    _, ent = losses.policy_loss_and_grad(x, tokens, adv, None, mask, entropy_coef=0.1, reduction="sum")
    dis, dgrad = losses.distillation_loss_and_grad(x, ids, teacher, mask, reduction="sum")
    for at in torch.arange(n, device=cuda_device).split(50):
        rows = torch.log_softmax(x[0, at].double(), -1)
        seen = mask[0, at].unsqueeze(-1)
        pick = rows.gather(-1, tokens[0, at].unsqueeze(-1))
        assert ((got.logprobs[0, at].double().unsqueeze(-1) - pick) * seen).abs().max() <= 2.5e-5
        p = rows.exp()
        hot = torch.zeros_like(p).scatter_(-1, tokens[0, at].unsqueeze(-1), 1.0)
        entropy = -(p * rows).sum(-1, keepdim=True)
        want = (p - hot) * adv[0, at].double().unsqueeze(-1)
        q = torch.softmax(teacher[0, at].double(), -1)
        each = ((grad, want), (ent, want + 0.1 * p * (rows + entropy)), (dgrad, p.scatter_add(-1, ids[0, at], -q)))
        for have, wanted in each:
            wanted = wanted * seen
            tol = wanted.abs() * (_half(dtype) + 2.5e-5) + 5e-5 * p + 2.0**-22 + (2.0**-25 if dtype == F16 else 0)
            assert ((have[0, at].double() - wanted).abs() <= tol).all()
        per = (q * (q.log() - rows.gather(-1, ids[0, at]))).sum(-1, keepdim=True)
        assert ((dis.kl[0, at].double().unsqueeze(-1) - per) * seen).abs().max() <= 5e-5


def test_the_mean_of_log_probabilities(cuda_device):
    """Their errors do not add up over a sequence: the mean error of 4 096 rows' is that of their float32 outputs.

    The outputs lie in (-4, -1): a rounding is uniform in +-2^-23 at the most, rms 2^-22 / sqrt(12) = 6.9e-8, of the
    mean of 4 096 1.1e-9; five times that is 5.5e-9.  The kernels' own mean error is held to 1e-8, and a log2f's
    rounding (a step of 6e-8, its mean a sixth of that at the most) adds 1e-8: 2.6e-8.  Without the low half of the
    scale, the correction of the approximate 2^y or the exact merges the mean is off by 4e-8 to 1e-7."""
    from randomrepo_b200 import losses

    n, v = 4096, 20011
    for dtype in (F32, BF16):
        for temperature in (1.0, 0.7):
            t = _float(temperature)
            g = torch.Generator(device=cuda_device).manual_seed(9)
            x = torch.randn(1, n, v, generator=g, device=cuda_device)
            spot = 0.5 * torch.rand(n, generator=g, device=cuda_device) - 2.0
            x[0, :, 0] = t * ((x[0, :, 1:].double() / t).logsumexp(-1).float() + spot)
            x = x.to(dtype)
            tokens = torch.zeros(1, n, dtype=torch.int64, device=cuda_device)
            want = torch.cat([torch.log_softmax(c.double() / t, -1)[..., 0] for c in x[0].split(512)])
            assert (want < -1).all() and (want > -4).all()
            adv = torch.zeros(1, device=cuda_device)
            for got in (losses.policy_loss_and_grad(x, tokens, adv, temperature=temperature)[0],
                        losses.policy_loss(x, tokens, adv, temperature=temperature)):
                off = (got.logprobs[0].double() - want).mean()
                assert abs(float(off)) <= 2.6e-8, (dtype, temperature, float(off))


@pytest.mark.parametrize("value", [torch.finfo(F32).min, torch.finfo(F32).max, -1e30, 1e20, -1e9, 0.0])
def test_a_teachers_list_of_one_value(cuda_device, value):
    """Entries that are all a mask's value are a uniform list, beside rows where one entry stands above them.

    kl = log p of the student against log q = -log k: 2.5e-5 for log p, 2^-22 for q; a gradient entry p - q likewise."""
    from randomrepo_b200 import losses

    v, k = 700, 12
    g = torch.Generator().manual_seed(8)
    x = torch.randn(1, 3, v, generator=g).to(cuda_device)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(3)]).unsqueeze(0).to(cuda_device)
    teacher = torch.full((1, 3, k), value, device=cuda_device)
    if value < 0:
        teacher[0, 1, 4] = torch.finfo(F32).max
    else:
        teacher[0, 1] = 0.0
    teacher[0, 2, 3:] = -math.inf
    for temperature in (1.0, 0.5):
        q = torch.softmax(teacher.double() / temperature, -1)
        rows = torch.log_softmax(x.double() / temperature, -1)
        per = temperature**2 * (torch.special.xlogy(q, q) - q * rows.gather(-1, ids)).sum(-1)
        want = temperature * rows.exp().scatter_add(-1, ids, -q)
        leaf = x.clone().requires_grad_()
        out = losses.distillation_loss(leaf, ids, teacher, temperature=temperature, reduction="sum")
        got, grad = losses.distillation_loss_and_grad(x, ids, teacher, temperature=temperature, reduction="sum")
        (own,) = torch.autograd.grad(out.loss, leaf)
        for res, d in ((got, grad), (out, own)):
            assert ((res.kl.double() - per).abs() <= 2.6e-5 + 2.0**-20 * per.abs()).all(), (res.kl, per)
            assert ((d.double() - want).abs() <= 2.6e-5 * (want.abs() + rows.exp()) + 2.0**-22).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_whole_rows_with_shifted_tokens(cuda_device, dtype):
    """Next-token rows without a slice: the tokens and per-row inputs shifted by one, the last position not scored.  The
    loss and the gradient down to the whole logits are those of ``logits[:, :-1]`` (each sum is off by 2.5e-5 at most)."""
    from torch.nn.functional import pad

    from randomrepo_b200 import losses

    b, t, v = 3, 9, 1003
    g = torch.Generator().manual_seed(4)
    data = (torch.randn(b, t, v, generator=g) * 2).to(dtype).to(cuda_device)
    input_ids = torch.randint(0, v, (b, t), generator=g).to(cuda_device)
    completion = (torch.rand(b, t, generator=g) < 0.7).to(cuda_device)
    adv = torch.randn(b, generator=g).to(cuda_device)
    old, ref = (-8 + 0.1 * torch.randn(b, t - 1, generator=g).to(cuda_device) for _ in range(2))
    kw = dict(kl_coef=0.05, entropy_coef=0.01)
    leaf = data.clone().requires_grad_()
    cut = losses.policy_loss(leaf[:, :-1], input_ids[:, 1:], adv, old, completion[:, 1:], ref_logprobs=ref, **kw)
    (want,) = torch.autograd.grad(cut.loss, leaf)
    mask = completion.roll(-1, 1)
    mask[:, -1] = False
    leaf = data.clone().requires_grad_()
    out = losses.policy_loss(leaf, input_ids.roll(-1, 1), adv, pad(old, (0, 1)), mask, ref_logprobs=pad(ref, (0, 1)), **kw)
    (got,) = torch.autograd.grad(out.loss, leaf)
    torch.testing.assert_close(out.logprobs[:, :-1], cut.logprobs, atol=5e-5, rtol=0)
    assert (out.logprobs[:, -1] == 0).all() and (got[:, -1] == 0).all()
    torch.testing.assert_close(out.loss, cut.loss, atol=1e-4, rtol=1e-4)
    torch.testing.assert_close(got.float(), want.float(), atol=1e-6, rtol=1e-4 + torch.finfo(dtype).eps)


def test_operators_hand_the_gradient_out(cuda_device):
    """``torch.ops.pkv`` losses return their gradient; to differentiate through them is an error, not a zero."""
    import randomrepo_b200.ops  # noqa: F401 - registers the operators

    leaf = torch.randn(2, 3, 65, device=cuda_device).requires_grad_()
    tokens = torch.zeros(2, 3, dtype=torch.int64, device=cuda_device)
    adv = torch.ones(2, device=cuda_device)
    rows = leaf * 2
    for out in (torch.ops.pkv.policy_loss(rows, tokens, adv, None, None, None, 0.2, 0.2, 0.0, 0.0, 1.0, "sum", 1.0),
                torch.ops.pkv.preference_loss(rows, tokens, None, None, 0.1, 0.0, False, 1.0),
                torch.ops.pkv.distillation_loss(rows, tokens.unsqueeze(-1), adv.view(2, 1, 1).expand(2, 3, 1), None, None,
                                                1.0, "sum", 1.0)):
        with pytest.raises(RuntimeError, match="autograd"):
            out[0].backward(retain_graph=True)
        leaf.grad = None
        rows.backward(out[-1].detach(), retain_graph=True)
        assert torch.equal(leaf.grad, 2 * out[-1].detach())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sums_of_rows_with_a_large_column(cuda_device, dtype):
    """Sums that are added up over a sequence: answers of one token that is much of its row.  A margin against the exact
    sums as the reference is two rows' errors (the float32 reference is taken off in 64 bits, the margin is rounded to
    2^-24 of itself).

    A column's exponent of 16 to 32 units is rounded twice, to 2^-20 at most: rms 5.4e-7 of its 2^y; a hundred columns
    and more share what the token leaves of the row: 5.4e-8.  A mean error of 2.6e-8: 6e-8 a row.  A sum of the token's
    2^y and the small ones beside it in 32 bits, or an approximate 2^y of the token, is off by 1e-7."""
    from randomrepo_b200 import losses

    n, v = 4096, 20011
    g = torch.Generator(device=cuda_device).manual_seed(3)
    tokens = torch.randint(0, v, (n, 1), generator=g, device=cuda_device)
    x = 2 * torch.randn(n, 1, v, generator=g, device=cuda_device)
    x.scatter_add_(-1, tokens.unsqueeze(-1), 6 + 7 * torch.rand(n, 1, 1, generator=g, device=cuda_device))
    x = x.to(dtype)
    exact = torch.cat([torch.log_softmax(c[:, 0].double(), -1).gather(-1, t) for c, t in zip(x.split(512), tokens.split(512))])
    ref = exact[:, 0].float()
    got = losses.preference_loss(x, tokens, None, ref, beta=1.0)
    left = exact[:, 0] - ref.double()
    off = got.margins.double() - (left[: n // 2] - left[n // 2:])
    assert off.pow(2).mean().sqrt() <= 6e-8 * math.sqrt(2), off.std()
