"""Losses over vocabulary rows, with their gradients, and a row's top logits (``libpkv_b200``).

What follows a rollout is training on it.  AgentRL's trainer does that with torch operations over a
[B, L, vocab] log_softmax (agentrl/core/trainer.py:72-167); here a row of logits is read once for its
statistics and, where a gradient is asked for, once more out of shared memory or L2 to write it:

* ``policy_loss`` -- the clipped policy loss of PPO / GRPO, with a KL term to a reference policy and an
  entropy bonus;
* ``preference_loss`` -- the paired log-ratio loss of chosen against rejected answers;
* ``distillation_loss`` -- a student's divergence from a teacher's top logits, as it keeps a speculative
  draft model close to the policy it drafts for; ``top_logits`` picks those logits from the teacher's rows.

Each loss comes in two forms.  ``*_loss(logits, ...)`` is differentiable in ``logits``: its backward pass
reads the logits a second time (once, in reverse mode; it frees them and the workspace, and reads what saved-tensor
hooks hand back).  ``*_loss_and_grad(logits, ...)`` returns the loss and its gradient from one
call, reading the logits from HBM once (policy and distillation): ``logits.backward(dlogits)`` continues
from there.  ``scale`` multiplies the loss and the gradient before its rounding to the logits' type (a
gradient accumulation factor, or a loss scale for float16).

``logits`` are ``[B, T, V]`` or ``[T, V]`` CUDA tensors of float32, float16 or bfloat16 with contiguous
columns (any batch and row strides); per-row inputs are ``[B, T]`` (``[T]``).  For next tokens give the whole rows,
tokens and per-row inputs shifted by one and the last position masked: ``logits[:, :-1]`` is read in place too, but the
slice's own gradient, PyTorch's, then zeroes and copies as much again (4 096 rows of 151 936 bfloat16 columns: 457 us,
with a slice 2 140).  A row whose mask is 0 is not scored: its logits are not read, its outputs and its gradient are
0; tokens there may be anything.  No scored row at all gives a loss of 0.  Losses and per-row outputs are
float32; sums over rows are taken in 64 bits, in a fixed order.  Calls launch on the current stream of the
logits' device, never synchronise, and can be captured in a CUDA graph (a captured training step best uses the
``*_and_grad`` forms: PyTorch cannot capture a backward pass into leaves that another, eager graph still holds).
There is no CPU path.
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import lib

__all__ = ["PolicyLoss", "PreferenceLoss", "DistillationLoss", "policy_loss", "policy_loss_and_grad",
           "preference_loss", "preference_loss_and_grad", "distillation_loss", "distillation_loss_and_grad",
           "top_logits"]

_DTYPES = {torch.float32: _lib.PKV_F32, torch.float16: _lib.PKV_F16, torch.bfloat16: _lib.PKV_BF16}
_REDUCTIONS = {"token_mean": 0, "sequence_mean": 1, "sum": 2}
_MAX_TOP = 256

# The structs of the C ABI (pkv_loss_rows and the terms of each loss), packed with native alignment.
_ROWS = struct.Struct("@PqqPqqPqqiiiif")
_POLICY = struct.Struct("@PqqPqqPqqPqqffffif")
_PREFERENCE = struct.Struct("@PqqPffif")
_DISTILLATION = struct.Struct("@PqqPqqiPqqif")
_NONE = (0, 0, 0)


class PolicyLoss(NamedTuple):
    """loss (scalar), and per row: the token's log-probability, the KL estimate against the reference
    (None without one) and the entropy (None unless ``entropy_coef`` is set)."""

    loss: torch.Tensor
    logprobs: torch.Tensor
    kl: torch.Tensor | None
    entropy: torch.Tensor | None


class PreferenceLoss(NamedTuple):
    """loss (scalar), the sequences' summed (or mean) log-probabilities [B], the pairs' margins [B / 2]."""

    loss: torch.Tensor
    logprobs: torch.Tensor
    margins: torch.Tensor


class DistillationLoss(NamedTuple):
    """loss (scalar) and each row's T^2-scaled divergence."""

    loss: torch.Tensor
    kl: torch.Tensor


def _logits(logits: torch.Tensor, what: str) -> torch.Tensor:
    """``logits`` as [B, T, V], checked."""
    if forward_ad._current_level >= 0 and isinstance(logits, torch.Tensor) and (
            forward_ad.unpack_dual(logits).tangent is not None):
        raise RuntimeError(f"{what}: the vocabulary rows have no forward-mode derivative")
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError(f"{what}: logits must be a CUDA tensor (the vocabulary kernels have no CPU path)")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"{what}: logits must be float32, float16 or bfloat16")
    if logits.dim() not in (2, 3) or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [batch, length, vocab] or [length, vocab]")
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        raise ValueError(f"{what}: logits must have a contiguous vocabulary dim")
    if logits.requires_grad:
        logits = logits.detach()
    return logits.unsqueeze(0) if logits.dim() == 2 else logits


def _rows_like(t: torch.Tensor, rows: torch.Size, dev: torch.device, dtype: torch.dtype, what: str,
               name: str) -> torch.Tensor:
    """A per-row input as [B, T] (``rows``) of ``dtype`` on ``dev`` ([T] for one sequence)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: {name} must be a tensor")
    if t.device != dev:
        raise ValueError(f"{what}: {name} must be on the logits' device")
    if t.shape != rows:
        if t.dim() == 1 and rows[0] == 1 and t.shape[0] == rows[1]:
            t = t.unsqueeze(0)
        else:
            raise ValueError(f"{what}: {name} must have one value per logits row, got {tuple(t.shape)}")
    if t.dtype != dtype:
        if dtype == torch.int64 and (t.is_floating_point() or t.dtype == torch.bool):
            raise ValueError(f"{what}: {name} must be integers")
        t = t.to(dtype)
    return t


def _advantages(t: torch.Tensor, rows: torch.Size, dev: torch.device, what: str) -> torch.Tensor:
    """Advantages [B, T], [B, 1] or [B] (one a sequence) as float32."""
    if isinstance(t, torch.Tensor) and t.shape != rows and t.device == dev and not (rows[0] == 1 and t.dim() == 1
                                                                                and t.shape[0] == rows[1]):
        if tuple(t.shape) not in ((rows[0],), (rows[0], 1)):
            raise ValueError(f"{what}: advantages must be [batch, length] or [batch], got {tuple(t.shape)}")
        return t if t.dtype == torch.float32 else t.to(torch.float32)
    return _rows_like(t, rows, dev, torch.float32, what, "advantages")


def _mask(mask: torch.Tensor | None, rows: torch.Size, dev: torch.device, what: str) -> torch.Tensor | None:
    """The mask as bytes [B, T] (anything but 0 is scored)."""
    if mask is None:
        return None
    if isinstance(mask, torch.Tensor) and mask.dtype not in (torch.bool, torch.uint8):
        mask = mask != 0
    # (a byte each, read as such)
    return _rows_like(mask, rows, dev, mask.dtype if isinstance(mask, torch.Tensor) else torch.bool, what, "mask")


def _array(t: torch.Tensor | None) -> tuple[int, int, int]:
    if t is None:
        return _NONE
    sb, st = t.stride()[:2]
    return t.data_ptr(), sb, st


def _reduction(name: str, what: str) -> int:
    if name not in _REDUCTIONS:
        raise ValueError(f"{what}: reduction must be one of {sorted(_REDUCTIONS)}, got {name!r}")
    return _REDUCTIONS[name]


def _grad_like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised gradient for logits [B, T, V] whose rows start as many bytes past a 16-byte boundary as
    the logits' do, so that both move in 16-byte vectors: dense where such rows are, else with the logits' strides
    (rows that overlap or lie far apart: dense, wherever they start)."""
    b, n, v = x.shape
    alike, at = x.is_contiguous(), x.data_ptr() % 16
    if alike and at == 0:
        return torch.empty(b, n, v, dtype=x.dtype, device=x.device)  # (faster than a tuple of sizes)
    size, numel = x.element_size(), x.numel()
    at //= size
    if not alike:
        sb, sn = (x.stride(0) if b > 1 else 0), (x.stride(1) if n > 1 else 0)
        alike = v * size % 16 == 0 and sb * size % 16 == 0 and sn * size % 16 == 0
    if alike:
        return torch.empty(numel + at, dtype=x.dtype, device=x.device)[at:].view(b, n, v)
    span = (n - 1) * sn + v
    if (n > 1 and sn < v) or (b > 1 and sb < span) or (b - 1) * sb + span > 2 * numel + 64:
        return torch.empty((b, n, v), dtype=x.dtype, device=x.device)  # overlapping or sparse rows
    flat = torch.empty((b - 1) * sb + span + 16, dtype=x.dtype, device=x.device)
    return flat.as_strided((b, n, v), (max(sb, span), max(sn, v), 1), at)


class _Kind(NamedTuple):
    """A loss: its entry points, inputs(rows, dev, what, *tensors): the terms' tensors, checked, terms(numbers, *tensors): the
    terms, packed."""

    what: str
    forward: object
    backward: object
    inputs: object
    terms: object


class _Call(NamedTuple):
    """One loss call, apart from its tensors: a differentiable call's graph node keeps it, and what that node keeps of
    tensors are saved ones alone (freed by the backward pass, and seen by saved-tensor hooks)."""

    kind: _Kind
    numbers: tuple
    temperature: float


class _Tensors(NamedTuple):
    """A call's tensors: rows [B, T, V], mask, the terms' inputs, outputs, and the workspace a backward pass reads."""

    x: torch.Tensor
    mask: torch.Tensor | None
    inputs: tuple
    outputs: tuple
    ws: torch.Tensor


def _temperature(temperature: float, what: str) -> float:
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{what}: the temperature must lie in [1e-6, 1e6]")
    return temperature


def _workspace(batch: int, length: int, dev: torch.device, what: str) -> torch.Tensor:
    nbytes = lib.pkv_loss_workspace_bytes(batch, length)
    if nbytes < 0:
        raise ValueError(f"{what}: too many rows")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def _on_device(x: torch.Tensor, fn, *args) -> None:
    """``fn(*args, stream)`` with the current stream of ``x``'s device, which is the current device meanwhile."""
    index = x.device.index
    if index == torch._C._cuda_getDevice():
        st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.raise_for_status(st)


def _launch(fn, x: torch.Tensor, temperature: float, grad: torch.Tensor | None, mask: tuple, terms: bytes,
            outputs: tuple, ws: torch.Tensor) -> None:
    """``fn(rows, terms, *outputs, workspace)`` on the logits' device and its current stream."""
    rows = _ROWS.pack(*_array(x), *_array(grad), *mask, *x.shape, _DTYPES[x.dtype], temperature)
    _on_device(x, fn, rows, terms, *[None if o is None else o.data_ptr() for o in outputs], ws.data_ptr(), ws.numel())


def _forward(c: _Call, t: _Tensors, grad: torch.Tensor | None) -> tuple:
    """The forward call; its packed mask and terms."""
    kind = c.kind
    mask, terms = _array(t.mask), kind.terms(c.numbers, *t.inputs)
    _launch(kind.forward, t.x, c.temperature, grad, mask, terms, t.outputs, t.ws)
    return mask, terms


def _unpacked(kind: _Kind, shape: torch.Size, dtype: torch.dtype, dev: torch.device, logits, mask, ws, inputs) -> tuple:
    """(rows, mask, inputs, workspace) of saved tensors that are not the call's own any more (a hook moved them to the
    host and back, or they were computed anew), checked as those were: the kernels would read past smaller ones."""
    if logits.shape != shape or logits.dtype != dtype or logits.device != dev:
        raise ValueError(f"logits {tuple(logits.shape)} of {logits.dtype} on {logits.device}")
    if ws.device != dev or ws.dtype != torch.uint8:
        raise ValueError("another workspace")
    x = logits if len(shape) == 3 else logits.unsqueeze(0)
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    rows = x.shape[:2]
    return x, _mask(mask, rows, dev, kind.what), kind.inputs(rows, dev, kind.what, *inputs), ws.contiguous()


class _RowLoss(torch.autograd.Function):
    """Forward: the loss call without a gradient.  Backward: the rows again, times the upstream gradient."""

    @staticmethod
    def forward(ctx, logits, call, t):
        at = logits.data_ptr(), logits.stride(), t.ws.data_ptr(), _forward(call, t, None)
        ctx.call = call, at, logits.shape, logits.dtype, t.x.device
        ctx.save_for_backward(logits, t.mask, t.ws, *t.inputs)
        return t.outputs[0]

    @staticmethod
    def backward(ctx, grad_loss):
        if torch.is_grad_enabled():  # (create_graph=True)
            raise RuntimeError("the vocabulary-row losses are differentiable once")
        (kind, numbers, temperature), at, shape, dtype, dev = ctx.call
        logits, mask, ws, *inputs = ctx.saved_tensors  # (also checks that nothing was changed in place since)
        try:
            packed = _array(mask), kind.terms(numbers, *inputs)
        except (ValueError, IndexError):  # (not even of as many dims)
            packed = None
        own = (logits.data_ptr(), logits.stride(), ws.data_ptr(), packed) == at
        if own and logits.shape == shape and logits.dtype == dtype:
            x = logits if len(shape) == 3 else logits.unsqueeze(0)
        else:
            try:
                x, mask, inputs, ws = _unpacked(kind, shape, dtype, dev, logits, mask, ws, inputs)
            except ValueError as e:
                raise RuntimeError(f"{kind.what}: a saved-tensor hook gave back something else: {e}") from e
            packed = _array(mask), kind.terms(numbers, *inputs)
        grad = _grad_like(x)
        if grad_loss.dtype != torch.float32 or grad_loss.device != dev:
            grad_loss = grad_loss.to(dtype=torch.float32, device=dev)
        _launch(kind.backward, x, temperature, grad, *packed, (grad_loss,), ws)
        return grad if len(shape) == 3 else grad.squeeze(0), None, None


def _run(c: _Call, logits: torch.Tensor, t: _Tensors) -> tuple:
    """The outputs of a differentiable call: the loss, and per-row values without a gradient."""
    if logits.requires_grad and torch.is_grad_enabled():
        return (_RowLoss.apply(logits, c, t), *t.outputs[1:])
    _forward(c, t, None)
    return t.outputs


def _run_with_grad(c: _Call, logits: torch.Tensor, t: _Tensors) -> torch.Tensor:
    grad = _grad_like(t.x)
    _forward(c, t, grad)
    return grad if grad.dim() == logits.dim() else grad.squeeze(0)


def _policy_inputs(rows, dev, what, tokens, advantages, old_logprobs, ref_logprobs) -> tuple:
    tok = _rows_like(tokens, rows, dev, torch.int64, what, "tokens")
    adv = _advantages(advantages, rows, dev, what)
    old = None if old_logprobs is None else _rows_like(old_logprobs, rows, dev, torch.float32, what, "old_logprobs")
    ref = None if ref_logprobs is None else _rows_like(ref_logprobs, rows, dev, torch.float32, what, "ref_logprobs")
    return tok, adv, old, ref


def _policy_terms(numbers, tok, adv, old, ref) -> bytes:
    each = adv.data_ptr(), adv.stride(0), adv.stride(1) if adv.shape == tok.shape else 0
    return _POLICY.pack(*_array(tok), *each, *_array(old), *_array(ref), *numbers)


_POLICY_KIND = _Kind("policy_loss", lib.pkv_policy_loss, lib.pkv_policy_loss_backward, _policy_inputs,
                    _policy_terms)


def _policy(logits, tokens, advantages, old_logprobs, mask, ref_logprobs, clip_low, clip_high, kl_coef, entropy_coef,
            temperature, reduction, scale):
    what = _POLICY_KIND.what
    x = _logits(logits, what)
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"{what}: clip_low and clip_high must be >= 0")
    rows, dev = x.shape[:2], x.device
    inputs = _policy_inputs(rows, dev, what, tokens, advantages, old_logprobs, ref_logprobs)
    m = _mask(mask, rows, dev, what)
    numbers = (float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef), _reduction(reduction, what),
               float(scale))
    c = _Call(_POLICY_KIND, numbers, _temperature(temperature, what))
    ws = _workspace(*rows, dev, what)
    lp = torch.empty(*logits.shape[:-1], dtype=torch.float32, device=dev)
    outputs = (lp.new_empty(()), lp, None if ref_logprobs is None else torch.empty_like(lp),
               torch.empty_like(lp) if entropy_coef else None)
    return c, _Tensors(x, m, inputs, outputs, ws)


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, advantages: torch.Tensor,
                old_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, *,
                ref_logprobs: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                reduction: str = "token_mean", scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss, differentiable in ``logits``.

    With z = logits / temperature, lp = log_softmax(z)[token] and r = exp(lp - old_logprobs) a scored row's loss is

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(ref - lp) - (ref - lp) - 1) - entropy_coef H

    ``advantages`` are [B, T], or [B] (one a sequence).  ``old_logprobs=None`` is the step right after the rollout:
    r is 1, with the gradient of lp.  ``reduction``: "token_mean" over all scored rows, "sequence_mean" the mean over
    sequences with a scored row of their rows' mean, or "sum".  All inputs but ``logits`` are constants.
    """
    c, t = _policy(logits, tokens, advantages, old_logprobs, mask, ref_logprobs, clip_low, clip_high, kl_coef,
                   entropy_coef, temperature, reduction, scale)
    return PolicyLoss(*_run(c, logits, t))


def policy_loss_and_grad(logits: torch.Tensor, tokens: torch.Tensor, advantages: torch.Tensor,
                         old_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, *,
                         ref_logprobs: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                         kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                         reduction: str = "token_mean", scale: float = 1.0) -> tuple[PolicyLoss, torch.Tensor]:
    """``policy_loss`` and its gradient with respect to ``logits`` (their type), in one pass over HBM."""
    c, t = _policy(logits, tokens, advantages, old_logprobs, mask, ref_logprobs, clip_low, clip_high, kl_coef,
                   entropy_coef, temperature, reduction, scale)
    grad = _run_with_grad(c, logits, t)
    return PolicyLoss(*t.outputs), grad


def _preference_inputs(rows, dev, what, tokens, ref) -> tuple:
    tok = _rows_like(tokens, rows, dev, torch.int64, what, "tokens")
    if ref is not None:
        if not isinstance(ref, torch.Tensor) or ref.device != dev or tuple(ref.shape) != (rows[0],):
            raise ValueError(f"{what}: ref_logprobs must be [2 * pairs] on the logits' device")
        ref = ref.to(torch.float32).contiguous()
    return tok, ref


def _preference_terms(numbers, tok, ref) -> bytes:
    return _PREFERENCE.pack(*_array(tok), 0 if ref is None else ref.data_ptr(), *numbers)


_PREFERENCE_KIND = _Kind("preference_loss", lib.pkv_preference_loss, lib.pkv_preference_loss_backward,
                         _preference_inputs, _preference_terms)


def _preference(logits, tokens, mask, ref_logprobs, beta, label_smoothing, length_normalised, scale):
    what = _PREFERENCE_KIND.what
    x = _logits(logits, what)
    if logits.dim() != 3 or x.shape[0] % 2:
        raise ValueError(f"{what}: logits must be [2 * pairs, length, vocab], the chosen answers first")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"{what}: label_smoothing must lie in [0, 1]")
    rows, dev = x.shape[:2], x.device
    inputs = _preference_inputs(rows, dev, what, tokens, ref_logprobs)
    m = _mask(mask, rows, dev, what)
    numbers = (float(beta), float(label_smoothing), int(bool(length_normalised)), float(scale))
    c = _Call(_PREFERENCE_KIND, numbers, 1.0)
    ws = _workspace(*rows, dev, what)
    sums = torch.empty(rows[0], dtype=torch.float32, device=dev)
    outputs = sums.new_empty(()), sums, torch.empty(rows[0] // 2, dtype=torch.float32, device=dev)
    return c, _Tensors(x, m, inputs, outputs, ws)


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None = None,
                    ref_logprobs: torch.Tensor | None = None, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    length_normalised: bool = False, scale: float = 1.0) -> PreferenceLoss:
    """Preference loss over pairs of answers, differentiable in ``logits`` [2P, T, V].

    Sequences 0 .. P-1 are the chosen answers, P .. 2P-1 the rejected ones.  S is the sum of a sequence's scored
    token log-probabilities (their mean with ``length_normalised``), R the reference policy's
    (``ref_logprobs`` [2P], None for 0), and a pair's loss

        m = beta ((S_c - R_c) - (S_r - R_r)),  -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m)

    averaged over the pairs (a term of weight 0 is 0 for infinite m too).  A sequence without a scored row has S = 0.
    """
    c, t = _preference(logits, tokens, mask, ref_logprobs, beta, label_smoothing, length_normalised, scale)
    return PreferenceLoss(*_run(c, logits, t))


def preference_loss_and_grad(logits: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None = None,
                             ref_logprobs: torch.Tensor | None = None, *, beta: float = 0.1,
                             label_smoothing: float = 0.0, length_normalised: bool = False,
                             scale: float = 1.0) -> tuple[PreferenceLoss, torch.Tensor]:
    """``preference_loss`` and its gradient with respect to ``logits`` (their type)."""
    c, t = _preference(logits, tokens, mask, ref_logprobs, beta, label_smoothing, length_normalised, scale)
    grad = _run_with_grad(c, logits, t)
    return PreferenceLoss(*t.outputs), grad


def _teacher_list(t: torch.Tensor, rows: torch.Size, dev: torch.device, dtype: torch.dtype, what: str,
                  name: str) -> torch.Tensor:
    """A teacher's list as [B, T, k] (``rows`` and k; [T, k] for one sequence) of ``dtype`` with contiguous entries."""
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{what}: {name} must be on the logits' device")
    if t.dim() == 2 and rows[0] == 1:
        t = t.unsqueeze(0)
    shape = t.shape
    if len(shape) != 3 or shape[:-1] != rows or not 1 <= shape[-1] <= _MAX_TOP:
        raise ValueError(f"{what}: {name} must be {list(rows)} + [k], k from 1 to {_MAX_TOP}, got {tuple(shape)}")
    if t.dtype != dtype:
        if dtype == torch.int64 and (t.is_floating_point() or t.dtype == torch.bool):
            raise ValueError(f"{what}: {name} must be integers")
        t = t.to(dtype)
    if t.stride(-1) != 1 and shape[-1] > 1:
        t = t.contiguous()
    return t


def _distillation_inputs(rows, dev, what, teacher_ids, teacher_logits, teacher_lse) -> tuple:
    ids = _teacher_list(teacher_ids, rows, dev, torch.int64, what, "teacher_ids")
    tl = _teacher_list(teacher_logits, rows, dev, torch.float32, what, "teacher_logits")
    if ids.shape != tl.shape:
        raise ValueError(f"{what}: teacher_ids and teacher_logits must have the same shape")
    lse = None if teacher_lse is None else _rows_like(teacher_lse, rows, dev, torch.float32, what, "teacher_lse")
    return ids, tl, lse


def _distillation_terms(numbers, ids, tl, lse) -> bytes:
    return _DISTILLATION.pack(*_array(ids), *_array(tl), ids.shape[-1], *_array(lse), *numbers)


_DISTILLATION_KIND = _Kind("distillation_loss", lib.pkv_distillation_loss, lib.pkv_distillation_loss_backward,
                           _distillation_inputs, _distillation_terms)


def _distillation(logits, teacher_ids, teacher_logits, mask, teacher_lse, temperature, reduction, scale):
    what = _DISTILLATION_KIND.what
    x = _logits(logits, what)
    rows, dev = x.shape[:2], x.device
    inputs = _distillation_inputs(rows, dev, what, teacher_ids, teacher_logits, teacher_lse)
    m = _mask(mask, rows, dev, what)
    c = _Call(_DISTILLATION_KIND, (_reduction(reduction, what), float(scale)), _temperature(temperature, what))
    ws = _workspace(*rows, dev, what)
    kl = torch.empty(*logits.shape[:-1], dtype=torch.float32, device=dev)
    return c, _Tensors(x, m, inputs, (kl.new_empty(()), kl), ws)


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      mask: torch.Tensor | None = None, *, teacher_lse: torch.Tensor | None = None,
                      temperature: float = 1.0, reduction: str = "token_mean", scale: float = 1.0) -> DistillationLoss:
    """Divergence of the student's rows from a teacher's top logits, differentiable in ``logits``.

    ``teacher_ids`` / ``teacher_logits`` [B, T, k] (k <= 256) list a row's likely tokens at the teacher and their
    logits (``top_logits`` makes them); an id below 0 or a logit of -inf is an absent entry, an id may come twice.
    q is the softmax of the list's logits / temperature, or, with ``teacher_lse`` (the log-sum-exp of the teacher's
    whole row / temperature), the teacher's own probabilities, which then sum to less than 1.  A scored row's loss is

        T^2 sum_k q_k (log q_k - log_softmax(logits / T)[id_k])

    and 0 for a row whose entries are all absent, or underflow (it counts in the means).  An id past the vocabulary makes the
    loss and its row's gradient NaN.  ``reduction`` as in ``policy_loss``.
    """
    c, t = _distillation(logits, teacher_ids, teacher_logits, mask, teacher_lse, temperature, reduction, scale)
    return DistillationLoss(*_run(c, logits, t))


def distillation_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                               mask: torch.Tensor | None = None, *, teacher_lse: torch.Tensor | None = None,
                               temperature: float = 1.0, reduction: str = "token_mean",
                               scale: float = 1.0) -> tuple[DistillationLoss, torch.Tensor]:
    """``distillation_loss`` and its gradient with respect to ``logits`` (their type), in one pass over HBM."""
    c, t = _distillation(logits, teacher_ids, teacher_logits, mask, teacher_lse, temperature, reduction, scale)
    grad = _run_with_grad(c, logits, t)
    return DistillationLoss(*t.outputs), grad


def top_logits(logits: torch.Tensor, k: int, *,
               temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The k largest logits of each row (k <= 256): (values float32 [..., k], tokens int64 [..., k], the log-sum-exp
    of logits / temperature [...]), largest first, equal ones by their column.  NaN counts as the
    largest value; a row with NaN or +inf has a NaN log-sum-exp."""
    what = "top_logits"
    x = _logits(logits, what)
    k = int(k)
    if not 1 <= k <= min(_MAX_TOP, x.shape[-1]):
        raise ValueError(f"{what}: k must be from 1 to {min(_MAX_TOP, x.shape[-1])}")
    temperature = _temperature(temperature, what)
    shape = logits.shape[:-1]
    values = torch.empty(*shape, k, dtype=torch.float32, device=x.device)
    tokens = torch.empty(*shape, k, dtype=torch.int64, device=x.device)
    lse = torch.empty(*shape, dtype=torch.float32, device=x.device)
    rows = _ROWS.pack(*_array(x), *_NONE, *_NONE, *x.shape, _DTYPES[x.dtype], temperature)
    _on_device(x, lib.pkv_top_logits, rows, k, values.data_ptr(), tokens.data_ptr(), lse.data_ptr())
    return values, tokens, lse
