"""Host side of the vocabulary-row losses on CPU: packed argument layouts, refusals, workspace sizes.

Every call below is rejected (or sized) before anything is launched; the kernels run in tests/test_gpu_losses.py.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from randomrepo_b200 import _lib, losses
from randomrepo_b200._lib import lib


class _Array(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64)]


class _Rows(ctypes.Structure):
    _fields_ = [("logits", _Array), ("grad", _Array), ("mask", _Array), ("batch", ctypes.c_int32),
                ("length", ctypes.c_int32), ("vocab", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("temperature", ctypes.c_float)]


class _Policy(ctypes.Structure):
    _fields_ = [("tokens", _Array), ("advantages", _Array), ("old", _Array), ("ref", _Array),
                ("clip_low", ctypes.c_float), ("clip_high", ctypes.c_float), ("kl", ctypes.c_float),
                ("entropy", ctypes.c_float), ("reduction", ctypes.c_int32), ("scale", ctypes.c_float)]


class _Preference(ctypes.Structure):
    _fields_ = [("tokens", _Array), ("ref", ctypes.c_void_p), ("beta", ctypes.c_float), ("smoothing", ctypes.c_float),
                ("normalised", ctypes.c_int32), ("scale", ctypes.c_float)]


class _Distillation(ctypes.Structure):
    _fields_ = [("ids", _Array), ("logits", _Array), ("k", ctypes.c_int32), ("lse", _Array),
                ("reduction", ctypes.c_int32), ("scale", ctypes.c_float)]


@pytest.mark.parametrize("packed,struct", [("_ROWS", _Rows), ("_POLICY", _Policy), ("_PREFERENCE", _Preference),
                                           ("_DISTILLATION", _Distillation)])
def test_packed_arguments_have_the_structs_layout(packed, struct):
    fmt = getattr(losses, packed)
    # struct.pack leaves out the padding behind the last member, which nothing reads.
    assert ctypes.sizeof(struct) - fmt.size in (0, 4)
    n = len(fmt.unpack(bytes(fmt.size)))
    raw = fmt.pack(*range(1, n + 1)) + bytes(8)
    got = struct.from_buffer_copy(raw)

    def flat(s):
        for name, _ in s._fields_:
            v = getattr(s, name)
            yield from flat(v) if isinstance(v, _Array) else (v,)

    assert list(flat(got)) == list(range(1, n + 1))


def test_workspace_sizes():
    assert lib.pkv_loss_workspace_bytes(-1, 4) == -1 and lib.pkv_loss_workspace_bytes(1 << 20, 1 << 20) == -1
    small, large = lib.pkv_loss_workspace_bytes(1, 1), lib.pkv_loss_workspace_bytes(16, 512)
    assert 0 < small < large and small % 256 == 0 and large >= 16 * 512 * (8 + 16 + 4)


def _rows(**kw):
    base = dict(logits=_Array(0x1000, 5120, 512), grad=_Array(), mask=_Array(), batch=2, length=10, vocab=512,
                dtype=_lib.PKV_F32, temperature=1.0)
    return _Rows(**(base | kw))


BAD_ROWS = [dict(batch=-1), dict(vocab=0), dict(dtype=7), dict(temperature=0.0), dict(temperature=math.inf),
            dict(temperature=math.nan), dict(logits=_Array(0, 5120, 512)), dict(logits=_Array(0x1002, 5120, 512)),
            dict(logits=_Array(0x1000, -5120, 512)), dict(grad=_Array(0x20000, 5120, 511)), dict(grad=_Array(0x1000, 5120, 512)),
            dict(grad=_Array(0x1000 + 2 * 5120 * 4 - 4, 5120, 512)),
            dict(grad=_Array(0x20000, 5119, 512)), dict(grad=_Array(0x20001, 5120, 512))]


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_entry_points_reject_bad_rows(bad):
    ws = 0x10000
    n = lib.pkv_loss_workspace_bytes(2, 10)
    tok = _Array(0x3000, 10, 1)
    rows = ctypes.byref(_rows(**bad))
    pol = ctypes.byref(_Policy(tokens=tok, advantages=tok, scale=1.0))
    pref = ctypes.byref(_Preference(tokens=tok, beta=0.1, scale=1.0))
    dis = ctypes.byref(_Distillation(ids=tok, logits=tok, k=1, scale=1.0))
    out = 0x4000
    assert lib.pkv_policy_loss(rows, pol, out, out, None, None, ws, n, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_preference_loss(rows, pref, out, out, out, ws, n, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_distillation_loss(rows, dis, out, out, ws, n, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_top_logits(rows, 1, out, out, out, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_policy_loss_backward(rows, pol, out, ws, n, None) == _lib.PKV_ERR_ARG
    assert _lib.last_error()


def test_entry_points_reject_bad_terms():
    ws, out, n = 0x10000, 0x4000, lib.pkv_loss_workspace_bytes(2, 10)
    tok = _Array(0x3000, 10, 1)
    rows = ctypes.byref(_rows())

    def policy(w=ws, size=n, logprobs=out, **kw):
        p = _Policy(**(dict(tokens=tok, advantages=tok, scale=1.0) | kw))
        return lib.pkv_policy_loss(rows, ctypes.byref(p), out, logprobs, None, None, w, size, None)

    for kw in (dict(tokens=_Array()), dict(advantages=_Array()), dict(reduction=3), dict(reduction=-1),
               dict(clip_low=-0.1), dict(clip_high=math.nan), dict(w=None), dict(w=ws + 128), dict(size=n - 1),
               dict(logprobs=None)):
        assert policy(**kw) == _lib.PKV_ERR_ARG, kw
    assert lib.pkv_policy_loss(rows, None, out, out, None, None, ws, n, None) == _lib.PKV_ERR_ARG
    pref = _Preference(tokens=tok, beta=0.1, scale=1.0)
    odd = _rows(batch=3)
    assert lib.pkv_preference_loss(ctypes.byref(odd), ctypes.byref(pref), out, out, out, ws, 1 << 20, None) == _lib.PKV_ERR_ARG
    pref.smoothing = 1.5
    assert lib.pkv_preference_loss(rows, ctypes.byref(pref), out, out, out, ws, n, None) == _lib.PKV_ERR_ARG
    for k, status in ((0, _lib.PKV_ERR_UNSUPPORTED), (257, _lib.PKV_ERR_UNSUPPORTED)):
        dis = _Distillation(ids=tok, logits=tok, k=k, scale=1.0)
        assert lib.pkv_distillation_loss(rows, ctypes.byref(dis), out, out, ws, n, None) == status
        assert lib.pkv_top_logits(rows, k, out, out, out, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_top_logits(ctypes.byref(_rows(vocab=5)), 6, out, out, out, None) == _lib.PKV_ERR_ARG
    assert lib.pkv_policy_loss_backward(rows, ctypes.byref(_Policy(tokens=tok)), out, ws, n, None) == _lib.PKV_ERR_ARG


def test_python_entry_points_have_no_cpu_path():
    x, tok = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: losses.policy_loss(x, tok, torch.zeros(2)), lambda: losses.policy_loss_and_grad(x, tok, torch.zeros(2)),
                 lambda: losses.preference_loss(x, tok), lambda: losses.preference_loss_and_grad(x, tok),
                 lambda: losses.distillation_loss(x, tok.unsqueeze(-1), x[..., :1]),
                 lambda: losses.distillation_loss_and_grad(x, tok.unsqueeze(-1), x[..., :1]),
                 lambda: losses.top_logits(x, 2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


class _OnDevice(torch.Tensor):
    """A host tensor that says it is on the device, to reach the checks behind the first one."""

    @property
    def is_cuda(self):
        return True


def _fake(t):
    return t.as_subclass(_OnDevice)


def test_python_entry_points_check_their_arguments():
    x, tok, adv = _fake(torch.zeros(2, 3, 8)), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    bad = [lambda: losses.policy_loss(_fake(torch.zeros(2, 3, 8, dtype=torch.float64)), tok, adv),
           lambda: losses.policy_loss(_fake(torch.zeros(8)), tok, adv),
           lambda: losses.policy_loss(_fake(torch.zeros(2, 8, 3).transpose(1, 2)), tok, adv),
           lambda: losses.policy_loss(x, tok[:, :2], adv), lambda: losses.policy_loss(x, adv, adv),
           lambda: losses.policy_loss(x, tok, torch.zeros(3)), lambda: losses.policy_loss(x, tok, torch.zeros(2, 2)),
           lambda: losses.policy_loss(x, tok, adv, torch.zeros(2)), lambda: losses.policy_loss(x, tok, adv, None, torch.ones(3, 2)),
           lambda: losses.policy_loss(x, tok, adv, clip_low=-1.0), lambda: losses.policy_loss(x, tok, adv, reduction="mean"),
           lambda: losses.policy_loss(x, tok, adv, temperature=0.0), lambda: losses.policy_loss(x, tok, adv, temperature=math.nan),
           lambda: losses.preference_loss(_fake(torch.zeros(3, 3, 8)), tok), lambda: losses.preference_loss(_fake(torch.zeros(3, 8)), tok[0]),
           lambda: losses.preference_loss(x, tok, label_smoothing=1.5), lambda: losses.preference_loss(x, tok, None, torch.zeros(3)),
           lambda: losses.distillation_loss(x, tok, adv), lambda: losses.distillation_loss(x, adv.unsqueeze(-1), adv.unsqueeze(-1)),
           lambda: losses.distillation_loss(x, tok.unsqueeze(-1), torch.zeros(2, 3, 2)),
           lambda: losses.distillation_loss(x, torch.zeros(2, 3, 257, dtype=torch.int64), torch.zeros(2, 3, 257)),
           lambda: losses.distillation_loss(x, torch.zeros(2, 3, 0, dtype=torch.int64), torch.zeros(2, 3, 0)),
           lambda: losses.distillation_loss(x, tok.unsqueeze(-1), adv.unsqueeze(-1), teacher_lse=torch.zeros(2)),
           lambda: losses.top_logits(x, 0), lambda: losses.top_logits(x, 9), lambda: losses.top_logits(x, 1, temperature=-1.0)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_gradients_are_laid_out_like_the_logits_rows():
    dense = torch.zeros(3, 4, 16, dtype=torch.bfloat16)
    assert losses._grad_like(dense[:, :-1]).is_contiguous()        # rows of whole vectors
    odd = torch.zeros(3, 4, 17, dtype=torch.bfloat16)
    assert losses._grad_like(odd).is_contiguous()
    for x in (odd[:, 1:], odd[:, :-1], odd[..., 1:17][:, ::2], odd[1:2], odd[:, 1:2], odd[..., :15]):
        g = losses._grad_like(x)
        assert g.shape == x.shape and g.stride(-1) == 1
        for i in range(x.shape[0]):
            for j in range(x.shape[1]):
                if x.shape[2] % 8:
                    assert (g[i, j].data_ptr() - x[i, j].data_ptr()) % 16 == 0
        g.copy_(torch.arange(g.numel()).view(g.shape).float())  # no two rows overlap
        assert len(g.float().unique()) > 1 or g.numel() == 1
        b, n, v = g.shape
        last = (b - 1) * g.stride(0) + (n - 1) * g.stride(1) + v + g.storage_offset()
        assert last <= g.untyped_storage().nbytes() // 2
    wide = torch.zeros(1, 1, 17).expand(3, 4, 17)
    assert losses._grad_like(wide).is_contiguous()


def test_operators_have_fake_shapes():
    """``torch.ops.pkv`` losses trace with fake tensors: shapes and types without running a kernel."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import randomrepo_b200.ops  # noqa: F401 - registers the operators

    with FakeTensorMode():
        dev = torch.device("cuda", 0)
        for shape in ((4, 9, 1001), (9, 1001)):
            x = torch.empty(shape, dtype=torch.bfloat16, device=dev)
            rows = shape[:-1]
            tok = torch.empty(rows, dtype=torch.int64, device=dev)
            f = torch.empty(rows, device=dev)
            loss, lp, kl, ent, grad = torch.ops.pkv.policy_loss(x, tok, f, f, None, f, 0.2, 0.2, 0.1, 0.0, 1.0, "sum", 1.0)
            assert loss.shape == () and lp.shape == rows and kl.shape == rows and ent.shape == (0,)
            assert grad.shape == shape and grad.dtype == torch.bfloat16 and lp.dtype == torch.float32
            ids = torch.empty((*rows, 5), dtype=torch.int64, device=dev)
            loss, kl, grad = torch.ops.pkv.distillation_loss(x, ids, torch.empty((*rows, 5), device=dev), None, None,
                                                             2.0, "token_mean", 1.0)
            assert loss.shape == () and kl.shape == rows and grad.shape == shape
            v, t, lse = torch.ops.pkv.top_logits(x, 7, 1.0)
            assert v.shape == (*rows, 7) and t.dtype == torch.int64 and lse.shape == rows
        x = torch.empty((4, 9, 1001), device=dev)
        loss, s, m, grad = torch.ops.pkv.preference_loss(x, torch.empty((4, 9), dtype=torch.int64, device=dev), None,
                                                         None, 0.1, 0.0, False, 1.0)
        assert loss.shape == () and s.shape == (4,) and m.shape == (2,) and grad.shape == x.shape


@pytest.mark.parametrize("slots", [4, 5, 8])
def test_the_rings_order_never_waits_for_itself(slots):
    """A model of the order in which a row's chunks are copied, looked at and freed when sums and gradient share a
    launch (csrc/losses.cu): rows of up to three rings' length, some a chunk shorter than others.  Copy l waits until
    the chunk of copy l - slots is free; every chunk that is looked at must have been copied by then."""
    import random

    for most in range(1, 3 * slots):
        whole = most <= slots - 1
        again = lambda n: 0 if whole else max(n - (slots - 1), min(n, 1))  # noqa: E731
        for seed in range(60):
            r = random.Random(seed)
            rows = [most - r.randint(0, 1) for _ in range(r.randint(1, 12))]
            copies, looks, begun = [], [], 0
            for i, n in enumerate(rows):
                following = i + 1 < len(rows) and rows[i + 1] > 0
                copies += [(i, c, 0) for c in range(begun, n)]
                for c in range(begun, n):
                    looks.append(((i, c, 0), c < again(n)))
                begun = int(following)
                if following:
                    copies.append((i + 1, 0, 0))
                    looks.append(((i + 1, 0, 0), again(rows[i + 1]) > 0))
                copies += [(i, c, 1) for c in range(again(n))]
                looks += [((i, c, 0), True) for c in range(again(n), n)] + [((i, c, 1), True) for c in range(again(n))]
            place = {c: k for k, c in enumerate(copies)}
            free, copied = set(), 0
            for chunk, done in looks:
                while copied < len(copies) and (copied < slots or copied - slots in free):
                    copied += 1
                assert place[chunk] < copied and place[chunk] not in free, (rows, chunk)
                if done:
                    free.add(place[chunk])
            assert len(free) == len(copies)


def test_the_graph_holds_no_tensor_beside_the_saved_ones(monkeypatch):
    """What a differentiable call leaves on its graph node is saved tensors: they go with the backward pass and pass
    through saved-tensor hooks.  (The launches are left out.)"""
    from torch.multiprocessing.reductions import StorageWeakRef

    packed = []
    monkeypatch.setattr(losses, "_on_device", lambda x, fn, *args: packed.append((fn, args)))
    tok, adv, per_row = torch.zeros(2, 3, dtype=torch.int64), torch.ones(2), torch.zeros(2, 3)
    ids = torch.zeros(2, 3, 4, dtype=torch.int64)
    for call in (lambda z: losses.policy_loss(z, tok, adv, per_row, per_row != 1, ref_logprobs=per_row),
                 lambda z: losses.preference_loss(z, tok, None, adv),
                 lambda z: losses.distillation_loss(z, ids, ids.float(), None, teacher_lse=per_row)):
        x = torch.randn(2, 3, 8).requires_grad_()
        logits = _fake(x * 2)
        gone = StorageWeakRef(logits.untyped_storage())
        loss = call(logits).loss
        del logits
        assert not gone.expired()
        packed.clear()
        (grad,) = torch.autograd.grad(loss, x)
        assert gone.expired() and grad.shape == x.shape
        assert len(packed) == 1


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    x, tok = _fake(torch.zeros(2, 3, 8)), torch.zeros(2, 3, dtype=torch.int64)
    with fwad.dual_level():
        dual = _fake(fwad.make_dual(torch.zeros(2, 3, 8), torch.ones(2, 3, 8)))
        for call in (lambda: losses.policy_loss(dual, tok, torch.zeros(2)), lambda: losses.preference_loss_and_grad(dual, tok),
                     lambda: losses.distillation_loss(dual, tok.unsqueeze(-1), x[..., :1]), lambda: losses.top_logits(dual, 2)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        with pytest.raises(ValueError, match="k must"):  # (others are taken, up to the next check)
            losses.top_logits(x, 9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_rows_of_whole_vectors_start_like_the_logits(dtype):
    """Rows of a multiple of 16 bytes that start elsewhere in their 16 bytes, all at the same place or each at its own."""
    wide, step = torch.zeros(3, 4, 32, dtype=dtype), torch.zeros(3, 4, 21, dtype=dtype)
    shifted = torch.zeros(3 * 4 * 16 + 1, dtype=dtype)[1:].view(3, 4, 16)
    for x in (wide[..., 1:17], wide[:, 1:, 3:19], wide[::2, ::3, 1:25], wide[:, :1, 5:13], step[..., :16], step[:, 1:, 2:18],
              step[:, :-1, 1:17].transpose(0, 1)[:, 1:2], shifted, shifted[1:], shifted[:, 1:]):
        g = losses._grad_like(x)
        assert g.shape == x.shape and g.stride(-1) == 1 and g.dtype == dtype
        for i in range(x.shape[0]):
            for j in range(x.shape[1]):
                assert (g[i, j].data_ptr() - x[i, j].data_ptr()) % 16 == 0, (x.shape, x.stride(), i, j)
        g.copy_(torch.arange(g.numel()).view(g.shape) % 251)
        assert torch.equal(g, (torch.arange(g.numel()).view(g.shape) % 251).to(dtype))  # no two rows overlap
