"""Refusals of the language-model operators: checked on the host, before any CUDA call."""
from __future__ import annotations

import contextlib
import ctypes
import math
import random
import weakref

import pytest
import torch

from gpa_b200 import _lib, ops, linear_cross_entropy, residual_norm, rms_norm


def _message():
    buf = ctypes.create_string_buffer(256)
    _lib.load().gpa_b200_last_error(buf, 256)
    return buf.value.decode()


def _args(**kw):
    a = _lib.GpaNormArgs()
    a.update = a.weight = 16
    a.outer, a.inner, a.width = 2, 3, 8
    a.update_outer, a.update_inner = 24, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_norms_refuse_cpu_tensors():
    x, w = torch.ones(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        residual_norm(x, x, w)


@pytest.mark.parametrize("change,code,word", [
    (dict(weight=None), 1, "weight"), (dict(update=None), 1, "update"),
    (dict(update_dtype=3), 1, "dtypes"), (dict(out_dtype=-1), 1, "dtypes"),
    (dict(width=0), 1, "width"), (dict(outer=-1), 1, "outer"),
    (dict(gate_mode=1), 1, "without a residual"), (dict(gate_mode=3), 1, "gate_mode"),
    (dict(scale=16), 1, "without a residual"), (dict(post_weight=16), 1, "without a residual"),
    (dict(residual=16, gate_mode=2), 1, "needs a gate"),
    (dict(width=16385), 2, "16384"), (dict(outer=1 << 31), 2, "rows"),
])
def test_norm_entry_points_refuse_bad_arguments(change, code, word):
    lib = _lib.load()
    if change.get("gate_mode") == 1:
        change = {**change, "gate": 16}
    a = _args(**change)
    assert lib.gpa_b200_norm_forward(a, None, 16, None) == code
    assert word in _message(), _message()
    g = _lib.GpaNormGrads()
    g.dupdate = 16
    assert lib.gpa_b200_norm_backward(a, None, None, None, g, None, 0, None) == code
    assert word in _message(), _message()
    assert lib.gpa_b200_norm_scratch_bytes(a) == 0


def test_norm_entry_points_refuse_missing_tensors():
    lib = _lib.load()
    assert lib.gpa_b200_norm_forward(None, None, None, None) == 1
    assert lib.gpa_b200_norm_forward(_args(), None, None, None) == 1 and "outputs" in _message()
    assert lib.gpa_b200_norm_forward(_args(residual=16), None, 16, None) == 1
    g = _lib.GpaNormGrads()
    assert lib.gpa_b200_norm_backward(_args(), None, None, None, None, None, 0, None) == 1
    assert lib.gpa_b200_norm_backward(_args(), None, None, None, g, None, 0, None) == 1  # no dupdate
    g.dresidual = 16
    assert lib.gpa_b200_norm_backward(_args(residual=16), None, None, None, g, None, 0, None) == 1
    g.dweight = 16  # a weight gradient over many rows needs scratch
    many = _args(residual=16, outer=1000)
    assert lib.gpa_b200_norm_backward(many, 16, None, None, g, None, 0, None) == 1
    assert "scratch" in _message()
    assert lib.gpa_b200_norm_backward(many, 16, None, None, g, 20, 1 << 30, None) == 1
    assert "16 bytes" in _message()
    assert lib.gpa_b200_norm_scratch_bytes(many) >= 5 * 8 * 4
    assert lib.gpa_b200_norm_scratch_bytes(_args()) == 0  # one block takes so few rows


@pytest.mark.parametrize("name", ["dpost_weight", "dscale", "dgate"])
def test_norm_backward_refuses_gradients_of_tensors_that_are_not_there(name):
    lib = _lib.load()
    g = _lib.GpaNormGrads()
    g.dresidual = 16
    setattr(g, name, 16)
    assert lib.gpa_b200_norm_backward(_args(residual=16), 16, None, None, g, 16, 1 << 30, None) == 1
    assert "not there" in _message()


def _loss_args(**kw):
    a = _lib.GpaLossArgs()
    a.hidden = a.weight = a.labels = 16
    a.outer, a.inner, a.width, a.vocab, a.weight_stride, a.dtype = 1, 3, 8, 10, 8, 1
    a.hidden_outer, a.hidden_inner = 24, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_loss_refuses_cpu_tensors():
    x, w, y = torch.ones(2, 8), torch.ones(5, 8), torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="CUDA"):
        linear_cross_entropy(x, w, y)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=3), 1, "dtype"), (dict(reduction=3), 1, "reduction"), (dict(width=0), 1, "width"),
    (dict(vocab=0), 1, "vocab"), (dict(outer=-1), 1, "outer"), (dict(weight_stride=7), 1, "overlap"),
    (dict(width=65537, weight_stride=65537), 2, "channels"), (dict(vocab=(1 << 29) + 1), 2, "vocabulary"),
    (dict(outer=1 << 21), 2, "rows"),
    (dict(outer=1 << 20, vocab=1 << 29), 2, "tiles"), (dict(weight=None), 1, "NULL"),
])
def test_loss_entry_points_refuse_bad_arguments(change, code, word):
    lib = _lib.load()
    a = _loss_args(**change)
    assert lib.gpa_b200_loss_forward(a, 16, 16, 1 << 40, 16, 1 << 40, None) == code
    assert word in _message(), _message()
    assert lib.gpa_b200_loss_backward(a, 16, 1 << 40, 16, 16, 16, 16, 1 << 40, None) == code
    assert word in _message(), _message()
    if word != "NULL":
        assert lib.gpa_b200_loss_saved_bytes(a) == 0
        assert lib.gpa_b200_loss_scratch_bytes(a, 0) == 0 and lib.gpa_b200_loss_scratch_bytes(a, 1) == 0


def test_loss_entry_points_refuse_small_workspaces():
    lib = _lib.load()
    for name in ("hidden", "labels"):
        a = _loss_args(**{name: None})
        assert lib.gpa_b200_loss_forward(a, 16, 16, 1 << 40, 16, 1 << 40, None) == 1 and "NULL" in _message()
    a = _loss_args()
    saved, fwd, bwd = (lib.gpa_b200_loss_saved_bytes(a), lib.gpa_b200_loss_scratch_bytes(a, 0),
                       lib.gpa_b200_loss_scratch_bytes(a, 1))
    assert saved > 0 and fwd > 0 and bwd > 0
    assert lib.gpa_b200_loss_forward(a, 16, 16, saved - 1, 16, fwd, None) == 1 and "size" in _message()
    assert lib.gpa_b200_loss_forward(a, 16, 16, saved, 16, fwd - 1, None) == 1
    assert lib.gpa_b200_loss_forward(a, None, 16, saved, 16, fwd, None) == 1
    assert lib.gpa_b200_loss_backward(a, 16, saved, 16, 16, 16, 16, bwd - 1, None) == 1
    assert lib.gpa_b200_loss_backward(a, 16, saved, 16, None, None, 16, bwd, None) == 1
    # the workspaces are read 32 bytes at a time
    assert lib.gpa_b200_loss_forward(a, 16, 16, saved, 32, fwd, None) == 1 and "32 bytes" in _message()
    assert lib.gpa_b200_loss_backward(a, 32, saved, 16, 16, 16, 48, bwd, None) == 1 and "32 bytes" in _message()


def test_loss_workspace_of_a_training_step_stays_small():
    """65536 tokens against 151936 entries: logits would take 19.9 GB in 16 bits."""
    lib = _lib.load()
    a = _loss_args(outer=8, inner=8192, width=1024, vocab=151936, weight_stride=1024)
    assert lib.gpa_b200_loss_scratch_bytes(a, 0) < 2.5e9 and lib.gpa_b200_loss_scratch_bytes(a, 1) < 2.5e9


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cut(rows, labelled, width, vocab, dtype):
    a = _loss_args(outer=1, inner=rows, width=width, vocab=vocab, weight_stride=width, dtype=dtype)
    cut = (ctypes.c_int64 * 4)()
    assert _lib.load().gpa_b200_loss_cut(a, labelled, cut) == 0
    return tuple(cut)


def test_every_part_of_dhidden_is_written():
    """The parts that are added up are fresh memory: each holds a block of the first piece, also
    where the vocabulary ends inside a tile of 256."""
    sizes = [(256, 256, 1024, 7000, 1), (17, 17, 640, 8000, 1), (256, 256, 384, 16000, 2), (1, 1, 384, 28996, 1),
             (256, 256, 512, 28996, 0), (512, 512, 512, 7000, 1), (768, 768, 512, 7000, 0), (4096, 200, 1024, 7000, 1)]
    rng = random.Random(5)
    for _ in range(20000):
        rows = _log(rng, 1, 20000)
        sizes.append((rows, max(1, int(rows * rng.choice([1, 0.4, 0.05]))), _log(rng, 8, 8192), _log(rng, 1, 300000),
                      rng.randrange(3)))
    for size in sizes:
        entries, blocks, parts, each = _cut(*size)
        assert 1 <= entries <= size[3] and blocks == -(-entries // 64)
        assert (parts - 1) * each < blocks <= parts * each, (size, blocks, parts, each)


def test_cut_refuses_bad_arguments():
    lib, cut = _lib.load(), (ctypes.c_int64 * 4)()
    assert lib.gpa_b200_loss_cut(_loss_args(), -1, cut) == 1 and "labelled" in _message()
    assert lib.gpa_b200_loss_cut(_loss_args(), 4, cut) == 1 and "labelled" in _message()
    assert lib.gpa_b200_loss_cut(_loss_args(), 3, None) == 1
    assert lib.gpa_b200_loss_cut(_loss_args(vocab=0), 3, cut) == 1 and "vocab" in _message()


class _Calls:
    """The operators on CPU tensors, with the library's launches recorded instead of made.  Each
    record holds the entry point's name and the arguments; the structures are copied."""

    def __init__(self, monkeypatch):
        self.made = []
        monkeypatch.setattr(ops, "_check_tensor", lambda name, t, device=None: None)
        monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(ops, "_call", self._record)

    def _record(self, fn, device, *args):
        copied = [type(a).from_buffer_copy(a) if isinstance(a, ctypes.Structure) else a for a in args]
        self.made.append((fn.__name__, copied))

    def last(self, name):
        return [a for n, a in self.made if n == name][-1]


def _rows_inside(pointer, tensor, outer, inner, strides, width):
    """Whether outer x inner rows at `strides` lie in the memory of `tensor`."""
    last = (outer - 1) * strides[0] + (inner - 1) * strides[1] + width
    end = tensor.untyped_storage().data_ptr() + tensor.untyped_storage().nbytes()
    return pointer == tensor.data_ptr() and pointer + last * tensor.element_size() <= end


def _packed(kept):
    """Saved tensors come back as dense copies, as tensors kept on another device do."""
    def back(t):
        kept.append(t.clone(memory_format=torch.contiguous_format))
        return kept[-1]
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, back)


def test_norm_backward_reads_saved_tensors_where_they_are(monkeypatch):
    calls, kept = _Calls(monkeypatch), []
    joint = torch.randn(3, 5, 96)
    x = joint[..., 16:48].detach().requires_grad_()  # rows 96 apart, inside the joint tensor
    assert not x.is_contiguous()
    w = torch.ones(32, requires_grad=True)
    with _packed(kept):
        y = rms_norm(x, w)
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    a = calls.last("gpa_b200_norm_backward")[0]
    assert a.width == 32 and a.outer * a.inner == 15
    back = next(t for t in kept if t.shape == x.shape)
    assert _rows_inside(a.update, back, a.outer, a.inner, (a.update_outer, a.update_inner), 32)


def test_residual_norm_backward_reads_saved_tensors_where_they_are(monkeypatch):
    calls, kept = _Calls(monkeypatch), []
    joint, wide = torch.randn(3, 5, 96), torch.randn(3, 5, 200)
    residual, update = torch.randn(3, 5, 32), joint[..., 16:48].detach().requires_grad_()
    gate = wide[..., 100:132].detach().requires_grad_()
    with _packed(kept):
        s, n = residual_norm(residual, update, torch.ones(32), gate=gate, post_weight=torch.ones(32))
    torch.autograd.grad((s, n), (update, gate), (torch.ones_like(s), torch.ones_like(n)))
    a = calls.last("gpa_b200_norm_backward")[0]
    inside = [t for t in kept if t.shape == update.shape]
    assert any(_rows_inside(a.update, t, a.outer, a.inner, (a.update_outer, a.update_inner), 32) for t in inside)
    assert any(_rows_inside(a.gate, t, a.outer, a.inner, (a.gate_outer, a.gate_inner), 32) for t in inside)


def test_loss_backward_reads_the_saved_weight_where_it_is(monkeypatch):
    calls, kept = _Calls(monkeypatch), []
    x = torch.randn(6, 32).bfloat16().requires_grad_()
    w = torch.randn(50, 96).bfloat16()[:, 16:48].detach().requires_grad_()  # rows 96 apart
    assert not w.is_contiguous()
    with _packed(kept):
        loss = linear_cross_entropy(x, w, torch.zeros(6, dtype=torch.long))
    torch.autograd.grad(loss, (x, w))
    a, saved, nbytes = calls.last("gpa_b200_loss_backward")[:3]
    back = next(t for t in kept if t.shape == w.shape)
    assert _rows_inside(a.weight, back, 1, 50, (0, a.weight_stride), 32)
    assert nbytes >= _lib.load().gpa_b200_loss_saved_bytes(a)


def test_loss_backward_of_a_weight_that_moved_off_its_alignment(monkeypatch):
    """The forward read the weight in place; the copy that comes back starts off 16 bytes."""
    calls, kept = _Calls(monkeypatch), []
    x = torch.randn(6, 32).bfloat16().requires_grad_()
    w = torch.randn(50, 32).bfloat16().requires_grad_()

    def back(t):
        if t.shape != w.shape:
            return t
        moved = torch.empty(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape)
        kept.append(moved.copy_(t))
        return moved

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        loss = linear_cross_entropy(x, w, torch.zeros(6, dtype=torch.long))
    assert kept == []
    torch.autograd.grad(loss, (x, w))
    assert kept[0].data_ptr() % 16
    a, saved, nbytes = calls.last("gpa_b200_loss_backward")[:3]
    assert a.weight % 16 == 0 and nbytes >= _lib.load().gpa_b200_loss_saved_bytes(a)


def test_loss_backward_of_a_weight_that_comes_back_strided(monkeypatch):
    calls, kept = _Calls(monkeypatch), []
    x = torch.randn(6, 32).bfloat16().requires_grad_()
    w = torch.randn(50, 32).bfloat16().requires_grad_()

    def back(t):
        if t.shape != w.shape:
            return t
        kept.append(torch.zeros(50, 43, dtype=t.dtype)[:, 3:35].copy_(t))
        return kept[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        loss = linear_cross_entropy(x, w, torch.zeros(6, dtype=torch.long))
    torch.autograd.grad(loss, (x, w))
    a, saved, nbytes = calls.last("gpa_b200_loss_backward")[:3]
    assert a.weight % 16 == 0 and a.weight_stride == 32
    assert nbytes >= _lib.load().gpa_b200_loss_saved_bytes(a)


@pytest.mark.parametrize("spoil", [lambda t: t.double() if t.is_floating_point() else t, lambda t: t[..., :-1]])
def test_saved_tensors_of_another_type_or_shape_are_refused(monkeypatch, spoil):
    _Calls(monkeypatch)
    x, w = torch.randn(4, 32, requires_grad=True), torch.ones(32, requires_grad=True)
    e = torch.randn(50, 32, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil):
        outs = [rms_norm(x, w), residual_norm(x, x, w, post_weight=w)[0],
                linear_cross_entropy(x, e, torch.zeros(4, dtype=torch.long))]
    for out in outs:
        with pytest.raises(RuntimeError, match="saved"):
            out.backward(torch.ones_like(out))


def test_forward_mode_derivatives_are_refused(monkeypatch):
    _Calls(monkeypatch)
    x, w, e = torch.randn(4, 32), torch.ones(32), torch.randn(50, 32)
    labels = torch.zeros(4, dtype=torch.long)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        dw = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: rms_norm(d, w), lambda: rms_norm(x, dw), lambda: residual_norm(d, x, w),
                     lambda: residual_norm(x, d, w), lambda: residual_norm(x, x, w, post_weight=dw),
                     lambda: residual_norm(x, x, w, gate=d), lambda: residual_norm(x, x, w, scale=dw),
                     lambda: linear_cross_entropy(d, e, labels),
                     lambda: linear_cross_entropy(x, torch.autograd.forward_ad.make_dual(e, e), labels)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        rms_norm(x, w)  # nothing to differentiate: as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: rms_norm(t, w), (x,), (x,))


def test_loss_backward_without_rows_needs_no_gradient_to_write():
    """The gradient of an empty hidden has no memory; with a frozen weight nothing is left to do."""
    lib = _lib.load()
    a = _loss_args(outer=0)
    saved, scratch = lib.gpa_b200_loss_saved_bytes(a), lib.gpa_b200_loss_scratch_bytes(a, 1)
    assert lib.gpa_b200_loss_backward(a, 32, saved, None, None, None, 32, scratch, None) == 0


def test_a_vocabulary_that_one_piece_holds_is_one_piece():
    for rows, vocab, dtype in ((1, 1, 1), (300, 151936, 1), (4096, 151936, 2), (2000, 100001, 0), (256, 1 << 21, 1)):
        assert _cut(rows, rows, 64, vocab, dtype)[0] == vocab
    assert _cut(65536, 65536, 64, 151936, 1)[0] < 151936


def test_nothing_is_kept_that_hooks_on_saved_tensors_took_away(monkeypatch):
    """What such a hook moves elsewhere is free for the allocator until the backward."""
    _Calls(monkeypatch)
    leaf, w, e = torch.randn(4, 32, requires_grad=True), torch.ones(32, requires_grad=True), torch.randn(50, 32)
    for op in (lambda t: rms_norm(t, w), lambda t: residual_norm(t.detach(), t, w, post_weight=w)[0],
               lambda t: linear_cross_entropy(t, e, torch.zeros(4, dtype=torch.long))):
        x = leaf * 1
        gone = weakref.ref(x)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
            out = op(x)
        del x
        assert gone() is None
        out.backward(torch.ones_like(out))


def test_loss_workspace_does_not_grow_with_the_weight():
    """Beside 1.5 GB of P and 256 MB of parts of dhidden: 512 MB of a wide weight's gradient at most."""
    lib = _lib.load()
    for rows, width, vocab, dtype in ((64, 8192, 151936, 1), (200, 4097, 151936, 1), (300, 8192, 151936, 0),
                                      (4096, 5001, 151936, 2)):
        a = _loss_args(outer=1, inner=rows, width=width, vocab=vocab, weight_stride=width, dtype=dtype)
        assert lib.gpa_b200_loss_scratch_bytes(a, 1) < 2.6e9, (rows, width)
