"""Operators of a language model round the DenseGPA core, as hand-written sm_100a kernels.

* :func:`residual_norm` -- the norm after a block, its gate and residual scale, the residual
  addition and the norm before the next block in one pass over the rows;
* :func:`rms_norm` -- the same norm without a residual stream;
* :func:`linear_cross_entropy` -- softmax cross entropy over a large vocabulary, in pieces of it
  and without keeping the logits.

They take CUDA tensors in float32, bfloat16 or float16 (the norms any mix of them), sum in fp32,
run on the current stream without synchronising, allocate through PyTorch, can be captured in a
CUDA graph and have first-order gradients in reverse mode; other derivatives are a
``RuntimeError``.  They raise ``ValueError`` for arguments they refuse.

As for any PyTorch operator, a backward that is captured must find no eager graph of the same
leaves alive: their gradient accumulators would belong to the eager stream.
"""
from __future__ import annotations

import contextlib
import functools
import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_NORM_WIDTH = 16384


def _on(device):
    """`device` as the current one: the library sizes the loss's workspaces for that."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


_HERE = contextlib.nullcontext()


class _Refuse(torch.autograd.Function):
    """Passes gradients on; whoever differentiates them again is told that there is no more."""

    @staticmethod
    def forward(ctx, token, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("second derivatives of this operator are not implemented")


def _first_order(backward):
    """A backward without a graph of its own.  With ``create_graph`` its results carry a node that
    refuses to be differentiated, so that a missing second derivative is an error, not a zero."""

    @functools.wraps(backward)
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        held = [g for g in out if g is not None]
        if not held:
            return out
        marked = iter(_Refuse.apply(torch.zeros((), device=held[0].device, requires_grad=True), *held))
        return tuple(None if g is None else next(marked) for g in out)

    return run


def _no_tangents(*tensors):
    """Without reverse-mode gradients an operator runs outside autograd, which would drop the
    tangents of forward-mode differentiation without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("forward-mode derivatives of this operator are not implemented")


def _call(fn, device, *args):
    """`fn(*args, stream)` on the current stream of `device`, made the current device."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, fn.__name__)


def _rows(t: Tensor):
    """`t` with unit stride along its last axis and its other axes as outer x inner rows:
    (tensor, outer stride, inner stride).  Copies only what these two strides cannot describe."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, (t.shape[-2] if t.ndim > 1 else 1) * width, width
    if t.stride(-1) == 1 or width == 1:
        outer, span = 0, None
        for size, stride in zip(reversed(t.shape[:-2]), reversed(t.stride()[:-2])):
            if size == 1:
                continue
            if span is None:
                outer, span = stride, stride * size
            elif stride == span:
                span = stride * size
            else:
                break
        else:
            return t, outer, t.stride(-2) if t.ndim > 1 else 0
    return _rows(t.contiguous())


def _places(*tensors):
    """Where the kernels find tensors, to tell whether saved ones are still there in the backward;
    None where hooks keep them meanwhile, which may bring anything back to the same place."""
    if torch._C._autograd._top_saved_tensors_default_hooks(False) is not None:
        return None
    return [None if t is None else t.data_ptr() for t in tensors]


def _altered(t, shape, dtype, index):
    """Whether a saved tensor is not what the kernels take from the forward: whoever kept it meanwhile
    (hooks on saved tensors, sharded parameters) may bring it back at another address and with other
    strides, but not with another shape, type or device."""
    return t is not None and (t.shape != shape or t.dtype is not dtype or t.get_device() != index)


_ALTERED = "a saved tensor came back with another shape, type or device than it was saved with"


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _check_tensor(name: str, t: Tensor, device=None):
    if t.is_cuda and t.dtype in _DTYPES and (device is None or t.device == device):
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (B200, sm_100a)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    raise ValueError(f"{name} is on {t.device}, the other tensors are on {device}")


def _vector(name: str, t: Tensor, width: int, device) -> Tensor:
    """A weight as the contiguous fp32 vector the kernels read (gradients flow back through)."""
    _check_tensor(name, t, device)
    if t.shape != (width,):
        raise ValueError(f"{name} must have shape [{width}], not {list(t.shape)}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _check_width(width: int):
    if not 1 <= width <= MAX_NORM_WIDTH:
        raise ValueError(f"the norms take 1 to {MAX_NORM_WIDTH} channels, not {width}")


_NONE = (None, 0, 0)  # no tensor, no strides


def _norm_args(residual, update, weight, post_weight, gate, scale, eps, const, stream_dtype,
               update_dtype, out_dtype, shape):
    """(GpaNormArgs, tensors that must outlive the launch)."""
    width = shape[-1]
    inner = shape[-2] if len(shape) > 1 else 1
    h, h0, h1 = _NONE if residual is None else _rows(residual)
    y, y0, y1 = _NONE if update is None else _rows(update)
    g, g0, g1 = _NONE if gate is None else _rows(gate)
    a = _lib.GpaNormArgs(
        _lib.ptr(h), _lib.ptr(y), _lib.ptr(g), weight.data_ptr(), _lib.ptr(post_weight),
        _lib.ptr(scale), math.prod(shape[:-2]) if inner else 0, inner, h0, h1, y0, y1, g0, g1,
        width, _DTYPES[stream_dtype], _DTYPES[update_dtype], 0 if g is None else _DTYPES[g.dtype],
        _DTYPES[out_dtype], 0 if g is None else 2 if g.shape[-1] == width else 1, eps, const)
    return a, (h, y, g)


def _norm_backward(a, device, stream_in, dstream, dnormed, grads):
    lib = _lib.load()
    g = _lib.GpaNormGrads(*[None if t is None else t.data_ptr() for t in grads])
    nbytes = lib.gpa_b200_norm_scratch_bytes(a)
    scratch = _scratch(nbytes, device) if nbytes else None
    _call(lib.gpa_b200_norm_backward, device, a, _lib.ptr(stream_in), _lib.ptr(dstream),
          _lib.ptr(dnormed), g, _lib.ptr(scratch), nbytes)


_DENSE = torch.contiguous_format


def _rms_args(x, weight, eps, out_dtype):
    return _norm_args(None, x, weight, None, None, None, eps, 1., x.dtype, x.dtype, out_dtype, x.shape)


def _rms_forward(x, weight, eps, out_dtype, args=None):
    out = torch.empty_like(x, dtype=out_dtype, memory_format=_DENSE)
    if out.numel():
        a, keep = _rms_args(x, weight, eps, out_dtype) if args is None else args
        _call(_lib.load().gpa_b200_norm_forward, x.device, a, None, out.data_ptr())
    return out


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, out_dtype):
        args = _rms_args(x, weight, eps, out_dtype)
        ctx.save_for_backward(x, weight)
        # the arguments serve the backward too, unless they point to a copy made for this call
        ctx.args = args[0] if args[1][1] is x else None
        ctx.places, ctx.stride = _places(x, weight), x.stride()
        ctx.dtype, ctx.eps, ctx.out_dtype = x.dtype, eps, out_dtype
        return _rms_forward(x, weight, eps, out_dtype, args)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        x, weight = ctx.saved_tensors
        a, keep = ctx.args, None
        if a is None or [x.data_ptr(), weight.data_ptr()] != ctx.places or x.stride() != ctx.stride:
            shape, index = dout.shape, dout.get_device()
            if _altered(x, shape, ctx.dtype, index) or _altered(weight, shape[-1:], torch.float32, index):
                raise RuntimeError(_ALTERED)
            weight = _dense(weight)
            a, keep = _rms_args(x, weight, ctx.eps, ctx.out_dtype)
        dx = torch.empty_like(x, memory_format=_DENSE)
        if not x.numel():
            return dx, torch.zeros_like(weight), None, None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        _norm_backward(a, x.device, None, None, dout.contiguous(), (None, dx, None, dw, None, None))
        return dx, dw, None, None


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, *,
             out_dtype: torch.dtype | None = None) -> Tensor:
    """``x / sqrt(mean(x^2, -1) + eps) * weight`` over the last axis, rounded once.

    x [..., D] (strided views are read in place where two strides describe their rows), weight
    [D], D up to 16384; returns a contiguous tensor of x's shape in ``out_dtype`` (x's dtype by
    default).  Gradients: x (in x's dtype) and weight.
    """
    _check_tensor("x", x)
    _no_tangents(x, weight)
    if x.ndim < 1:
        raise ValueError("x must have at least one axis")
    _check_width(x.shape[-1])
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    weight = _vector("weight", weight, x.shape[-1], x.device)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _RMSNorm.apply(x, weight, float(eps), out_dtype)
    return _rms_forward(x, weight, eps, out_dtype)


def _residual_args(residual, update, weight, post_weight, gate, scale, eps, const, out_dtype):
    return _norm_args(residual, update, weight, post_weight, gate, scale, eps, const, residual.dtype,
                      update.dtype, out_dtype, residual.shape)


def _residual_forward(residual, update, weight, post_weight, gate, scale, eps, const, out_dtype,
                      args=None):
    stream = torch.empty_like(residual, memory_format=_DENSE)
    normed = torch.empty_like(residual, dtype=out_dtype, memory_format=_DENSE)
    if stream.numel():
        a, keep = args or _residual_args(residual, update, weight, post_weight, gate, scale, eps,
                                         const, out_dtype)
        _call(_lib.load().gpa_b200_norm_forward, residual.device, a, stream.data_ptr(),
              normed.data_ptr())
    return stream, normed


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, update, weight, post_weight, gate, scale, eps, const, out_dtype):
        given = (residual, update, weight, post_weight, gate, scale, eps, const, out_dtype)
        args = _residual_args(*given)
        stream, normed = _residual_forward(*given, args)
        # the update itself is needed only where the residual's share depends on it
        read = post_weight is not None or gate is not None or scale is not None
        ctx.save_for_backward(stream, update if read else None, weight, post_weight, gate, scale)
        # the arguments serve the backward too, unless they point to a copy made for this call
        ctx.args = args[0] if args[1][1] is update and args[1][2] is gate else None
        ctx.places = _places(stream, update if read else None, weight, post_weight, gate, scale)
        ctx.strides = update.stride() if read else None, None if gate is None else gate.stride()
        ctx.dtype, ctx.update_dtype = residual.dtype, update.dtype
        ctx.gate = None if gate is None else (gate.shape, gate.dtype)
        ctx.eps, ctx.const, ctx.out_dtype = eps, const, out_dtype
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    @_first_order
    def backward(ctx, dstream, dnormed):
        if dstream is None and dnormed is None:
            return (None,) * 9
        saved = ctx.saved_tensors
        stream, update, weight, post_weight, gate, scale = saved
        a, keep = ctx.args, None
        strides = None if update is None else update.stride(), None if gate is None else gate.stride()
        if a is None or [None if t is None else t.data_ptr() for t in saved] != ctx.places or strides != ctx.strides:
            up = dnormed if dstream is None else dstream
            shape, index = up.shape, up.get_device()
            vector = shape[-1:]
            if (_altered(stream, shape, ctx.dtype, index) or _altered(weight, vector, torch.float32, index) or
                    _altered(update, shape, ctx.update_dtype, index) or
                    _altered(post_weight, vector, torch.float32, index) or
                    _altered(scale, vector, torch.float32, index) or
                    gate is not None and _altered(gate, *ctx.gate, index)):
                raise RuntimeError(_ALTERED)
            stream, weight, post_weight, scale = map(_dense, (stream, weight, post_weight, scale))
            a, keep = _norm_args(stream, update, weight, post_weight, gate, scale, ctx.eps, ctx.const,
                                 stream.dtype, ctx.update_dtype, ctx.out_dtype, stream.shape)
        need = ctx.needs_input_grad
        dres = torch.empty_like(stream) if need[0] else None
        dupd = torch.empty_like(stream, dtype=ctx.update_dtype) if need[1] else None
        dw, dpw, dscale = (torch.empty_like(weight) if need[i] else None for i in (2, 3, 5))
        dgate = torch.empty_like(gate, memory_format=_DENSE) if need[4] else None
        if not stream.numel():
            for t in (dw, dpw, dscale):
                if t is not None:
                    t.zero_()
            return dres, dupd, dw, dpw, dgate, dscale, None, None, None
        dstream = None if dstream is None else dstream.contiguous()
        dnormed = None if dnormed is None else dnormed.contiguous()
        _norm_backward(a, stream.device, stream, dstream, dnormed, (dres, dupd, dgate, dw, dpw, dscale))
        return dres, dupd, dw, dpw, dgate, dscale, None, None, None


def residual_norm(residual: Tensor, update: Tensor, weight: Tensor, eps: float = 1e-6, *,
                  post_weight: Tensor | None = None, gate: Tensor | None = None,
                  scale: Tensor | float | None = None,
                  out_dtype: torch.dtype | None = None) -> tuple[Tensor, Tensor]:
    """The residual addition between two blocks, with the norms on both sides of it.

    With ``rms(x) = sqrt(mean(x^2, -1) + eps)``::

        u      = update / rms(update) * post_weight     (update itself without post_weight)
        stream = residual + scale * sigmoid(gate) * u   (rounded to residual's dtype)
        normed = stream / rms(stream) * weight          (rounded to out_dtype)

    residual, update [..., D] with D up to 16384; weight, post_weight [D]; gate broadcastable to
    update, with a last axis of D (one gate for each channel) or 1 (one for each row); scale a
    number, or a tensor of D values or one.  ``out_dtype`` defaults to update's dtype.  Returns
    ``(stream, normed)``, both contiguous and of residual's shape; ``normed`` is computed from
    the rounded stream.  Gradients: every tensor argument.
    """
    _check_tensor("residual", residual)
    _no_tangents(residual, update, weight, post_weight, gate, scale)
    dev = residual.device
    _check_tensor("update", update, dev)
    if residual.ndim < 1 or residual.shape != update.shape:
        raise ValueError(f"residual {list(residual.shape)} and update {list(update.shape)} must "
                         "have the same shape [..., D]")
    width = residual.shape[-1]
    _check_width(width)
    out_dtype = update.dtype if out_dtype is None else out_dtype
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    weight = _vector("weight", weight, width, dev)
    if post_weight is not None:
        post_weight = _vector("post_weight", post_weight, width, dev)
    if gate is not None:
        _check_tensor("gate", gate, dev)
        if gate.ndim < 1 or gate.shape[-1] not in (1, width):
            raise ValueError(f"gate {list(gate.shape)} must end in 1 or {width}")
        want = update.shape[:-1] + gate.shape[-1:]
        if gate.shape != want:
            try:
                gate = gate.expand(want)
            except RuntimeError:
                raise ValueError(f"gate {list(gate.shape)} does not broadcast to update "
                                 f"{list(update.shape)}") from None
    const = 1.
    if isinstance(scale, Tensor):
        _check_tensor("scale", scale, dev)
        if scale.numel() == 1:
            scale = scale.reshape(1).expand(width)
        scale = _vector("scale", scale, width, dev)
    elif scale is not None:
        const, scale = float(scale), None
    args = (residual, update, weight, post_weight, gate, scale, float(eps), const, out_dtype)
    if torch.is_grad_enabled() and (
            residual.requires_grad or update.requires_grad or weight.requires_grad or
            (post_weight is not None and post_weight.requires_grad) or
            (gate is not None and gate.requires_grad) or (scale is not None and scale.requires_grad)):
        return _ResidualNorm.apply(*args)
    return _residual_forward(*args)


def loss_limits(tokens: int, width: int, vocab: int) -> str | None:
    """What `linear_cross_entropy` says of sizes it does not take, or None."""
    if not 1 <= width <= 65536 or not 1 <= vocab <= 1 << 29:
        return f"1 to 65536 channels and 1 to 2^29 vocabulary entries, not {width} and {vocab}"
    if tokens > 1 << 22:
        return f"at most 2^22 tokens in a call, not {tokens}"
    if -(-tokens // 256) * -(-vocab // 256) > 1 << 30:
        return f"at most 2^30 tiles of 256 x 256 logits in a call, not {tokens} x {vocab}"
    return None


_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def _loss_args(weight, shape, dtype, ignore_index, reduction, hidden=_NONE, labels=None):
    """(GpaLossArgs, the weight it points to); only the forward gives hidden and labels."""
    w = weight if weight.stride(-1) == 1 and weight.stride(0) >= weight.shape[1] else weight.contiguous()
    inner = shape[-2] if len(shape) > 1 else 1
    vocab, width = weight.shape
    return _lib.GpaLossArgs(
        _lib.ptr(hidden[0]), w.data_ptr(), labels, math.prod(shape[:-2]) if inner else 0, inner,
        hidden[1], hidden[2], w.stride(0), vocab, ignore_index, width, _DTYPES[dtype], reduction), w


def _scratch(nbytes, device):
    return torch.empty(nbytes, device=device, dtype=torch.uint8)


def _loss_forward(hidden, weight, labels, ignore_index, reduction, keep_rows):
    """(loss, what the backward reads or None, GpaLossArgs or None where it points to a copy)."""
    lib = _lib.load()
    dev = hidden.device
    rows = _rows(hidden)
    a, w = _loss_args(weight, hidden.shape, hidden.dtype, ignore_index, reduction, rows,
                      labels.data_ptr())
    if reduction == 2:
        loss = torch.empty_like(labels, dtype=torch.float32)
    else:
        loss = torch.empty((), device=dev, dtype=torch.float32)
    with _on(dev):
        kept, more = lib.gpa_b200_loss_saved_bytes(a), lib.gpa_b200_loss_scratch_bytes(a, 0)
        saved = _scratch(kept if keep_rows else kept + more, dev)
        scratch = _scratch(more, dev) if keep_rows else None  # else behind what the backward would read
        at = saved.data_ptr()
        _call(lib.gpa_b200_loss_forward, dev, a, loss.data_ptr(), at, kept,
              scratch.data_ptr() if keep_rows else at + kept, more)
    return loss, saved if keep_rows else None, a if w is weight else None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        loss, saved, ctx.args = _loss_forward(hidden, weight, labels, ignore_index, reduction, True)
        # the labelled rows are packed into `saved`: hidden and labels are not needed again
        ctx.save_for_backward(weight, saved)
        ctx.hidden, ctx.weight, ctx.saved = (hidden.shape, hidden.dtype), (weight.shape, weight.stride()), saved.numel()
        ctx.places = _places(weight, saved)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        weight, saved = ctx.saved_tensors
        (shape, dtype), (weight_shape, stride) = ctx.hidden, ctx.weight
        lib = _lib.load()
        dev = weight.device
        a, keep = ctx.args, None
        if a is None or [weight.data_ptr(), saved.data_ptr()] != ctx.places or weight.stride() != stride:
            index = dloss.get_device()
            if _altered(weight, weight_shape, dtype, index) or _altered(saved, (ctx.saved,), torch.uint8, index):
                raise RuntimeError(_ALTERED)
            saved = _dense(saved)
            a, keep = _loss_args(weight, shape, dtype, ctx.ignore_index, ctx.reduction)
            if lib.gpa_b200_loss_saved_bytes(a) > saved.numel():
                # the forward read the weight in place; where it is now that takes a copy of it
                a, keep = _loss_args(weight.clone(memory_format=_DENSE), shape, dtype, ctx.ignore_index,
                                     ctx.reduction)
        dx = torch.empty(shape, device=dev, dtype=dtype) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight, memory_format=_DENSE) if ctx.needs_input_grad[1] else None
        dloss = dloss.contiguous()
        with _on(dev):
            nbytes = lib.gpa_b200_loss_scratch_bytes(a, 1)
            scratch = _scratch(nbytes, dev)
            _call(lib.gpa_b200_loss_backward, dev, a, saved.data_ptr(), saved.numel(),
                  dloss.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), scratch.data_ptr(), nbytes)
        return dx, dw, None, None, None


def linear_cross_entropy(hidden: Tensor, weight: Tensor, labels: Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T`` against ``labels``, in fp32.

    hidden [..., D] and weight [V, D] of one dtype (float32, bfloat16, float16), labels [...]
    integers; D up to 65536, V up to 2^29, 2^22 tokens.  The logits are formed tile by tile and
    never stored; the backward forms them again.  Tokens labelled ``ignore_index`` have no loss
    and zero gradients, cost nothing and are not read.  A label outside [0, V) makes its loss,
    and every gradient it reaches, NaN.

    ``reduction``: "mean" over the labelled tokens (0 when there is none), "sum", or "none" (a
    loss for each token, 0 where ignored).  Gradients: hidden and weight, rounded once to their
    dtype; with 16-bit inputs the gradient of each logit is rounded to that type on the way, and
    under "none" so are the hidden rows times their own gradients, for the weight's.
    """
    _check_tensor("hidden", hidden)
    _no_tangents(hidden, weight)
    dev = hidden.device
    _check_tensor("weight", weight, dev)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    if hidden.dtype != weight.dtype:
        raise ValueError(f"hidden ({hidden.dtype}) and weight ({weight.dtype}) must share a dtype")
    if hidden.ndim < 1 or weight.ndim != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"expected hidden [..., D] and weight [V, D], not {list(hidden.shape)} and "
                         f"{list(weight.shape)}")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {list(labels.shape)} must have hidden's leading shape "
                         f"{list(hidden.shape[:-1])}")
    if labels.device != dev:
        raise ValueError(f"labels is on {labels.device}, the other tensors are on {dev}")
    if labels.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise ValueError(f"labels must be integers, not {labels.dtype}")
    too_large = loss_limits(labels.numel(), weight.shape[1], weight.shape[0])
    if too_large:
        raise ValueError(too_large)
    if labels.dtype != torch.int64 or not labels.is_contiguous():
        labels = labels.long().contiguous()
    args = (hidden, weight, labels, int(ignore_index), _REDUCTIONS[reduction])
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(*args)
    return _loss_forward(*args, False)[0]


__all__ = ["linear_cross_entropy", "rms_norm", "residual_norm"]
