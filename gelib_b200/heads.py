"""Both ends of a network over discrete things, species of atoms or the entries of a vocabulary: the lookup of an embedding table, and the losses
behind a last dense layer.

What the reference leaves to torch.nn, as the readout (its Python layer ends with the products, python/src/gelib).  A table row per species
makes the l=0 part of a network's input; the invariants of its last product go through the readout to a vector per atom, whose products with
a matrix of classes are scored against the class that was there, or against what a larger network holds likely.  The products are never kept.
All compute on CUDA tensors in float32, bfloat16 or float16 with float32 sums; losses are float32.  They can be differentiated once, and
not in forward mode, which is refused.  Calls whose operands need nothing special are made by the native host side.
"""
import ctypes

import torch

from ._lib import LinearLossArgs, check, device_guard, lib, native, stream_of
from .gelib_common import plain
from .readout import _TYPES, _checked, _dense, _ptr, _rows, _workspace, linear

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _numbers(fn, name, t, x, shape):
    """t holds numbers of rows or classes on x's device."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise RuntimeError("%s: %s must be an int64 or int32 tensor" % (fn, name))
    if t.device != x.device:
        raise RuntimeError("%s: %s must be on the device of %s" % (fn, name, "weight" if fn == "embedding" else "x"))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError("%s: %s must have shape %s, got %s" % (fn, name, tuple(shape), tuple(t.shape)))


def _differentiable_once(name, grads):
    """Gradients of a call whose own gradient is asked for: an error when that is wanted, not zeros."""
    some = [g for g in grads if g is not None]
    if not torch.is_grad_enabled() or not some:
        return grads
    marked = torch._C._functions.DelayedError(name + " can be differentiated once", len(some))(*[g.detach().requires_grad_() for g in some])
    marked = iter((marked,) if len(some) == 1 else marked)
    return tuple(None if g is None else next(marked) for g in grads)


class EmbeddingFn(torch.autograd.Function):
    """embedding with its gradient; ids (n), weight (v, d)."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        ids, weight = ids.contiguous(), _rows(weight)
        v, d = weight.shape
        n = ids.numel()
        y = torch.empty(n, d, dtype=weight.dtype, device=weight.device)
        state = _workspace(lib().gelib_embedding_state_bytes(n, v), weight) if ctx.needs_input_grad[1] else None
        with device_guard(weight):
            check(lib().gelib_embedding(_ptr(y), _ptr(ids), _ptr(weight), n, v, d, max(weight.stride(0), d), scale, padding, ids.element_size(),
                                        _TYPES[weight.dtype], _ptr(state), stream_of(weight)))
        ctx.save_for_backward(state)
        ctx.sizes, ctx.scale = (n, v, d), scale
        return y

    @staticmethod
    def backward(ctx, gy):
        with torch.no_grad():
            gw = EmbeddingFn.gradient(ctx, gy)
        return _differentiable_once("embedding", (None, gw, None, None))

    @staticmethod
    def gradient(ctx, gy):
        state, = ctx.saved_tensors
        gy = _dense(gy)
        n, v, d = ctx.sizes
        gw = torch.empty(v, d, dtype=gy.dtype, device=gy.device)
        with device_guard(gy):
            w = _workspace(lib().gelib_embedding_workspace(n, v, d, _TYPES[gy.dtype]), gy)
            check(lib().gelib_embedding_back(_ptr(gw), _ptr(gy), _ptr(state), n, v, d, ctx.scale, _TYPES[gy.dtype], _ptr(w), stream_of(gy)))
        return gw


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids]: the rows of weight (v, d) that ids, of any shape, names; the result has shape ids.shape + (d,).

    weight is real or complex64, whose rows then are those of an l=0 part.  The gradient of weight is dense; what falls on a row is added in the
    order of ids, in float32, and rounded once, so that it repeats bit for bit.  Row padding_idx has no gradient.  An id outside [0, v)
    gives a row of NaN, and no gradient.  Where weight requires a gradient the ids are sorted for it in this call (16 bytes an id are kept): a
    validation pass that needs none runs under ``torch.no_grad()``.
    """
    scale = float(scale)
    if isinstance(ids, torch.Tensor) and isinstance(weight, torch.Tensor) and (padding_idx is None or type(padding_idx) is int):
        y = native().embedding(ids, weight, scale, padding_idx)
        if y is not None:
            return y
    with plain():
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
            raise RuntimeError("embedding: weight must have 2 dimensions (entries, channels)")
        if weight.dtype == torch.complex64:
            y = embedding(ids, torch.view_as_real(weight.resolve_conj()).reshape(weight.size(0), 2 * weight.size(1)), scale, padding_idx)
            return torch.view_as_complex(y.view(y.shape[:-1] + (weight.size(1), 2)))
        _checked("embedding", weight, ())
        _numbers("embedding", "ids", ids, weight, None)
        v, d = weight.shape
        padding = -1
        if padding_idx is not None:
            padding = int(padding_idx)
            if not -v <= padding < v:
                raise RuntimeError("embedding: padding_idx %d is none of the %d rows" % (padding, v))
            padding %= v
        wanted = weight if torch.is_grad_enabled() else weight.detach()   # needs_input_grad does not tell: nothing is sorted where no gradient follows
        return EmbeddingFn.apply(ids.reshape(-1), wanted, scale, padding).view(ids.shape + (d,))


def _loss_args(x, w, bias, target, teacher, transposed, reduction, ignore_index, temperature):
    a = LinearLossArgs()
    a.x, a.w, a.bias, a.target, a.teacher = _ptr(x), _ptr(w), _ptr(bias), _ptr(target), _ptr(teacher)
    a.m, a.k, a.n = x.size(0), w.size(0), w.size(1)
    a.ldx = max(x.stride(0), a.k)
    a.ldw = max(w.stride(1) if transposed else w.stride(0), a.k if transposed else a.n)
    a.top = 1 if teacher is None else teacher.size(1)
    a.w_transposed, a.reduction, a.ignore_index, a.temperature = transposed, reduction, ignore_index, temperature
    a.type, a.teacher_type, a.index_bytes = _TYPES[x.dtype], 0 if teacher is None else _TYPES[teacher.dtype], target.element_size()
    return a


def _call(fn, a, backward, like):
    with device_guard(like):
        w = _workspace(lib().gelib_linear_loss_workspace(ctypes.byref(a), backward), like)
        check(fn(ctypes.byref(a), _ptr(w), stream_of(like)))


class LinearLossFn(torch.autograd.Function):
    """linear_cross_entropy (teacher None) and linear_distillation with their gradients; x (m, k), target (m) or (m, top)."""

    @staticmethod
    def forward(ctx, x, w, bias, target, teacher, reduction, ignore_index, temperature):
        x, bias, target, teacher = _rows(x), _dense(bias), target.contiguous(), _dense(teacher)
        transposed = w.stride(0) == 1 and w.stride(1) != 1 and w.stride(1) >= w.size(0) and not w.is_neg()   # the view w.t() of a matrix (n_out, n_in)
        w = w if transposed else _rows(w)
        a = _loss_args(x, w, bias, target, teacher, transposed, reduction, ignore_index, temperature)
        loss = torch.empty(x.size(0) if reduction == 0 else 1, dtype=torch.float32, device=x.device)
        state = torch.empty(lib().gelib_linear_loss_state_bytes(ctypes.byref(a)), dtype=torch.uint8, device=x.device)
        a.loss, a.state = _ptr(loss), _ptr(state)
        _call(lib().gelib_linear_loss, a, 0, x)
        ctx.save_for_backward(x, w, bias, target, teacher, state)
        ctx.rest = transposed, reduction, ignore_index, temperature
        return loss if reduction == 0 else loss.view(())

    @staticmethod
    def backward(ctx, gy):
        with torch.no_grad():
            grads = LinearLossFn.gradients(ctx, gy)
        return _differentiable_once("linear_cross_entropy" if ctx.saved_tensors[4] is None else "linear_distillation", grads + (None,) * 5)

    @staticmethod
    def gradients(ctx, gy):
        x, w, bias, target, teacher, state = ctx.saved_tensors
        transposed = ctx.rest[0]
        a = _loss_args(x, w, bias, target, teacher, *ctx.rest)
        gy = _dense(gy)
        need = ctx.needs_input_grad
        like = dict(dtype=x.dtype, device=x.device)
        gx = torch.empty(a.m, a.k, **like) if need[0] else None
        gw = torch.empty((a.n, a.k) if transposed else (a.k, a.n), **like) if need[1] else None
        gb = torch.empty(a.n, **like) if need[2] else None
        a.gy, a.state, a.gx, a.gw, a.gb = _ptr(gy), _ptr(state), _ptr(gx), _ptr(gw), _ptr(gb)
        _call(lib().gelib_linear_loss_back, a, 1, x)
        return gx, gw.t() if need[1] and transposed else gw, gb


def _linear_loss(fn, x, w, bias, target, teacher, reduction, ignore_index, temperature):
    with plain():
        if not isinstance(x, torch.Tensor) or x.dim() < 1 or not isinstance(w, torch.Tensor) or w.dim() != 2 or x.size(-1) != w.size(0):
            raise RuntimeError("%s: x must be (..., n_in) and w (n_in, n_classes)" % fn)
        k, n = w.shape
        if k < 1 or n < 1:
            raise RuntimeError("%s: w must have at least one input channel and one class, got %s" % (fn, tuple(w.shape)))
        _checked(fn, x, (("w", w, (k, n)), ("bias", bias, (n,))))
        lead = x.shape[:-1]
        m = lead.numel()
        if teacher is None:
            _numbers(fn, "target", target, x, lead)
            shaped = target.reshape(m)
        else:
            if not isinstance(teacher, torch.Tensor) or teacher.device != x.device or teacher.dtype not in _TYPES:
                raise RuntimeError("%s: logits must be a float32, bfloat16 or float16 tensor on the device of x" % fn)
            if teacher.dim() != x.dim() or teacher.shape[:-1] != lead or not 1 <= teacher.size(-1) <= 1024:
                raise RuntimeError("%s: logits must have shape %s with 1 to 1024 entries, got %s" % (fn, tuple(lead) + ("entries",), tuple(teacher.shape)))
            if teacher.requires_grad and torch.is_grad_enabled():
                raise RuntimeError("%s: the teacher's logits have no gradient here; detach them" % fn)
            _numbers(fn, "ids", target, x, teacher.shape)
            shaped, teacher = target.reshape(m, -1 if m else teacher.size(-1)), teacher.reshape(m, -1 if m else teacher.size(-1))
        loss = LinearLossFn.apply(x.reshape(m, k), w, bias, shaped, teacher, reduction, ignore_index, temperature)
        return loss.view(lead) if reduction == 0 else loss


def _reduction(fn, name):
    if name not in REDUCTIONS:
        raise ValueError("%s: reduction is one of %s; got %r" % (fn, ", ".join(REDUCTIONS), name))
    return REDUCTIONS[name]


def linear_cross_entropy(x, w, target, bias=None, ignore_index=-100, reduction="mean"):
    """The cross entropy of the rows of x w + bias, with x (..., n_in) and w (n_in, n_classes), and the classes target (...), int64 or int32.

    A row's loss is log(sum of exp z) - z[target].  Rows whose target is ignore_index have none: they count as 0, their gradients are zero, and
    nothing that x holds there matters.  reduction: "mean" over the rows that have a loss (0 when none has), "sum", or "none" for a loss per row.
    Losses are float32.  z is never kept; the gradients are computed from it a second time, in pieces of the classes.  w may be the view ``v.t()`` of a
    matrix (n_classes, n_in), such as an embedding's table: it is used as it lies, and so is its gradient.  x may have strided rows; other
    strides are copied.  A target that is no class makes its row's loss and gradients NaN.
    """
    r, ignore_index = _reduction("linear_cross_entropy", reduction), int(ignore_index)
    if isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and isinstance(target, torch.Tensor):
        y = native().linear_loss(x, w, bias, target, None, r, ignore_index, 1.0)
        if y is not None:
            return y
    return _linear_loss("linear_cross_entropy", x, w, bias, target, None, r, ignore_index, 1.0)


def linear_distillation(x, w, ids, logits, bias=None, temperature=1.0, reduction="mean"):
    """The divergence of the rows of x w + bias from a teacher's largest logits: logits (..., entries) of the classes ids (..., entries).

    With q = softmax(logits / temperature) over a row's entries and p = softmax((x w + bias) / temperature) over all classes, a row's loss is
    temperature^2 times the sum of q (log q - log p).  Entries whose id is negative, and those whose logit is -infinity, are missing; rows
    without entries have no loss, like those of linear_cross_entropy that are ignored.  The same class may come twice.  At most 1024 entries;
    logits may be of another type than x, and have no gradient.  An id of n_classes or more makes its row's loss and gradients NaN.
    The rest is as for linear_cross_entropy.
    """
    fn = "linear_distillation"
    r, temperature = _reduction(fn, reduction), float(temperature)
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError("%s: the temperature is between 1e-15 and 1e15; got %r" % (fn, temperature))
    if isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and isinstance(ids, torch.Tensor) and isinstance(logits, torch.Tensor):
        y = native().linear_loss(x, w, bias, ids, logits, r, 0, temperature)
        if y is not None:
            return y
    if logits is None:
        raise RuntimeError("%s: logits must be a float32, bfloat16 or float16 tensor on the device of x" % fn)
    return _linear_loss(fn, x, w, bias, ids, logits, r, 0, temperature)


class Embedding(torch.nn.Module):
    """Module form of :func:`embedding`: weight (entries, channels) with normal entries, complex ones for an l=0 part."""

    def __init__(self, entries, channels, scale=1.0, padding_idx=None, device='cpu', dtype=torch.float32):
        super().__init__()
        if padding_idx is not None and not -entries <= padding_idx < entries:
            raise RuntimeError("embedding: padding_idx %d is none of the %d rows" % (padding_idx, entries))
        self.scale, self.padding_idx = scale, padding_idx
        weight = torch.randn(entries, channels, device=device, dtype=dtype)
        if padding_idx is not None:
            weight[padding_idx] = 0
        self.weight = torch.nn.Parameter(weight)

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)


class Classifier(torch.nn.Module):
    """A last layer over classes: its outputs by :func:`linear`, and its losses without them.  Weight (n_in, n_classes) with normal entries
    of variance 1 / n_in, bias zero."""

    def __init__(self, n_in, n_classes, bias=True, device='cpu', dtype=torch.float32):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.randn(n_in, n_classes, device=device, dtype=dtype) / max(1, n_in) ** 0.5)
        self.bias = torch.nn.Parameter(torch.zeros(n_classes, device=device, dtype=dtype)) if bias else None

    def forward(self, x):
        return linear(x, self.weight, self.bias)

    def cross_entropy(self, x, target, ignore_index=-100, reduction="mean"):
        return linear_cross_entropy(x, self.weight, target, self.bias, ignore_index, reduction)

    def distillation(self, x, ids, logits, temperature=1.0, reduction="mean"):
        return linear_distillation(x, self.weight, ids, logits, self.bias, temperature, reduction)
