"""The readout of an equivariant network: group norm with an activation, and the dense layer with its epilogue.

What the reference leaves to torch.nn (its Python layer ends with the products, python/src/gelib): the invariants of a network -- the l=0
parts of its last product, (b, [grid...], channels) with the channels last as in every part -- are normalised and go through dense layers.
Both operators compute on CUDA tensors in float32, bfloat16 or float16 with float32 sums, and have gradients; they can be differentiated once, and
not in forward mode, which is refused.  Calls whose operands need nothing special are made by the native host side.
"""
import ctypes

import torch

from ._lib import LinearArgs, check, device_guard, lib, native, stream_of
from .gelib_common import plain

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3}


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation is one of %s; got %r" % (", ".join(str(a) for a in ACTIVATIONS), name))
    return ACTIVATIONS[name]


def _checked(fn, x, others):
    """x is a real CUDA tensor, the others go with it."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("gelib_b200 computes on CUDA tensors only (this build has no CPU path); got a %s tensor"
                           % (x.device.type if isinstance(x, torch.Tensor) else type(x).__name__))
    if x.dtype not in _TYPES:
        raise RuntimeError("%s: expected a float32, bfloat16 or float16 tensor, got %s" % (fn, x.dtype))
    for name, t, shape in others:
        if t is None:
            continue
        if t.device != x.device or t.dtype != x.dtype:
            raise RuntimeError("%s: %s must be of x's type on x's device" % (fn, name))
        if tuple(t.shape) != tuple(shape):
            raise RuntimeError("%s: %s must have shape %s, got %s" % (fn, name, tuple(shape), tuple(t.shape)))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n > 0 else None


def _dense(t):
    return None if t is None else t.resolve_neg().contiguous()


class GroupNormFn(torch.autograd.Function):
    """group_norm with its gradients; x (b, s, n)."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        x, weight, bias = _dense(x), _dense(weight), _dense(bias)
        b, s, n = x.shape
        y = torch.empty_like(x)
        stats = torch.empty(2, b, groups, device=x.device) if any(ctx.needs_input_grad[:3]) else None
        with device_guard(x):
            w = _workspace(lib().gelib_group_norm_workspace(b, s, n, groups, _TYPES[x.dtype], 0), x)
            check(lib().gelib_group_norm(_ptr(y), _ptr(stats) and _ptr(stats[0]), _ptr(stats) and _ptr(stats[1]), _ptr(x), _ptr(weight), _ptr(bias),
                                         b, s, n, groups, eps, act, _TYPES[x.dtype], _ptr(w), stream_of(x)))
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, weight, bias, stats = ctx.saved_tensors
        gy = _dense(gy)
        b, s, n = x.shape
        gx, gw, gb = (torch.empty_like(t) if t is not None and need else None for t, need in zip((x, weight, bias), ctx.needs_input_grad))
        with device_guard(x):
            w = _workspace(lib().gelib_group_norm_workspace(b, s, n, ctx.groups, _TYPES[x.dtype], 1), x)
            check(lib().gelib_group_norm_back(_ptr(gx), _ptr(gw), _ptr(gb), _ptr(gy), _ptr(x), _ptr(weight), _ptr(bias), _ptr(stats[0]),
                                              _ptr(stats[1]), b, s, n, ctx.groups, ctx.act, _TYPES[x.dtype], _ptr(w), stream_of(x)))
        return gx, gw, gb, None, None, None


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None):
    """act((x - mean) / sqrt(var + eps) * weight + bias) of x (b, [grid...], n), channels last.

    Each batch index has its own mean and (biased) variance for each of the `groups` groups of n / groups neighbouring channels, over the
    grid and the group.  weight, bias: (n,) of x's type, or None.  activation: None, "relu", "silu" or "gelu_tanh" (the tanh form).
    x with other strides than a dense tensor's is copied first.  n is at most 16384.
    """
    act, groups, eps = _activation(activation), int(groups), float(eps)
    if isinstance(x, torch.Tensor):
        y = native().group_norm(x, groups, weight, bias, eps, act)
        if y is not None:
            return y
    with plain():
        if not isinstance(x, torch.Tensor) or x.dim() < 2:
            raise RuntimeError("group_norm: x must have at least 2 dimensions (batch, channels)")
        n = x.size(-1)
        if groups < 1 or n % groups:
            raise RuntimeError("group_norm: %d channels do not divide into %d groups" % (n, groups))
        _checked("group_norm", x, (("weight", weight, (n,)), ("bias", bias, (n,))))
        shape = x.shape
        y = GroupNormFn.apply(x.reshape(shape[0], -1 if x.numel() else shape[1:-1].numel(), n), weight, bias, groups, eps, act)
        return y.view(shape)


def _linear_args(x, w, transposed, act):
    a = LinearArgs()
    a.x, a.w, a.m, a.k, a.n = x.data_ptr(), w.data_ptr(), x.size(0), w.size(0), w.size(1)
    a.ldx, a.ldw = max(x.stride(0), a.k) if a.m == 1 else x.stride(0), w.stride(1) if transposed else w.stride(0)
    a.ldw = max(a.ldw, a.k if transposed else a.n)   # the stride of a dimension of one element may be anything
    a.w_transposed, a.act, a.type = transposed, act, _TYPES[x.dtype]
    return a


def _rows(t):
    """t, or a dense copy, as a matrix of dense rows that do not overlap."""
    t = t.resolve_neg()
    return t if (t.stride(1) == 1 or t.size(1) == 1) and (t.stride(0) >= t.size(1) or t.size(0) == 1) else t.contiguous()


def _call(fn, a, backward, like):
    with device_guard(like):
        w = _workspace(lib().gelib_linear_workspace(ctypes.byref(a), backward), like)
        check(fn(ctypes.byref(a), _ptr(w), stream_of(like)))


class LinearFn(torch.autograd.Function):
    """linear with its gradients; x (m, k), residual (m, n)."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, act):
        x, bias, residual = _rows(x), _dense(bias), _dense(residual)
        transposed = w.stride(0) == 1 and w.stride(1) != 1 and not w.is_neg()   # the view w.t() of a matrix (n_out, n_in)
        w = w if transposed and w.stride(1) >= w.size(0) else _rows(w)
        transposed = transposed and w.stride(0) == 1 and w.stride(1) != 1
        a = _linear_args(x, w, transposed, act)
        y = torch.empty(a.m, a.n, dtype=x.dtype, device=x.device)
        z = torch.empty_like(y) if act and any(ctx.needs_input_grad[:3]) else None
        a.y, a.z, a.bias, a.residual = _ptr(y), _ptr(z), _ptr(bias), _ptr(residual)
        _call(lib().gelib_linear, a, 0, x)
        ctx.save_for_backward(x, w, z)
        ctx.transposed, ctx.act = transposed, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, w, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        gr = gy if need[3] else None
        gx = gw = gb = None
        if any(need[:3]):
            gy = _dense(gy)
            a = _linear_args(x, w, ctx.transposed, ctx.act)
            if need[0]:
                gx = torch.empty(a.m, a.k, dtype=x.dtype, device=x.device)
            if need[1]:
                gw = torch.empty((a.n, a.k) if ctx.transposed else (a.k, a.n), dtype=x.dtype, device=x.device)
            if need[2]:
                gb = torch.empty(a.n, dtype=x.dtype, device=x.device)
            a.gy, a.z, a.gx, a.gw, a.gb = _ptr(gy), _ptr(z), _ptr(gx), _ptr(gw), _ptr(gb)
            _call(lib().gelib_linear_back, a, 1, x)
            gw = gw.t() if need[1] and ctx.transposed else gw
        return gx, gw, gb, gr, None


def linear(x, w, bias=None, residual=None, activation=None):
    """act(x w + bias) + residual, with x (..., n_in) and w (n_in, n_out), laid out as the matrices of SO3weights.

    bias: (n_out,); residual: (..., n_out); all of x's type.  activation: None, "relu", "silu" or "gelu_tanh" (the tanh form).  Sums
    are float32 and a result is rounded once.  w may be the view ``v.t()`` of a matrix (n_out, n_in): it is used as it lies, and so is its
    gradient.  x may have strided rows; other strides are copied.  With an activation and gradients, x w + bias is kept in x's type.
    """
    act = _activation(activation)
    if isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor):
        y = native().linear(x, w, bias, residual, act)
        if y is not None:
            return y
    with plain():
        if not isinstance(x, torch.Tensor) or x.dim() < 1 or not isinstance(w, torch.Tensor) or w.dim() != 2 or x.size(-1) != w.size(0):
            raise RuntimeError("linear: x must be (..., n_in) and w (n_in, n_out)")
        k, n = w.shape
        shape = x.shape[:-1] + (n,)
        _checked("linear", x, (("w", w, (k, n)), ("bias", bias, (n,)), ("residual", residual, shape)))
        m = x.shape[:-1].numel()
        y = LinearFn.apply(x.reshape(m, k), w, bias, None if residual is None else residual.reshape(m, n), act)
        return y.view(shape)


class Linear(torch.nn.Module):
    """Module form of :func:`linear`: weight (n_in, n_out) with normal entries of variance 1 / n_in, bias zero."""

    def __init__(self, n_in, n_out, bias=True, activation=None, device='cpu', dtype=torch.float32):
        super().__init__()
        _activation(activation)
        self.activation = activation
        self.weight = torch.nn.Parameter(torch.randn(n_in, n_out, device=device, dtype=dtype) / max(1, n_in) ** 0.5)
        self.bias = torch.nn.Parameter(torch.zeros(n_out, device=device, dtype=dtype)) if bias else None

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual, self.activation)


class GroupNorm(torch.nn.Module):
    """Module form of :func:`group_norm`, with a weight and a bias."""

    def __init__(self, groups, channels, eps=1e-5, activation=None, device='cpu', dtype=torch.float32):
        super().__init__()
        _activation(activation)
        self.groups, self.eps, self.activation = groups, eps, activation
        self.weight = torch.nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))

    def forward(self, x):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps, self.activation)
