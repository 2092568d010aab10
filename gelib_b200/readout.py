"""The readout of an equivariant network: group norm with an activation, and the dense layer with its epilogue.

What the reference leaves to torch.nn (its Python layer ends with the products, python/src/gelib): the invariants of a network -- the l=0
parts of its last product, (b, [grid...], channels) with the channels last as in every part -- are normalised and go through dense layers.
Both operators compute on CUDA tensors in float32, bfloat16 or float16 with float32 sums, and have gradients.
"""
import torch

from ._lib import check, device_guard, lib, stream_of
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
