"""The optimizer step of a network's weights: AdamW over all of them in one launch, moments in 32 or in 8 bits.

GElib's networks are trained with torch.optim (python/src/gelib has no optimizer), whose step is a handful of launches per
kind of tensor.  The weights are many small tensors -- a complex mixing matrix per l and layer, dense matrices, biases -- so here one
launch takes them all.
"""
import ctypes
import math

import torch

from ._lib import AdamwOptions, AdamwTensor, check, device_guard, lib, native, stream_of
from .gelib_common import plain

_TYPES = {torch.float32: 0, torch.complex64: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK8 = 256  # elements of an 8-bit state that share a scale


def _reals(t):
    return t.numel() * (2 if t.is_complex() else 1)


def _scalar(name, value):
    if isinstance(value, torch.Tensor):
        raise TypeError("adamw_step: %s is a number on the host, not a tensor" % name)
    return float(value)


def _dense(what, t, device, types, n):
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in types or not t.is_contiguous() or t.is_conj() or t.is_neg():
        raise RuntimeError("adamw_step: %s must be a contiguous tensor of %s on %s"
                           % (what, " or ".join(str(d).replace("torch.", "") for d in types), device))
    if _reals(t) != n:
        raise RuntimeError("adamw_step: %s has %d numbers where %d are needed" % (what, _reals(t), n))
    return t.data_ptr()


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, exp_avg_scale=None,
               exp_avg_sq_scale=None, master=None, seed=0, grad_scale=None, refresh_master=False):
    """One AdamW step, in place, on lists of tensors of one CUDA device:

        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - lr weight_decay) - lr m / (1 - b1^step) / (sqrt(v / (1 - b2^step)) + eps)

    params: contiguous float32, complex64 (taken as pairs of real numbers), bfloat16 or float16; grads: the same shapes and types.
    exp_avg, exp_avg_sq: m and v, as many float32 numbers as the parameter has (complex64 serves too).  With exp_avg_scale and
    exp_avg_sq_scale they are states in 8 bits: float8_e4m3fn codes, of which each 256 consecutive ones share a float32 scale; of v the
    root is held (:func:`block8_values` gives what they stand for).  They are rounded stochastically, by `seed` (another one each
    step) and an element's place in the lists, so the same call gives the same result.  master: float32 copies of the 16-bit parameters, which
    take the step and of which these are the rounded values; None for the others.  refresh_master: a copy whose rounding is not its parameter
    becomes the parameter before the step, element by element, so that what was written to parameters in between stays.  grad_scale: a float32
    tensor of one element on the device that gradients are multiplied by (the inverse of a loss scale, the factor of a clipping).

    step, lr and the rest are numbers on the host: a captured graph would repeat them, so a stream that is being captured is refused.
    No two tensors of a call may overlap.
    """
    lr, eps, weight_decay = _scalar("lr", lr), _scalar("eps", eps), _scalar("weight_decay", weight_decay)
    beta1, beta2 = (_scalar("betas", b) for b in betas)
    step, seed = int(step), int(seed) % (1 << 64)
    if len(params) == 0 and not (len(grads) or len(exp_avg) or len(exp_avg_sq)):
        return
    if native().adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, master, step, lr, beta1, beta2, eps, weight_decay,
                           seed, grad_scale, bool(refresh_master)) is not None:
        return
    with torch.no_grad(), plain():
        _adamw_step(list(params), list(grads), list(exp_avg), list(exp_avg_sq), exp_avg_scale, exp_avg_sq_scale, master, step, lr, beta1, beta2, eps,
                    weight_decay, seed, grad_scale, refresh_master)
        # what autograd has saved of these tensors is no longer what they hold
        for written in (params, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, master):
            torch.autograd.graph.increment_version([t for t in written or () if t is not None])


def _adamw_step(params, grads, m, v, ms, vs, master, step, lr, beta1, beta2, eps, weight_decay, seed, grad_scale, refresh_master):
    k = len(params)
    if (ms is None) != (vs is None):
        raise RuntimeError("adamw_step: states in 8 bits need exp_avg_scale and exp_avg_sq_scale")
    for name, other in (("grads", grads), ("exp_avg", m), ("exp_avg_sq", v), ("exp_avg_scale", ms), ("exp_avg_sq_scale", vs), ("master", master)):
        if other is not None and len(other) != k:
            raise RuntimeError("adamw_step: %d params and %d %s" % (k, len(other), name))
    device = params[0].device
    if device.type != "cuda":
        raise RuntimeError("gelib_b200 computes on CUDA tensors only (this build has no CPU path); got a %s tensor" % device.type)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adamw_step: the step's number and its rate are host values, which a captured graph would repeat")
    options = AdamwOptions(lr, beta1, beta2, eps, weight_decay, step, seed, None, 32 if ms is None else 8, bool(refresh_master))
    if grad_scale is not None:
        options.grad_scale = _dense("grad_scale", grad_scale, device, (torch.float32,), 1)
    real, codes = (torch.float32, torch.complex64), (torch.float8_e4m3fn,)
    entries, keep = (AdamwTensor * k)(), []
    for i, (p, g, e) in enumerate(zip(params, grads, entries)):
        n, scales = _reals(p), -(-_reals(p) // BLOCK8)
        e.p, e.n = _dense("a parameter", p, device, tuple(_TYPES), n), n
        e.type = _TYPES[p.dtype]
        if g.layout != torch.strided or g.shape != p.shape:
            raise RuntimeError("adamw_step: a gradient must be a dense tensor of its parameter's shape")
        keep.append(g.resolve_conj().resolve_neg().contiguous())
        e.g = _dense("a gradient", keep[-1], device, (p.dtype,), n)
        e.m, e.v = (_dense(what, t[i], device, real if ms is None else codes, n) for what, t in (("exp_avg", m), ("exp_avg_sq", v)))
        if ms is not None:
            e.m_scale, e.v_scale = (_dense(what, t[i], device, (torch.float32,), scales) for what, t in
                                    (("exp_avg_scale", ms), ("exp_avg_sq_scale", vs)))
        copy = master[i] if master is not None else None
        if (copy is None) != (e.type == 0):
            raise RuntimeError("adamw_step: a master copy goes with 16-bit parameters, and only with these")
        if copy is not None:
            e.master = _dense("a master copy", copy, device, (torch.float32,), n)
    with device_guard(params[0]):
        check(lib().gelib_adamw_step(k, entries, ctypes.byref(options), stream_of(params[0])))


def block8_values(codes, scale):
    """What an 8-bit state stands for (of exp_avg_sq: its root): codes times the scale of their block of 256, as a bfloat16 tensor of the codes'
    shape, exactly."""
    out = native().block8_values(codes, scale)
    if out is not None:
        return out
    with torch.no_grad(), plain():
        device = codes.device
        if device.type != "cuda":
            raise RuntimeError("gelib_b200 computes on CUDA tensors only (this build has no CPU path); got a %s tensor" % device.type)
        n = codes.numel()
        if codes.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32 or scale.device != device or scale.numel() != -(-n // BLOCK8):
            raise RuntimeError("block8_values: float8_e4m3fn codes, and a float32 scale for each 256 of them on the same device")
        codes, scale = codes.contiguous(), scale.contiguous()
        out = torch.empty(codes.shape, dtype=torch.bfloat16, device=device)
        with device_guard(codes):
            check(lib().gelib_block8_values(out.data_ptr(), codes.data_ptr(), scale.data_ptr(), n, stream_of(codes)))
        return out


class AdamW(torch.optim.Optimizer):
    """torch.optim's AdamW on :func:`adamw_step`: one launch per param group and device.

    state_bits: 32, or 8 for moments of one byte an element (and 4 bytes per 256).  Parameters of 16 bits get float32 master
    copies in the state; a step begins from the copies, and from the parameter where it was written since the last one.  seed: of the
    stochastic rounding of 8-bit states.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        if state_bits not in (32, 8):
            raise ValueError("state_bits is 32 or 8")
        if not (math.isfinite(lr) and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError("AdamW: lr must be finite, eps and weight_decay not negative, betas in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))

    def _state_of(self, p, bits):
        state = self.state[p]
        if not state:
            if p.dtype not in _TYPES or not p.is_contiguous():
                raise RuntimeError("AdamW: parameters must be contiguous and float32, complex64, bfloat16 or float16")
            n, dtype = _reals(p), torch.float32 if bits == 32 else torch.float8_e4m3fn
            state["step"] = 0
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(n, dtype=torch.uint8 if bits == 8 else dtype, device=p.device).view(dtype)
                if bits == 8:
                    state[name + "_scale"] = torch.ones(-(-n // BLOCK8), device=p.device)
            if _TYPES[p.dtype] != 0:
                state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for number, group in enumerate(self.param_groups):
            bits, calls = group["state_bits"], {}
            for p in group["params"]:
                if p.grad is not None:
                    state = self._state_of(p, bits)
                    calls.setdefault((p.device, state["step"]), []).append((p, state))
            for (device, step), members in calls.items():
                states = [s for _, s in members]
                scales = {name: [s[name] for s in states] for name in ("exp_avg_scale", "exp_avg_sq_scale")} if bits == 8 else {}
                adamw_step([p for p, _ in members], [p.grad for p, _ in members], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], step=step + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], master=[s.get("master") for s in states],
                           seed=group["seed"] + step + 1 + (number << 32), grad_scale=grad_scale, refresh_master=True,
                           **scales)
                for s in states:
                    s["step"] = step + 1
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but states keep their own types: torch would turn codes and master copies into the parameter's type.

        Hooks see what they would of torch's: those before it the whole dict, which they may replace, those after it the loaded state.  So the state is taken
        out behind the last hook before torch loads, and put in ahead of the first one after.
        """
        held = {}

        def take(_, given):
            held.update(given)
            return {"state": {}, "param_groups": given["param_groups"]}

        def put(_):
            numbers = [i for group in held["param_groups"] for i in group["params"]]
            params = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(numbers, params):
                if i in held["state"]:
                    self.state[p] = {name: value.detach().to(p.device, copy=True) if isinstance(value, torch.Tensor) else value
                                     for name, value in held["state"][i].items()}

        hooks = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(put, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
