"""Clipping the gradients of a network by their common norm (extension; the reference has none)."""
import math

import numpy as np

from .. import backend_api
from ..backend_selection import BackendTensor
from ..parallel import _ArrayView
from ..tensor import Tensor

_ALIGN = 64         # a gradient's place in the common array begins at a multiple of this many elements (256 bytes)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, grad_scale=1.0, error_if_nonfinite=False):
    """Scales the gradients of `parameters` down to a common norm of at most `max_norm`; returns that norm as it was before, a
    tensor of shape (1,).

    norm_type 2: the square root of the sum of all squares, held in double; norm_type inf: the largest magnitude.  Every
    gradient is multiplied by min(1, max_norm / (norm + 1e-6)).  A NaN in one of them makes the norm and all of them NaN; an infinity
    makes the norm infinite, hence the factor 0: itself NaN, everything finite 0.
    Parameters without a gradient are passed over, one that is listed twice counts once.  `grad_scale` is the factor the
    optimizer applies when it steps (`optimizer.grad_scale`, 1/world behind a gradient exchange): the norm is that of the scaled
    gradients.  error_if_nonfinite reads the norm back and raises RuntimeError instead of scaling, which a captured step cannot.

    Gradients are not modified in place: p.grad is replaced (nodes of a retained graph and parameters with a common gradient
    keep reading the arrays they have)."""
    params = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    max_norm, norm_type, grad_scale = float(max_norm), float(norm_type), float(grad_scale)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must be >= 0, got {max_norm}")
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"clip_grad_norm_: norm_type is 2 or inf, got {norm_type}")
    if not 0.0 <= grad_scale < math.inf:
        raise ValueError(f"clip_grad_norm_: grad_scale must be finite and >= 0, got {grad_scale}")
    seen, live, grads = set(), [], []
    for p in params:
        g = p.grad
        if g is not None and id(p) not in seen:
            seen.add(id(p))
            live.append(p)
            grads.append((g.data if isinstance(g, Tensor) else g).compact())
    device = grads[0]._device if grads else (params[0].device if params else backend_api.default_device())
    for g in grads:
        if g._device is not device and g._device != device:
            raise ValueError("clip_grad_norm_: the gradients are on different devices")
    mod = device.mod
    if error_if_nonfinite and getattr(mod, "capturing", False):
        raise RuntimeError("clip_grad_norm_: error_if_nonfinite reads the norm back, which a captured step cannot")
    if not hasattr(mod, "clip_grad_norm"):
        return _primitive(live, grads, device, max_norm, norm_type, grad_scale, error_if_nonfinite)
    norm = BackendTensor.make((1,), device=device)
    handles = [g._handle for g in grads]
    sizes = [h.size for h in handles]
    flat = mod.Array(sum([-(-n // _ALIGN) for n in sizes]) * _ALIGN)
    outs, at = [], 0
    for n in sizes:
        outs.append(_ArrayView(flat, at, n))
        at += -(-n // _ALIGN) * _ALIGN
    mod.clip_grad_norm(handles, outs, norm._handle, max_norm, norm_type == math.inf, grad_scale)
    if error_if_nonfinite:
        _refuse_nonfinite(float(norm.numpy()[0]))
    for p, g, out in zip(live, grads, outs):
        new = BackendTensor.make(g._shape, g._strides, device, out)      # (compact, as g is)
        p.grad = Tensor(new) if isinstance(p.grad, Tensor) else new
    return Tensor(norm)


def _like(old, new):
    return Tensor(new) if isinstance(old, Tensor) else new


def _refuse_nonfinite(norm):
    if not math.isfinite(norm):
        raise RuntimeError(f"clip_grad_norm_: the norm of the gradients is {norm}")


def _primitive(live, grads, device, max_norm, norm_type, grad_scale, error_if_nonfinite):
    """the same over the device primitives, every gradient read back: the squares of fp32 values need double"""
    if norm_type == math.inf:
        parts = [float((g.maximum(-g)).max().numpy().reshape(-1)[0]) for g in grads if g.size]
        total = math.nan if any(math.isnan(v) for v in parts) else max(parts, default=0.0)
    else:
        total = math.sqrt(sum(float(np.square(g.numpy(), dtype=np.float64).sum()) for g in grads if g.size))
    total *= grad_scale
    if error_if_nonfinite:
        with np.errstate(over="ignore"):
            _refuse_nonfinite(float(np.float32(total)))      # (the norm as it is returned)
    coef = max_norm / (total + 1e-6)
    coef = 1.0 if coef > 1.0 else coef
    for p, g in zip(live, grads):
        p.grad = _like(p.grad, g * coef)
    return Tensor(device.full((1,), total))
