"""Bindings of csrc/muon.hip: orthogonalised matrices (Newton-Schulz iterations) and the update of weight matrices along an
orthogonalised momentum.  ``optim.Muon`` is the optimiser on top of it."""
import ctypes
import functools
import math

import torch

from . import _lib

_FIELDS = 11       # int64 fields of a matrix stack: in, out, momentum, rows, cols, batch, row / matrix strides of in and out, type
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_SIDE, MAX_SHORT_SIDE, MAX_STEPS = 1 << 24, 16384, 64


def _coefficients(coefficients, steps):
    """float[3 * steps]: one triple for every step, or a triple for each."""
    if type(coefficients) is tuple and len(coefficients) == 3 and all(type(v) is float for v in coefficients):
        return _same_coefficients(coefficients, int(steps))
    return _coefficient_array(coefficients, int(steps))


@functools.lru_cache(maxsize=32)
def _same_coefficients(coefficients, steps):
    return _coefficient_array(coefficients, steps)


def _coefficient_array(coefficients, steps):
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps: 1 to {MAX_STEPS}, got {steps}")
    rows = list(coefficients)
    if len(rows) == 3 and not any(isinstance(v, (tuple, list)) for v in rows):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients: (a, b, c), or {steps} such triples")
    return (ctypes.c_float * (3 * steps))(*(float(v) for r in rows for v in r)), steps


def _check_side(name, rows, cols):
    if max(rows, cols) > MAX_SIDE or min(rows, cols) > MAX_SHORT_SIDE:
        raise ValueError(f"{name}: [{rows}, {cols}]: sides up to {MAX_SIDE}, the shorter one up to {MAX_SHORT_SIDE}")


def _run(entry, table, count, device, *args):
    """One call over `count` matrix stacks; workspace from the current stream's pool of the tensors' device."""
    if device.index != _lib.current_device():
        with torch.cuda.device(device):
            return _run(entry, table, count, device, *args)
    fields = (ctypes.c_longlong * len(table))(*table)
    size = _lib.size_call("agb_ns_workspace_bytes", fields, count)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    _lib.call(entry, fields, count, *args, work.data_ptr(), size, _lib.stream())


def _pointer(t):
    if not t.is_cuda:
        _lib.ptr(t)        # (refuses host tensors)
    return t.data_ptr()


@torch.no_grad()
def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The matrices x [..., rows, cols] with their singular values brought near one: X = x / (|x|_F + eps), then `steps` times
    X <- a X + (b G + c G G) X with G = X X^T.

    x: fp32, bf16 or fp16, one tensor or a sequence of tensors of any shapes (handled together, which is what the small ones
    need); rows may be strided.  coefficients: (a, b, c), or a triple for each step; such that singular values from [0, 1] stay
    in a range where sigma^2 and b sigma^2 + c sigma^4 are below 7.  The products are accumulated in fp32 from operands of 22
    bits and more; the result has x's type, rounded once.  A zero matrix stays zero; a matrix with a NaN or an infinity is NaN
    throughout.  Not differentiable."""
    many = isinstance(x, (list, tuple))
    xs = list(x) if many else [x]
    coef, steps = _coefficients(coefficients, steps)
    if not eps >= 0:
        raise ValueError(f"orthogonalize: eps {eps}")
    outs, table, count, keep = [], [], 0, []
    for t in xs:
        if t.dim() < 2:
            raise ValueError(f"orthogonalize: matrices [..., rows, cols], got {list(t.shape)}")
        if t.dtype not in TYPES:
            raise _lib.AgbError(f"orthogonalize: fp32, bf16 or fp16 matrices (got {t.dtype})")
        if t.requires_grad:
            raise ValueError("orthogonalize: not differentiable: pass a detached tensor")
        if t.device != xs[0].device:
            raise _lib.AgbError(f"orthogonalize: matrices on {xs[0].device} and {t.device} in one call")
        rows, cols = t.shape[-2:]
        _check_side("orthogonalize", rows, cols)
        _pointer(t)
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        outs.append(out)
        if not t.numel():
            continue
        v = t.reshape(-1, rows, cols)
        if (cols > 1 and v.stride(2) != 1) or (rows > 1 and v.stride(1) < cols):
            v = v.contiguous()
        keep.append(v)
        table += [v.data_ptr(), out.data_ptr(), 0, rows, cols, v.shape[0], v.stride(1) if rows > 1 else cols, v.stride(0), cols,
                  rows * cols, TYPES[t.dtype]]
        count += 1
    if count:
        _run("agb_orthogonalize", table, count, xs[0].device, steps, coef, float(eps))
    return outs if many else outs[0]


def matrix_shape(p):
    """(rows, cols) of a parameter as a matrix: leading axes merged (a convolution kernel [offsets, Cin, Cout] maps offsets * Cin
    inputs to Cout outputs); None where that leaves no matrix (vectors, and single rows or columns such as biases [1, C])."""
    if p.dim() < 2:
        return None
    cols = p.shape[-1]
    rows = p.numel() // cols if cols else 0
    return (rows, cols) if rows > 1 and cols > 1 else None


def adjust_factor(adjust, rows, cols):
    """Factor of the learning rate: "rms": 0.2 sqrt(longer side), which gives an update of that shape the root mean square of
    about 0.2; "none": 1."""
    if adjust == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    if adjust in (None, "none"):
        return 1.0
    raise ValueError(f"adjust '{adjust}': choose rms or none")


@torch.no_grad()
def muon_update(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
                eps=1e-7, adjust="rms", clip_value=None):
    """One step of a list of weight matrices, in place:
        m <- momentum m + (1 - momentum) g;   u = (1 - momentum) g + momentum m  (nesterov)  or  m
        p <- (1 - lr weight_decay) p - lr adjust orthogonalize(u)

    params, momenta: fp32, contiguous, each taken as a matrix (``matrix_shape``); grads: fp32, bf16 or fp16 of the same shapes,
    left as they are; clip_value limits each of their elements first.  All matrices go through the same launches.  A parameter or a
    momentum may not be listed twice, nor be a gradient.  In a captured graph lr and the list are fixed; what a model keeps of its
    weights in other forms is renewed by sparse_ops.bump_weight_epoch() after a replay."""
    _update(params, grads, momenta, lr, 1.0 - lr * weight_decay, momentum, nesterov, steps, coefficients, eps, adjust, clip_value)


def _update(params, grads, momenta, lr, decay, momentum, nesterov, steps, coefficients, eps, adjust, clip_value):
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"muon_update: {len(params)} parameters, {len(grads)} gradients, {len(momenta)} momenta")
    coef, steps = _coefficients(coefficients, steps)
    if not 0 <= momentum < 1:
        raise ValueError(f"muon_update: momentum {momentum}")
    if clip_value is not None and not clip_value > 0:
        raise ValueError(f"muon_update: clip_value {clip_value}")
    if not eps >= 0:
        raise ValueError(f"muon_update: eps {eps}")
    table, sizes, keep, seen = [], [], [], set()
    for p, g, m in zip(params, grads, momenta):
        shape = matrix_shape(p)
        if shape is None:
            raise ValueError(f"muon_update: {list(p.shape)} is no matrix")
        if g.shape != p.shape or m.shape != p.shape:
            raise ValueError(f"muon_update: parameter {list(p.shape)}, gradient {list(g.shape)}, momentum {list(m.shape)}")
        if p.dtype != torch.float32 or m.dtype != torch.float32 or g.dtype not in TYPES:
            raise _lib.AgbError(f"muon_update: fp32 parameters and momenta, fp32 / bf16 / fp16 gradients (got {p.dtype}, "
                                f"{m.dtype}, {g.dtype})")
        if not (p.is_contiguous() and m.is_contiguous()):
            raise _lib.AgbError("muon_update: parameters and momenta are contiguous")
        if not p.device == g.device == m.device == params[0].device:
            raise _lib.AgbError("muon_update: tensors on several devices in one call")
        _check_side("muon_update", *shape)
        rows, cols = shape
        g = g.contiguous()
        keep.append(g)
        pp, mp = _pointer(p), _pointer(m)
        if pp in seen or mp in seen or pp == mp:
            raise ValueError("muon_update: a tensor is listed twice")
        seen.update((pp, mp))
        table += [g.data_ptr(), pp, mp, rows, cols, 1, cols, rows * cols, cols, rows * cols, TYPES[g.dtype]]
        sizes.append(shape)
    if any(f in seen for f in table[0::_FIELDS]):
        raise ValueError("muon_update: a gradient is a parameter or a momentum of the list")
    steplen = (ctypes.c_float * max(1, len(params)))(*(lr * adjust_factor(adjust, r, c) for r, c in sizes))
    if params:
        _run("agb_muon_update", table, len(params), params[0].device, steps, coef, float(eps), steplen,
             float(decay), float(momentum), int(bool(nesterov)), float(clip_value or 0.0))
        # (the parameters were rewritten through raw pointers: torch's version counters did not move)
        from .sparse_ops import bump_weight_epoch
        bump_weight_epoch()
