"""Root-mean-square norm over the last axis with the residual's addition, on MI355X: the entry of a block around
`fm_memory` or `fm_selective_scan`.

    fm_norm             differentiable, output in the inputs' dtype
    fm_norm_quantized   output in 8 bits (e4m3) with one scale a row, for a product in 8 bits

float32, float16 and bfloat16; statistics and gradient sums in float32. The kernels are in libfmscan_hip.so
(include/fmselective.h); there is no CPU implementation behind them. The reference normalises inside its layer alone
(fm/scan/fm_scan.py:124-127).
"""
from __future__ import annotations

import torch

from .. import _lib
from .fm_scan import _ptr, _raw, _require
from .fm_selective import _call, _dense, _gpu, _no_derivative, _once, _parameter, _tracked, _type_of

__all__ = ["fm_norm", "fm_norm_quantized", "FM_Norm"]


def _check(inputs, weight, residual, eps):
    """(rows, D, dtype code, flags)"""
    _gpu("inputs", inputs)
    if inputs.dim() < 1 or weight.dim() != 1:
        _require(False, "inputs must be (..., D) and weight (D,)")
    shape, dtype, dev = inputs.shape, inputs.dtype, inputs.device
    D = shape[-1]
    code = _type_of(inputs)
    if D > _lib.SELECTIVE_MAX_NORM:
        _require(False, f"the last axis must have at most {_lib.SELECTIVE_MAX_NORM} elements, got {D}")
    if not eps >= 0:
        _require(False, f"eps must be >= 0, got {eps}")
    _dense("inputs", inputs, shape, dtype, dev)
    flags = _parameter("weight", weight, (D,), dtype, dev, _lib.SELECTIVE_NARROW_WEIGHT)
    if residual is not None:
        _dense("residual", residual, shape, dtype, dev)
    return inputs.numel() // D if D else 0, D, code, flags


def _forward(inputs, weight, residual, eps, save=False, quantized=False):
    """(out, residual_out or None, inv_rms or None, scales or None, the checked sizes)"""
    sizes = rows, D, code, flags = _check(inputs, weight, residual, eps)
    dev, shape = inputs.device, inputs.shape
    out = torch.empty(shape, dtype=torch.float8_e4m3fn if quantized else inputs.dtype, device=dev)
    stream_out = None if residual is None else torch.empty(shape, dtype=inputs.dtype, device=dev)
    inv_rms = torch.empty(rows, dtype=torch.float32, device=dev) if save else None
    scales = torch.empty(shape[:-1], dtype=torch.float32, device=dev) if quantized else None
    if rows:
        _call(dev, _raw.fmselective_norm_forward, inputs.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(stream_out),
              out.data_ptr(), _ptr(scales), _ptr(inv_rms), rows, D, code, flags, float(eps))
    elif quantized:
        scales.zero_()
    return out, stream_out, inv_rms, scales, sizes


class FM_Norm(torch.autograd.Function):
    """out, residual_out = FM_Norm.apply(inputs, weight, residual, eps); residual_out is None without a residual."""

    @staticmethod
    def forward(ctx, inputs, weight, residual=None, eps=1e-6):
        save = any(ctx.needs_input_grad)
        out, stream_out, inv_rms, _, ctx.sizes = _forward(inputs, weight, residual, eps, save=save)
        if save:
            ctx.save_for_backward(inputs if residual is None else stream_out, weight, inv_rms)
        ctx.set_materialize_grads(False)
        return out, stream_out

    @staticmethod
    def backward(ctx, out_grad, residual_grad):
        return _once(_norm_gradients, ctx, out_grad, residual_grad)


def _norm_gradients(ctx, out_grad, residual_grad):
    if out_grad is None and residual_grad is None:
        return None, None, None, None
    stream_in, weight, inv_rms = ctx.saved_tensors
    if out_grad is None:  # nothing goes through the norm
        return residual_grad, torch.zeros_like(weight), residual_grad, None
    rows, D, code, flags = ctx.sizes
    dev = stream_in.device
    grad, d_weight = torch.empty_like(stream_in), torch.empty_like(weight)
    if not rows:
        return grad, d_weight.zero_(), grad, None
    out_grad = out_grad.contiguous()
    residual_grad = None if residual_grad is None else residual_grad.contiguous()
    need = _raw.fmselective_norm_workspace_bytes(rows, D, code)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(dev, _raw.fmselective_norm_backward, out_grad.data_ptr(), _ptr(residual_grad), stream_in.data_ptr(),
          weight.data_ptr(), inv_rms.data_ptr(), grad.data_ptr(), d_weight.data_ptr(), rows, D, code, flags,
          workspace.data_ptr(), need)
    return grad, d_weight, grad if ctx.needs_input_grad[2] else None, None


def fm_norm(inputs, weight, residual=None, eps=1e-6):
    """Root-mean-square norm of inputs + residual over the last axis, and the sum itself.

        r = inputs + residual (in the inputs' dtype),  out = r / sqrt(mean(r ** 2) + eps) * weight

    Arguments:
        inputs, residual (..., D): contiguous, one dtype; residual may be omitted (r is inputs then). D up to 16384.
        weight (D,): float32 or the inputs' dtype.

    Squares are summed in float32. With eps = 0 a row whose mean square is zero there (zeros, or a root mean square below
    2^-75) gives zeros, and nothing goes back through its norm; the same holds for a row of finite values whose sum of squares
    is infinite there (from 2^128 on).

    Returns (out (..., D), r (..., D)): r is the residual of the next block. What the norm sees is r as it is
    stored, rounded. Differentiable once, backwards, in inputs, weight and residual.
    """
    if _tracked(inputs, weight, residual):
        out, stream_out = FM_Norm.apply(inputs, weight, residual, eps)
    else:
        out, stream_out, _, _, _ = _forward(inputs, weight, residual, eps)
    return out, (inputs if residual is None else stream_out)


def fm_norm_quantized(inputs, weight, residual=None, eps=1e-6):
    """fm_norm with its output in 8 bits, one scale a row. Not differentiable: an argument that requires a gradient is refused
    outside torch.no_grad().

    Returns (values (..., D) torch.float8_e4m3fn, scales (...) float32, r (..., D)): out is values * scales, scales are
    max |out| / 448 of each row, values are out / scales in float32, rounded to nearest even (float32's own roundings decide
    where the quotient of unrounded numbers is halfway between two values). A row of zeros, or of values below 2^-100, has
    scale 0; a row with a NaN among its outputs has a NaN scale.
    """
    if _tracked(inputs, weight, residual):
        _no_derivative("fm_norm_quantized")
    out, stream_out, _, scales, _ = _forward(inputs, weight, residual, eps, quantized=True)
    return out, scales, (inputs if residual is None else stream_out)
