"""The operators of a selective state space layer on MI355X, beside the Factorization-Memory scan.

    fm_conv, fm_conv_step              short depthwise convolution along time: sequences, one token
    fm_selective_scan, fm_selective_step
                                       the recurrence whose decay depends on channel, state and input

Sequences are time last, (B, D, L), as in `fm_scan`. The calls on sequences are differentiable; the single-token
forms update their state in place (or write it to `state_out`). float32, float16 and bfloat16; every sum, state and
gradient sum is held in float32. The kernels are in libfmscan_hip.so (include/fmselective.h); there is no CPU
implementation behind them. The reference has no counterpart of these operators.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .fm_scan import _dtype_code, _on_device, _on_gpu, _ptr, _raw, _require

__all__ = ["fm_conv", "fm_conv_step", "FM_Conv"]


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _sequence(name, t, shape, like):
    """A (B, D, L) input: any batch and channel stride, time dense."""
    _on_gpu(name, t, like.device)
    _require(t.dtype == like.dtype, f"{name} has dtype {t.dtype}, expected {like.dtype}")
    _require(t.shape == shape, f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    _require(t.stride(-1) == 1 or t.shape[-1] <= 1, f"{name} must have a time stride of 1, got strides {t.stride()}")


def _dense(name, t, shape, dtype, dev):
    _on_gpu(name, t, dev)
    _require(t.dtype == dtype, f"{name} has dtype {t.dtype}, expected {dtype}")
    _require(t.shape == shape, f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    _require(t.is_contiguous(), f"{name} must be contiguous")


def _parameter(name, t, shape, like, narrow):
    """A parameter in float32 or in the inputs' type; `narrow` is the flag for the latter."""
    _on_gpu(name, t, like.device)
    _require(t.dtype == torch.float32 or t.dtype == like.dtype,
             f"{name} has dtype {t.dtype}, expected torch.float32 or {like.dtype}")
    _require(t.shape == shape, f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    _require(t.is_contiguous(), f"{name} must be contiguous")
    return 0 if t.dtype == torch.float32 else narrow


def _lengths(lengths, B, dev):
    if lengths is not None:
        _dense("lengths", lengths, (B,), torch.int32, dev)


def _slots(slots, B, dev):
    """The flag for the slots' type."""
    if slots is None:
        return 0
    _on_gpu("slots", slots, dev)
    _require(slots.dtype in (torch.int32, torch.int64), f"slots has dtype {slots.dtype}, expected int32 or int64")
    _require(slots.shape == (B,) and slots.is_contiguous(), f"slots must be a dense {(B,)}, got {tuple(slots.shape)}")
    return _lib.SELECTIVE_SLOTS_64 if slots.dtype == torch.int64 else 0


def _pool(state, state_out, slots, B, each, dtype, dev):
    """State pool of a single-token call: (S, *each), and where the new states go."""
    _on_gpu("state", state, dev)
    _require(state.dtype == dtype, f"state has dtype {state.dtype}, expected {dtype}")
    _require(state.dim() == 3 and state.shape[1:] == each, f"state must be (S, {each[0]}, {each[1]}), got {tuple(state.shape)}")
    _require(state.is_contiguous(), "state must be contiguous")
    _require(slots is not None or state.shape[0] == B, f"without slots the state must hold {B} rows, got {state.shape[0]}")
    if state_out is None:
        return state
    _dense("state_out", state_out, state.shape, dtype, dev)
    return state_out


def _conv_check(inputs, weight, bias, initial_state, lengths, silu):
    _require(inputs.dim() == 3 and weight.dim() == 2, "inputs must be (B, D, L) and weight (D, W)")
    B, D, L = inputs.shape
    W = weight.shape[1]
    _require(2 <= W <= 4, f"weight must have 2, 3 or 4 taps, got {W}")
    _sequence("inputs", inputs, inputs.shape, inputs)
    code = _dtype_code(inputs)
    flags = (_lib.SELECTIVE_SILU if silu else 0) | _parameter("weight", weight, (D, W), inputs, _lib.SELECTIVE_NARROW_WEIGHT)
    if bias is not None:
        flags |= _parameter("bias", bias, (D,), inputs, _lib.SELECTIVE_NARROW_BIAS)
    if initial_state is not None:
        _dense("initial_state", initial_state, (B, D, W - 1), inputs.dtype, inputs.device)
    _lengths(lengths, B, inputs.device)
    return B, D, L, W, code, flags


def _carried(initial_state, shape, like, dtype):
    """The final state where no step counts anywhere: the initial state, or zeros."""
    return torch.zeros(shape, dtype=dtype, device=like.device) if initial_state is None else initial_state.clone()


def _conv_forward(inputs, weight, bias, initial_state, lengths, silu, return_state):
    B, D, L, W, code, flags = _conv_check(inputs, weight, bias, initial_state, lengths, silu)
    out = torch.empty((B, D, L), dtype=inputs.dtype, device=inputs.device)
    if not out.numel():
        return out, _carried(initial_state, (B, D, W - 1), inputs, inputs.dtype) if return_state else None
    final = torch.empty((B, D, W - 1), dtype=inputs.dtype, device=inputs.device) if return_state else None
    with _on_device(inputs.device):
        _lib.check(_raw.fmselective_conv_forward(
            inputs.data_ptr(), inputs.stride(0), inputs.stride(1), weight.data_ptr(), _ptr(bias), _ptr(initial_state),
            _ptr(lengths), out.data_ptr(), _ptr(final), B, D, L, W, code, flags, _stream(inputs.device)))
    return out, final


def _conv_backward(inputs, weight, bias, initial_state, lengths, silu, out_grad, final_grad, want_state):
    B, D, L, W, code, flags = _conv_check(inputs, weight, bias, initial_state, lengths, silu)
    dev = inputs.device
    if out_grad is None:
        out_grad = torch.zeros((B, D, L), dtype=inputs.dtype, device=dev)
    elif out_grad.stride(-1) != 1:
        out_grad = out_grad.contiguous()
    _sequence("the output's gradient", out_grad, (B, D, L), inputs)
    if final_grad is not None:
        final_grad = final_grad.contiguous()
        _dense("the final state's gradient", final_grad, (B, D, W - 1), inputs.dtype, dev)
    if not inputs.numel():
        d_state = None
        if want_state:
            d_state = torch.zeros((B, D, W - 1), dtype=inputs.dtype, device=dev) if final_grad is None else final_grad
        return (torch.zeros_like(inputs), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), d_state)
    d_inputs = torch.empty((B, D, L), dtype=inputs.dtype, device=dev)
    d_weight = torch.empty_like(weight)
    d_bias = None if bias is None else torch.empty_like(bias)
    d_state = torch.empty((B, D, W - 1), dtype=inputs.dtype, device=dev) if want_state else None
    need = _raw.fmselective_conv_workspace_bytes(B, D, L, W, code)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    with _on_device(dev):
        _lib.check(_raw.fmselective_conv_backward(
            inputs.data_ptr(), inputs.stride(0), inputs.stride(1), out_grad.data_ptr(), out_grad.stride(0),
            out_grad.stride(1), weight.data_ptr(), _ptr(bias), _ptr(initial_state), _ptr(final_grad), _ptr(lengths),
            d_inputs.data_ptr(), d_weight.data_ptr(), _ptr(d_bias), _ptr(d_state), B, D, L, W, code, flags,
            workspace.data_ptr(), need, _stream(dev)))
    return d_inputs, d_weight, d_bias, d_state


class FM_Conv(torch.autograd.Function):
    """out, final_state = FM_Conv.apply(inputs, weight, bias, initial_state, lengths, silu, return_state)

    final_state is None unless asked for. See fm_conv.
    """

    @staticmethod
    def forward(ctx, inputs, weight, bias=None, initial_state=None, lengths=None, silu=True, return_state=False):
        ctx.save_for_backward(inputs, weight, bias, initial_state, lengths)
        ctx.silu = bool(silu)
        ctx.set_materialize_grads(False)
        return _conv_forward(inputs, weight, bias, initial_state, lengths, silu, return_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, out_grad, final_grad):
        inputs, weight, bias, initial_state, lengths = ctx.saved_tensors
        if out_grad is None and final_grad is None:
            return (None,) * 7
        grads = _conv_backward(inputs, weight, bias, initial_state, lengths, ctx.silu, out_grad, final_grad,
                               ctx.needs_input_grad[3])
        return (*grads, None, None, None)


def fm_conv(inputs, weight, bias=None, initial_state=None, lengths=None, silu=True, return_state=False):
    """Short causal depthwise convolution along time, with the activation that follows it.

        out[b, d, t] = act(bias[d] + sum_j weight[d, j] * inputs[b, d, t - W + 1 + j])

    Arguments:
        inputs (B, D, L): time stride 1, any batch and channel stride.
        weight (D, W), W = 2, 3 or 4, and bias (D,): float32 or the inputs' dtype.
        initial_state (B, D, W - 1): the inputs before the first, oldest first; zeros if omitted.
        lengths (B,) int32: the steps that count of each row of a padded batch (clamped to [0, L]); the output is
            zero beyond them, and nothing is read there.
        silu: out = s * sigmoid(s) of the sum s, else the sum itself.
        return_state: also return the last W - 1 inputs that count, the state that continues the sequence.

    Returns (B, D, L), or that and the final state (B, D, W - 1). Differentiable once, in everything but lengths.
    """
    out, final = FM_Conv.apply(inputs, weight, bias, initial_state, lengths, silu, return_state)
    return (out, final) if return_state else out


def fm_conv_step(inputs, state, weight, bias=None, slots=None, silu=True, state_out=None):
    """fm_conv for one token of every row; moves the state on by it. Not differentiable.

    Arguments:
        inputs (B, D): channel stride 1.
        state (S, D, W - 1): pool of states, updated in place.
        slots (B,) int32 or int64: which state a row has; S = B and row b has state b if omitted. A row whose slot
            lies outside [0, S) is skipped: its output is zero and no state is touched. Where a slot is named more
            than once the first row has it and the others are skipped.
        state_out (S, D, W - 1): where the named states are written instead (`state` then stays as it is).

    Returns (B, D).
    """
    _require(inputs.dim() == 2 and weight.dim() == 2, "inputs must be (B, D) and weight (D, W)")
    B, D = inputs.shape
    W = weight.shape[1]
    dev = inputs.device
    _require(2 <= W <= 4, f"weight must have 2, 3 or 4 taps, got {W}")
    _sequence("inputs", inputs, inputs.shape, inputs)
    code = _dtype_code(inputs)
    flags = (_lib.SELECTIVE_SILU if silu else 0) | _parameter("weight", weight, (D, W), inputs, _lib.SELECTIVE_NARROW_WEIGHT)
    if bias is not None:
        flags |= _parameter("bias", bias, (D,), inputs, _lib.SELECTIVE_NARROW_BIAS)
    new = _pool(state, state_out, slots, B, (D, W - 1), inputs.dtype, dev)
    flags |= _slots(slots, B, dev)
    if slots is not None and state.shape[0] == 0:
        return torch.zeros((B, D), dtype=inputs.dtype, device=dev)
    out = torch.empty((B, D), dtype=inputs.dtype, device=dev)
    if out.numel():
        with _on_device(dev):
            _lib.check(_raw.fmselective_conv_step(
                inputs.data_ptr(), inputs.stride(0), state.data_ptr(), new.data_ptr(), weight.data_ptr(), _ptr(bias),
                _ptr(slots), out.data_ptr(), B, D, W, state.shape[0], code, flags, _stream(dev)))
    return out
