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
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .. import _lib
from .fm_scan import _DTYPES, _dtype_code, _on_gpu, _ptr, _raw, _require

__all__ = ["fm_conv", "fm_conv_step", "FM_Conv", "fm_selective_scan", "fm_selective_step", "FM_Selective"]


# The checks come as one condition for the usual case and a function that says what is wrong: a call for one
# token takes a few microseconds, and messages that are put together beforehand would double that.

def _gpu(name, t):
    if not t.is_cuda:
        _on_gpu(name, t, t.device)


def _wrong(name, t, shape, dtypes, dev, strides):
    _require(t.device == dev, f"{name} is on {t.device}, expected {dev}")
    _require(t.dtype in dtypes, f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    _require(t.shape == shape, f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    _require(False, f"{name} must {strides}, got strides {t.stride()}")


def _sequence(name, t, shape, dtype, dev):
    """A (B, D, L) input, or one like it: any strides but the last axis', which is 1."""
    if t.dtype != dtype or t.shape != shape or t.device != dev or (t.stride(-1) != 1 and shape[-1] > 1):
        _wrong(name, t, shape, (dtype,), dev, "have a time stride of 1")


def _dense(name, t, shape, dtype, dev):
    if t.dtype != dtype or t.shape != shape or t.device != dev or not t.is_contiguous():
        _wrong(name, t, shape, (dtype,), dev, "be contiguous")


def _parameter(name, t, shape, dtype, dev, narrow):
    """A parameter in float32 or in the inputs' type; `narrow` is the flag for the latter."""
    own = t.dtype
    if (own != torch.float32 and own != dtype) or t.shape != shape or t.device != dev or not t.is_contiguous():
        _wrong(name, t, shape, (torch.float32, dtype), dev, "be contiguous")
    return 0 if own == torch.float32 else narrow


def _type_of(t):
    code = _DTYPES.get(t.dtype)
    return _dtype_code(t) if code is None else code


def _slots(slots, B, dev):
    """The flag for the slots' type."""
    if slots is None:
        return 0
    wide = slots.dtype == torch.int64
    if (not wide and slots.dtype != torch.int32) or slots.shape != (B,) or slots.device != dev or not slots.is_contiguous():
        _wrong("slots", slots, (B,), (torch.int32, torch.int64), dev, "be contiguous")
    return _lib.SELECTIVE_SLOTS_64 if wide else 0


def _pool(state, state_out, slots, B, D, each, dtype, dev):
    """State pool of a single-token call, (S, D, each), and where the new states go."""
    _require(state.dim() == 3, "state must be (S, channels, values)")
    S = state.shape[0]
    _dense("state", state, (S, D, each), dtype, dev)
    if slots is None and S != B:
        _require(False, f"without slots the state must hold {B} rows, got {S}")
    new = state
    if state_out is not None:
        _dense("state_out", state_out, (S, D, each), dtype, dev)
        new = state_out
    if not new.is_inference():
        increment_version(new)  # a graph that holds the states as they were refuses its backward pass
    return new


def _call(dev, entry, *args):
    """An entry point of the library on `dev` and its current stream."""
    index = dev.index
    if torch.cuda.current_device() == index:
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _dual(tensors):
    """Whether one of them carries a tangent of forward-mode differentiation."""
    if forward_ad._current_level < 0:  # (an attribute, where unpack_dual would cost a microsecond a tensor)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _once(gradients, ctx, *grads):
    """A node's gradients, differentiable once: the guard against a second time is only put up where one could follow.
    (This runs on autograd's own thread, where every Python object that the forward call has just used is in another
    core's cache: the arguments are not checked a second time either.)"""
    if _dual(grads):
        _require(False, "the gradient has no forward-mode derivative, but the output's gradient carries a tangent")
    return once_differentiable(gradients)(ctx, *grads) if torch.is_grad_enabled() else gradients(ctx, *grads)


def _tracked(*tensors):
    """Whether autograd follows a call with these arguments: backwards, or forwards, where a dual tensor requires no gradient
    and the node raises (it has no forward derivative)."""
    # (one call for all of them: a loop over a step's ten takes a microsecond more)
    if torch.is_grad_enabled() and torch._C._any_requires_grad(*tensors):
        return True
    return forward_ad._current_level >= 0 and _dual(tensors)


def _no_derivative(call):
    """For a call that autograd follows and that has no derivative: detached quietly, the gradient would be lost."""
    _require(False, f"{call} is not differentiable, but a tensor it was given requires a gradient or carries a tangent: "
                    "call it under torch.no_grad(), or detach the tensor")


def _conv_check(inputs, weight, bias, initial_state, lengths, silu):
    _gpu("inputs", inputs)
    if inputs.dim() != 3 or weight.dim() != 2:
        _require(False, "inputs must be (B, D, L) and weight (D, W)")
    shape, dtype, dev = inputs.shape, inputs.dtype, inputs.device
    B, D, L = shape
    W = weight.shape[1]
    if not 2 <= W <= 4:
        _require(False, f"weight must have 2, 3 or 4 taps, got {W}")
    _sequence("inputs", inputs, shape, dtype, dev)
    code = _type_of(inputs)
    flags = _parameter("weight", weight, (D, W), dtype, dev, _lib.SELECTIVE_NARROW_WEIGHT)
    if silu:
        flags |= _lib.SELECTIVE_SILU
    if bias is not None:
        flags |= _parameter("bias", bias, (D,), dtype, dev, _lib.SELECTIVE_NARROW_BIAS)
    if initial_state is not None:
        _dense("initial_state", initial_state, (B, D, W - 1), dtype, dev)
    if lengths is not None:
        _dense("lengths", lengths, (B,), torch.int32, dev)
    return B, D, L, W, code, flags


def _carried(initial_state, shape, like, dtype):
    """The final state where no step counts anywhere: the initial state, or zeros."""
    return torch.zeros(shape, dtype=dtype, device=like.device) if initial_state is None else initial_state.clone()


def _conv_forward(inputs, weight, bias, initial_state, lengths, silu, return_state):
    """(out, final state or None, the checked sizes)"""
    sizes = _conv_check(inputs, weight, bias, initial_state, lengths, silu)
    B, D, L, W, code, flags = sizes
    out = torch.empty((B, D, L), dtype=inputs.dtype, device=inputs.device)
    if not out.numel():
        return out, _carried(initial_state, (B, D, W - 1), inputs, inputs.dtype) if return_state else None, sizes
    final = torch.empty((B, D, W - 1), dtype=inputs.dtype, device=inputs.device) if return_state else None
    _call(inputs.device, _raw.fmselective_conv_forward, inputs.data_ptr(), inputs.stride(0), inputs.stride(1), weight.data_ptr(),
          _ptr(bias), _ptr(initial_state), _ptr(lengths), out.data_ptr(), _ptr(final), B, D, L, W, code, flags)
    return out, final, sizes


def _conv_backward(inputs, weight, bias, initial_state, lengths, sizes, out_grad, final_grad, want_state):
    B, D, L, W, code, flags = sizes
    dev = inputs.device
    if out_grad is None:
        out_grad = torch.zeros((B, D, L), dtype=inputs.dtype, device=dev)
    elif out_grad.stride(-1) != 1:
        out_grad = out_grad.contiguous()
    _sequence("the output's gradient", out_grad, (B, D, L), inputs.dtype, dev)
    if final_grad is not None:
        final_grad = final_grad.contiguous()
        _dense("the final state's gradient", final_grad, (B, D, W - 1), inputs.dtype, dev)
    if not inputs.numel():
        d_state = None
        if want_state:
            d_state = torch.zeros((B, D, W - 1), dtype=inputs.dtype, device=dev) if final_grad is None else final_grad
        return (torch.zeros_like(inputs), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), d_state)
    d_inputs = torch.empty_like(inputs, memory_format=torch.contiguous_format)
    d_weight = torch.empty_like(weight)
    d_bias = None if bias is None else torch.empty_like(bias)
    d_state = torch.empty((B, D, W - 1), dtype=inputs.dtype, device=dev) if want_state else None
    need = _raw.fmselective_conv_workspace_bytes(B, D, L, W, code)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(dev, _raw.fmselective_conv_backward, inputs.data_ptr(), inputs.stride(0), inputs.stride(1), out_grad.data_ptr(),
          out_grad.stride(0), out_grad.stride(1), weight.data_ptr(), _ptr(bias), _ptr(initial_state), _ptr(final_grad),
          _ptr(lengths), d_inputs.data_ptr(), d_weight.data_ptr(), _ptr(d_bias), _ptr(d_state), B, D, L, W, code, flags,
          workspace.data_ptr(), need)
    return d_inputs, d_weight, d_bias, d_state


class FM_Conv(torch.autograd.Function):
    """out, final_state = FM_Conv.apply(inputs, weight, bias, initial_state, lengths, silu, return_state)

    final_state is None unless asked for. See fm_conv.
    """

    @staticmethod
    def forward(ctx, inputs, weight, bias=None, initial_state=None, lengths=None, silu=True, return_state=False):
        out, final, ctx.sizes = _conv_forward(inputs, weight, bias, initial_state, lengths, silu, return_state)
        ctx.save_for_backward(inputs, weight, bias, initial_state, lengths)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, out_grad, final_grad):
        return _once(_conv_gradients, ctx, out_grad, final_grad)


def _conv_gradients(ctx, out_grad, final_grad):
    if out_grad is None and final_grad is None:
        return (None,) * 7
    grads = _conv_backward(*ctx.saved_tensors, ctx.sizes, out_grad, final_grad, ctx.needs_input_grad[3])
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

    Returns (B, D, L), or that and the final state (B, D, W - 1). Differentiable once, backwards, in everything but lengths.
    """
    if _tracked(inputs, weight, bias, initial_state):
        out, final = FM_Conv.apply(inputs, weight, bias, initial_state, lengths, silu, return_state)
    else:
        out, final, _ = _conv_forward(inputs, weight, bias, initial_state, lengths, silu, return_state)
    return (out, final) if return_state else out


def fm_conv_step(inputs, state, weight, bias=None, slots=None, silu=True, state_out=None):
    """fm_conv for one token of every row; moves the state on by it. Not differentiable: an argument that requires a
    gradient is refused outside torch.no_grad().

    Arguments:
        inputs (B, D): channel stride 1.
        state (S, D, W - 1): pool of states, updated in place.
        slots (B,) int32 or int64: which state a row has; S = B and row b has state b if omitted. A row whose slot
            lies outside [0, S) is skipped: its output is zero and no state is touched. Where a slot is named more
            than once the first row has it and the others are skipped.
        state_out (S, D, W - 1): where the named states are written instead (`state` then stays as it is).

    Returns (B, D).
    """
    _gpu("inputs", inputs)
    if inputs.dim() != 2 or weight.dim() != 2:
        _require(False, "inputs must be (B, D) and weight (D, W)")
    shape, dtype, dev = inputs.shape, inputs.dtype, inputs.device
    B, D = shape
    W = weight.shape[1]
    if not 2 <= W <= 4:
        _require(False, f"weight must have 2, 3 or 4 taps, got {W}")
    _sequence("inputs", inputs, shape, dtype, dev)
    code = _type_of(inputs)
    flags = _parameter("weight", weight, (D, W), dtype, dev, _lib.SELECTIVE_NARROW_WEIGHT) | _slots(slots, B, dev)
    if silu:
        flags |= _lib.SELECTIVE_SILU
    if bias is not None:
        flags |= _parameter("bias", bias, (D,), dtype, dev, _lib.SELECTIVE_NARROW_BIAS)
    if _tracked(inputs, state, weight, bias, state_out):
        _no_derivative("fm_conv_step")
    new = _pool(state, state_out, slots, B, D, W - 1, dtype, dev)
    S = state.shape[0]
    if slots is not None and S == 0:
        return torch.zeros((B, D), dtype=dtype, device=dev)
    out = torch.empty(shape, dtype=dtype, device=dev)
    if B and D:
        _call(dev, _raw.fmselective_conv_step, inputs.data_ptr(), inputs.stride(0), state.data_ptr(), new.data_ptr(),
              weight.data_ptr(), _ptr(bias), _ptr(slots), out.data_ptr(), B, D, W, S, code, flags)
    return out


def _channels(tokens, delta, A, skip, gate, delta_bias, G, softplus):
    """What calls on sequences and for one token check alike: (N, dtype code, flags)."""
    shape, dtype, dev = tokens.shape, tokens.dtype, tokens.device
    D, N = shape[1], A.shape[1]
    _sequence("tokens", tokens, shape, dtype, dev)
    code = _type_of(tokens)
    _sequence("delta", delta, shape, dtype, dev)
    if not 1 <= N <= _lib.SELECTIVE_MAX_STATES:
        _require(False, f"A must have 1 to {_lib.SELECTIVE_MAX_STATES} states, got {N}")
    _dense("A", A, (D, N), torch.float32, dev)
    if G < 1 or D % G:
        _require(False, f"the groups of write must divide the {D} channels, got {G}")
    flags = _lib.SELECTIVE_SOFTPLUS if softplus else 0
    if skip is not None:
        flags |= _parameter("skip", skip, (D,), dtype, dev, _lib.SELECTIVE_NARROW_SKIP)
    if delta_bias is not None:
        flags |= _parameter("delta_bias", delta_bias, (D,), dtype, dev, _lib.SELECTIVE_NARROW_BIAS)
    if gate is not None:
        _sequence("gate", gate, shape, dtype, dev)
    return N, code, flags


def _scan_check(tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths, softplus):
    """Checks the arguments of a call on sequences; ((B, D, L, N, G, dtype code), flags)."""
    _gpu("tokens", tokens)
    if tokens.dim() != 3 or A.dim() != 2 or write.dim() != 4:
        _require(False, "tokens must be (B, D, L), A (D, N), write (B, G, N, L)")
    B, D, L = tokens.shape
    G, dtype, dev = write.shape[1], tokens.dtype, tokens.device
    N, code, flags = _channels(tokens, delta, A, skip, gate, delta_bias, G, softplus)
    _sequence("write", write, (B, G, N, L), dtype, dev)
    _sequence("read", read, (B, G, N, L), dtype, dev)
    if initial_state is not None:
        _dense("initial_state", initial_state, (B, D, N), torch.float32, dev)
    if lengths is not None:
        _dense("lengths", lengths, (B,), torch.int32, dev)
    return (B, D, L, N, G, code), flags


def _scan_packed(sizes, flags, tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths):
    """The arguments as the library takes them."""
    B, D, L, N, G, code = sizes
    z_b, z_d = (0, 0) if gate is None else gate.stride()[:2]
    return _lib.SCAN_INPUTS.pack(
        tokens.data_ptr(), delta.data_ptr(), _at(gate), write.data_ptr(), read.data_ptr(), _at(skip), _at(delta_bias),
        A.data_ptr(), _at(initial_state), _at(lengths), *tokens.stride()[:2], *delta.stride()[:2], z_b, z_d,
        *write.stride()[:3], *read.stride()[:3], B, D, L, N, G, code, flags)


def _at(t):
    return 0 if t is None else t.data_ptr()


def _scan_forward(tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths, softplus, return_state, save):
    """(out, final state or None, the states that backward starts from or None, the checked sizes and flags)"""
    inputs = (tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths)
    checked = sizes, flags = _scan_check(*inputs, softplus)
    B, D, L, N, G, code = sizes
    dev = tokens.device
    out = torch.empty((B, D, L), dtype=tokens.dtype, device=dev)
    if not (B and D and L):
        return out, _carried(initial_state, (B, D, N), tokens, torch.float32) if return_state else None, None, checked
    final = torch.empty((B, D, N), dtype=torch.float32, device=dev) if return_state else None
    marks = None
    if save:
        marks = torch.empty((B, D, -(-L // _lib.SELECTIVE_MARK), N), dtype=torch.float32, device=dev)
    need = _raw.fmselective_scan_workspace_bytes(*sizes, 0)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, _raw.fmselective_scan_forward, _scan_packed(sizes, flags, *inputs), out.data_ptr(), _ptr(final), _ptr(marks),
          _ptr(workspace), need)
    return out, final, marks, checked


def _scan_backward(inputs, checked, marks, out_grad, final_grad, want_state):
    """Gradients in the order of the inputs, None for absent ones."""
    tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths = inputs
    sizes, flags = checked
    B, D, L, N, G, code = sizes
    dev, dtype = tokens.device, tokens.dtype
    if out_grad is None:
        out_grad = torch.zeros((B, D, L), dtype=dtype, device=dev)
    elif out_grad.stride(-1) != 1:
        out_grad = out_grad.contiguous()
    _sequence("the output's gradient", out_grad, (B, D, L), dtype, dev)
    if final_grad is not None:
        final_grad = final_grad.contiguous()
        _dense("the final state's gradient", final_grad, (B, D, N), torch.float32, dev)
    if not (B and D and L):
        d_state = None
        if want_state:
            d_state = torch.zeros((B, D, N), dtype=torch.float32, device=dev) if final_grad is None else final_grad
        zeros = [None if t is None else torch.zeros_like(t) for t in (tokens, delta, A, write, read, skip, gate, delta_bias)]
        return (*zeros, d_state)
    grads = [None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
             for t in (tokens, delta, A, write, read, skip, gate, delta_bias)]
    d_tokens, d_delta, d_A, d_write, d_read, d_skip, d_gate, d_bias = grads
    d_state = torch.empty((B, D, N), dtype=torch.float32, device=dev) if want_state else None
    need = _raw.fmselective_scan_workspace_bytes(*sizes, 1)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    o = _lib.SCAN_GRADS.pack(out_grad.data_ptr(), *out_grad.stride()[:2], _at(final_grad), marks.data_ptr(),
                             d_tokens.data_ptr(), d_delta.data_ptr(), _at(d_gate), d_write.data_ptr(), d_read.data_ptr(),
                             d_A.data_ptr(), _at(d_state), _at(d_skip), _at(d_bias))
    _call(dev, _raw.fmselective_scan_backward, _scan_packed(sizes, flags, *inputs), o, workspace.data_ptr(), need)
    return (*grads, d_state)


class FM_Selective(torch.autograd.Function):
    """out, final_state = FM_Selective.apply(tokens, delta, A, write, read, skip, gate, delta_bias, initial_state,
    lengths, softplus, return_state): fm_selective_scan with write and read (B, G, N, L); final_state is None
    unless asked for."""

    @staticmethod
    def forward(ctx, tokens, delta, A, write, read, skip=None, gate=None, delta_bias=None, initial_state=None, lengths=None,
                softplus=True, return_state=False):
        inputs = (tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths)
        save = any(ctx.needs_input_grad)
        out, final, marks, checked = _scan_forward(*inputs, softplus, return_state, save)
        if save:
            ctx.save_for_backward(*inputs, marks)
            ctx.checked = checked
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, out_grad, final_grad):
        return _once(_scan_gradients, ctx, out_grad, final_grad)


def _scan_gradients(ctx, out_grad, final_grad):
    if out_grad is None and final_grad is None:
        return (None,) * 12
    *inputs, marks = ctx.saved_tensors
    grads = _scan_backward(inputs, ctx.checked, marks, out_grad, final_grad, ctx.needs_input_grad[8])
    return (*grads, None, None, None)


def fm_selective_scan(tokens, delta, A, write, read, skip=None, gate=None, delta_bias=None, initial_state=None, lengths=None,
                      softplus=True, return_state=False):
    """Selective state space scan: N states a channel, whose decay depends on channel, state and step.

        dt = softplus(delta + delta_bias)
        h[b, d, n] <- exp(dt * A[d, n]) * h[b, d, n] + dt * tokens[b, d, t] * write[b, g, n, t]
        out[b, d, t] = (sum_n read[b, g, n, t] * h[b, d, n] + skip[d] * tokens[b, d, t]) * silu(gate[b, d, t])

    Arguments:
        tokens, delta (B, D, L) and gate (B, D, L) or None: one dtype, time stride 1, any batch and channel stride.
        A (D, N): float32, negative in a model whose states decay (minus infinity: the state forgets at once); N up to 256. Where
            a state grows, its growth over the call's steps must be finite in float32, even while the state itself is zero.
        write, read (B, G, N, L), or (B, N, L) for one group: of the tokens' dtype, time stride 1; channel d is in
            group g = d // (D / G).
        skip, delta_bias (D,): float32 or the tokens' dtype; absent is zero.
        initial_state (B, D, N): float32; zeros if omitted.
        lengths (B,) int32: the steps that count of each row of a padded batch (clamped to [0, L]); nothing is read
            beyond them, the output is zero there, and the final state is that after the last step that counts.
        softplus: apply it to delta + delta_bias, else the sum is dt itself.
        return_state: also return the state after the last step that counts, float32 (B, D, N).

    Returns (B, D, L) of the tokens' dtype, or that and the final state. Differentiable once, backwards, in everything but
    lengths. Where a gradient is wanted the forward call keeps a state every 128 steps, B D L N / 32 bytes, and the backward call
    holds partial sums of B D L N / 2 bytes while it runs (269 MB at (8, 2048, 2048), N = 16): more where groups are not multiples
    of 16 channels or L not one of 128, which count as if they were.
    """
    if write.dim() == 3 and read.dim() == 3:
        write, read = write.unsqueeze(1), read.unsqueeze(1)
    inputs = (tokens, delta, A, write, read, skip, gate, delta_bias, initial_state, lengths)
    if _tracked(*inputs):
        out, final = FM_Selective.apply(*inputs, softplus, return_state)
    else:
        out, final, _, _ = _scan_forward(*inputs, softplus, return_state, False)
    return (out, final) if return_state else out


def fm_selective_step(tokens, state, delta, A, write, read, skip=None, gate=None, delta_bias=None, slots=None, softplus=True,
                      state_out=None):
    """fm_selective_scan for one token of every row; moves the state on by it. Not differentiable: an argument that requires a
    gradient is refused outside torch.no_grad().

    Arguments:
        tokens, delta, gate (B, D): channel stride 1. write, read (B, G, N) or (B, N): state stride 1.
        state (S, D, N): float32 pool of states, updated in place.
        slots (B,) int32 or int64: which state a row has; S = B and row b has state b if omitted. A row whose slot
            lies outside [0, S) is skipped: its output is zero and no state is touched. Where a slot is named more
            than once the first row has it and the others are skipped.
        state_out (S, D, N): where the named states are written instead (`state` then stays as it is: the way back
            when a token is not accepted).

    Returns (B, D) of the tokens' dtype.
    """
    if write.dim() == 2 and read.dim() == 2:
        write, read = write.unsqueeze(1), read.unsqueeze(1)
    _gpu("tokens", tokens)
    if tokens.dim() != 2 or A.dim() != 2 or write.dim() != 3:
        _require(False, "tokens must be (B, D), A (D, N), write (B, G, N)")
    shape, dtype, dev = tokens.shape, tokens.dtype, tokens.device
    B, D = shape
    G = write.shape[1]
    N, code, flags = _channels(tokens, delta, A, skip, gate, delta_bias, G, softplus)
    _sequence("write", write, (B, G, N), dtype, dev)
    _sequence("read", read, (B, G, N), dtype, dev)
    flags |= _slots(slots, B, dev)
    if _tracked(tokens, state, delta, A, write, read, skip, gate, delta_bias, state_out):
        _no_derivative("fm_selective_step")
    new = _pool(state, state_out, slots, B, D, N, torch.float32, dev)
    S = state.shape[0]
    if slots is not None and S == 0:
        return torch.zeros(shape, dtype=dtype, device=dev)
    out = torch.empty(shape, dtype=dtype, device=dev)
    if B and D:
        packed = _lib.SCAN_INPUTS.pack(
            tokens.data_ptr(), delta.data_ptr(), _at(gate), write.data_ptr(), read.data_ptr(), _at(skip), _at(delta_bias),
            A.data_ptr(), state.data_ptr(), 0, tokens.stride(0), 0, delta.stride(0), 0, 0 if gate is None else gate.stride(0), 0,
            *write.stride(), *read.stride(), B, D, 1, N, G, code, flags)
        _call(dev, _raw.fmselective_scan_step, packed, new.data_ptr(), _ptr(slots), S, out.data_ptr())
    return out
