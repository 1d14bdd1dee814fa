"""Plain implementations of the selective layer's operators in float64 on the CPU, one step of time after the other,
and the comparison that the tests make. Gradients come from the formulas; a test holds them to differences.

Tolerances. A result is held to |got - ref| <= eps / 2 |ref| + c 2^-24 mag + tiny: one rounding to the result's type
(half a step of it, torch.finfo(t).eps / 2 of the value), and c roundings to float32 of terms whose absolute values
add up to `mag`. `mag` is computed here, beside the result, with every term's absolute value; each test derives its c
from the number of float32 operations that a term passes through.
"""
import torch

F32 = 2.0 ** -24
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}  # half the smallest subnormal


def close(got, ref, mag, c, what=""):
    """`got` (any dtype, any device) against `ref` in float64 with magnitudes `mag`, c float32 roundings."""
    t = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)}, expected {tuple(ref.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bound = torch.finfo(t).eps / 2 * ref.abs() + c * F32 * mag * (1 + torch.finfo(t).eps) + TINY[t]
    over = (got - ref).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, (f"{what}: off by {(got - ref).abs().max().item():.3g}, over the bound by {worst:.3g} at "
                        f"{tuple(int(i) for i in (over == over.max()).nonzero()[0])}")


def f64(t):
    return None if t is None else t.detach().cpu().double()


def conv(x, w, bias=None, state=None, lengths=None, silu=True, dy=None, dfinal=None):
    """Results and magnitudes: {name: (value, magnitude)}."""
    x, w, bias, state, dy, dfinal = (f64(v) for v in (x, w, bias, state, dy, dfinal))
    (B, D, L), W = x.shape, w.shape[1]
    ends = [L] * B if lengths is None else [max(0, min(L, int(n))) for n in lengths.tolist()]
    live = torch.zeros(B, 1, L, dtype=torch.float64)
    for b, n in enumerate(ends):
        live[b, :, :n] = 1
    before = torch.zeros(B, D, W - 1, dtype=torch.float64) if state is None else state
    xs = torch.cat([before, torch.where(live > 0, x, 0.0)], -1)
    pre = torch.zeros(B, D, L, dtype=torch.float64)
    mag = torch.zeros_like(pre)
    for j in range(W):
        pre += w[:, j, None] * xs[..., j:j + L]
        mag += (w[:, j, None] * xs[..., j:j + L]).abs()
    if bias is not None:
        pre += bias[:, None]
        mag += bias.abs()[:, None]
    sig = torch.sigmoid(pre)
    y = pre * sig if silu else pre
    final = torch.stack([xs[b, :, n:n + W - 1] for b, n in enumerate(ends)])
    out = {"y": (y * live, mag * live), "final": (final, final.abs())}
    if dy is None and dfinal is None:
        return out
    dy = torch.zeros_like(x) if dy is None else torch.where(live > 0, dy, 0.0)
    slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
    dpre = dy * slope
    # the slope moves with the sum (|second derivative| <= 1/2), and is itself a few operations on it
    dmag = dy.abs() * (slope.abs() + 0.5 * mag + pre.abs()) if silu else dy.abs()
    dxs, gmag = torch.zeros_like(xs), torch.zeros_like(xs)
    dw, wmag = torch.zeros_like(w), torch.zeros_like(w)
    for j in range(W):
        dxs[..., j:j + L] += w[:, j, None] * dpre
        gmag[..., j:j + L] += w[:, j, None].abs() * dmag
        dw[:, j] = (dpre * xs[..., j:j + L]).sum((0, 2))
        wmag[:, j] = (dmag * xs[..., j:j + L].abs()).sum((0, 2))
    if dfinal is not None:
        for b, n in enumerate(ends):
            dxs[b, :, n:n + W - 1] += dfinal[b]
            gmag[b, :, n:n + W - 1] += dfinal[b].abs()
    # (taps of steps that count reach inputs that count, or the state)
    out["dx"] = (dxs[..., W - 1:] * live, gmag[..., W - 1:])
    out["dstate"] = (dxs[..., :W - 1], gmag[..., :W - 1])
    out["dweight"], out["dbias"] = (dw, wmag), (dpre.sum((0, 2)), dmag.sum((0, 2)))
    return out
