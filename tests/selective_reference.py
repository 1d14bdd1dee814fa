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


def scan(u, delta, A, write, read, skip=None, gate=None, bias=None, state=None, lengths=None, softplus=True, dy=None,
         dfinal=None):
    """Results and magnitudes of the selective scan: {name: (value, magnitude)}; write, read (B, G, N, L).

    A state's magnitude runs through the same recurrence with every term's absolute value, and with each step's
    decay counted with the relative error that float32 leaves in its exponent: a few roundings of dt A. `roundings`
    of a state is that sum, in units of one rounding of one term; see test_gpu_selective.py for the factors.
    """
    u, delta, A, write, read, skip, gate, bias, state, dy, dfinal = (
        f64(v) for v in (u, delta, A, write, read, skip, gate, bias, state, dy, dfinal))
    (B, D, L), (_, G, N, _) = u.shape, write.shape
    ends = [L] * B if lengths is None else [max(0, min(L, int(n))) for n in lengths.tolist()]
    live = torch.zeros(B, 1, L, dtype=torch.float64)
    for b, n in enumerate(ends):
        live[b, :, :n] = 1
    mask = lambda v: torch.where(live.reshape(B, *[1] * (v.dim() - 2), L) > 0, v, 0.0)  # noqa: E731
    u, delta, write, read = (mask(v) for v in (u, delta, write, read))
    gate = None if gate is None else mask(gate)
    pre = delta if bias is None else delta + bias[:, None]
    dt = mask(torch.nn.functional.softplus(pre, threshold=100) if softplus else pre)
    write, read = (v.repeat_interleave(D // G, 1) for v in (write, read))  # (B, D, N, L)
    h = torch.zeros(B, D, N, dtype=torch.float64) if state is None else state
    h0 = h
    mag = h.abs()
    hs, ms, ys, ymags = [], [], [], []
    for t in range(L):
        x = dt[..., t, None] * A
        a = torch.exp(x)
        b = (dt[..., t] * u[..., t])[..., None] * write[..., t]
        # a new term, and what the decay's own error does to the old state: (2 |x| + 2) of a rounding, and one a step
        mag = a * mag + b.abs() + (2 * x.abs() + 3) * a * h.abs()
        h = a * h + b
        hs.append(h), ms.append(mag)
        ys.append((h * read[..., t]).sum(-1)), ymags.append((mag * read[..., t].abs()).sum(-1))
    y, ymag = (torch.stack(v, -1) if L else torch.zeros(B, D, 0, dtype=torch.float64) for v in (ys, ymags))
    if skip is not None:
        y = y + skip[:, None] * u
        ymag = ymag + (skip[:, None] * u).abs()
    sig = None if gate is None else torch.sigmoid(gate)
    act = torch.ones_like(u) if gate is None else gate * sig
    out = {"y": (mask(y * act), mask(ymag * act.abs() + (y * act).abs() * (1 + (gate.abs() if gate is not None else 0)))),
           "final": (h, mag)}
    if dy is None and dfinal is None:
        return out
    dy = torch.zeros_like(u) if dy is None else mask(dy)
    g = dy * act
    grow = 1 if gate is None else 3 + gate.abs()  # what the gate's own operations add to a term of g
    carry = torch.zeros_like(h) if dfinal is None else dfinal
    cmag = carry.abs()
    new = {k: torch.zeros_like(v) for k, v in (("du", u), ("ddt", u), ("dwrite", write), ("dread", write))}
    mags = {k: torch.zeros_like(v) for k, v in new.items()}
    dA, dAmag = torch.zeros(B, D, N, dtype=torch.float64), torch.zeros(B, D, N, dtype=torch.float64)
    for t in reversed(range(L)):
        x = dt[..., t, None] * A
        a, gt, dtt, ut = torch.exp(x), g[..., t, None], dt[..., t], u[..., t]
        gm = gt.abs() * (grow if isinstance(grow, int) else grow[..., t, None])
        dh = gt * read[..., t] + carry
        dm = gm * read[..., t].abs() + cmag
        new["dread"][..., t], mags["dread"][..., t] = gt * hs[t], gm * ms[t]
        new["dwrite"][..., t] = dh * (dtt * ut)[..., None]
        mags["dwrite"][..., t] = dm * (dtt * ut).abs()[..., None]
        before, bm = (hs[t - 1], ms[t - 1]) if t else (h0, h0.abs())
        sw, swm = (dh * write[..., t]).sum(-1), (dm * write[..., t].abs()).sum(-1)
        p = dh * a * before
        pm = a * (dm * before.abs() + dh.abs() * bm) + (2 * x.abs() + 3) * p.abs()
        new["du"][..., t], mags["du"][..., t] = dtt * sw, dtt * swm
        new["ddt"][..., t] = ut * sw + (A * p).sum(-1)
        mags["ddt"][..., t] = ut.abs() * swm + (A.abs() * pm).sum(-1)
        dA += dtt[..., None] * p
        dAmag += dtt[..., None] * pm
        carry, cmag = a * dh, a * dm + (2 * x.abs() + 3) * (a * dh).abs()
    slope = torch.sigmoid(pre) if softplus else torch.ones_like(pre)
    per = lambda v: v.view(B, G, D // G, N, L).sum(2)  # noqa: E731
    gmag = g.abs() * grow
    if skip is not None:
        new["du"] += skip[:, None] * g
        mags["du"] += skip.abs()[:, None] * gmag
    ddelta = mask(new["ddt"] * slope)
    dmag = mask(mags["ddt"] * slope * (1 + pre.abs()))
    out.update({"du": (mask(new["du"]), mags["du"]), "ddelta": (ddelta, dmag), "dbias": (ddelta.sum((0, 2)), dmag.sum((0, 2))),
                "dA": (dA.sum(0), dAmag.sum(0)), "dwrite": (mask(per(new["dwrite"])), per(mags["dwrite"])),
                "dread": (mask(per(new["dread"])), per(mags["dread"])), "dskip": ((g * u).sum((0, 2)), (gmag * u.abs()).sum((0, 2))),
                "dstate": (carry, cmag)})
    if gate is not None:
        z = gate
        dslope = sig * (1 + z * (1 - sig))
        out["dgate"] = (mask(dy * y * dslope), mask(dy.abs() * ymag * (dslope.abs() + z.abs() + 1)))
    return out


def norm(r, w, eps, dy=None, dr=None):
    """The norm of the stored stream r (..., D) and its gradients: {name: (value, magnitude)}."""
    r, w, dy, dr = (f64(v) for v in (r, w, dy, dr))
    inv = 1 / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    y = r * inv * w
    out = {"y": (y, y.abs())}
    if dy is None and dr is None:
        return out
    x, gw = r * inv, (torch.zeros_like(r) if dy is None else dy) * w
    dr = torch.zeros_like(r) if dr is None else dr
    out["dr"] = (dr + inv * (gw - x * (gw * x).mean(-1, keepdim=True)),
                 dr.abs() + inv * (gw.abs() + x.abs() * (gw * x).abs().mean(-1, keepdim=True)))
    rows = lambda v: v.reshape(-1, v.shape[-1]).sum(0)  # noqa: E731
    out["dweight"] = (rows(dy * x), rows((dy * x).abs()))
    return out
