"""What is measured of the selective layer's operators: the cases, their plain forms, and the calls a user makes.

Plain forms are elementary torch operations in 32 bits, rounded once at the end; the recurrence along time is a
scan by doubling (log2 L sweeps over whole tensors). `exact` walks the time steps one by one in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
E4M3_MAX = 448.0


# ---- cases -------------------------------------------------------------------------------------------

def listed():
    return [
        # the short convolution in a training step of a wide layer: forward and backward
        dict(name="conv_train", op="conv_train", B=8, D=4096, L=2048, W=4, dtype="bf16", bias=True, state=False),
        # a padded batch of prompts that continue earlier ones, odd length, rows off the 16-byte grid
        dict(name="conv_prompt", op="conv_prompt", B=5, D=1536, L=1021, W=4, dtype="f16", bias=True, state=True, ragged=True),
        # one token of one sequence: nothing but latency
        dict(name="conv_step_one", op="conv_step", B=1, D=2048, W=4, dtype="bf16", slots=False),
        # one token each of a full serving batch, states picked out of a pool
        dict(name="conv_step_batch", op="conv_step", B=256, D=4096, W=4, dtype="f16", slots=True),
        # the scan in a training step: forward and backward, gate, skip and softplus
        dict(name="scan_train", op="scan_train", B=8, D=2048, L=2048, N=16, G=1, dtype="bf16", gate=True, state=False, ragged=False),
        # a small training step with odd sizes, several groups and a state carried in
        dict(name="scan_train_odd", op="scan_train", B=2, D=400, L=1023, N=24, G=2, dtype="f32", gate=False, state=True, ragged=False),
        # one long prompt
        dict(name="scan_prompt_long", op="scan_prompt", B=1, D=4096, L=16384, N=16, G=1, dtype="bf16", gate=True, state=False, ragged=False),
        # a padded batch of short prompts that continue earlier ones
        dict(name="scan_prompt_ragged", op="scan_prompt", B=7, D=1024, L=515, N=16, G=1, dtype="f16", gate=True, state=True, ragged=True),
        # one token of one sequence
        dict(name="scan_step_one", op="scan_step", B=1, D=2048, N=16, G=1, dtype="bf16", slots=False),
        # one token each of a full serving batch
        dict(name="scan_step_batch", op="scan_step", B=256, D=4096, N=16, G=1, dtype="bf16", slots=True),
        # the block's entry in training: residual's addition and norm, forward and backward
        dict(name="norm_train", op="norm_train", T=8192, D=4096, dtype="bf16"),
        # the same before a product in 8 bits, for a prompt
        dict(name="norm_quantized", op="norm_quantized", T=4096, D=5120, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_train", "conv_prompt", "conv_step", "scan_train", "scan_train", "scan_prompt", "scan_prompt",
                     "scan_step", "norm_train", "norm_quantized"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm_train", "norm_quantized"):
        D = _log(rng, 64, 8192)
        return dict(op=op, T=min(_log(rng, 1, 16384), (1 << 24) // D), D=D, dtype=dtype)
    if op == "conv_step":
        return dict(op=op, B=_log(rng, 1, 256), D=_log(rng, 64, 4096), W=rng.choice([2, 3, 4]), dtype=dtype,
                    slots=rng.random() < 0.5)
    G = rng.choice([1, 1, 2, 4])
    D = G * _log(rng, 16, 4096 // G)
    if op == "scan_step":
        return dict(op=op, B=_log(rng, 1, 256), D=D, N=rng.choice([4, 8, 16, 16, 20, 32]) if D <= 2048 else 16, G=G, dtype=dtype,
                    slots=rng.random() < 0.5)
    B = _log(rng, 1, 16)
    most = 1 << 25
    L = max(1, min(_log(rng, 1, 16384), most // (B * D)))
    if op in ("conv_train", "conv_prompt"):
        return dict(op=op, B=B, D=D, L=L, W=rng.choice([2, 3, 4]), dtype=dtype, bias=rng.random() < 0.7,
                    state=rng.random() < 0.5, **({"ragged": rng.random() < 0.5} if op == "conv_prompt" else {}))
    N = rng.choice([4, 8, 16, 16, 16, 20, 32])
    L = max(1, min(L, (most * 16) // (B * D * N)))
    return dict(op=op, B=B, D=D, L=L, N=N, G=G, dtype=dtype, gate=rng.random() < 0.7, state=rng.random() < 0.5,
                ragged=rng.random() < 0.3)


# ---- inputs ------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _lengths(g, B, L):
    n = torch.randint(0, L + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    n[0] = L  # a batch is padded to its longest
    return n


def _slots(g, B, S):
    s = torch.randperm(S, generator=g, device=DEV)[:B].to(torch.int32)
    if B > 3:
        s[B // 2] = -1  # a row of the batch that holds no sequence at the moment
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, t = case["op"], TYPES[case["dtype"]]
    s = {"op": op, "dtype": t}
    if op.startswith("norm"):
        T, D = case["T"], case["D"]
        s["x"], s["residual"] = _randn(g, T, D).to(t), (3 * _randn(g, T, D)).to(t)
        s["weight"] = (1 + 0.1 * _randn(g, D)).to(t)
        if op == "norm_train":
            s["dy"], s["dresidual"] = _randn(g, T, D).to(t), _randn(g, T, D).to(t)
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_()
        return s
    B, D = case["B"], case["D"]
    if op.startswith("conv"):
        W = case["W"]
        s["weight"] = (_randn(g, D, W) / math.sqrt(W)).to(t)
        s["bias"] = (0.1 * _randn(g, D)).to(t) if case.get("bias", True) else None
        if op == "conv_step":
            S = B + 64 if case["slots"] else B
            s["x"], s["state"] = _randn(g, B, D).to(t), _randn(g, S, D, W - 1).to(t)
            s["slots"] = _slots(g, B, S) if case["slots"] else None
            s["new_state"] = s["state"].clone()
            return s
        L = case["L"]
        s["x"] = _randn(g, B, D, L).to(t)
        s["state"] = _randn(g, B, D, W - 1).to(t) if case["state"] else None
        if op == "conv_train":
            s["dy"] = _randn(g, B, D, L).to(t)
            s["leaves"] = [k for k in ("x", "weight", "bias", "state") if s[k] is not None]
            for k in s["leaves"]:
                s[k].requires_grad_()
        else:
            s["lengths"] = _lengths(g, B, L) if case["ragged"] else None
        return s
    N, G = case["N"], case["G"]
    s["A"] = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32) * torch.exp(0.1 * _randn(g, D, N))
    dt = torch.exp(torch.rand(D, generator=g, device=DEV) * math.log(100.0) + math.log(0.001))  # steps from 0.001 to 0.1
    s["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
    s["skip"] = 1 + 0.1 * _randn(g, D)
    if op == "scan_step":
        S = B + 64 if case["slots"] else B
        s["u"], s["delta"], s["z"] = _randn(g, B, D).to(t), (0.5 * _randn(g, B, D)).to(t), _randn(g, B, D).to(t)
        s["write"], s["read"] = _randn(g, B, G, N).to(t), _randn(g, B, G, N).to(t)
        s["state"] = 0.1 * _randn(g, S, D, N)
        s["new_state"] = s["state"].clone()
        s["slots"] = _slots(g, B, S) if case["slots"] else None
        return s
    L = case["L"]
    s["u"], s["delta"] = _randn(g, B, D, L).to(t), (0.5 * _randn(g, B, D, L)).to(t)
    s["z"] = _randn(g, B, D, L).to(t) if case["gate"] else None
    s["write"], s["read"] = _randn(g, B, G, N, L).to(t), _randn(g, B, G, N, L).to(t)
    s["state"] = 0.1 * _randn(g, B, D, N) if case["state"] else None
    s["lengths"] = _lengths(g, B, L) if case["ragged"] else None
    if op == "scan_train":
        s["dy"] = _randn(g, B, D, L).to(t)
        s["leaves"] = [k for k in ("u", "delta", "A", "write", "read", "skip", "z", "delta_bias", "state") if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_()
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    op = s["op"]
    if op == "norm_train":
        from fm.scan.fm_norm import fm_norm

        y, r = fm_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        dx, dr, dw = torch.autograd.grad([y, r], [s["x"], s["residual"], s["weight"]], [s["dy"], s["dresidual"]])
        return {"y": y, "residual": r, "dx": dx, "dresidual": dr, "dweight": dw}
    if op == "norm_quantized":
        from fm.scan.fm_norm import fm_norm_quantized

        q, scale, r = fm_norm_quantized(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return {"q": q, "scale": scale, "residual": r}
    from fm.scan import fm_selective as m

    if op == "conv_train":
        y = m.fm_conv(s["x"], s["weight"], s["bias"], initial_state=s["state"])
        grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
    if op == "conv_prompt":
        y, final = m.fm_conv(s["x"], s["weight"], s["bias"], initial_state=s["state"], lengths=s["lengths"], return_state=True)
        return {"y": y, "final": final}
    if op == "conv_step":
        y = m.fm_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"], state_out=s["new_state"])
        return {"y": y, "state": s["new_state"]}
    if op == "scan_step":
        y = m.fm_selective_step(s["u"], s["state"], s["delta"], s["A"], s["write"], s["read"], skip=s["skip"], gate=s["z"],
                                delta_bias=s["delta_bias"], slots=s["slots"], state_out=s["new_state"])
        return {"y": y, "state": s["new_state"]}
    y = m.fm_selective_scan(s["u"], s["delta"], s["A"], s["write"], s["read"], skip=s["skip"], gate=s["z"],
                            delta_bias=s["delta_bias"], initial_state=s["state"], lengths=s["lengths"],
                            return_state=op == "scan_prompt")
    if op == "scan_prompt":
        return {"y": y[0], "final": y[1]}
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
    return {"y": y, **{"d" + k: v for k, v in zip(s["leaves"], grads)}}


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _plain(s):
    with torch.no_grad():
        return {"norm_train": _plain_norm, "norm_quantized": _plain_norm, "conv_train": _plain_conv, "conv_prompt": _plain_conv,
                "conv_step": _plain_conv_step, "scan_train": _plain_scan, "scan_prompt": _plain_scan,
                "scan_step": _plain_scan_step}[s["op"]](s)


def _plain_norm(s):
    t = s["dtype"]
    res = (s["x"].float() + s["residual"].float()).to(t)  # the stream as it is stored is what the norm sees
    r, w = res.float(), s["weight"].float()
    inv = 1 / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS)
    y = r * inv * w
    if s["op"] == "norm_quantized":
        top = y.abs().amax(-1, keepdim=True)
        return {"q": (y * (E4M3_MAX / top)).to(torch.float8_e4m3fn), "scale": (top / E4M3_MAX).squeeze(-1), "residual": res}
    gw = s["dy"].float() * w
    dr = s["dresidual"].float() + inv * (gw - r * inv * inv * (gw * r).mean(-1, keepdim=True))
    dw = (s["dy"].float() * r * inv).sum(0)
    return {"y": y.to(t), "residual": res, "dx": dr.to(t), "dresidual": dr.to(t), "dweight": dw.to(t)}


def _inside(lengths, B, L):
    if lengths is None:
        return None
    return (torch.arange(L, device=DEV) < lengths[:, None])[:, None, :]  # (B, 1, L)


def _plain_conv(s):
    t, x, w = s["dtype"], s["x"].float(), s["weight"].float()
    (B, D, L), W = x.shape, w.shape[1]
    before = torch.zeros(B, D, W - 1, device=DEV) if s["state"] is None else s["state"].float()
    xs = torch.cat([before, x], -1)
    windows = xs.unfold(-1, W, 1)  # (B, D, L, W)
    pre = (windows * w[:, None, :]).sum(-1)
    if s["bias"] is not None:
        pre = pre + s["bias"].float()[:, None]
    sig = _sigmoid(pre)
    y = pre * sig
    if s["op"] == "conv_prompt":
        inside = _inside(s["lengths"], B, L)
        at = torch.arange(W - 1, device=DEV) + (L if inside is None else s["lengths"].long()[:, None, None])
        final = torch.gather(xs, -1, at.expand(B, D, W - 1))
        return {"y": (y if inside is None else torch.where(inside, y, 0.0)).to(t), "final": final.to(t)}
    dpre = s["dy"].float() * (sig * (1 + pre * (1 - sig)))
    out = {"y": y.to(t)}
    around = torch.cat([torch.zeros(B, D, W - 1, device=DEV), dpre, torch.zeros(B, D, W - 1, device=DEV)], -1)
    dxs = (around.unfold(-1, W, 1) * w.flip(1)[:, None, :]).sum(-1)  # (B, D, L + W - 1)
    out["dx"] = dxs[..., W - 1:].to(t)
    out["dweight"] = (windows * dpre[..., None]).sum((0, 2)).to(t)
    if s["bias"] is not None:
        out["dbias"] = dpre.sum((0, 2)).to(t)
    if s["state"] is not None:
        out["dstate"] = dxs[..., :W - 1].to(t)
    return out


def _put(s, new, y):
    """Rows of a step without a slot give zeros and leave every state alone."""
    t, out = s["dtype"], s["new_state"]
    if s["slots"] is None:
        out.copy_(new)
        return {"y": y.to(t), "state": out}
    held = s["slots"] >= 0
    out.index_copy_(0, s["slots"][held].long(), new[held].to(out.dtype))
    return {"y": torch.where(held[:, None], y, 0.0).to(t), "state": out}


def _plain_conv_step(s):
    x, w = s["x"].float(), s["weight"].float()
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].clamp(min=0).long()]
    window = torch.cat([old.float(), x[:, :, None]], -1)
    pre = (window * w).sum(-1) + s["bias"].float()
    return _put(s, window[..., 1:], pre * _sigmoid(pre))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_scan_step(s):
    u = s["u"].float()
    B, D = u.shape
    per = D // s["write"].shape[1]
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].clamp(min=0).long()]
    write, read = (s[k].float().repeat_interleave(per, 1) for k in ("write", "read"))
    new = torch.exp(dt[..., None] * s["A"]) * old + (dt * u)[..., None] * write
    z = s["z"].float()
    y = ((new * read).sum(-1) + s["skip"] * u) * z * _sigmoid(z)
    return _put(s, new, y)


def _scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the last axis, by doubling."""
    step = 1
    while step < a.shape[-1]:
        b = torch.cat([b[..., :step], b[..., step:] + a[..., step:] * b[..., :-step]], -1)
        a = torch.cat([a[..., :step], a[..., step:] * a[..., :-step]], -1)
        step *= 2
    return b


def _plain_scan(s):
    t, u, delta, A = s["dtype"], s["u"].float(), s["delta"].float(), s["A"]
    (B, D, L), (_, G, N, _) = u.shape, s["write"].shape
    per = D // G
    inside = _inside(s["lengths"], B, L)
    mask = (lambda v: v) if inside is None else (lambda v: torch.where(inside, v, 0.0))
    pre = delta + s["delta_bias"][:, None]
    dt = mask(_softplus(pre))  # a step of length zero leaves the state as it is
    write, read = (s[k].float().repeat_interleave(per, 1) for k in ("write", "read"))  # (B, D, N, L)
    a = torch.exp(dt[:, :, None] * A[:, :, None])
    b = (dt * u)[:, :, None] * write
    if s["state"] is not None:
        b = torch.cat([b[..., :1] + a[..., :1] * s["state"][..., None], b[..., 1:]], -1)
    h = _scan(a, b)
    del b
    y = (h * read).sum(2) + s["skip"][:, None] * u
    z = None if s["z"] is None else s["z"].float()
    out = mask(y if z is None else y * z * _sigmoid(z))
    if s["op"] == "scan_prompt":
        return {"y": out.to(t), "final": h[..., -1].contiguous()}
    dy = mask(s["dy"].float())
    res = {"y": out.to(t)}
    g = dy
    if z is not None:
        sig = _sigmoid(z)
        g = dy * z * sig
        res["dz"] = (dy * y * sig * (1 + z * (1 - sig))).to(t)
    c = g[:, :, None] * read
    later = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1)  # dh[t] = c[t] + a[t+1] dh[t+1]
    dh = _scan(later.flip(-1), c.flip(-1)).flip(-1)
    del c, later
    first = torch.zeros(B, D, N, device=DEV) if s["state"] is None else s["state"]
    back = dh * a * torch.cat([first[..., None], h[..., :-1]], -1)
    sum_write = (dh * write).sum(2)
    ddelta = mask((u * sum_write + (back * A[:, :, None]).sum(2)) * _sigmoid(pre))
    res["du"] = mask(dt * sum_write + s["skip"][:, None] * g).to(t)
    res["ddelta"], res["ddelta_bias"] = ddelta.to(t), ddelta.sum((0, 2))
    res["dA"] = (back * dt[:, :, None]).sum((0, 3))
    res["dskip"] = (g * u).sum((0, 2))
    res["dwrite"] = (dh * (dt * u)[:, :, None]).view(B, G, per, N, L).sum(2).to(t)
    res["dread"] = (h * g[:, :, None]).view(B, G, per, N, L).sum(2).to(t)
    if s["state"] is not None:
        res["dstate"] = (a[..., 0] * dh[..., 0]).contiguous()
    return {k: res[k] for k in ["y"] + ["d" + k for k in s["leaves"]]}


# ---- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op.startswith("norm"):
        n = case["T"] * case["D"]
        if op == "norm_train":  # forward: two in, two out; backward: two gradients and the stream in, one gradient out, to two places
            return {"bytes": 9 * n * e, "flops": 15 * n}
        return {"bytes": n * (3 * e + 1) + 4 * case["T"], "flops": 7 * n}
    B, D = case["B"], case["D"]
    if op == "conv_step":
        return {"bytes": B * D * e * (2 + 2 * (case["W"] - 1)) + D * e * (case["W"] + 1), "flops": B * D * (2 * case["W"] + 5)}
    if op.startswith("conv"):
        n, W = B * D * case["L"], case["W"]
        if op == "conv_train":
            return {"bytes": 5 * n * e, "flops": n * (6 * W + 18)}
        return {"bytes": 2 * n * e, "flops": n * (2 * W + 5)}
    N, G = case["N"], case["G"]
    if op == "scan_step":
        return {"bytes": 8 * B * D * N + 4 * B * D * e + 2 * B * G * N * e + 4 * D * N, "flops": B * D * (8 * N + 20)}
    L, z = case["L"], int(case["gate"])
    streams, shared = B * D * L * e, 2 * B * G * N * L * e
    if op == "scan_prompt":
        return {"bytes": (3 + z) * streams + shared, "flops": B * D * L * (8 * N + 20)}
    return {"bytes": (3 + z + 5 + 2 * z) * streams + 3 * shared, "flops": B * D * L * (30 * N + 60)}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        d = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
        op = s["op"]
        if op.startswith("norm"):
            return _exact_norm(s, d)
        if op == "conv_step":
            return _exact_step(s, d, True)
        if op == "scan_step":
            return _exact_step(s, d, False)
        return _exact_conv(s, d) if op.startswith("conv") else _exact_scan(s, d)


def _exact_norm(s, d):
    r = (d["x"] + d["residual"]).to(s["dtype"]).double()
    D = r.shape[-1]
    rms = (r.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
    unit = r / rms
    y = unit * d["weight"]
    if s["op"] == "norm_quantized":
        top = y.abs().max(-1, keepdim=True).values
        # the quotient before it is rounded to 8 bits
        return {"q": y / top * E4M3_MAX, "scale": top[:, 0] / E4M3_MAX, "residual": r}
    gw = d["dy"] * d["weight"]
    dr = d["dresidual"] + (gw - unit * (gw * unit).sum(-1, keepdim=True) / D) / rms
    return {"y": y, "residual": r, "dx": dr, "dresidual": dr, "dweight": (d["dy"] * unit).sum(0)}


def _exact_conv(s, d):
    x, w = d["x"], d["weight"]
    (B, D, L), W = x.shape, w.shape[1]
    xs = torch.zeros(B, D, L + W - 1, device=DEV, dtype=torch.float64)
    if d["state"] is not None:
        xs[..., :W - 1] = d["state"]
    xs[..., W - 1:] = x
    pre = torch.zeros_like(x)
    for j in range(W):
        pre += w[:, j, None] * xs[..., j:j + L]
    if d["bias"] is not None:
        pre += d["bias"][:, None]
    sig = torch.sigmoid(pre)
    y = pre * sig
    if s["op"] == "conv_prompt":
        final = torch.empty(B, D, W - 1, device=DEV, dtype=torch.float64)
        ends = [L] * B if s["lengths"] is None else s["lengths"].tolist()
        for b, n in enumerate(ends):
            final[b] = xs[b, :, n:n + W - 1]
            y[b, :, n:] = 0
        return {"y": y, "final": final}
    dpre = d["dy"] * (sig + y * (1 - sig))
    dxs = torch.zeros_like(xs)
    dw = torch.empty_like(w)
    for j in range(W):
        dxs[..., j:j + L] += w[:, j, None] * dpre
        dw[:, j] = (dpre * xs[..., j:j + L]).sum((0, 2))
    grads = {"x": dxs[..., W - 1:], "weight": dw, "bias": dpre.sum((0, 2)), "state": dxs[..., :W - 1]}
    return {"y": y, **{"d" + k: grads[k] for k in s["leaves"]}}


def _exact_step(s, d, conv):
    B, D = (d["x"] if conv else d["u"]).shape
    y = torch.zeros(B, D, device=DEV, dtype=torch.float64)
    state = d["new_state"].clone()
    slots = list(range(B)) if s["slots"] is None else s["slots"].tolist()
    for b, slot in enumerate(slots):
        if slot < 0:
            continue
        if conv:
            window = torch.cat([d["state"][slot], d["x"][b, :, None]], -1)
            pre = (window * d["weight"]).sum(-1) + d["bias"]
            y[b], state[slot] = pre * torch.sigmoid(pre), window[:, 1:]
            continue
        G = d["write"].shape[1]
        dt = torch.nn.functional.softplus(d["delta"][b] + d["delta_bias"], threshold=60)
        w, r = (d[k][b][:, None].expand(G, D // G, -1).reshape(D, -1) for k in ("write", "read"))
        h = torch.exp(dt[:, None] * d["A"]) * d["state"][slot] + (dt * d["u"][b])[:, None] * w
        y[b] = ((h * r).sum(-1) + d["skip"] * d["u"][b]) * d["z"][b] * torch.sigmoid(d["z"][b])
        state[slot] = h
    return {"y": y, "state": state}


def _exact_scan(s, d):
    (B, D, L), (_, G, N, _) = d["u"].shape, d["write"].shape
    if B * D * N * L > 1 << 31:
        return None
    ends = torch.full((B,), L, device=DEV) if s["lengths"] is None else s["lengths"].long()
    live = (torch.arange(L, device=DEV)[:, None] < ends).double()[:, :, None]  # (L, B, 1)
    first = lambda v: v.permute(2, 0, 1).contiguous()  # noqa: E731  (L, B, D)
    u, pre = first(d["u"]), first(d["delta"]) + d["delta_bias"]
    dt = torch.nn.functional.softplus(pre, threshold=60) * live
    w, r = (d[k].permute(3, 0, 1, 2).contiguous() for k in ("write", "read"))  # (L, B, G, N)
    wide = lambda v: v[:, :, None].expand(B, G, D // G, N).reshape(B, D, N)  # noqa: E731
    train = s["op"] == "scan_train"
    h0 = torch.zeros(B, D, N, device=DEV, dtype=torch.float64) if d["state"] is None else d["state"]
    h, y = h0, torch.empty_like(u)
    hs = torch.empty(L, B, D, N, device=DEV, dtype=torch.float64) if train else None
    for i in range(L):
        h = torch.exp(dt[i][..., None] * d["A"]) * h + (dt[i] * u[i])[..., None] * wide(w[i])
        y[i] = (h * wide(r[i])).sum(-1)
        if train:
            hs[i] = h
    y += d["skip"] * u
    z = None if d["z"] is None else first(d["z"])
    gate = 1.0 if z is None else z * torch.sigmoid(z)
    last = lambda v: v.permute(1, 2, 0)  # noqa: E731
    if not train:
        return {"y": last(y * gate * live), "final": h}
    dy = first(d["dy"]) * live
    g = dy * gate
    du, ddt, dz = torch.empty_like(u), torch.empty_like(u), None
    if z is not None:
        sig = torch.sigmoid(z)
        dz = last(dy * y * sig * (1 + z * (1 - sig)))
    dw, dr = torch.empty(L, B, G, N, device=DEV, dtype=torch.float64), torch.empty(L, B, G, N, device=DEV, dtype=torch.float64)
    dA, carry = torch.zeros_like(d["A"]), torch.zeros_like(h0)
    per_group = lambda v: v.view(B, G, D // G, N).sum(2)  # noqa: E731
    for i in reversed(range(L)):
        a = torch.exp(dt[i][..., None] * d["A"])
        dh = g[i][..., None] * wide(r[i]) + carry
        dr[i] = per_group(g[i][..., None] * hs[i])
        dw[i] = per_group(dh * (dt[i] * u[i])[..., None])
        sw = (dh * wide(w[i])).sum(-1)
        carry = dh * a
        p = carry * (hs[i - 1] if i else h0)
        du[i] = dt[i] * sw + d["skip"] * g[i]
        ddt[i] = u[i] * sw + (p * d["A"]).sum(-1)
        dA += (p * dt[i][..., None]).sum(0)
    ddelta = ddt * torch.sigmoid(pre) * live
    move = lambda v: v.permute(1, 2, 3, 0)  # noqa: E731
    grads = {"u": last(du * live), "delta": last(ddelta), "A": dA, "write": move(dw), "read": move(dr), "skip": (g * u).sum((0, 1)),
             "z": dz, "delta_bias": ddelta.sum((0, 1)), "state": carry}
    return {"y": last(y * gate * live), **{"d" + k: grads[k] for k in s["leaves"]}}
