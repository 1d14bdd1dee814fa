"""The selective layer's operators on the GPU against plain implementations in float64 (selective_reference.py)."""
import math

import pytest
import torch

import selective_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def m():
    import fm.scan.fm_selective as m

    assert torch.cuda.is_available(), "these tests need the GPU"
    return m


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


def strided(t, pad_channel=3, pad_batch=1):
    """The same values in a wider buffer: other batch and channel strides, off the 16-byte grid."""
    B, D, L = t.shape
    wide = torch.full((B + pad_batch, D + pad_batch, L + pad_channel), float("nan"), dtype=t.dtype, device=t.device)
    view = wide[:B, 1:D + 1, 1:L + 1] if pad_batch else wide[:, :, 1:L + 1]
    view.copy_(t)
    return view


def spoil(t, lengths):
    """NaN in the steps that do not count."""
    for b, n in enumerate(lengths.tolist()):
        t[b, ..., max(0, min(n, t.shape[-1])):] = float("nan")
    return t


# ---- short convolution ------------------------------------------------------------------------------
# forward: W + 1 roundings of the sum, 10 and the size of the sum for the silu: c = 32 at sums below 10
# gradients: the slope takes about 16 operations, the taps W more: c = 48; sums over time add a rounding a term
# in a lane (L / 64 + 8), the lanes' tree and the column sums (6 + B segments / 8 + 8)

CONV_SHAPES = [(1, 1, 1, 2), (2, 3, 2, 4), (1, 5, 3, 3), (3, 7, 8, 4), (2, 4, 9, 2), (2, 3, 64, 4), (2, 65, 127, 3),
               (1, 3, 511, 4), (2, 2, 513, 4), (1, 2, 2049, 4), (1, 1, 9000, 4), (700, 3, 5, 4),
               (170, 6400, 1, 3), (500, 640, 9, 4), (330, 210, 65, 2)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", CONV_SHAPES, ids=str)
def test_conv(m, shape, dtype):
    B, D, L, W = shape
    for variant in range(4):
        g = gen(B * 1000 + L + variant)
        x, w = rand(g, B, D, L, dtype=dtype), rand(g, D, W, dtype=dtype if variant % 2 else F32, scale=0.5)
        bias = rand(g, D, dtype=F32 if variant == 3 else dtype, scale=0.1) if variant != 1 else None
        state = rand(g, B, D, W - 1, dtype=dtype) if variant >= 2 else None
        lengths = None
        if variant == 3:
            lengths = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
            lengths[0] = (L, 0, L + 7, -2)[L % 4]
            lengths = lengths.to(DEV)
            x = spoil(x, lengths)
        if variant in (1, 3):
            x = strided(x)
        dy, dfinal = rand(g, B, D, L, dtype=dtype), rand(g, B, D, W - 1, dtype=dtype)
        if lengths is not None:
            dy = spoil(dy, lengths)
        silu = variant != 2
        leaves = [t for t in (x, w, bias, state) if t is not None]
        for t in leaves:
            t.requires_grad_()
        y, final = m.fm_conv(x, w, bias, initial_state=state, lengths=lengths, silu=silu, return_state=True)
        ref = R.conv(x, w, bias, state, lengths, silu, dy, dfinal)
        what = f"{shape} {dtype} variant {variant}"
        R.close(y, *ref["y"], 32, what + " y")
        R.close(final, *ref["final"], 0, what + " final")
        grads = torch.autograd.grad([y, final], leaves, [dy, dfinal])
        names = [n for n, t in (("dx", x), ("dweight", w), ("dbias", bias), ("dstate", state)) if t is not None]
        c = 48 + L / 64 + 8 + 6 + B + 8
        for n, t in zip(names, grads):
            R.close(t, *ref[n], 48 if n in ("dx", "dstate") else c, f"{what} {n}")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv_in_pieces_is_the_whole(m, dtype):
    """A prompt in two calls, the state handed on: bit for bit the one call."""
    g = gen(3)
    x, w, bias = rand(g, 2, 5, 300, dtype=dtype), rand(g, 5, 4, dtype=dtype), rand(g, 5, dtype=dtype)
    whole, last = m.fm_conv(x, w, bias, return_state=True)
    for cut in (1, 2, 8, 131):
        a, s = m.fm_conv(x[..., :cut], w, bias, return_state=True)
        b, s = m.fm_conv(x[..., cut:], w, bias, initial_state=s, return_state=True)
        assert torch.equal(torch.cat([a, b], -1), whole) and torch.equal(s, last)


def test_conv_other_uses_of_its_gradients(m):
    """Only the final state used; an expanded gradient (of a sum); a gradient of the final state alone."""
    g = gen(4)
    x, w = rand(g, 2, 3, 40), rand(g, 3, 4)
    x.requires_grad_(), w.requires_grad_()
    y = m.fm_conv(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    ref = R.conv(x, w, dy=torch.ones(2, 3, 40))
    R.close(dx, *ref["dx"], 48, "dx"), R.close(dw, *ref["dweight"], 80, "dw")
    y, s = m.fm_conv(x, w, return_state=True)
    (dx,) = torch.autograd.grad(s, [x], torch.ones_like(s))
    assert torch.equal(dx[..., -3:], torch.ones_like(dx[..., -3:])) and not dx[..., :-3].any()


def test_conv_gradients_are_the_differences(m):
    """The reference's gradients, which the kernels are held to, against central differences in float64."""
    g = gen(5)
    x, w, b, s = (torch.randn(*n, generator=g, dtype=torch.float64) for n in ((2, 2, 6), (2, 3), (2,), (2, 2, 2)))
    dy, df = torch.randn(2, 2, 6, generator=g, dtype=torch.float64), torch.randn(2, 2, 2, generator=g, dtype=torch.float64)
    lengths = torch.tensor([6, 4])
    loss = lambda *a: sum((r * d).sum() for r, d in zip(  # noqa: E731
        [v[0] for v in list(R.conv(a[0], a[1], a[2], a[3], lengths).values())[:2]], (dy, df)))
    ref = R.conv(x, w, b, s, lengths, True, dy, df)
    for n, v in (("dx", x), ("dweight", w), ("dbias", b), ("dstate", s)):
        for at in ([0] * v.dim(), [k - 1 for k in v.shape]):
            at, h = tuple(at), 1e-5
            args = [x, w, b, s]
            ends = []
            for sign in (1, -1):
                moved = v.clone()
                moved[at] += sign * h
                ends.append(loss(*[moved if a is v else a for a in args]))
            # second-order differences: h^2 and 1e-16 / h
            assert abs((ends[0] - ends[1]) / (2 * h) - ref[n][0][at]) < 1e-8


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,D,W", [(1, 1, 2), (1, 300, 4), (5, 64, 3), (64, 257, 4)])
def test_conv_step(m, B, D, W, dtype):
    g = gen(B + D)
    S = B + 3
    x, w, bias = rand(g, B, D, dtype=dtype), rand(g, D, W, dtype=dtype, scale=0.5), rand(g, D)
    pool = rand(g, S, D, W - 1, dtype=dtype)
    for slots in (None, torch.randperm(S, generator=g)[:B].to(torch.int32).to(DEV), torch.randperm(S, generator=g)[:B].to(DEV)):
        state = pool[:B].clone() if slots is None else pool.clone()
        at = torch.arange(B) if slots is None else slots.cpu().long()
        if slots is not None and B > 3:
            slots[1], slots[2], slots[B - 1] = -1, S, slots[0]  # skipped: out of range, and named a second time
        skipped = [1, 2, B - 1] if slots is not None and B > 3 else []
        before = state.clone()
        ref = R.conv(x[..., None], w, bias, pool[at.to(DEV)])
        aside = torch.full_like(state, 7)
        y = m.fm_conv_step(x, state, w, bias, slots=slots, state_out=aside)
        assert torch.equal(state, before)
        y2 = m.fm_conv_step(x, state, w, bias, slots=slots)
        assert torch.equal(y, y2)
        rows = [b for b in range(B) if b not in skipped]
        R.close(y[rows], ref["y"][0][rows][..., 0], ref["y"][1][rows][..., 0], 32, "y")
        assert not y[skipped].any()
        want, want_aside = before.clone(), torch.full_like(state, 7)
        for b in rows:
            new = ref["final"][0][b].to(dtype).to(DEV)
            want[at[b]], want_aside[at[b]] = new, new
        assert torch.equal(state, want) and torch.equal(aside, want_aside)


def test_conv_steps_are_the_sequence(m):
    g = gen(9)
    x, w, bias = rand(g, 3, 70, 12, dtype=BF16), rand(g, 70, 4, dtype=BF16), rand(g, 70, dtype=BF16)
    whole, last = m.fm_conv(x, w, bias, return_state=True)
    state = torch.zeros(3, 70, 3, dtype=BF16, device=DEV)
    for t in range(12):
        assert torch.equal(m.fm_conv_step(x[..., t].contiguous(), state, w, bias), whole[..., t])
    assert torch.equal(state, last)


# ---- selective scan ---------------------------------------------------------------------------------
# The reference's magnitudes follow every term through the recurrence, a rounding a step and the decay's own error
# included. On top of those a result passes through the composition of 8 steps, of 16 or 64 lanes and of the tiles
# (products of decays in place of one step after the other: at most 6 levels of two roundings each and the total's
# exponent, three roundings of |dt A| summed), the sum over N, and about ten operations of softplus (twice) and
# gate: c = 40 + N. A gradient multiplies two such quantities and runs both ways: c = 80 + 2 N; sums over time, channels
# and batch add a rounding for every term that one thread adds: 8 steps a tile, L / 128 tiles, 16 blocks.

SCAN_SHAPES = [  # B, D, L, N, G
    (1, 1, 1, 1, 1), (2, 3, 2, 2, 1), (1, 4, 7, 3, 2), (2, 6, 9, 16, 3), (3, 17, 40, 5, 1), (1, 8, 127, 16, 2),
    (1, 33, 128, 8, 1), (2, 20, 129, 17, 1), (1, 5, 300, 33, 1), (2, 4, 513, 4, 4), (1, 2, 1100, 16, 1), (70, 2, 3, 4, 1),
    (1, 2, 2700, 3, 1), (2, 3, 5000, 2, 1),  # rows cut along time
    (260, 40, 140, 3, 1), (130, 70, 21, 3, 1), (120, 160, 33, 5, 2), (90, 256, 150, 2, 1)]  # 16 lanes a channel; 4: one tile, two, five


def scan_case(shape, dtype, variant, seed=0):
    B, D, L, N, G = shape
    g = gen(B * 100 + D * 10 + L + N + variant + seed)
    a = {"tokens": rand(g, B, D, L, dtype=dtype), "delta": rand(g, B, D, L, dtype=dtype, scale=0.5),
         "A": -torch.exp(rand(g, D, N)) * (1 + torch.arange(N, device=DEV)) / 4,
         "write": rand(g, B, G, N, L, dtype=dtype), "read": rand(g, B, G, N, L, dtype=dtype)}
    a["skip"] = rand(g, D, dtype=dtype if variant == 2 else F32) if variant else None
    a["gate"] = rand(g, B, D, L, dtype=dtype) if variant != 1 else None
    a["delta_bias"] = rand(g, D, dtype=dtype if variant == 1 else F32) - 3 if variant != 2 else None
    a["initial_state"] = rand(g, B, D, N) if variant >= 2 else None
    a["lengths"] = None
    dy, dfinal = rand(g, B, D, L, dtype=dtype), rand(g, B, D, N)
    if variant == 3:
        n = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        n[0] = (L, 0, L + 7, -2)[L % 4]
        a["lengths"] = n.to(DEV)
        for k in ("tokens", "delta", "gate", "write", "read"):
            spoil(a[k], n)
        spoil(dy, n)
    if variant in (1, 3):
        for k in ("tokens", "delta", "gate"):
            if a[k] is not None:
                a[k] = strided(a[k])
        for k in ("write", "read"):
            a[k] = strided(a[k].flatten(1, 2), pad_batch=0).unflatten(1, (G, N))
        dy = strided(dy)
    return a, dy, dfinal, variant != 2 or None


REF = {"tokens": "u", "initial_state": "state", "delta_bias": "bias"}
GRADS = {"tokens": "du", "delta": "ddelta", "A": "dA", "write": "dwrite", "read": "dread", "skip": "dskip", "gate": "dgate",
         "delta_bias": "dbias", "initial_state": "dstate"}


def scan_reference(a, softplus, dy=None, dfinal=None):
    return R.scan(**{REF.get(k, k): v for k, v in a.items()}, softplus=softplus, dy=dy, dfinal=dfinal)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SCAN_SHAPES, ids=str)
def test_selective_scan(m, shape, dtype):
    B, D, L, N, G = shape
    for variant in range(4):
        a, dy, dfinal, softplus = scan_case(shape, dtype, variant)
        softplus = bool(softplus)
        if not softplus:
            a["delta"] = a["delta"].abs() * 0.2
        what = f"{shape} {dtype} variant {variant}"
        ref = scan_reference(a, softplus, dy, dfinal)
        y, final = m.fm_selective_scan(**a, softplus=softplus, return_state=True)
        R.close(y, *ref["y"], 40 + N, what + " y")
        R.close(final, *ref["final"], 40 + N, what + " final")
        leaves = {k: v.requires_grad_() for k, v in a.items() if v is not None and k != "lengths"}
        y2, final2 = m.fm_selective_scan(**a, softplus=softplus, return_state=True)
        assert torch.equal(y, y2) and torch.equal(final, final2)
        grads = torch.autograd.grad([y2, final2], list(leaves.values()), [dy, dfinal])
        c = 80 + 2 * N + 16 + 8 + L / 128 + B
        for k, t in zip(leaves, grads):
            assert t.dtype == a[k].dtype
            R.close(t, *ref[GRADS[k]], c, f"{what} {GRADS[k]}")


def test_selective_scan_reference_gradients_are_the_differences():
    """The formulas that the kernels are held to, against central differences in float64."""
    g = gen(11)
    r = lambda *n: torch.randn(*n, generator=g, dtype=torch.float64)  # noqa: E731
    B, D, L, N, G = 2, 4, 5, 3, 2
    a = dict(u=r(B, D, L), delta=r(B, D, L), A=-r(D, N).abs(), write=r(B, G, N, L), read=r(B, G, N, L), skip=r(D), gate=r(B, D, L),
             bias=r(D), state=r(B, D, N))
    lengths, dy, df = torch.tensor([5, 3]), r(B, D, L), r(B, D, N)

    def loss(**k):
        out = R.scan(**k, lengths=lengths)
        return (out["y"][0] * dy).sum() + (out["final"][0] * df).sum()

    ref = R.scan(**a, lengths=lengths, dy=dy, dfinal=df)
    names = dict(u="du", delta="ddelta", A="dA", write="dwrite", read="dread", skip="dskip", gate="dgate", bias="dbias", state="dstate")
    for k, name in names.items():
        for at in ([0] * a[k].dim(), [n - 1 for n in a[k].shape], [n // 2 for n in a[k].shape]):
            at, h = tuple(at), 1e-5
            ends = []
            for sign in (1, -1):
                moved = a[k].clone()
                moved[at] += sign * h
                ends.append(loss(**{**a, k: moved}))
            # the third derivatives are of order ten: 1e-9 from h squared, 1e-11 from the rounding over h
            assert abs((ends[0] - ends[1]) / (2 * h) - ref[name][0][at]) < 1e-7 * (1 + abs(ref[name][0][at])), (k, at)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_selective_scan_in_pieces_is_the_whole(m, dtype):
    """Two calls, the state handed on, against the one call: the same recurrence composed elsewhere."""
    a, *_ = scan_case((2, 5, 300, 16, 1), dtype, 0)
    ref = scan_reference(a, True)
    for cut in (1, 128, 200):
        part = lambda lo, hi: {k: v[..., lo:hi] if k in ("tokens", "delta", "gate", "write", "read") else v  # noqa: E731
                               for k, v in a.items()}
        y1, s = m.fm_selective_scan(**part(0, cut), return_state=True)
        y2, s = m.fm_selective_scan(**{**part(cut, 300), "initial_state": s}, return_state=True)
        R.close(torch.cat([y1, y2], -1), *ref["y"], 56, "y")
        R.close(s, *ref["final"], 56, "final")


def test_selective_scan_more_channels_than_a_wave_row(m):
    """Enough channels for 16 lanes each, several tiles, a group's end inside a block; for 4 lanes each, many states."""
    for dtype, (B, D, L, N, G) in ((BF16, (4, 2100, 200, 4, 1)), (F32, (3, 2802, 131, 3, 2)), (F16, (130, 70, 9, 250, 1))):
        a, *_ = scan_case((B, D, L, N, G), dtype, 3)
        y, final = m.fm_selective_scan(**a, return_state=True)
        ref = scan_reference(a, True)
        R.close(y, *ref["y"], 40 + N, "y")
        R.close(final, *ref["final"], 40 + N, "final")


def test_selective_scan_gives_the_same_bits_again(m):
    a, dy, dfinal, _ = scan_case((2, 40, 400, 16, 1), BF16, 3)
    leaves = {k: v.requires_grad_() for k, v in a.items() if v is not None and k != "lengths"}
    got = []
    for _ in range(2):
        out = m.fm_selective_scan(**a, return_state=True)
        got.append([*out, *torch.autograd.grad(out, list(leaves.values()), [dy, dfinal])])
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_selective_scan_three_axes_are_one_group(m):
    a, dy, *_ = scan_case((2, 6, 50, 4, 1), F32, 0)
    w3, r3 = a["write"].squeeze(1).clone().requires_grad_(), a["read"].squeeze(1).clone().requires_grad_()
    a["write"].requires_grad_(), a["read"].requires_grad_()
    y = m.fm_selective_scan(**a)
    y3 = m.fm_selective_scan(**{**a, "write": w3, "read": r3})
    assert torch.equal(y, y3)
    for p, q in zip(torch.autograd.grad(y, [a["write"], a["read"]], dy), torch.autograd.grad(y3, [w3, r3], dy)):
        assert torch.equal(p.squeeze(1), q)


def test_selective_scan_large_and_small_steps(m):
    """Steps so large that the state is forgotten at once, and so small that softplus is the exponential alone."""
    B, D, L, N = 1, 4, 40, 4
    g = gen(17)
    for shift in (-16.0, -9.0, 30.0):
        a = {"tokens": rand(g, B, D, L), "delta": rand(g, B, D, L) + shift, "A": -torch.ones(D, N, device=DEV),
             "write": rand(g, B, 1, N, L), "read": rand(g, B, 1, N, L)}
        ref = R.scan(*[a[k] for k in ("tokens", "delta", "A", "write", "read")])
        y, final = m.fm_selective_scan(**a, return_state=True)
        R.close(y, *ref["y"], 48, f"{shift} y")
        R.close(final, *ref["final"], 48, f"{shift} final")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (2, 6, 3, 2), (5, 64, 16, 1), (3, 130, 20, 2), (33, 65, 64, 1), (2, 8, 250, 1),
                                     (64, 4100, 4, 2), (64, 4097, 3, 1)])  # many: two channels a lane
def test_selective_step(m, B, D, N, G, dtype):
    g = gen(B + D + N)
    S = B + 2
    a, *_ = scan_case((B, D, 1, N, G), dtype, 0)
    a["delta_bias"], a["skip"] = a["delta_bias"].to(dtype), rand(g, D)
    pool = rand(g, S, D, N)
    one = {k: a[k][..., 0].contiguous() for k in ("tokens", "delta", "gate", "write", "read")}
    for slots in (None, torch.randperm(S, generator=g)[:B].to(torch.int32).to(DEV), torch.randperm(S, generator=g)[:B].to(DEV)):
        state = pool[:B].clone() if slots is None else pool.clone()
        at = torch.arange(B) if slots is None else slots.cpu().long()
        skipped = []
        if slots is not None and B > 3:
            slots[1], slots[2], slots[B - 1] = -7, S, slots[0]
            skipped = [1, 2, B - 1]
        ref = R.scan(a["tokens"], a["delta"], a["A"], a["write"], a["read"], a["skip"], a["gate"], a["delta_bias"],
                     pool[at.to(DEV)])
        call = dict(one, A=a["A"], skip=a["skip"], delta_bias=a["delta_bias"], slots=slots)
        before, aside = state.clone(), torch.full_like(state, 7)
        y = m.fm_selective_step(state=state, state_out=aside, **call)
        assert torch.equal(state, before)
        assert torch.equal(m.fm_selective_step(state=state, **call), y)
        rows = [b for b in range(B) if b not in skipped]
        R.close(y[rows], ref["y"][0][rows][..., 0], ref["y"][1][rows][..., 0], 40 + N, "y")
        assert not y[skipped].any()
        R.close(state[at[rows]], ref["final"][0][rows], ref["final"][1][rows], 40, "state")
        assert torch.equal(aside[at[rows]], state[at[rows]])
        rest = [s for s in range(state.shape[0]) if s not in set(at[rows].tolist())]
        assert torch.equal(state[rest], before[rest]) and (aside[rest] == 7).all()


def test_selective_step_views(m):
    """Rows of wider buffers (a projection's slices), states that lie off the 16-byte grid."""
    g = gen(21)
    B, D, N = 3, 37, 8
    wide = rand(g, B, 2 * D + 2 * N + 1, dtype=BF16)
    u, z, w, r = (wide[:, i:i + n] for i, n in ((0, D), (D, D), (2 * D, N), (2 * D + N, N)))
    delta, A = rand(g, B, D, dtype=BF16), -torch.exp(rand(g, D, N))
    buf = rand(g, B * D * N + 1)
    state = buf[1:].view(B, D, N)
    kept = state.clone()
    y = m.fm_selective_step(u, state, delta, A, w, r, gate=z)
    assert torch.equal(y, m.fm_selective_step(u.contiguous(), kept, delta, A, w.contiguous(), r.contiguous(), gate=z.contiguous()))
    assert torch.equal(state, kept)


def test_steps_are_seen_by_a_graph_that_holds_the_states(m):
    """States that an eager graph keeps for its backward pass and that a step then moves on."""
    g = gen(22)
    a = scan_case((2, 4, 9, 3, 1), F32, 0)[0]
    state = rand(g, 2, 4, 3)
    tokens = a["tokens"].requires_grad_()
    y = m.fm_selective_scan(tokens, a["delta"], a["A"], a["write"], a["read"], initial_state=state)
    token, delta, write, read = (t[..., 0].detach().contiguous() for t in (tokens, a["delta"], a["write"], a["read"]))
    m.fm_selective_step(token, state, delta, a["A"], write, read)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    carried, w = rand(g, 2, 4, 3), rand(g, 4, 4)
    y = m.fm_conv(tokens, w, initial_state=carried)
    other = torch.empty_like(carried)
    m.fm_conv_step(rand(g, 2, 4), carried, w, state_out=other)  # leaves `carried` as it is
    y.sum().backward(retain_graph=True)
    m.fm_conv_step(rand(g, 2, 4), carried, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        m.fm_conv_step(rand(g, 2, 4), rand(g, 2, 4, 3), w)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_channel_that_is_not_finite_stays_alone(m, bad):
    """Channels side by side in a wave: the others' outputs and gradients keep their bits."""
    g = gen(61)
    for B, D, L in ((3, 70, 5), (2, 70, 65), (2, 9, 700)):
        x, w, dy = rand(g, B, D, L, dtype=BF16), rand(g, D, 4), rand(g, B, D, L, dtype=BF16)
        got = []
        for spoiled in (False, True):
            mine = x.clone()
            if spoiled:
                mine[:, 4, L // 2] = bad
            leaves = [mine.requires_grad_(), w.detach().clone().requires_grad_()]
            y = m.fm_conv(*leaves)
            got.append([y, *torch.autograd.grad(y, leaves, dy)])
        keep = [d for d in range(D) if d != 4]
        assert not torch.isfinite(got[1][0][:, 4]).all()
        for p, q in zip(*got):
            axis = 1 if p.dim() == 3 else 0
            assert torch.equal(p.index_select(axis, torch.tensor(keep, device=DEV)), q.index_select(axis, torch.tensor(keep, device=DEV)))
    for shape in ((130, 70, 21, 3, 1), (9, 1030, 140, 2, 1), (1, 9, 700, 3, 1)):  # 4, 16, 64 lanes a channel
        a, dy, *_ = scan_case(shape, F32, 0)
        got = []
        for spoiled in (False, True):
            mine = {k: v.clone().requires_grad_() for k, v in a.items() if v is not None}
            if spoiled:
                with torch.no_grad():
                    mine["tokens"][:, 4, shape[2] // 2] = bad
            y = m.fm_selective_scan(**mine)
            own = ("tokens", "delta", "gate", "A", "delta_bias")  # (write's and read's gradients are sums over the channels)
            got.append([y, *torch.autograd.grad(y, [mine[k] for k in own], dy)])
        keep = torch.tensor([d for d in range(shape[1]) if d != 4], device=DEV)
        assert not torch.isfinite(got[1][0][:, 4]).all()
        for p, q in zip(*got):
            axis = 1 if p.dim() == 3 else 0
            assert torch.equal(p.index_select(axis, keep), q.index_select(axis, keep))


# ---- norm -------------------------------------------------------------------------------------------
# sum of squares: at most 4 chunks of 8 in a thread and 10 levels, halved by the root; a few operations after it: c = 40
# the row's second sum, of products: c = 80; weight's gradient: a rounding a row in a slot (8 to rows / 512), then
# slots / 16 and 16 more

NORM_SHAPES = [(1, 1), (3, 5), (2, 64), (5, 511), (9, 513), (4, 1030), (3, 2049), (2, 4097), (2, 8193), (1, 16384), (130, 96), (600, 40)]


@pytest.fixture(scope="module")
def nm():
    import fm.scan.fm_norm as nm

    return nm


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm(nm, shape, dtype):
    T, D = shape
    g = gen(T + D)
    for variant in range(3):
        x, w = rand(g, T, D, dtype=dtype), 1 + rand(g, D, dtype=F32 if variant == 1 else dtype, scale=0.2)
        res = None if variant == 1 else rand(g, T, D, dtype=dtype, scale=3.0)
        eps = (1e-6, 0.0, 1e-2)[variant]
        dy, dr = rand(g, T, D, dtype=dtype), rand(g, T, D, dtype=dtype)
        leaves = [t.requires_grad_() for t in (x, w, res) if t is not None]
        y, r = nm.fm_norm(x, w, residual=res, eps=eps)
        stored = x if res is None else (x.float() + res.float()).to(dtype)
        assert torch.equal(r, stored)
        q, scales, rq = nm.fm_norm_quantized(x.detach(), w.detach(), residual=None if res is None else res.detach(), eps=eps)
        assert torch.equal(rq, stored)
        with_r = res is not None and variant == 0
        ref = R.norm(stored, w, eps, dy, dr if with_r else None)
        R.close(y, *ref["y"], 40, f"{shape} {dtype} y")
        grads = torch.autograd.grad([y, r] if with_r else [y], leaves, [dy, dr] if with_r else [dy])
        R.close(grads[0], *ref["dr"], 80, f"{shape} {dtype} dx")
        c = 48 + max(8, T / 512) + T / 128
        R.close(grads[1], *ref["dweight"], c, f"{shape} {dtype} dw")
        if res is not None:
            assert torch.equal(grads[2], grads[0])
        exact = ref["y"][0]
        top = exact.abs().amax(-1)
        assert ((scales.cpu().double() - top / 448).abs() <= 48 * 2.0 ** -24 * top / 448).all()
        # half a step of e4m3: 2^-4 of a normal value, 2^-10 scales of a subnormal one
        off = (q.cpu().float().double() * scales.cpu().double()[:, None] - exact).abs()
        bound = torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -10 * (top / 448)[:, None]) + 100 * 2.0 ** -24 * top[:, None]
        assert (off <= bound).all()
        assert torch.equal(q.cpu().float().abs().amax(-1), torch.full((T,), 448.0))


def test_norm_quantized_rows_without_a_scale(nm):
    """Zeros, values whose scale leaves float32, a NaN, an infinity: the other rows are as they would be alone."""
    x = torch.randn(6, 300, generator=gen(1)).to(DEV)
    alone = nm.fm_norm_quantized(x, torch.ones(300, device=DEV))
    x[1] = 0
    x[2] *= 1e-36
    x[3, 7], x[4, 9] = float("nan"), float("inf")
    q, s, _ = nm.fm_norm_quantized(x, torch.ones(300, device=DEV))
    assert s[1] == 0 and not q[1].float().any() and s[2] == 0 and not q[2].float().any()
    assert torch.isnan(s[3]) and torch.isnan(q[3].float()).all() and torch.isnan(s[4]) and torch.isnan(q[4, 9].float())
    for i in (0, 5):
        assert torch.equal(q[i].float(), alone[0][i].float()) and s[i] == alone[1][i]


def test_norm_of_a_subnormal_mean(nm):
    """Without eps, values whose mean square is subnormal: squares near 2^-132 are off by 2^-150, the root by half of that."""
    x = torch.randn(3, 300, generator=gen(5)) * 2.0 ** -66
    y, _ = nm.fm_norm(x.to(DEV), torch.ones(300, device=DEV), eps=0.0)
    exact = x.double() / x.double().pow(2).mean(-1, keepdim=True).sqrt()
    assert ((y.cpu().double() - exact).abs() <= 2.0 ** -17 * exact.abs()).all()


def test_norm_uses_of_its_outputs(nm):
    g = gen(2)
    x, res, w = rand(g, 2, 3, 50), rand(g, 2, 3, 50), rand(g, 50)
    for t in (x, res, w):
        t.requires_grad_()
    y, r = nm.fm_norm(x, w, residual=res)
    assert y.shape == r.shape == (2, 3, 50)
    dx, dw = torch.autograd.grad(r.sum(), [x, w], retain_graph=True)
    assert (dx == 1).all() and not dw.any()
    dx, dres = torch.autograd.grad((y * 2).sum() + r.sum(), [x, res])
    ref = R.norm(r, w, 1e-6, torch.full((2, 3, 50), 2.0), torch.ones(2, 3, 50))
    R.close(dx, *ref["dr"], 80, "dx")
    assert torch.equal(dx, dres)


# ---- all together -------------------------------------------------------------------------------------

def layer_weights(g, C, D, N, R_, dtype):
    w = lambda *s: rand(g, *s, dtype=dtype, scale=s[-1] ** -0.5)  # noqa: E731
    return {"norm": 1 + rand(g, C, dtype=dtype, scale=0.1), "into": w(2 * D, C), "conv": w(D, 4), "conv_bias": rand(g, D, dtype=dtype, scale=0.1),
            "x": w(R_ + 2 * N, D), "dt": w(D, R_), "dt_bias": rand(g, D) - 3, "A": -torch.exp(rand(g, D, N)), "skip": rand(g, D), "out": w(C, D)}


def block(m, nm, p, x, res, N, R_, lengths=None, conv_state=None, state=None):
    """A block of a selective model on (B, L, C): norm, projections, convolution, scan. Returns out, stream, states."""
    y, res = nm.fm_norm(x, p["norm"], residual=res)
    u, z = (p["into"] @ y.transpose(1, 2)).chunk(2, 1)  # (B, D, L) each, views of one buffer
    u, conv_state = m.fm_conv(u, p["conv"], p["conv_bias"], initial_state=conv_state, lengths=lengths, return_state=True)
    dt, write, read = (p["x"] @ u).split([R_, N, N], 1)
    y, state = m.fm_selective_scan(u, p["dt"] @ dt, p["A"], write, read, skip=p["skip"], gate=z, delta_bias=p["dt_bias"],
                                   initial_state=state, lengths=lengths, return_state=True)
    return (p["out"] @ y).transpose(1, 2).contiguous(), res, conv_state, state


def block_step(m, nm, p, x, res, N, R_, conv_state, state, slots):
    y, res = nm.fm_norm(x, p["norm"], residual=res)
    u, z = (y @ p["into"].t()).chunk(2, 1)
    u = m.fm_conv_step(u, conv_state, p["conv"], p["conv_bias"], slots=slots)
    dt, write, read = (u @ p["x"].t()).split([R_, N, N], 1)
    y = m.fm_selective_step(u, state, dt @ p["dt"].t(), p["A"], write, read, skip=p["skip"], gate=z, delta_bias=p["dt_bias"],
                            slots=slots)
    return y @ p["out"].t(), res


def test_block_for_prompts_then_tokens(m, nm):
    """A padded batch of prompts, then token by token out of a pool of states, against the whole sequences at once."""
    g = gen(31)
    B, L, C, D, N, R_ = 3, 40, 24, 48, 8, 4
    p = layer_weights(g, C, D, N, R_, F32)
    x, res = rand(g, B, L, C), rand(g, B, L, C)
    whole, stream, *_ = block(m, nm, p, x, res, N, R_)
    n = torch.tensor([17, 1, 30], dtype=torch.int32, device=DEV)
    out, _, conv_state, state = block(m, nm, p, x[:, :30].contiguous(), res[:, :30].contiguous(), N, R_, lengths=n)
    scale = whole.abs().max().item()
    # the same operations in another order through a few products of up to 48 terms: 2^-24 of each, times their number
    near = lambda a, b: (a - b).abs().max().item() < 4096 * 2.0 ** -24 * scale  # noqa: E731
    for b in range(B):
        assert near(out[b, :n[b]], whole[b, :n[b]])
    pool_c, pool_s = torch.zeros(5, D, 3, device=DEV), torch.zeros(5, D, N, device=DEV)
    slots = torch.tensor([4, 0, 2], device=DEV)
    pool_c[slots], pool_s[slots] = conv_state, state
    at = n.long().clone()
    for _ in range(9):
        rows = torch.arange(B, device=DEV)
        y, r = block_step(m, nm, p, x[rows, at].contiguous(), res[rows, at].contiguous(), N, R_, pool_c, pool_s, slots)
        assert near(y, whole[rows, at]) and torch.equal(r, stream[rows, at])
        at += 1
    assert not pool_s[[1, 3]].any() and not pool_c[[1, 3]].any()


def test_block_trains(m, nm):
    """Gradients of a whole block in float32 against differences along a direction for every weight."""
    g = gen(32)
    B, L, C, D, N, R_ = 2, 70, 16, 24, 4, 3
    p = layer_weights(g, C, D, N, R_, F32)
    x, res = rand(g, B, L, C), rand(g, B, L, C)
    for v in (*p.values(), x, res):
        v.requires_grad_()
    G1, G2 = rand(g, B, L, C), rand(g, B, L, C)

    def loss(q, x, res):
        out, stream, *_ = block(m, nm, q, x, res, N, R_)
        return (out.double() * G1.double()).sum() + (stream.double() * G2.double()).sum()

    names = [*p, "inputs", "residual"]
    values = [*p.values(), x, res]
    grads = torch.autograd.grad(loss(p, x, res), values)
    for name, v, d in zip(names, values, grads):
        along = rand(g, *v.shape)
        h = 2.0 ** -8 * v.detach().abs().mean().item()
        with torch.no_grad():
            ends = [loss({k: (w + s * h * along if k == name else w) for k, w in p.items()},
                         x + s * h * along if name == "inputs" else x, res + s * h * along if name == "residual" else res)
                    for s in (1, -1)]
        slope, want = ((ends[0] - ends[1]) / (2 * h)).item(), (d.double() * along.double()).sum().item()
        size = (d.double().pow(2).sum().sqrt() * along.double().pow(2).sum().sqrt()).item()
        # second order in h (2^-16, times derivatives of order ten) and float32 results over h: one part in 100 of the
        # gradient's size bounds both
        assert abs(slope - want) < 0.01 * size, (name, slope, want, size)


# ---- where and when they run ---------------------------------------------------------------------------

def test_other_streams(m, nm):
    a, dy, dfinal, _ = scan_case((2, 20, 300, 8, 1), BF16, 2)
    cw = rand(gen(3), 20, 4, dtype=BF16)
    for t in (a["tokens"], a["A"], a["write"]):
        t.requires_grad_()

    def work():
        u = m.fm_conv(a["tokens"], cw)
        y, s = m.fm_selective_scan(u, *[a[k] for k in ("delta", "A", "write", "read")], gate=a["gate"], return_state=True)
        n, _ = nm.fm_norm(y, cw.new_ones(300))
        grads = torch.autograd.grad([n, s], [a["tokens"], a["A"], a["write"]], [dy, dfinal])
        return [t.detach() for t in (y, s, n, *grads)]

    want = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def test_steps_in_a_graph(m, nm):
    """Single tokens captured once and replayed on changing inputs, with other work in between."""
    g = gen(41)
    B, D, N = 4, 96, 16
    a, *_ = scan_case((B, D, 1, N, 1), BF16, 0)
    one = {k: a[k][..., 0].contiguous() for k in ("delta", "gate", "write", "read")}
    x, cw, w = rand(g, B, D, dtype=BF16), rand(g, D, 4, dtype=BF16), 1 + rand(g, D, dtype=BF16, scale=0.1)
    slots = torch.tensor([3, 1, -1, 0], device=DEV)
    start_c, start_s = rand(g, 5, D, 3, dtype=BF16), rand(g, 5, D, N)
    pool_c, pool_s = start_c.clone(), start_s.clone()

    def token():
        q, s, _ = nm.fm_norm_quantized(x, w)
        u = m.fm_conv_step(x, pool_c, cw, slots=slots)
        return q, s, m.fm_selective_step(u, pool_s, one["delta"], a["A"], one["write"], one["read"], gate=one["gate"], slots=slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = token()
    xs = [rand(g, B, D, dtype=BF16) for _ in range(4)]
    pool_c.copy_(start_c), pool_s.copy_(start_s)
    want = []
    for t in xs:
        x.copy_(t)
        want.append([v.clone() for v in token()])
    last = pool_c.clone(), pool_s.clone()
    pool_c.copy_(start_c), pool_s.copy_(start_s)
    for t, w_ in zip(xs, want):
        x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for got, expect in zip(captured, w_):
            assert torch.equal(got.view(torch.uint8), expect.view(torch.uint8))
        torch.randn(1000, device=DEV).sum().item()
    assert torch.equal(pool_c, last[0]) and torch.equal(pool_s, last[1])


def test_training_step_in_a_graph(m, nm):
    g = gen(42)
    a, dy, *_ = scan_case((2, 20, 200, 8, 1), BF16, 0)
    cw, w = rand(g, 20, 4, dtype=BF16), 1 + rand(g, 200, dtype=BF16, scale=0.1)
    leaves = [a["tokens"], a["delta"], a["A"], a["write"], a["read"], a["gate"], a["delta_bias"], cw, w]

    def step():
        mine = [t.detach().requires_grad_() for t in leaves]
        u = m.fm_conv(mine[0], mine[7])
        y = m.fm_selective_scan(u, *mine[1:5], gate=mine[5], delta_bias=mine[6])
        n, _ = nm.fm_norm(y, mine[8])
        return [n, *torch.autograd.grad(n, mine, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        a["tokens"].copy_(rand(g, 2, 20, 200, dtype=BF16))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(captured, want):
            assert torch.equal(x, y)


def test_nothing_to_do(m, nm):
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    s0 = torch.ones(2, 3, 3, device=DEV)
    y, s = m.fm_conv(z(2, 3, 0), z(3, 4), initial_state=s0, return_state=True)
    assert y.shape == (2, 3, 0) and torch.equal(s, s0)
    h0 = torch.ones(2, 3, 4, device=DEV, requires_grad=True)
    y, h = m.fm_selective_scan(z(2, 3, 0), z(2, 3, 0), z(3, 4), z(2, 1, 4, 0), z(2, 1, 4, 0), initial_state=h0, return_state=True)
    assert y.shape == (2, 3, 0) and torch.equal(h, h0)
    (d,) = torch.autograd.grad(h, [h0], torch.full_like(h, 3))
    assert (d == 3).all()
    assert m.fm_selective_scan(z(0, 3, 5), z(0, 3, 5), z(3, 4), z(0, 1, 4, 5), z(0, 1, 4, 5)).shape == (0, 3, 5)
    assert m.fm_selective_step(z(0, 3), z(0, 3, 4), z(0, 3), z(3, 4), z(0, 4), z(0, 4)).shape == (0, 3)
    assert m.fm_conv_step(z(0, 3), z(0, 3, 3), z(3, 4)).shape == (0, 3)
    y, r = nm.fm_norm(z(0, 8).requires_grad_(), z(8))
    assert y.shape == (0, 8)
    q, s, _ = nm.fm_norm_quantized(z(2, 0, 8), z(8))
    assert q.shape == (2, 0, 8) and s.shape == (2, 0)


def test_broadcast_inputs_get_summed_gradients(m):
    """write and read shared by the batch, one gate for all channels: views of stride zero, whose gradients are sums."""
    g = gen(51)
    B, D, L, N = 3, 10, 150, 4
    a, dy, *_ = scan_case((B, D, L, N, 1), F32, 0)
    shared = {"write": rand(g, 1, 1, N, L), "read": rand(g, 1, 1, N, L), "gate": rand(g, B, 1, L)}
    wide = {"write": (B, 1, N, L), "read": (B, 1, N, L), "gate": (B, D, L)}
    for t in shared.values():
        t.requires_grad_()
    a.update({k: t.expand(wide[k]) for k, t in shared.items()})
    y = m.fm_selective_scan(**a)
    grads = torch.autograd.grad(y, list(shared.values()), dy)
    ref = scan_reference(a, True, dy)
    R.close(y, *ref["y"], 44, "y")
    for (k, t), got in zip(shared.items(), grads):
        axis = 1 if k == "gate" else 0
        v, mag = (x.sum(axis, keepdim=True) for x in ref[GRADS[k]])
        R.close(got, v, mag, 80 + 2 * N + 40 + D, k)  # (the sum adds at most ten roundings)


def test_offsets_beyond_32_bits(m, nm):
    """Strides, pools and outputs whose elements lie more than 2^31 apart."""
    g = gen(52)
    far = (1 << 31) + 24
    B, D, L, N = 2, 3, 40, 4
    a, *_ = scan_case((B, D, L, N, 1), BF16, 0)
    buf = torch.zeros(far + (1 << 16), dtype=BF16, device=DEV)
    def apart(t, at):  # batch element 1 lies `far` elements behind batch element 0
        shape = t.shape
        strides = [far] + [math.prod(shape[i + 1:]) for i in range(1, t.dim())]
        view = buf.as_strided(shape, strides, at)
        view.copy_(t)
        return view
    near = m.fm_selective_scan(**a)
    at, moved = 0, dict(a)
    for k in ("tokens", "delta", "gate", "write", "read"):
        moved[k] = apart(a[k], at)
        at += 4096
    assert torch.equal(m.fm_selective_scan(**moved), near)
    w = rand(g, D, 4, dtype=BF16)
    assert torch.equal(m.fm_conv(moved["tokens"], w), m.fm_conv(a["tokens"], w))
    del buf, moved
    # a pool of states of more than 2^31 values: the named slots alone are touched
    D, N = 4096, 16
    S = (1 << 31) // (D * N) + 3
    pool = torch.zeros(S, D, N, device=DEV)
    a, *_ = scan_case((2, D, 1, N, 1), BF16, 0)
    one = {k: a[k][..., 0].contiguous() for k in ("tokens", "delta", "gate", "write", "read")}
    slots = torch.tensor([S - 1, 1], device=DEV)
    small = torch.zeros(2, D, N, device=DEV)
    y = m.fm_selective_step(state=pool, A=a["A"], slots=slots, **one)
    assert torch.equal(y, m.fm_selective_step(state=small, A=a["A"], **one))
    assert torch.equal(pool[slots], small)
    pool[slots] = 0
    assert not pool.any()
    del pool
    # outputs of more than 2^31 values
    D, L = 4099, 1 << 19
    x = torch.zeros(1, D, L, dtype=BF16, device=DEV)
    x[0, -1] = rand(g, L, dtype=BF16)
    w = rand(g, D, 4, dtype=BF16)
    y = m.fm_conv(x, w)
    assert torch.equal(y[:, -1:], m.fm_conv(x[:, -1:].contiguous(), w[-1:].contiguous())) and not y[0, -2].any()
    rows = x.view(-1, 4096)
    y, _ = nm.fm_norm(rows, w.new_ones(4096))
    assert torch.equal(y[-128:], nm.fm_norm(rows[-128:].contiguous(), w.new_ones(4096))[0])


def test_calls_from_two_threads(m):
    """Two threads, each on a stream of its own: what each gets is what it gets alone."""
    import threading

    cases = [scan_case((2, 20, 300, 8, 1), BF16, 2, seed=s)[0] for s in (1, 2)]
    w = [rand(gen(s), 20, 4, dtype=BF16) for s in (1, 2)]
    work = lambda i: m.fm_selective_scan(**{**cases[i], "tokens": m.fm_conv(cases[i]["tokens"], w[i])}, return_state=True)  # noqa: E731
    want = [work(i) for i in (0, 1)]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = work(i)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not bad


def test_gradients_are_differentiable_once(m, nm):
    """create_graph gives the same gradients, and a second derivative is an error, not a wrong number."""
    g = gen(61)
    x, w = rand(g, 2, 3, 20).requires_grad_(), rand(g, 3, 4).requires_grad_()
    n = (1 + rand(g, 20, scale=0.1)).requires_grad_()
    a, *_ = scan_case((2, 3, 20, 2, 1), F32, 0)
    for out in (m.fm_conv(x, w), nm.fm_norm(x, n)[0], m.fm_selective_scan(**{**a, "tokens": x})):
        (once,) = torch.autograd.grad(out.square().sum(), [x], retain_graph=True)
        (graph,) = torch.autograd.grad(out.square().sum(), [x], create_graph=True)
        assert torch.equal(once, graph)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            graph.sum().backward()
