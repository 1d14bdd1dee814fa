"""The selective layer's operators on the GPU against plain implementations in float64 (selective_reference.py)."""
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
               (1, 3, 511, 4), (2, 2, 513, 4), (1, 2, 2049, 4), (1, 1, 9000, 4), (700, 3, 5, 4)]


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
    (1, 33, 128, 8, 1), (2, 20, 129, 17, 1), (1, 5, 300, 33, 1), (2, 4, 513, 4, 4), (1, 2, 1100, 16, 1), (70, 2, 3, 4, 1)]


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
