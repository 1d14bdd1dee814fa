"""The forms of the selective layer's kernels that large calls take: rows of many tiles, blocks that walk over many rows,
states beyond one chunk and beyond 64 KiB of LDS, sums that several waves share. Against float64 (selective_reference.py)."""
import pytest
import torch

import selective_reference as R
from test_gpu_selective import BF16, DEV, F16, F32, GRADS, gen, rand, scan_case, scan_reference, spoil, strided

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m():
    import fm.scan.fm_selective as m

    assert torch.cuda.is_available(), "these tests need the GPU"
    return m


@pytest.fixture(scope="module")
def nm():
    import fm.scan.fm_norm as nm

    return nm


# ---- convolution: segments of four tiles and more ------------------------------------------------------
# A tile is 64 chunks of 16 bytes: 512 steps, in float32 256. 4096 rows and more are walked whole: 4, 6 (8, 11) tiles, the
# first four in flight together; 1024 rows in four segments of 5 (9) tiles.
# Roundings: those of a result are 32 forward (sum and silu at sums below 10) and 48 in the gradients (slope and taps); a
# parameter's gradient adds one a step of a lane (L / 64 and a chunk's 8), 6 across the lanes, and the column sums' parts
# (8 for 2 batch elements of 4 segments, 16 waves).

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(2, 2050, 2600, 4), (1, 4096, 2048, 3), (1, 1024, 8292, 2)], ids=str)
@pytest.mark.parametrize("full", [False, True], ids=["plain", "padded"])
def test_conv_rows_of_many_tiles(m, shape, dtype, full):
    B, D, L, W = shape
    g = gen(L + full)
    x, w, dy = rand(g, B, D, L, dtype=dtype), rand(g, D, W, scale=0.5), rand(g, B, D, L, dtype=dtype)
    bias = state = lengths = dfinal = None
    if full:
        bias, state, dfinal = rand(g, D, scale=0.1), rand(g, B, D, W - 1, dtype=dtype), rand(g, B, D, W - 1, dtype=dtype)
        lengths = torch.tensor([L - 1, 1801][-B:], dtype=torch.int32)
        x, dy = strided(spoil(x, lengths)), strided(spoil(dy, lengths))
        lengths = lengths.to(DEV)
    leaves = [t.requires_grad_() for t in (x, w, bias, state) if t is not None]
    y, final = m.fm_conv(x, w, bias, initial_state=state, lengths=lengths, return_state=True)
    grads = torch.autograd.grad([y, final] if full else [y], leaves, [dy, dfinal] if full else [dy])
    ref = R.conv(x, w, bias, state, lengths, True, dy, dfinal)
    R.close(y, *ref["y"], 32, "y")
    R.close(final, *ref["final"], 0, "final")
    c = 48 + L / 64 + 8 + 6 + 8 + 16
    for n, t in zip(["dx", "dweight"] + ["dbias", "dstate"] * full, grads):
        R.close(t, *ref[n], 48 if n in ("dx", "dstate") else c, n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1025, 2050])
def test_conv_step_of_several_blocks_a_row(m, D, dtype):
    g = gen(D)
    B, S, W = 5, 7, 4
    x, w, bias, pool = rand(g, B, D, dtype=dtype), rand(g, D, W, dtype=dtype, scale=0.5), rand(g, D), rand(g, S, D, W - 1, dtype=dtype)
    slots = torch.tensor([6, -1, 2, 6, 0], device=DEV)  # row 1 has no slot, row 3 names one that is taken
    rows, at = [0, 2, 4], [6, 2, 0]
    ref = R.conv(x[rows][..., None], w, bias, pool[at])
    state = pool.clone()
    y = m.fm_conv_step(x, state, w, bias, slots=slots)
    R.close(y[rows], ref["y"][0][..., 0], ref["y"][1][..., 0], 32, "y")
    assert not y[[1, 3]].any()
    pool[at] = ref["final"][0].to(dtype).to(DEV)
    assert torch.equal(state, pool)


# ---- scan ------------------------------------------------------------------------------------------------
# Roundings as in test_gpu_selective.py (40 + N forward, 80 + 2 N in the gradients); sums over channels add 2 across the
# quarters of a wave, 3 over the waves, the blocks that one wave of the last launch takes (at most 7, or a sixteenth) and the
# waves that share a sum (at most 16); sums over time 8 steps and L / 128 tiles; over batch and segments B 2 / 16 + 16.

FORMS = [  # B, D, L, N, G
    (2, 6, 100, 24, 1), (4, 1100, 150, 20, 1),       # 16 lanes a channel, two chunks of states; the second with two tiles
    (2, 6, 128, 256, 1), (1, 3, 2100, 130, 1),       # more than 64 KiB of LDS; the second cut along time in both directions
    (130, 70, 9, 140, 1),                            # 4 lanes a channel, five chunks of states
    (1, 1030, 9, 3, 1), (2, 1200, 20, 2, 2), (1, 300, 140, 3, 1), (3, 150, 17, 4, 1)]  # 16, 8, 4, 2 waves a sum of the last launch


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_selective_scan_forms(m, shape, dtype):
    B, D, L, N, G = shape
    for variant in (2, 3):
        a, dy, dfinal, softplus = scan_case(shape, dtype, variant)
        softplus = bool(softplus)
        if not softplus:
            a["delta"] = a["delta"].abs() * 0.2
        ref = scan_reference(a, softplus, dy, dfinal)
        leaves = {k: v.requires_grad_() for k, v in a.items() if v is not None and k != "lengths"}
        y, final = m.fm_selective_scan(**a, softplus=softplus, return_state=True)
        R.close(y, *ref["y"], 40 + N, f"{variant} y")
        R.close(final, *ref["final"], 40 + N, f"{variant} final")
        grads = torch.autograd.grad([y, final], list(leaves.values()), [dy, dfinal])
        c = 80 + 2 * N + 2 + 3 + 7 + 16 + 8 + L / 128 + B * 2 / 16 + 16
        for k, t in zip(leaves, grads):
            R.close(t, *ref[GRADS[k]], c, f"{variant} {GRADS[k]}")


# ---- norm: blocks that walk over several rows --------------------------------------------------------------
# Backward has at most 512 blocks, of a row or of four waves with a row each. weight's gradient: 48 roundings of a term, one a row
# of a block or wave (T / 512 and one at most), 3 over the block's waves, then 512 parts over 16 waves, 32 each, and those 16.

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(4100, 96), (2300, 600), (5000, 1030), (1541, 2049), (600, 4097), (1100, 8193)], ids=str)
def test_norm_blocks_of_many_rows(nm, shape, dtype):
    T, D = shape
    g = gen(T + D)
    x, res, dy, dr = (rand(g, T, D, dtype=dtype) for _ in range(4))
    w = 1 + rand(g, D, dtype=dtype, scale=0.2)
    leaves = [t.requires_grad_() for t in (x, w, res)]
    y, r = nm.fm_norm(x, w, residual=res)
    grads = torch.autograd.grad([y, r], leaves, [dy, dr])
    ref = R.norm(r, w, 1e-6, dy, dr)
    R.close(y, *ref["y"], 40, "y")
    R.close(grads[0], *ref["dr"], 80, "dx")
    R.close(grads[1], *ref["dweight"], 48 + T / 512 + 1 + 3 + 32 + 16, "dw")
    assert torch.equal(grads[2], grads[0])
