"""Values at the edges of what the selective layer's operators accept."""
import pytest
import torch

import selective_reference as R
from test_gpu_selective import BF16, DEV, F16, F32, GRADS, gen, rand, scan_case, scan_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m():
    import fm.scan.fm_selective as m

    assert torch.cuda.is_available(), "these tests need the GPU"
    return m


@pytest.fixture(scope="module")
def nm():
    import fm.scan.fm_norm as nm

    assert torch.cuda.is_available(), "these tests need the GPU"
    return nm


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [5, 300, 2049, 9000])
def test_norm_of_a_row_of_zeros_without_eps(nm, D, dtype):
    """Nothing to scale: zeros, in 8 bits too, and the row adds nothing to any gradient but hands the stream's on."""
    g = gen(D)
    x, dy, dr, w = rand(g, 3, D, dtype=dtype), rand(g, 3, D, dtype=dtype), rand(g, 3, D, dtype=dtype), 1 + rand(g, D, scale=0.1)
    res = torch.zeros_like(x)
    alone, _ = nm.fm_norm(x, w, residual=res, eps=0.0)
    x[1] = 0
    leaves = [t.requires_grad_() for t in (x, w, res)]
    y, r = nm.fm_norm(x, w, residual=res, eps=0.0)
    assert not y[1].any() and torch.equal(y[[0, 2]], alone[[0, 2]])
    dx, dw, _ = torch.autograd.grad([y, r], leaves, [dy, dr])
    assert torch.equal(dx[1], dr[1])
    ref = R.norm(x[[0, 2]], w, 0.0, dy[[0, 2]], dr[[0, 2]])
    R.close(dx[[0, 2]], *ref["dr"], 80, "dx")
    R.close(dw, *ref["dweight"], 64, "dw")
    q, s, _ = nm.fm_norm_quantized(x.detach(), w.detach(), residual=res.detach(), eps=0.0)
    assert s[1] == 0 and not q[1].float().any() and (s[[0, 2]] > 0).all()


@pytest.mark.parametrize("shape", [(2, 5, 21, 3, 1), (1, 4, 300, 3, 1), (1, 2, 2700, 3, 1), (130, 70, 21, 3, 1)], ids=str)
def test_scan_states_that_forget_at_once(m, shape):
    """A of minus infinity: a state is the last step's term alone, also where rows end inside a tile. The decay is zero as it is
    for A = -1e30 (every dt here is above 1e-4), whose gradients are the formulas' with p = 0."""
    a, dy, dfinal, _ = scan_case(shape, F32, 2)
    n = torch.full((shape[0],), shape[2], dtype=torch.int32)
    n[0] -= 4
    a["lengths"] = n.to(DEV)
    a["A"][0, 1] = a["A"][1, 2] = -1e30
    ref = scan_reference(a, True, dy, dfinal)
    a["A"][0, 1] = a["A"][1, 2] = float("-inf")
    leaves = {k: v.requires_grad_() for k, v in a.items() if v is not None and k != "lengths"}
    y, final = m.fm_selective_scan(**a, return_state=True)
    R.close(y, *ref["y"], 43, "y")
    R.close(final, *ref["final"], 43, "final")
    grads = torch.autograd.grad([y, final], list(leaves.values()), [dy, dfinal])
    for k, t in zip(leaves, grads):
        R.close(t, *ref[GRADS[k]], 80 + 6 + 24 + 16 + shape[2] / 128 + shape[0], GRADS[k])


def test_step_of_length_zero_of_a_state_that_forgets_at_once(m):
    g = gen(7)
    x, w, r, state = rand(g, 2, 3), rand(g, 2, 4), rand(g, 2, 4), rand(g, 2, 3, 4)
    A, dt = torch.full((3, 4), float("-inf"), device=DEV), rand(g, 2, 3).abs() + 0.1
    dt[0] = 0
    before = state.clone()
    y = m.fm_selective_step(x, state, dt, A, w, r, softplus=False)
    assert torch.equal(state[0], before[0]) and torch.isfinite(y).all()
    assert torch.equal(state[1], (dt[1] * x[1])[:, None] * w[1])
