"""Values at the edges of what the selective layer's operators accept."""
import pytest
import torch

import selective_reference as R
from test_gpu_selective import BF16, F16, F32, gen, rand

pytestmark = pytest.mark.gpu


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
