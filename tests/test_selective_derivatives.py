"""What autograd asks of the selective layer's calls and they do not have is an error, never a derivative of zero. On the CPU: the
device test is taken out, and no kernel is launched."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

B, D, L, N = 2, 4, 8, 3


@pytest.fixture
def calls(monkeypatch):
    """name: (call, its tensors by name) of every operator; the results are not computed."""
    import fm_amd.scan.fm_norm as norm
    import fm_amd.scan.fm_selective as selective

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0

    for module in (norm, selective):
        monkeypatch.setattr(module, "_raw", Library())
        monkeypatch.setattr(module, "_gpu", lambda name, t: None)
        monkeypatch.setattr(module, "_call", lambda *args: None)
    r = torch.rand
    return {
        "conv": (selective.fm_conv, dict(inputs=r(B, D, L), weight=r(D, 4), bias=r(D), initial_state=r(B, D, 3))),
        "scan": (selective.fm_selective_scan, dict(tokens=r(B, D, L), delta=r(B, D, L), A=r(D, N), write=r(B, N, L), read=r(B, N, L),
                                                   skip=r(D), gate=r(B, D, L), delta_bias=r(D), initial_state=r(B, D, N))),
        "norm": (norm.fm_norm, dict(inputs=r(B, L, D), weight=r(D), residual=r(B, L, D))),
        "conv_step": (selective.fm_conv_step, dict(inputs=r(B, D), state=r(B, D, 3), weight=r(D, 4), bias=r(D), state_out=r(B, D, 3))),
        "step": (selective.fm_selective_step, dict(tokens=r(B, D), state=r(B, D, N), delta=r(B, D), A=r(D, N), write=r(B, N), read=r(B, N),
                                                   skip=r(D), gate=r(B, D), delta_bias=r(D), state_out=r(B, D, N))),
        "quantized": (norm.fm_norm_quantized, dict(inputs=r(B, L, D), weight=r(D), residual=r(B, L, D))),
    }


SEQUENCES = ["conv", "scan", "norm"]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", SEQUENCES)
def test_forward_mode_is_refused(calls, name, grad_mode):
    """A dual tensor requires no gradient: the tangent would be dropped."""
    call, tensors = calls[name]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        call(**tensors)  # (none of them is one)
        for k, t in tensors.items():
            with pytest.raises(NotImplementedError, match="jvp"):
                call(**{**tensors, k: forward_ad.make_dual(t, torch.ones_like(t))})
    call(**tensors)


@pytest.mark.parametrize("name", SEQUENCES)
def test_each_tensor_that_requires_a_gradient_makes_a_node(calls, name):
    call, tensors = calls[name]
    for k, t in tensors.items():
        mine = {**tensors, k: t.clone().requires_grad_()}
        out = call(**mine)
        assert (out[0] if isinstance(out, tuple) else out).requires_grad, k
        with torch.no_grad():
            out = call(**mine)
            assert not (out[0] if isinstance(out, tuple) else out).requires_grad


@pytest.mark.parametrize("name", ["conv_step", "step", "quantized"])
def test_calls_without_a_derivative_refuse_what_needs_one(calls, name):
    """As torch refuses an `out=` among tensors that require gradients."""
    call, tensors = calls[name]
    for k, t in tensors.items():
        mine = {**tensors, k: t.clone().requires_grad_()}
        with pytest.raises(RuntimeError, match="not differentiable"):
            call(**mine)
        with torch.no_grad():
            call(**mine)
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="not differentiable"):
            call(**{**tensors, k: forward_ad.make_dual(t, torch.ones_like(t))})
    version = tensors["state"]._version if "state" in tensors else 0
    with pytest.raises(RuntimeError, match="not differentiable"):
        call(**{k: v.clone().requires_grad_() if k in ("tokens", "inputs") else v for k, v in tensors.items()})
    assert "state" not in tensors or tensors["state"]._version == version  # (nothing was moved on)
    call(**tensors)


@pytest.mark.parametrize("name", SEQUENCES)
def test_a_tangent_of_the_gradient_is_refused(calls, name):
    """Forward over reverse: the output's gradient is the dual tensor."""
    call, tensors = calls[name]
    mine = {k: t.clone().requires_grad_() for k, t in tensors.items()}
    out = call(**mine)
    out = out[0] if isinstance(out, tuple) else out
    dy = torch.ones_like(out)
    torch.autograd.grad(out, list(mine.values()), dy, retain_graph=True)
    with forward_ad.dual_level():
        torch.autograd.grad(out, list(mine.values()), dy, retain_graph=True)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, list(mine.values()), forward_ad.make_dual(dy, torch.ones_like(dy)))
