"""The selective layer's entry points without a GPU: what include/fmselective.h declares is exported, and calls that
are wrong come back as errors before anything touches a GPU."""
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
HEADER = (ROOT / "include" / "fmselective.h").read_text()
CODES = (ROOT / "include" / "fmscan.h").read_text()
P = 1 << 40  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    from fm_amd import _lib

    return _lib.load()


def code(name):
    return int(re.search(r"#define\s+FMSCAN_E_%s\s+\(?(-?\w+)\)?" % name, CODES).group(1), 0)


def test_every_declared_symbol_is_exported(lib):
    names = set(re.findall(r"\b(fmselective_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)))
    assert names
    for name in names:
        assert hasattr(lib, name), name


def test_python_constants_match_the_header():
    from fm_amd import _lib

    flags = dict(re.findall(r"#define\s+FMSELECTIVE_(\w+)\s+(0x[0-9a-f]+)u", HEADER))
    assert flags
    for name, value in flags.items():
        assert getattr(_lib, "SELECTIVE_" + name) == int(value, 16), name


def test_conv_rejects(lib):
    def fwd(x=P, sb=64, sd=8, w=2 * P, bias=None, s=None, n=None, out=3 * P, f=None, B=2, D=3, L=8, W=4, dtype=2, flags=0):
        return lib.fmselective_conv_forward(x, sb, sd, w, bias, s, n, out, f, B, D, L, W, dtype, flags, None)

    assert fwd(x=None) == code("NULL") and fwd(w=None) == code("NULL") and fwd(out=None) == code("NULL")
    assert fwd(W=1) == code("SHAPE") and fwd(W=5) == code("SHAPE") and fwd(L=0) == code("SHAPE") and fwd(B=0) == code("SHAPE")
    assert fwd(B=1 << 20, D=1 << 20) == code("SHAPE") and fwd(L=1 << 31) == code("SHAPE") and fwd(sb=-1) == code("SHAPE")
    assert fwd(dtype=3) == code("DTYPE") and fwd(flags=1) == code("FLAGS") and fwd(flags=0x100) == code("FLAGS")
    assert fwd(out=P + 16) == code("ALIAS") and fwd(f=3 * P + 8) == code("ALIAS") and fwd(s=4 * P, f=4 * P) == code("ALIAS")
    assert b"overlaps" in lib.fmscan_last_error()
    need = lib.fmselective_conv_workspace_bytes
    assert need(2, 3, 8, 4, 2) == 2 * 3 * 5 * 4 and need(2, 3, 8, 5, 2) == 0 and need(2, 3, 0, 4, 2) == 0

    def bwd(x=P, dy=2 * P, w=3 * P, dx=4 * P, dw=5 * P, ws=6 * P, ws_bytes=1 << 20, ds=None, L=8):
        return lib.fmselective_conv_backward(x, 64, 8, dy, 64, 8, w, None, None, None, None, dx, dw, None, ds, 2, 3, L, 4, 2,
                                             0, ws, ws_bytes, None)

    assert bwd(dy=None) == code("NULL") and bwd(dw=None) == code("NULL") and bwd(L=0) == code("SHAPE")
    assert bwd(ws=None) == code("WORKSPACE") and bwd(ws_bytes=8) == code("WORKSPACE") and bwd(ws=6 * P + 2) == code("WORKSPACE")
    assert bwd(dx=2 * P) == code("ALIAS") and bwd(ds=4 * P + 8) == code("ALIAS") and bwd(ws=5 * P) == code("ALIAS")

    def step(x=P, s=2 * P, so=2 * P, w=3 * P, slots=None, out=4 * P, B=2, D=3, W=4, S=2, flags=0):
        return lib.fmselective_conv_step(x, 3, s, so, w, None, slots, out, B, D, W, S, 2, flags, None)

    assert step(s=None) == code("NULL") and step(S=3) == code("SHAPE") and step(S=0) == code("SHAPE") and step(W=9) == code("SHAPE")
    assert step(S=1 << 31, slots=9 * P) == code("SHAPE") and step(flags=1) == code("FLAGS")
    assert step(so=2 * P + 2) == code("ALIAS") and step(out=2 * P) == code("ALIAS") and step(out=P) == code("ALIAS")


def on_cpu(monkeypatch, modules):
    """The Python checks on CPU tensors: the device test relaxed to "the same device", no library behind it."""
    class NoLaunch:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called before the arguments were checked")

    def same_device(name, t, dev):
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, expected {dev}")

    for mod in modules:
        monkeypatch.setattr(mod, "_raw", NoLaunch())
        monkeypatch.setattr(mod, "_on_gpu", same_device)


def refuses(call, good, changes):
    for change, message in changes:
        with pytest.raises(RuntimeError, match=message):
            call(**{**good, **change})


def test_cpu_tensors_are_rejected():
    import fm.scan.fm_selective as m

    x = torch.rand(2, 3, 8)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        m.fm_conv(x, torch.rand(3, 4))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        m.fm_conv_step(x[..., 0].contiguous(), torch.rand(2, 3, 3), torch.rand(3, 4))


def test_conv_checks_its_arguments(monkeypatch):
    import fm_amd.scan.fm_selective as m

    on_cpu(monkeypatch, [m])
    B, D, L = 2, 3, 8
    good = dict(inputs=torch.rand(B, D, L), weight=torch.rand(D, 4), bias=torch.rand(D), initial_state=torch.rand(B, D, 3),
                lengths=torch.tensor([1, 8], dtype=torch.int32))
    refuses(m.fm_conv, good, [
        (dict(inputs=torch.rand(B, L, D).transpose(1, 2)), "time stride"),
        (dict(inputs=torch.rand(B, D)), "must be"),
        (dict(inputs=torch.rand(B, D, L).double()), "dtype"),
        (dict(weight=torch.rand(D, 5)), "taps"),
        (dict(weight=torch.rand(D + 1, 4)), "weight must be"),
        (dict(weight=torch.rand(D, 4).half()), "weight has dtype"),
        (dict(weight=torch.rand(4, D).t()), "weight must be contiguous"),
        (dict(bias=torch.rand(D + 1)), "bias must be"),
        (dict(bias=torch.rand(D).to("meta")), "bias is on meta"),
        (dict(initial_state=torch.rand(B, D, 4)), "initial_state must be"),
        (dict(initial_state=torch.rand(B, D, 3).half()), "initial_state has dtype"),
        (dict(lengths=torch.tensor([1, 8])), "lengths has dtype"),
        (dict(lengths=torch.tensor([1], dtype=torch.int32)), "lengths must be"),
    ])
    good = dict(inputs=torch.rand(B, D), weight=torch.rand(D, 4), state=torch.rand(5, D, 3), slots=torch.tensor([1, 0]))
    refuses(m.fm_conv_step, good, [
        (dict(slots=None), "without slots"),
        (dict(slots=torch.tensor([1.0, 0.0])), "slots has dtype"),
        (dict(slots=torch.tensor([1])), "slots must be"),
        (dict(state=torch.rand(5, D, 4)), "state must be"),
        (dict(state=torch.rand(5, D, 3).half()), "state has dtype"),
        (dict(state=torch.rand(5, 3, D).transpose(1, 2)), "state must be contiguous"),
        (dict(state_out=torch.rand(4, D, 3)), "state_out must be"),
        (dict(inputs=torch.rand(D, B).t()), "time stride"),
    ])
