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
    assert fwd(B=1 << 20, D=1 << 20) == code("SHAPE") and fwd(L=(1 << 30) + 1) == code("SHAPE") and fwd(sb=-1) == code("SHAPE")
    assert fwd(B=1, D=(1 << 30) + 1) == code("SHAPE") and fwd(B=1 << 15, D=1 << 15, L=1 << 11) == code("SHAPE")
    assert fwd(dtype=3) == code("DTYPE") and fwd(flags=1) == code("FLAGS") and fwd(flags=0x100) == code("FLAGS")
    assert fwd(out=P + 16) == code("ALIAS") and fwd(f=3 * P + 8) == code("ALIAS") and fwd(s=4 * P, f=4 * P) == code("ALIAS")
    assert b"overlaps" in lib.fmscan_last_error()
    assert fwd(out=2 * P + 2 * 3 * 4) == code("ALIAS") and fwd(bias=3 * P - 8) == code("ALIAS")  # float32 parameters: 48 and 12 bytes
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

    for mod in modules:
        monkeypatch.setattr(mod, "_raw", NoLaunch())
        monkeypatch.setattr(mod, "_gpu", lambda name, t: None)


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


def scan_inputs(_lib, **change):
    a = dict(tokens=P, delta=2 * P, gate=0, write=3 * P, read=4 * P, skip=0, delta_bias=0, A=5 * P, initial_state=0, lengths=0,
             tokens_strides=(24, 8), delta_strides=(24, 8), gate_strides=(24, 8), write_strides=(32, 32, 8),
             read_strides=(32, 32, 8), B=2, D=3, L=8, N=4, G=1, dtype=2, flags=0)
    return packed(_lib.SCAN_INPUTS, {**a, **{k: v or 0 for k, v in change.items()}}, len(a))


def packed(form, fields, count):
    assert len(fields) == count  # no field by a wrong name
    return form.pack(*[x for v in fields.values() for x in (v if isinstance(v, tuple) else (v,))])


def test_scan_rejects(lib):
    from fm_amd import _lib

    def fwd(out=7 * P, final=None, marks=None, ws=None, ws_bytes=0, **change):
        p = scan_inputs(_lib, **change)
        return lib.fmselective_scan_forward(p, out, final, marks, ws, ws_bytes, None)

    assert lib.fmselective_scan_forward(None, P, None, None, None, 0, None) == code("NULL")
    assert fwd(out=None) == code("NULL") and fwd(tokens=None) == code("NULL") and fwd(read=None) == code("NULL")
    assert fwd(N=0) == code("SHAPE") and fwd(N=257) == code("SHAPE") and fwd(G=2) == code("SHAPE") and fwd(L=0) == code("SHAPE")
    assert fwd(write_strides=(32, 32, -8)) == code("SHAPE") and fwd(B=1 << 30, D=4) == code("SHAPE")
    assert fwd(dtype=5) == code("DTYPE") and fwd(flags=0x4) == code("FLAGS") and fwd(flags=0x2) == code("FLAGS")
    assert fwd(out=P + 32) == code("ALIAS") and fwd(final=5 * P) == code("ALIAS") and fwd(marks=7 * P) == code("ALIAS")
    assert fwd(initial_state=6 * P, final=6 * P) == code("ALIAS")
    need = lib.fmselective_scan_workspace_bytes
    assert need(2, 3, 8, 4, 1, 2, 1) > 0 and need(2, 3, 8, 4, 2, 2, 1) == 0 and need(2, 3, 0, 4, 1, 2, 1) == 0
    assert need(2, 3, 8, 4, 1, 2, 0) == 0 and need(1, 3, 1 << 16, 4, 1, 2, 0) > 0 and need(8, 4096, 1 << 16, 4, 1, 2, 0) == 0
    long = dict(L=1 << 16, tokens_strides=(3 << 16, 1 << 16), delta_strides=(3 << 16, 1 << 16))
    assert fwd(ws=P, ws_bytes=1 << 30, **long) == code("ALIAS") and fwd(ws=7 * P + 64, ws_bytes=1 << 30, **long) == code("ALIAS")

    def bwd(ws=20 * P, ws_bytes=1 << 30, inputs={}, **change):
        g = dict(out_grad=7 * P, out_grad_strides=(24, 8), final_state_grad=0, marks=8 * P, tokens=9 * P, delta=10 * P, gate=0,
                 write=11 * P, read=12 * P, A=13 * P, initial_state=0, skip=0, delta_bias=0)
        o = packed(_lib.SCAN_GRADS, {**g, **{k: v or 0 for k, v in change.items()}}, len(g))
        return lib.fmselective_scan_backward(scan_inputs(_lib, **inputs), o, ws, ws_bytes, None)

    assert bwd(marks=None) == code("NULL") and bwd(write=None) == code("NULL")
    assert bwd(gate=14 * P) == code("NULL") and bwd(inputs=dict(skip=15 * P)) == code("NULL")
    assert bwd(ws=None) == code("WORKSPACE") and bwd(ws_bytes=64) == code("WORKSPACE") and bwd(ws=20 * P + 4) == code("WORKSPACE")
    assert bwd(tokens=7 * P) == code("ALIAS") and bwd(delta=9 * P) == code("ALIAS") and bwd(ws=13 * P) == code("ALIAS")

    def step(state=6 * P, new=6 * P, slots=None, S=2, out=7 * P, **change):
        p = scan_inputs(_lib, initial_state=state, **change)
        return lib.fmselective_scan_step(p, new, slots, S, out, None)

    assert step(state=None) == code("NULL") and step(out=None) == code("NULL")
    assert step(S=3) == code("SHAPE") and step(S=0, slots=16 * P) == code("SHAPE") and step(new=6 * P + 16) == code("ALIAS")
    # more threads than a launch counts, and strides whose span passes 64 bits
    assert step(B=1 << 24, S=1 << 24, new=1 << 50, out=1 << 52, state=1 << 50) == code("SHAPE")
    assert b"one launch" in lib.fmscan_last_error()
    assert fwd(B=1 << 20, tokens_strides=(1 << 44, 8), out=P + (1 << 50)) == code("ALIAS")
    assert step(out=6 * P) == code("ALIAS") and step(N=300) == code("SHAPE") and step(flags=0x8) == code("FLAGS")


def test_norm_rejects(lib):
    def fwd(x=P, r=None, w=2 * P, ro=None, out=3 * P, s=None, inv=None, rows=4, D=8, dtype=2, flags=0, eps=1e-6):
        return lib.fmselective_norm_forward(x, r, w, ro, out, s, inv, rows, D, dtype, flags, eps, None)

    assert fwd(x=None) == code("NULL") and fwd(r=4 * P) == code("NULL") and fwd(rows=0) == code("SHAPE") and fwd(D=16385) == code("SHAPE")
    assert fwd(eps=-1.0) == code("SHAPE") and fwd(eps=float("nan")) == code("SHAPE") and fwd(dtype=9) == code("DTYPE")
    assert fwd(flags=1) == code("FLAGS") and fwd(out=P) == code("ALIAS") and fwd(r=4 * P, ro=4 * P) == code("ALIAS")
    assert fwd(s=3 * P + 8) == code("ALIAS") and fwd(inv=2 * P) == code("ALIAS")
    assert fwd(rows=1 << 25, D=4096, x=P, out=1 << 50, w=1 << 52) == code("SHAPE") and b"one launch" in lib.fmscan_last_error()

    def bwd(dy=P, dr=None, x=2 * P, w=3 * P, inv=4 * P, g=5 * P, dw=6 * P, ws=7 * P, n=1 << 20):
        return lib.fmselective_norm_backward(dy, dr, x, w, inv, g, dw, 4, 8, 2, 0, ws, n, None)

    assert bwd(inv=None) == code("NULL") and bwd(ws=None) == code("WORKSPACE") and bwd(n=4) == code("WORKSPACE")
    assert bwd(g=P) == code("ALIAS") and bwd(dr=5 * P) == code("ALIAS") and bwd(ws=6 * P) == code("ALIAS")


def test_scan_checks_its_arguments(monkeypatch):
    import fm_amd.scan.fm_selective as m

    on_cpu(monkeypatch, [m])
    B, D, L, N = 2, 6, 8, 4
    r = torch.rand
    good = dict(tokens=r(B, D, L), delta=r(B, D, L), A=r(D, N), write=r(B, 2, N, L), read=r(B, 2, N, L), skip=r(D), gate=r(B, D, L),
                delta_bias=r(D), initial_state=r(B, D, N), lengths=torch.tensor([1, 8], dtype=torch.int32))
    refuses(m.fm_selective_scan, good, [
        (dict(tokens=r(B, L, D).transpose(1, 2)), "tokens must have a time stride"),
        (dict(delta=r(B, D, L + 1)), "delta must be"),
        (dict(delta=r(B, D, L).half()), "delta has dtype"),
        (dict(A=r(D, N).half()), "A has dtype"),
        (dict(A=r(D, 257), write=r(B, 2, 257, L), read=r(B, 2, 257, L)), "states"),
        (dict(write=r(B, 4, N, L), read=r(B, 4, N, L)), "groups"),
        (dict(read=r(B, 1, N, L)), "read must be"),
        (dict(write=r(B, N, L)), "write"),
        (dict(write=r(B, 2, L, N).transpose(2, 3)), "write must have a time stride"),
        (dict(skip=r(D + 1)), "skip must be"),
        (dict(gate=r(B, D, L).to("meta")), "gate is on meta"),
        (dict(delta_bias=r(D).double()), "delta_bias has dtype"),
        (dict(initial_state=r(B, D, N).half()), "initial_state has dtype"),
        (dict(initial_state=r(B, N, D).transpose(1, 2)), "initial_state must be contiguous"),
        (dict(lengths=torch.tensor([1, 8])), "lengths has dtype"),
    ])
    good = dict(tokens=r(B, D), state=r(5, D, N), delta=r(B, D), A=r(D, N), write=r(B, N), read=r(B, N), gate=r(B, D),
                slots=torch.tensor([0, 4]))
    refuses(m.fm_selective_step, good, [
        (dict(slots=None), "without slots"),
        (dict(slots=torch.tensor([0, 4], dtype=torch.int16)), "slots has dtype"),
        (dict(state=r(5, D, N).half()), "state has dtype"),
        (dict(state=r(5, N, D).transpose(1, 2)), "state must be contiguous"),
        (dict(state_out=r(5, D, N + 1)), "state_out must be"),
        (dict(write=r(B, N + 1)), "write must be"),
        (dict(gate=r(D, B).t()), "gate must have"),
        (dict(tokens=r(B, D, 1)), "must be"),
    ])


def test_norm_checks_its_arguments(monkeypatch):
    import fm_amd.scan.fm_norm as m

    on_cpu(monkeypatch, [m])
    r = torch.rand
    good = dict(inputs=r(2, 3, 8), weight=r(8), residual=r(2, 3, 8))
    for call in (m.fm_norm, m.fm_norm_quantized):
        refuses(call, good, [
            (dict(inputs=r(2, 8, 3).transpose(1, 2)), "inputs must be contiguous"),
            (dict(inputs=r(2, 3, 8).double()), "dtype"),
            (dict(weight=r(9)), "weight must be"),
            (dict(weight=r(8).half()), "weight has dtype"),
            (dict(residual=r(2, 3, 9)), "residual must be"),
            (dict(residual=r(2, 3, 8).half()), "residual has dtype"),
            (dict(residual=r(2, 8, 3).transpose(1, 2)), "residual must be contiguous"),
            (dict(eps=-1e-6), "eps"),
            (dict(inputs=r(1, 16385), weight=r(16385), residual=None), "16384"),
        ])
