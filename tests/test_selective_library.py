"""What the built library holds of the selective layer's kernels."""
import re


def test_every_norm_kernel_has_rows_that_need_it():
    """A form takes rows of up to threads * chunks * 16 bytes, and the next smaller one half of that at least."""
    from fm_amd import _lib, build

    _lib.load()
    names = set(re.findall(rb"norm_(forward|backward)_kernelI(f|DF16_|DF16b)Li(\d+)ELi(\d+)E", build.LIB.read_bytes()))
    assert {n[1] for n in names} == {b"f", b"DF16_", b"DF16b"} and {n[0] for n in names} == {b"forward", b"backward"}
    for way, kind, threads, chunks in names:
        most = int(threads) * int(chunks) * (4 if kind == b"f" else 8)
        assert most // 2 < _lib.SELECTIVE_MAX_NORM, (way, kind, threads, chunks)
