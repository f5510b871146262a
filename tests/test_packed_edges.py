"""Corners of the paged caches' C-ABI, on the CPU (no kernel runs)."""
import ctypes

from prism_amd import _lib


def test_both_appends_check_alike():
    """The two entry points differ in their amplitude's type alone."""
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    st, cs = (ctypes.c_int64 * 4)(*[64] * 4), (ctypes.c_int64 * 6)(*[64] * 6)
    ps, ends = (ctypes.c_int64 * 2)(1, 1), (ctypes.c_int32 * 4)(32)

    def append(f, dtype=1, T=4, D=64, page=16, R=64, inter=1, pos=None, axes=1):
        return f(one, one, dtype, T, 2, D, st, one, one, 16, 4, page, cs, one, 2, 2, one, 2, None, one, R, inter, pos, 0, ps, axes,
                 ends, 1.25, None)

    for f in (lib.prism_paged_append, lib.prism_paged_append_f64):
        assert append(f, T=0) == 0
        assert [append(f, dtype=0), append(f, T=3), append(f, D=96), append(f, page=24), append(f, R=63), append(f, R=24, inter=0),
                append(f, pos=one, axes=5), append(f, pos=one, R=32)] == [1] * 8
