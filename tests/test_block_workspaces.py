"""CPU tests of the workspaces of attention over all keys and of group norm: how many bytes a problem asks for."""
import ctypes as C

import pytest

from e_natten_b200 import _lib

lib = _lib.lib
SMS, ROWS = 148, 128                                     # (without a device the library counts a B200's)
BF16, F16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32


def attention(B, N, Nk, Tq, Tk, channels, dtype=BF16, causal=False, backward=False, halves="qkv", path=0):
    a = _lib.AttentionArgs()
    a.struct_size = C.sizeof(a)
    a.B, a.N, a.Nk, a.Tq, a.Tk, a.C, a.dtype, a.causal, a.path, a.scale = B, N, Nk, Tq, Tk, channels, dtype, causal, path, 1.0
    for name in ("q", "k", "v", "o", "d_o") + tuple("d_" + x for x in halves):
        setattr(a, name, _lib.Heads(256, 0, 0, 0))       # dummy, never dereferenced
    return lib.na2d_attention_workspace(C.byref(a), backward)


def norm(B, P, channels, groups, dtype=F32, backward=False):
    a = _lib.NormArgs()
    a.struct_size = C.sizeof(a)
    a.B, a.C, a.groups, a.dtype, a.param_dtype, a.P, a.eps = B, channels, groups, dtype, F32, P, 1e-5
    a.x = _lib.Pixels(256, 0, 0)
    return lib.na2d_group_norm_workspace(C.byref(a), backward)


def test_no_parts_no_workspace():
    """CUDA cores; a tile of keys; more tiles than groups; causal calls with more tiles than SMs."""
    assert attention(2, 4, 2, 300, 5000, 64, F32) == attention(2, 4, 2, 300, 5000, 64, F32, backward=True) == 0
    assert attention(2, 4, 2, 300, 5000, 64, BF16, path=_lib.PATH_SIMT) == 0
    assert attention(4, 8, 8, 1, 128, 64) == 0
    assert attention(16, 16, 16, 256, 256, 64) == 0
    assert attention(8, 8, 8, 4096, 4096, 64, causal=True, backward=True) == 0


@pytest.mark.parametrize("Tk", [1 << 14, 1 << 17, 1 << 20])
def test_on_a_line_the_device_bounds_it(Tk):
    """Whatever the number of keys: at most two parts a CTA or a group, and one for each unit."""
    rows = (2 * SMS + 8) * 4 * 129 * 4
    assert 0 < attention(4, 8, 2, 1, Tk, 128) <= rows
    assert 0 < attention(1, 2, 2, 40, Tk, 128) <= (2 * SMS + 2) * 40 * 129 * 4
    assert attention(2, 8, 2, 300, Tk, 128, backward=True, halves="q") == 2 * SMS * ROWS * 128 * 4
    assert attention(2, 8, 2, 300, Tk, 128, backward=True) in (2 * SMS * ROWS * 128 * 4, 2 * 2 * SMS * ROWS * 128 * 4)


def test_fp16_keeps_its_rows_norms_there():
    for shape in ((2, 4, 2, 300, 5000, 64), (1, 2, 1, 77, 90, 128), (16, 16, 16, 196, 196, 64)):
        for halves in ("qkv", "q", "kv"):
            B, N, Nk, Tq = shape[:4]
            more = attention(*shape, F16, backward=True, halves=halves) - attention(*shape, BF16, backward=True, halves=halves)
            assert 0 <= more - 4 * (B * N * Tq + 2 * B * Nk) <= 24
            assert attention(*shape, F16) == attention(*shape, BF16)


def test_group_norm():
    """None for a forward on the chip or of wide groups, the entries' channel sums for such a backward; in two passes what the device
    bounds."""
    assert norm(4, 49, 64, 8) == 0 and norm(4, 49, 64, 8, backward=True) == 4 * 64 * 8
    assert norm(2, 100, 1542, 1) == 0 and norm(2, 100, 1542, 1, backward=True) == 2 * 1542 * 8
    for P in (1 << 16, 1 << 20, 1 << 24):
        assert 0 < norm(2, P, 256, 16) <= 3 * SMS * 256 * 8 + 4096
        assert 0 < norm(2, P, 256, 16, backward=True) <= 3 * SMS * 256 * 8 + 4096 + SMS * 256 * 8
