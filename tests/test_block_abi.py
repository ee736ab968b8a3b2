"""CPU tests of the C ABI of group normalisation, rotary positions and attention over all keys, and of a rule of their source: bad
arguments are refused before any CUDA call, and the structures are the header's.  No compute runs here."""
import ctypes as C
import glob
import os
import re
import subprocess

import pytest
import torch

import e_natten_b200 as na
from e_natten_b200 import _lib
from test_kernel_source import CSRC, scopes_of

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GPU_WANTED = (_lib.ERR_CUDA, _lib.ERR_NO_DEVICE)         # past validation
lib = _lib.lib


def attention(backward=False, **kw):
    a = _lib.AttentionArgs()
    a.struct_size = C.sizeof(_lib.AttentionArgs)
    a.B, a.N, a.Nk, a.Tq, a.Tk, a.C, a.dtype, a.path, a.device, a.scale = 2, 4, 2, 16, 32, 64, 1, 0, 0, 1.0
    for name in ("q", "k", "v", "o") + (("d_o", "d_q", "d_k", "d_v") if backward else ()):
        setattr(a, name, _lib.Heads(256, 0, 0, 0))       # dummy, never dereferenced
    a.lse = 256
    a.delta = 256 if backward else None
    for name, value in kw.items():
        setattr(a, name, value)
    return (lib.na2d_attention_backward if backward else lib.na2d_attention_forward)(C.byref(a))


def norm(backward=False, **kw):
    a = _lib.NormArgs()
    a.struct_size = C.sizeof(_lib.NormArgs)
    a.B, a.C, a.groups, a.dtype, a.param_dtype, a.activation, a.device, a.eps, a.P = 2, 64, 8, 1, 0, 0, 0, 1e-5, 100
    a.x = a.d_y = _lib.Pixels(256, 0, 0)
    a.y = a.d_x = a.mean = a.rstd = a.workspace = 256
    a.workspace_bytes = 1 << 30
    for name, value in kw.items():
        setattr(a, name, value)
    return (lib.na2d_group_norm_backward if backward else lib.na2d_group_norm_forward)(C.byref(a))


def rotary(**kw):
    a = _lib.RotaryArgs()
    a.struct_size = C.sizeof(_lib.RotaryArgs)
    a.B, a.N, a.Nk, a.T, a.C, a.dims, a.dtype, a.device = 2, 4, 2, 16, 64, 64, 1, 0
    a.q = a.k = _lib.Heads(256, 0, 0, 0)
    a.out_q = a.out_k = a.table = 4096
    a.table_rows = 16
    for name, value in kw.items():
        setattr(a, name, value)
    return lib.na2d_rotary(C.byref(a))


@pytest.mark.parametrize("backward", [False, True])
def test_attention_refuses_bad_arguments_without_touching_cuda(backward):
    call = lambda **kw: attention(backward, **kw)
    assert (lib.na2d_attention_backward if backward else lib.na2d_attention_forward)(None) == _lib.ERR_BAD_ARG
    nothing = _lib.Heads(0, 0, 0, 0)
    for kw in (dict(struct_size=8), dict(B=-1), dict(Tq=-1), dict(Tk=-3), dict(N=5), dict(Nk=0), dict(C=0), dict(scale=0.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(path=9), dict(B=0), dict(q=nothing), dict(v=nothing), dict(lse=None)):
        assert call(**kw) == _lib.ERR_BAD_ARG, kw
    if backward:
        for kw in (dict(d_o=nothing), dict(delta=None), dict(d_k=nothing), dict(d_q=nothing, d_k=nothing, d_v=nothing)):
            assert call(**kw) == _lib.ERR_BAD_ARG, kw
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED
    assert call(C=300) == _lib.ERR_UNSUPPORTED
    assert call(dtype=0, path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert call(C=68, path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert call(q=_lib.Heads(258, 0, 0, 0), path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert call() in GPU_WANTED and call(device=-1) in GPU_WANTED


@pytest.mark.parametrize("backward", [False, True])
def test_group_norm_refuses_bad_arguments_without_touching_cuda(backward):
    call = lambda **kw: norm(backward, **kw)
    assert (lib.na2d_group_norm_backward if backward else lib.na2d_group_norm_forward)(None) == _lib.ERR_BAD_ARG
    for kw in (dict(struct_size=8), dict(B=-1), dict(P=-1), dict(groups=7), dict(groups=0), dict(C=0), dict(eps=-1.0), dict(eps=float("nan")),
               dict(activation=5), dict(B=0), dict(x=_lib.Pixels(0, 0, 0)), dict(mean=None), dict(rstd=None)):
        assert call(**kw) == _lib.ERR_BAD_ARG, kw
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED
    assert call(param_dtype=2, weight=256) == _lib.ERR_UNSUPPORTED       # fp16 parameters of a bf16 map
    assert call() in GPU_WANTED and call(device=-1) in GPU_WANTED


def test_rotary_refuses_bad_arguments_without_touching_cuda():
    assert lib.na2d_rotary(None) == _lib.ERR_BAD_ARG
    for kw in (dict(struct_size=8), dict(B=-1), dict(T=-1), dict(dims=7), dict(dims=66), dict(table=None), dict(table_rows=15),
               dict(out_q=None), dict(B=0), dict(q=_lib.Heads(0, 0, 0, 0))):
        assert rotary(**kw) == _lib.ERR_BAD_ARG, kw
    assert rotary(dtype=7) == _lib.ERR_UNSUPPORTED
    assert rotary() in GPU_WANTED and rotary(device=-1) in GPU_WANTED


def test_workspaces():
    """None where a unit has its rows and keys to itself; bounded by the device, not by the problem, where the parts lie on a line."""
    a = _lib.AttentionArgs()
    a.struct_size = C.sizeof(_lib.AttentionArgs)
    assert lib.na2d_attention_workspace(None, 0) == 0
    assert lib.na2d_attention_workspace(C.byref(a), 0) == 0              # not a problem
    n = _lib.NormArgs()
    n.struct_size = C.sizeof(_lib.NormArgs)
    assert lib.na2d_group_norm_workspace(None, 0) == 0
    assert lib.na2d_group_norm_workspace(C.byref(n), 1) == 0


def test_structures_are_the_headers(tmp_path):
    """Sizes and offsets as a C compiler sees them."""
    structures = {"na2d_heads": _lib.Heads, "na2d_attention_args": _lib.AttentionArgs, "na2d_pixels": _lib.Pixels,
                  "na2d_norm_args": _lib.NormArgs, "na2d_rotary_args": _lib.RotaryArgs}
    lines, want = [], []
    for name, mirror in structures.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(mirror))
        for field, _ in mirror._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(mirror, field).offset)
    source, program = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "na2d.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(program)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 4, 8)
    for call in (lambda: na.attention(q, q, q), lambda: na.group_norm(q, 4), lambda: na.rotary(q, q, torch.zeros(4, 4, 2)),
                 lambda: na.rotary_table(torch.arange(4), na.rotary_frequencies(8))):
        with pytest.raises(ValueError):
            call()


def test_frequencies():
    f = na.rotary_frequencies(16, base=100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([100.0 ** (-2 * i / 16) for i in range(8)], dtype=torch.float64), rtol=1e-15)
    for bad in (dict(dims=0), dict(dims=5), dict(dims=8, base=0.0), dict(dims=8, original_length=0), dict(dims=8, original_length=10, slow=3, fast=2)):
        with pytest.raises(ValueError):
            na.rotary_frequencies(**bad)


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "na2d_attn_*.cuh"))), ids=os.path.basename)
def test_a_wait_that_decides_a_branch_decides_it_for_its_warp(path):
    for call, heads in scopes_of(open(path).read(), r"\blt\.acquire(_warp)?\("):
        one_lane = any(re.search(r"\bif \(lane == 0\)\s*$", head) for head in heads)
        assert one_lane == (call == "lt.acquire(")
