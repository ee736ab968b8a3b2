"""CPU tests of the C ABI of attention over a prefix and of beam search: bad arguments are refused before any CUDA call, workspaces, and
the structures are the header's.  No compute runs here."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import e_natten_b200 as na
from e_natten_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GPU_WANTED = (_lib.ERR_CUDA, _lib.ERR_NO_DEVICE)         # past validation
lib = _lib.lib
NOTHING = _lib.Heads(0, 0, 0, 0)


def prefix_args(backward=False, **kw):
    a = _lib.PrefixAttentionArgs()
    a.struct_size = C.sizeof(_lib.PrefixAttentionArgs)
    a.B, a.S, a.N, a.Nk, a.Tq, a.Tk, a.P, a.C, a.dtype, a.path, a.device, a.causal, a.scale = 6, 2, 4, 2, 16, 32, 100, 64, 1, 0, 0, 1, 1.0
    for name in ("q", "k", "v", "prefix_k", "prefix_v", "o") + (("d_o", "d_q", "d_k", "d_v", "d_prefix_k", "d_prefix_v") if backward else ()):
        setattr(a, name, _lib.Heads(256, 0, 0, 0))       # dummy, never dereferenced
    a.lse = a.workspace = 256
    a.workspace_bytes = 1 << 40
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def prefix(backward=False, **kw):
    return (lib.na2d_prefix_attention_backward if backward else lib.na2d_prefix_attention_forward)(C.byref(prefix_args(backward, **kw)))


def select_args(**kw):
    a = _lib.BeamSelectArgs()
    a.struct_size = C.sizeof(_lib.BeamSelectArgs)
    a.B, a.K, a.V, a.count, a.dtype, a.device, a.end = 2, 4, 1000, 8, 1, 0, 3
    a.logits = a.scores = a.out_scores = a.out_parents = a.out_words = a.workspace = 256
    a.workspace_bytes = 1 << 30
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def select(**kw):
    return lib.na2d_beam_select(C.byref(select_args(**kw)))


def reorder(given=None, **kw):
    a = _lib.BeamReorderArgs()
    a.struct_size = C.sizeof(_lib.BeamReorderArgs)
    given = [dict()] if given is None else given
    table = (_lib.Cache * max(1, len(given)))()
    for entry, change in zip(table, given):
        entry.ptr, entry.stride_e, entry.stride_h, entry.stride_t, entry.heads, entry.tokens, entry.row_bytes = 256, 4096, 2048, 256, 2, 8, 256
        for name, value in change.items():
            setattr(entry, name, value)
    a.B, a.K, a.caches, a.device, a.cache, a.parents = 2, 4, len(given), 0, table, 256
    for name, value in kw.items():
        setattr(a, name, value)
    return lib.na2d_beam_reorder(C.byref(a))


@pytest.mark.parametrize("backward", [False, True])
def test_prefix_attention_refuses_bad_arguments_without_touching_cuda(backward):
    call = lambda **kw: prefix(backward, **kw)
    assert (lib.na2d_prefix_attention_backward if backward else lib.na2d_prefix_attention_forward)(None) == _lib.ERR_BAD_ARG
    for kw in (dict(struct_size=8), dict(B=-1), dict(B=0), dict(S=0), dict(S=4), dict(Tq=0), dict(P=0), dict(Tk=-1), dict(N=5), dict(Nk=0), dict(C=0),
               dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(path=9), dict(q=NOTHING), dict(prefix_v=NOTHING), dict(v=NOTHING),
               dict(o=NOTHING), dict(lse=None), dict(workspace=None), dict(workspace=264), dict(workspace_bytes=100)):
        assert call(**kw) == _lib.ERR_BAD_ARG, kw
    if backward:
        for kw in (dict(d_o=NOTHING), dict(d_k=NOTHING), dict(d_prefix_v=NOTHING), dict(Tk=0),
                   dict(d_q=NOTHING, d_k=NOTHING, d_v=NOTHING, d_prefix_k=NOTHING, d_prefix_v=NOTHING)):
            assert call(**kw) == _lib.ERR_BAD_ARG, kw
    assert call(dtype=7) == _lib.ERR_UNSUPPORTED
    assert call(C=300) == _lib.ERR_UNSUPPORTED
    assert call(dtype=0, path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert call(C=68, path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert call(prefix_k=_lib.Heads(258, 0, 0, 0), path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    strided = _lib.Heads(256, 1 << 16, 64, 256)
    assert call(**{"d_q" if backward else "o": strided}) == _lib.ERR_UNSUPPORTED
    for kw in (dict(P=(1 << 29) + 1), dict(Tk=(1 << 29) + 1), dict(Tq=1 << 28), dict(B=1 << 22, S=1 << 22, N=8, Tq=1)):
        assert call(**kw) == _lib.ERR_TOO_LARGE, kw
    assert call() in GPU_WANTED and call(device=-1) in GPU_WANTED
    assert prefix(False, Tk=0, k=NOTHING, v=NOTHING) in GPU_WANTED


@pytest.mark.parametrize("name", ["d_k", "d_v", "d_prefix_k", "d_prefix_v"])
def test_prefix_attention_asks_for_key_gradients_on_16_bytes_for_tensor_cores(name):
    assert prefix(True, **{name: _lib.Heads(258, 0, 0, 0)}, path=_lib.PATH_TENSOR) == _lib.ERR_UNSUPPORTED
    assert prefix(True, d_q=_lib.Heads(258, 0, 0, 0), path=_lib.PATH_TENSOR) in GPU_WANTED        # (written by the join, in pieces that fit)


def test_prefix_attention_workspaces():
    """Bounded by the rows and the device: the partial results of few rows do not grow with the keys."""
    room = lambda backward=0, **kw: lib.na2d_prefix_attention_workspace(C.byref(prefix_args(bool(backward), **kw)), backward)
    assert lib.na2d_prefix_attention_workspace(None, 0) == 0 and room(C=0) == 0
    assert room() > 0 and room(1) > 0
    assert room(P=1 << 20) <= 4 * room(P=1 << 14)
    rows = 6 * 4 * 16
    assert room(dtype=0) >= 2 * rows * 64 * 4            # both halves in fp32
    assert room(1) >= 2 * rows * 64 * 4
    need = room()
    assert prefix(workspace_bytes=need - 1) == _lib.ERR_BAD_ARG and prefix(workspace_bytes=need) in GPU_WANTED


def test_beam_select_refuses_bad_arguments_without_touching_cuda():
    assert lib.na2d_beam_select(None) == _lib.ERR_BAD_ARG and lib.na2d_beam_select_workspace(None) == 0
    for kw in (dict(struct_size=8), dict(B=0), dict(K=0), dict(V=0), dict(count=0), dict(count=-1), dict(end=-1), dict(end=1000), dict(logits=None),
               dict(scores=None), dict(out_scores=None), dict(out_parents=None), dict(out_words=None), dict(workspace=None), dict(workspace=260),
               dict(workspace_bytes=64)):
        assert select(**kw) == _lib.ERR_BAD_ARG, kw
    for kw in (dict(dtype=7), dict(K=33), dict(count=65)):
        assert select(**kw) == _lib.ERR_UNSUPPORTED, kw
    for kw in (dict(V=(1 << 24) + 1), dict(B=1 << 19)):
        assert select(**kw) == _lib.ERR_TOO_LARGE, kw
    assert select() in GPU_WANTED and select(device=-1) in GPU_WANTED
    need = lib.na2d_beam_select_workspace(C.byref(select_args()))
    assert need >= 2 * 4 * (8 + 8 * 8)
    assert select(workspace_bytes=need - 1) == _lib.ERR_BAD_ARG and select(workspace_bytes=need) in GPU_WANTED
    assert lib.na2d_beam_select_workspace(C.byref(select_args(V=1 << 24, B=64))) < 64 << 20


def test_beam_reorder_refuses_bad_arguments_without_touching_cuda():
    assert lib.na2d_beam_reorder(None) == _lib.ERR_BAD_ARG
    for kw in (dict(struct_size=8), dict(B=0), dict(K=0), dict(caches=-1), dict(parents=None), dict(cache=None)):
        assert reorder(**kw) == _lib.ERR_BAD_ARG, kw
    for change in (dict(ptr=None), dict(heads=0), dict(tokens=0), dict(row_bytes=0)):
        assert reorder([{}, change]) == _lib.ERR_BAD_ARG, change
    assert reorder(K=33) == _lib.ERR_UNSUPPORTED
    assert reorder(B=1 << 23) == _lib.ERR_TOO_LARGE
    assert reorder([dict(row_bytes=1 << 40)]) == _lib.ERR_TOO_LARGE
    assert reorder([dict(row_bytes=1 << 32, tokens=8)]) == _lib.ERR_TOO_LARGE
    assert reorder([dict(row_bytes=(1 << 27) + 1, tokens=8)]) == _lib.ERR_TOO_LARGE        # in single bytes
    assert reorder([]) == 0
    assert reorder(K=1) == 0                             # nothing can move
    assert reorder() in GPU_WANTED and reorder(device=-1) in GPU_WANTED


def test_structures_are_the_headers(tmp_path):
    """Sizes and offsets as a C compiler sees them."""
    structures = {"na2d_prefix_attention_args": _lib.PrefixAttentionArgs, "na2d_beam_select_args": _lib.BeamSelectArgs, "na2d_cache": _lib.Cache,
                  "na2d_beam_reorder_args": _lib.BeamReorderArgs}
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
    q = torch.zeros(2, 2, 4, 8)
    for call in (lambda: na.prefix_attention(q, q, q), lambda: na.beam_select(torch.zeros(1, 2, 3), torch.zeros(1, 2)),
                 lambda: na.beam_reorder(q, torch.zeros(1, 2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            call()
