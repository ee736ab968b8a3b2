"""CPU tests of the C ABI of attention over a prefix and of beam search: calls whose caches, pointers or strides are unlike one another.  No
compute runs here."""
import ctypes as C

import pytest

from test_answers_abi import GPU_WANTED, _lib, lib, prefix, prefix_args, reorder


def test_beam_reorder_takes_a_list_where_it_takes_each_cache():
    """The pieces that a cache goes in, and the limit on their number, are its own."""
    large, odd = dict(row_bytes=1 << 28), dict(row_bytes=13, stride_t=13, stride_h=104, stride_e=208)
    assert reorder([large]) in GPU_WANTED and reorder([odd]) in GPU_WANTED
    assert reorder([large, odd]) in GPU_WANTED and reorder([odd, large]) in GPU_WANTED
    too_large = dict(row_bytes=(1 << 27) + 1, tokens=8)
    for given in ([too_large], [large, too_large], [too_large, odd]):
        assert reorder(given) == _lib.ERR_TOO_LARGE


@pytest.mark.parametrize("backward", [False, True])
def test_prefix_attention_workspace_goes_by_where_operands_lie(backward):
    """Operands off 16-byte boundaries are the CUDA cores', with a workspace of their own: a query that has the call's pointers is enough, one
    that has others need not be, and the call says so."""
    room = lambda **kw: lib.na2d_prefix_attention_workspace(C.byref(prefix_args(backward, **kw)), int(backward))
    shape = dict(B=2, S=1, N=1, Nk=1, Tq=30, Tk=40, P=1 << 15, C=64, causal=0)
    odd = dict(shape, prefix_k=_lib.Heads(258, 0, 0, 0))
    assert room(**odd) != room(**shape)
    for kw in (shape, odd):
        assert prefix(backward, **kw, workspace_bytes=room(**kw)) in GPU_WANTED
        assert prefix(backward, **kw, workspace_bytes=room(**kw) - 1) == _lib.ERR_BAD_ARG
    less, more = sorted((shape, odd), key=lambda kw: room(**kw))
    assert prefix(backward, **more, workspace_bytes=room(**less)) == _lib.ERR_BAD_ARG


@pytest.mark.parametrize("backward", [False, True])
def test_prefix_attention_counts_rows_of_whole_blocks_in_32_bits(backward):
    """A block of the joins has up to 256 rows, the last one some beyond the last row."""
    rows = lambda Tq, **kw: prefix(backward, B=4, S=4, N=1, Nk=1, Tq=Tq, Tk=0, P=1, C=3, k=_lib.Heads(0, 0, 0, 0), v=_lib.Heads(0, 0, 0, 0),
                                   **(dict(d_k=_lib.Heads(0, 0, 0, 0), d_v=_lib.Heads(0, 0, 0, 0)) if backward else {}), workspace_bytes=1 << 60, **kw)
    assert rows((1 << 29) - 1) == _lib.ERR_TOO_LARGE     # 2^31 - 4
    assert rows((1 << 29) - 64) in GPU_WANTED            # 2^31 - 256
