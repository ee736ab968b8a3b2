"""CPU tests of the C ABI of attention over a prefix and of beam search: calls whose caches, pointers or strides are unlike one another.  No
compute runs here."""
from test_answers_abi import GPU_WANTED, _lib, reorder


def test_beam_reorder_takes_a_list_where_it_takes_each_cache():
    """The pieces that a cache goes in, and the limit on their number, are its own."""
    large, odd = dict(row_bytes=1 << 28), dict(row_bytes=13, stride_t=13, stride_h=104, stride_e=208)
    assert reorder([large]) in GPU_WANTED and reorder([odd]) in GPU_WANTED
    assert reorder([large, odd]) in GPU_WANTED and reorder([odd, large]) in GPU_WANTED
    too_large = dict(row_bytes=(1 << 27) + 1, tokens=8)
    for given in ([too_large], [large, too_large], [too_large, odd]):
        assert reorder(given) == _lib.ERR_TOO_LARGE
