"""Host side of the paged cache: calls that its documentation allows, or refuses, beyond the plain ones."""
import pytest
import torch

import tiga as tg


def parts(sequences=2, width=3, page_size=4, heads=2, dim=16):
    key = torch.zeros(sequences * width * page_size, heads, dim, dtype=torch.bfloat16)
    shape = (sequences, heads, width * page_size)
    return {"key": key, "value": key.clone(), "lengths": torch.zeros(sequences, dtype=torch.int32), "page_size": page_size,
            "page_table": torch.arange(sequences * width, dtype=torch.int32).reshape(sequences, width),
            "weight": torch.zeros(shape), "position": torch.zeros(shape, dtype=torch.int32),
            "seen": torch.zeros(sequences, dtype=torch.int32)}


@pytest.mark.parametrize("name", ("key", "value", "page_table", "lengths", "weight", "position", "seen", "page_size",
                                  "capacity", "sequences", "heads", "dim", "device"))
def test_what_the_kernels_read_cannot_be_exchanged(name):
    """The kernels have the tensors' addresses: another tensor in their place would be seen by the host alone."""
    cache = tg.PagedCache(**parts())
    kept = getattr(cache, name)
    other = kept + 1 if isinstance(kept, (torch.Tensor, int)) else torch.device("meta")
    with pytest.raises(AttributeError, match=name):
        setattr(cache, name, other)
    with pytest.raises(AttributeError, match=name):
        delattr(cache, name)
    assert getattr(cache, name) is kept


def test_contents_change_in_place():
    cache = tg.PagedCache(**parts())
    lengths = cache.lengths
    cache.lengths += 2                                  # an in-place addition, then the same tensor again
    assert cache.lengths is lengths and lengths.tolist() == [2, 2]
    cache.lengths[1] = 5
    assert cache.relation().resolve_csr()[0].tolist() == [0, 2, 7]


@pytest.mark.parametrize("lengths,table,what", (
    ([5, 3], [[0, 1, 2], [-1, 4, 5]], "table"), ([5, 3], [[0, 6, 2], [3, 4, 5]], "table"),
    ([13, 3], [[0, 1, 2], [3, 4, 5]], "length"), ([5, -1], [[0, 1, 2], [3, 4, 5]], "length")))
def test_a_snapshot_follows_no_contents_out_of_range(lengths, table, what):
    """What the kernels skip and report must not become indexes of the relation's snapshot either."""
    cache = tg.PagedCache(**parts())
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    cache.page_table.copy_(torch.tensor(table, dtype=torch.int32))
    for call in (cache.resolve_csr, cache.relation().resolve_csr, cache.relation().transpose,
                 cache.relation().degree_bounds):
        with pytest.raises(RuntimeError, match=what):
            call()


def test_a_snapshot_looks_at_no_page_behind_the_lengths():
    cache = tg.PagedCache(**parts())
    cache.lengths.copy_(torch.tensor([5, 0], dtype=torch.int32))
    cache.page_table.copy_(torch.tensor([[2, 1, -7], [99, 99, 99]], dtype=torch.int32))
    row_ptr, col_idx = cache.resolve_csr()
    assert row_ptr.tolist() == [0, 5, 5] and col_idx.tolist() == [8, 9, 10, 11, 4]


def test_tracked_state_does_not_follow_the_default_dtype():
    default = torch.get_default_dtype()
    try:
        for dtype in (torch.bfloat16, torch.float64):
            torch.set_default_dtype(dtype)
            cache = tg.PagedCache.empty(2, 8, 1, 16, page_size=4, device="cpu", track=True)
            assert cache.weight.dtype == torch.float32
            assert tg.rotary_frequencies(8, sections=(1, 3)).dtype == torch.float32
    finally:
        torch.set_default_dtype(default)
