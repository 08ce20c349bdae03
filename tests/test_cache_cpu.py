"""Host side of the paged cache and of norm_rotary: argument checks, the relation, the helper tables."""
import pytest
import torch

import tiga as tg
from tiga import _native


def parts(pages=6, page_size=4, heads=2, dim=16, sequences=2, width=3, dtype=torch.bfloat16):
    key = torch.zeros(pages * page_size, heads, dim, dtype=dtype)
    return {"key": key, "value": key.clone(), "page_table": torch.arange(sequences * width, dtype=torch.int32).reshape(
        sequences, width), "lengths": torch.zeros(sequences, dtype=torch.int32), "page_size": page_size}


def tracked(given):
    sequences, width = given["page_table"].shape
    shape = (sequences, given["key"].shape[1], width * given["page_size"])
    return {**given, "weight": torch.zeros(shape), "position": torch.zeros(shape, dtype=torch.int32),
            "seen": torch.zeros(sequences, dtype=torch.int32)}


def test_cache_accepts_views_and_reports_its_sizes():
    given = tracked(parts())
    both = torch.zeros(24, 2, 2, 16, dtype=torch.float16)          # keys and values side by side
    cache = tg.PagedCache(both[:, 0], both[:, 1], given["page_table"], given["lengths"], page_size=4)
    assert (cache.sequences, cache.capacity, cache.heads, cache.dim, cache.tracked) == (2, 12, 2, 16, False)
    assert tg.PagedCache(**given).tracked
    made = tg.PagedCache.empty(3, 5, 2, 8, page_size=4, device="cpu", track=True)
    assert made.capacity == 8 and made.weight.shape == (3, 2, 8) and made.page_table.tolist() == [[0, 1], [2, 3], [4, 5]]


@pytest.mark.parametrize("change,error", (
    ({"page_size": 0}, ValueError),
    ({"page_size": 5}, ValueError),                                            # 24 slots are no whole pages
    ({"key": torch.zeros(24, 2, 16)}, NotImplementedError),                    # float32
    ({"key": torch.zeros(24, 2, 8, dtype=torch.bfloat16)}, ValueError),        # not the value's shape
    ({"page_table": torch.zeros(2, 3, dtype=torch.int64)}, ValueError),
    ({"page_table": torch.zeros(3, 2, dtype=torch.int32).t()}, ValueError),    # not contiguous
    ({"page_table": torch.zeros(3, 3, dtype=torch.int32)}, ValueError),        # lengths of another count
    ({"lengths": torch.zeros(2, dtype=torch.int64)}, ValueError),
    ({"key": torch.zeros(24, 2, 20, dtype=torch.bfloat16), "value": torch.zeros(24, 2, 20, dtype=torch.bfloat16)},
     NotImplementedError),                                                     # 20 is no multiple of 8
    ({"key": torch.zeros(24, 2, 264, dtype=torch.bfloat16), "value": torch.zeros(24, 2, 264, dtype=torch.bfloat16)},
     NotImplementedError),
    ({"key": torch.zeros(24, 2, 17, dtype=torch.bfloat16)[:, :, :16]}, ValueError),      # rows not 16-byte aligned
    ({"key": torch.zeros(24, 2, 16, dtype=torch.bfloat16, requires_grad=True)}, NotImplementedError),
))
def test_cache_refuses_what_the_kernels_cannot_read(change, error):
    with pytest.raises(error):
        tg.PagedCache(**{**parts(), **change})


@pytest.mark.parametrize("change", (
    {"weight": None}, {"seen": torch.zeros(3, dtype=torch.int32)}, {"weight": torch.zeros(2, 2, 11)},
    {"position": torch.zeros(2, 2, 12)},
))
def test_tracked_state_comes_together_and_fits(change):
    with pytest.raises(ValueError):
        tg.PagedCache(**{**tracked(parts()), **change})


def test_cpu_cache_is_refused_not_emulated():
    cache = tg.PagedCache(**parts())
    row = torch.zeros(2, 2, 16, dtype=torch.bfloat16)
    for call in (lambda: cache.append(row, row), lambda: cache.attend(row), lambda: cache.evict(4), cache.check):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError):
        tg.norm_rotary(row, row, torch.zeros(2, dtype=torch.int64), tg.rotary_frequencies(16))


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


def test_relation_follows_the_cache():
    cache = tg.PagedCache(**parts())
    cache.page_table.copy_(torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32))
    relation = cache.relation()
    assert relation is cache.relation() and relation.num_src == 24 and relation.num_dst == 2
    assert relation.degree_bounds() == (0, 0)
    cache.lengths.copy_(torch.tensor([5, 0], dtype=torch.int32))
    row_ptr, col = relation.resolve_csr()
    assert row_ptr.tolist() == [0, 5, 5] and col.tolist() == [16, 17, 18, 19, 4]
    assert relation.degree_bounds() == (0, 5)
    cache.lengths.copy_(torch.tensor([1, 6], dtype=torch.int32))
    assert relation.resolve_csr()[1].tolist() == [16, 8, 9, 10, 11, 20, 21]
    assert relation.transpose().num_dst == 24 and relation.degree_statistics() == (1, 6, 7)
    with pytest.raises(NotImplementedError):
        relation.native_plan(transpose=False)
    with pytest.raises(NotImplementedError):
        relation.halo(tg.DeviceMesh("cpu", 2))


def test_reference_evaluator_over_the_relation():
    cache = tg.PagedCache(**parts())
    gen = torch.Generator().manual_seed(0)
    cache.key.copy_(torch.randn(cache.key.shape, generator=gen))
    cache.value.copy_(torch.randn(cache.value.shape, generator=gen))
    cache.lengths.copy_(torch.tensor([7, 0], dtype=torch.int32))
    query = torch.randn(2, 2, 16, generator=gen).to(torch.bfloat16)
    out = Attention().reference(graph=cache.relation(), src={"key": cache.key, "value": cache.value},
                                dst={"query": query}, scale=0.25)
    k, v = cache.key[:7].float(), cache.value[:7].float()
    p = torch.softmax(torch.einsum("hd,thd->ht", query[0].float(), k) * 0.25, dim=-1)
    torch.testing.assert_close(out[0].float(), torch.einsum("ht,thd->hd", p, v), rtol=2e-2, atol=2e-2)
    assert bool((out[1] == 0).all())


def test_relation_does_not_outlive_or_hold_its_cache():
    import gc
    import weakref

    gc.disable()
    try:
        cache = tg.PagedCache(**parts())
        watch = weakref.ref(cache)
        cache.relation()
        del cache
        assert watch() is None                      # no reference cycle: memory is free at once
    finally:
        gc.enable()


def test_rotary_frequencies():
    plain = tg.rotary_frequencies(8)
    torch.testing.assert_close(plain, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    split = tg.rotary_frequencies(8, sections=(1, 0, 3))
    assert split.shape == (3, 4) and torch.equal(split.sum(0), plain) and bool((split[1] == 0).all())
    for bad in ({"dim": 7}, {"dim": 0}, {"dim": 8, "sections": (2, 1)}, {"dim": 8, "sections": (5, -1)},
                {"dim": 8, "base": 0.0}):
        with pytest.raises(ValueError):
            tg.rotary_frequencies(**bad)


def test_native_argument_errors_without_gpu():
    lib = _native.lib()
    import ctypes

    assert lib.tgb_norm_rotary_fwd(None, 0) == _native.INVALID_ARGUMENT

    def block(dim, pairs, axes, bits=64, dtype=0):
        return _native.NORM_ROTARY.pack(*[0] * 18, 1, 1, 1, dim, pairs, axes, bits, dtype, dtype, 1, 0, 1e-6)

    assert lib.tgb_norm_rotary_fwd(block(2000, 0, 1), 0) == _native.UNSUPPORTED
    assert lib.tgb_norm_rotary_fwd(block(8, 5, 1), 0) == _native.INVALID_ARGUMENT
    assert lib.tgb_norm_rotary_fwd(block(8, 4, 1, bits=16), 0) == _native.INVALID_ARGUMENT
    assert lib.tgb_norm_rotary_fwd(block(8, 4, 1, dtype=7), 0) == _native.UNSUPPORTED
    assert lib.tgb_norm_rotary_fwd(block(8, 4, 1), 0) == _native.INVALID_ARGUMENT          # null fields
    assert lib.tgb_norm_rotary_bwd(block(8, 4, 9), None, None, None, 0, 0) == _native.UNSUPPORTED
    assert lib.tgb_norm_rotary_scratch_bytes(0) == 0
    size = ctypes.c_uint64()
    assert lib.tgb_cache_attend_scratch_bytes(None, 8, 0, ctypes.byref(size)) == _native.INVALID_ARGUMENT
    block = _native.PagedCacheArguments(dtype=_native.DTYPE_F32)
    assert lib.tgb_cache_evict_scratch_bytes(ctypes.addressof(block), 8, ctypes.byref(size)) == _native.UNSUPPORTED
    block = _native.PagedCacheArguments(key=16, value=16, fault=16, num_pages=1, page_size=4, pages_per_sequence=1,
                                        page_table=16, lengths=16, sequences=1, heads=2, dim=16,
                                        dtype=_native.DTYPE_BF16)
    assert lib.tgb_cache_evict_scratch_bytes(ctypes.addressof(block), 8, ctypes.byref(size)) == _native.OK
    assert lib.tgb_cache_evict(ctypes.addressof(block), None, 8, 0, None, 0, 0) == _native.INVALID_ARGUMENT
    assert b"track" in lib.tgb_last_error()
    for change in ({"dim": 20}, {"heads": 0}, {"num_pages": 0}, {"key": 8}, {"key_head_stride": 4}, {"weight": 16}):
        broken = _native.PagedCacheArguments.from_buffer_copy(block)
        for name, value in change.items():
            setattr(broken, name, value)
        assert lib.tgb_cache_append(ctypes.addressof(broken), 16, 16, 32, 16, 32, 16, 1, None, None, 0) != _native.OK
