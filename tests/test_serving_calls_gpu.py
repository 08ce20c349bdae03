"""Paged cache and head rotation: calls that their documentation allows, or refuses, beyond the plain ones."""
import pytest
import torch

import tiga as tg
from test_cache_gpu import Attention, make, slots

pytestmark = pytest.mark.gpu


def run_threads(*bodies):
    """Every body in a thread and on a stream of its own; the first exception is raised again."""
    import threading

    errors = []

    def run(body):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                body()
        except Exception as error:                      # noqa: BLE001
            errors.append(error)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(body,)) for body in bodies]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]


def test_two_threads_evict_caches_of_different_sizes():
    """The selection keeps ranks in as much shared memory as the capacity asks for, 32 KB and 160 KB here. (The entry
    point itself is called, so that the threads are in it most of the time.)"""
    caches = [tg.PagedCache.empty(1, places, 1, 8, track=True) for places in (8000, 40000)]
    statuses = []
    for cache in caches:
        cache.lengths.fill_(100)
        cache.evict(200)

    def body(cache):
        def run():
            scratch = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
            arguments = (cache._address, None, 200, 0, scratch.data_ptr(), scratch.numel(),
                         torch.cuda.current_stream().cuda_stream)
            evict = cache._lib.tgb_cache_evict
            statuses.extend({evict(*arguments) for _ in range(20000)})
            torch.cuda.current_stream().synchronize()
        return run

    run_threads(*(body(cache) for cache in caches))
    for cache in caches:
        cache.check()
        assert cache.lengths.tolist() == [100]
    assert statuses == [0, 0]


def test_two_threads_rotate_heads_of_different_sizes():
    """Heads above 256 values are staged in shared memory, 50 KB and 64 KB here."""
    from tiga import _native, rotary

    positions, statuses = torch.zeros(1, device="cuda", dtype=torch.int64), []

    def body(dim):
        x, frequencies = torch.ones(1, 1, dim, device="cuda"), tg.rotary_frequencies(dim, device="cuda")
        assert torch.equal(tg.norm_rotary(x, None, positions, frequencies, eps=None), x)

        def run():
            out = torch.zeros_like(x)
            block = rotary._pack(x, None, None, (out, None), None, None, positions, frequencies, None, False)
            forward, stream = _native.lib().tgb_norm_rotary_fwd, torch.cuda.current_stream().cuda_stream
            statuses.extend({forward(block, stream) for _ in range(20000)})
            torch.cuda.current_stream().synchronize()
            assert torch.equal(out, x)
        return run

    run_threads(body(800), body(1024))
    assert statuses == [0, 0]


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode derivative: an input that carries a tangent is refused, not taken without it."""
    import torch.autograd.forward_ad as forward_ad

    cache, _ = make([5, 6], 2, 64, 16, torch.bfloat16, 1, capacity=32, spare=0.0)
    row = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    positions, frequencies = torch.zeros(2, device="cuda", dtype=torch.int64), tg.rotary_frequencies(64, device="cuda")
    weight = torch.ones(64, device="cuda")
    lengths = cache.lengths.tolist()
    with forward_ad.dual_level():
        dual, dual_weight = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (row, weight))
        dual_wide, dual_slots = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (row.new_zeros(2, 2, 67), cache.key))
        dual_frequencies = forward_ad.make_dual(frequencies, torch.ones_like(frequencies))
        for call in (
            lambda: cache.attend(dual), lambda: cache.append(dual, row), lambda: cache.append(row, dual),
            lambda: cache.append(dual_wide[:, :, 3:], row), lambda: cache.attend(dual_wide[:, :, 3:]),
            lambda: cache.over(dual_slots, cache.value),
            lambda: Attention()(graph=cache.relation(), src={"key": cache.key, "value": cache.value}, dst={"query": dual},
                                scale=1.0),
            lambda: tg.norm_rotary(dual, row, positions, frequencies),
            lambda: tg.norm_rotary(row, dual, positions, frequencies),
            lambda: tg.norm_rotary(row, row, positions, frequencies, query_weight=dual_weight),
            lambda: tg.norm_rotary(row, row, positions, frequencies, key_weight=dual_weight),
            lambda: tg.norm_rotary(row, row, positions, dual_frequencies),
            lambda: tg.norm_rotary(dual.detach().requires_grad_(), dual, positions, frequencies),
        ):
            with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                call()
            with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                call()
        assert cache.lengths.tolist() == lengths
        # without a tangent a call inside the level is like any other
        got = cache.attend(row), *tg.norm_rotary(row, row, positions, frequencies, query_weight=weight)
    want = cache.attend(row), *tg.norm_rotary(row, row, positions, frequencies, query_weight=weight)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
