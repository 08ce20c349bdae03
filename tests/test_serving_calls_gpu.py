"""Paged cache and head rotation: calls that their documentation allows, or refuses, beyond the plain ones."""
import pytest
import torch

import test_cache_gpu as plain
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


def one_place_ahead(places, dtype, ahead, at, roomy):
    """`places` places of which the one `at` has a score `ahead` larger (base 2) than the others' 0; a query and a scale."""
    cache, _ = make([places], 1, 64, 64, dtype, 3, capacity=200000 if roomy else None)
    rows = slots(cache, 0, places)
    cache.key[rows] = 0
    cache.key[rows[at], 0, 0] = 1
    cache.value[rows] = 0
    query = torch.zeros(1, 1, 64, device="cuda", dtype=dtype)
    query[0, 0, 0] = 1
    return cache, rows, query, ahead * 0.6931471805599453


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("ahead", (30, 39, 60, 100))
@pytest.mark.parametrize("places,at", ((3, 0), (700, 699), (700, 5), (5000, 64)))
@pytest.mark.parametrize("roomy", (False, True))
def test_infinite_values_of_places_with_small_weights(dtype, ahead, places, at, roomy):
    """A place whose weight float32 holds, however small, takes its infinite value into the column; the others do not."""
    cache, rows, query, scale = one_place_ahead(places, dtype, ahead, at, roomy)
    near = at + 1 if at + 1 < places else at - 1           # of the same warp, mostly
    cache.value[rows[near], 0, 7] = float("inf")
    cache.value[rows[near], 0, 40] = -float("inf")
    cache.value[rows[at], 0, 9] = 2
    want = torch.zeros(64, device="cuda", dtype=dtype)
    want[7], want[40], want[9] = float("inf"), -float("inf"), 2
    assert torch.equal(cache.attend(query, scale)[0, 0], want)


@pytest.mark.parametrize("dtype,largest", ((torch.bfloat16, 2.0 ** 110), (torch.float16, 65504.0)))
@pytest.mark.parametrize("places", (300, 70000))
def test_places_without_weight_add_nothing(dtype, largest, places):
    """Scores of -inf, and scores that float32 has no weight for: large values add exactly 0."""
    cache, rows, query, scale = one_place_ahead(places, dtype, 200, 17, False)
    others = torch.cat([rows[:17], rows[18:]])
    cache.value[others] = largest
    cache.value[rows[17]] = 0
    assert bool((cache.attend(query, scale) == 0).all())
    cache.key[others, 0, 0] = -float("inf")
    assert bool((cache.attend(query, 1.0) == 0).all())


def test_places_with_next_to_no_weight_add_next_to_nothing():
    """fp16 parts of a weight are multiples of 2^-39 of the largest one, and neither is 0 where the weight is not: a
    weight below that is held as 2^-38 at most, 2^-38 too much. 70000 places of the largest value, all of weight
    2^-100, then add no more than 70000 * 2^-38 * 65504 = 0.0167."""
    cache, rows, query, scale = one_place_ahead(70000, torch.float16, 100, 17, False)
    cache.value[rows] = 65504
    cache.value[rows[17]] = 0
    got = cache.attend(query, scale).double()
    assert bool((got >= 0).all()) and bool((got <= 70000 * 2.0 ** -38 * 65504).all())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("places", (2, 700, 70000))
@pytest.mark.parametrize("accumulate", (False, True))
def test_averages_of_the_largest_values_are_finite(dtype, places, accumulate):
    """n equal weights of the type's largest value: the numerator is held with room for 2^24 of them. (The result is off
    by a rounding, and by n + 64 additions in float32.)"""
    cache, _ = make([places], 1, 64, 64, dtype, 3, track=True)
    rows, largest = slots(cache, 0, places), torch.finfo(dtype).max
    cache.key[rows] = 0
    cache.value[rows] = largest
    cache.value[rows, 0, 1] = -largest
    cache.weight.zero_()
    got = cache.attend(torch.ones(1, 3, 64, device="cuda", dtype=dtype), accumulate=accumulate).double()
    want = torch.full_like(got, largest)
    want[:, :, 1] = -largest
    half = torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= (half + (places + 64) * 2.0 ** -23) * largest).all())
    if accumulate:
        weight = cache.weight[0, 0, :places].double()
        assert bool(((weight - 3 / places).abs() <= 3 / places * (places + 64) * 2.0 ** -23).all())


@pytest.mark.parametrize("places", (300, 70000))
def test_the_largest_values_of_places_without_weight_add_nothing(places):
    cache, rows, query, scale = one_place_ahead(places, torch.bfloat16, 200, 17, False)
    cache.value[rows] = torch.finfo(torch.bfloat16).max
    cache.value[rows[17]] = 0
    assert bool((cache.attend(query, scale) == 0).all())


@pytest.mark.parametrize("bounds", ([0, 30, 10, 40], [0, 10, 20, 41], [-1, 10, 20, 40], [40, 0, 0, 0]))
def test_runs_that_overlap_or_leave_the_tokens_are_reported(bounds):
    """Bounds that run backwards would move lengths over places that no token was written to."""
    cache = tg.PagedCache.empty(3, 64, 2, 64, page_size=16)
    rows = torch.ones(40, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache.append(rows, rows, cu_seqlens=torch.tensor(bounds, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        cache.check()
    lengths = cache.lengths.clone()
    assert bool(((0 <= lengths) & (lengths <= 64)).all())
    cache.append(rows[:0], rows[:0], cu_seqlens=torch.zeros(4, device="cuda", dtype=torch.int32))
    cache.append(rows, rows, cu_seqlens=torch.tensor([3, 3, 8, 8], device="cuda", dtype=torch.int32))
    cache.check()
    assert torch.equal(cache.lengths, lengths + torch.tensor([0, 5, 0], device="cuda", dtype=torch.int32))


def test_a_fault_is_reported_by_the_cache_it_happened_in():
    def fresh():
        return make([10, 20], 2, 64, 16, torch.bfloat16, 3, capacity=32, spare=0.0)[0]

    bad, good = fresh(), fresh()
    row = torch.ones(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    want = good.attend(row)
    bad.page_table[0, 0] = -1
    bad.attend(row)
    torch.cuda.synchronize()
    assert torch.equal(good.attend(row), want)
    good.append(row, row)
    good.check()
    with pytest.raises(RuntimeError, match="table"):
        bad.check()
    # a later layer under the same table reports to the cache whose table it is
    layer = Attention()
    layer(graph=bad.relation(), src={"key": good.key, "value": good.value}, dst={"query": row}, scale=1.0)
    torch.cuda.synchronize()
    good.check()
    with pytest.raises(RuntimeError, match="table"):
        bad.attend(row)
    other = bad.over(good.key, good.value)
    bad.attend(row)
    with pytest.raises(RuntimeError, match="table"):
        other.check()
    # an eviction's faults: of the cache it reads, and of the one it writes
    source = make([40, 20], 2, 64, 16, torch.bfloat16, 3, capacity=48, spare=0.0, track=True)[0]
    into = tg.PagedCache.empty(2, 32, 2, 64, page_size=16)
    into.page_table[1, 0] = 10 ** 9
    source.evict(24, into=into)
    source.check()
    with pytest.raises(RuntimeError, match="table"):
        into.check()


def test_caches_that_come_and_go_report_no_faults_of_others():
    row = torch.ones(1, 1, 8, device="cuda", dtype=torch.bfloat16)
    for i in range(3000):
        cache = tg.PagedCache.empty(1, 1, 1, 8, page_size=1)
        if i % 3 == 0:
            cache.page_table.fill_(-1)
        cache.append(row, row)
        if i % 7 == 0:
            if i % 3 == 0:
                with pytest.raises(RuntimeError, match="table"):
                    cache.check()
            else:
                cache.check()


class Counted(Attention):
    staged = 0

    def edge(self, src, dst, edge, scale):
        type(self).staged += 1
        return super().edge(src, dst, edge, scale)


def test_one_layer_object_over_many_caches():
    """The program is staged once for all relations that differ only in the caches they stand for."""
    class Layer(Counted):
        pass

    layer = Layer()
    made = [make([30 + i, 500], 2, 64, (16, 32)[i % 2], torch.bfloat16, i, capacity=512)[0] for i in range(12)]
    # the same number of slots, whatever the page size
    slots_of = {cache.key.shape for cache in made}
    query = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    relations = [cache.relation() for cache in made]
    for turn in range(3):
        for cache, relation in zip(made, relations):
            out = layer(graph=relation, src={"key": cache.key, "value": cache.value}, dst={"query": query}, scale=0.125)
            assert torch.equal(out, cache.attend(query, 0.125))
        if turn == 0:
            first = Layer.staged
    assert Layer.staged == first and first <= 2 * len(slots_of)
    # another type, scale, number of sequences or kind of relation is another program
    half = make([9], 2, 64, 16, torch.float16, 1)[0]
    q = torch.randn(1, 4, 64, device="cuda").half()
    for scale in (0.125, 0.5):
        assert torch.equal(layer(graph=half.relation(), src={"key": half.key, "value": half.value}, dst={"query": q}, scale=scale),
                           half.attend(q, scale))
    packed = torch.randn(7, 2, 64, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 7], device="cuda", dtype=torch.int32)
    out = layer(graph=tg.Graph.cu_seqlens(cu), src={"key": packed, "value": packed}, dst={"query": packed}, scale=0.125)
    assert out.shape == (7, 2, 64)


def test_a_layer_holds_no_cache():
    import gc
    import weakref

    layer = Attention()
    query = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    gc.collect()
    gc.disable()
    try:
        for _ in range(3):
            cache, _ = make([30, 500], 2, 64, 16, torch.bfloat16, 3)
            watch = weakref.ref(cache), weakref.ref(cache.key)
            for _ in range(2):
                layer(graph=cache.relation(), src={"key": cache.key, "value": cache.value}, dst={"query": query}, scale=0.125)
            del cache
            assert watch[0]() is None and watch[1]() is None        # memory is free at once
    finally:
        gc.enable()


def test_threads_share_a_layer_object():
    made = [make([300 + i, 500], 2, 64, 16, torch.bfloat16, i, capacity=512)[0] for i in range(4)]
    query = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    want = [cache.attend(query, 0.125) for cache in made]
    layer = Attention()

    def body(i):
        def run():
            relation = made[i].relation()
            for _ in range(300):
                got = layer(graph=relation, src={"key": made[i].key, "value": made[i].value}, dst={"query": query}, scale=0.125)
                assert torch.equal(got, want[i])
        return run

    run_threads(*(body(i) for i in range(4)))


def test_eviction_between_caches_without_elements():
    """Tensors without elements share an address, and nothing else."""
    rows = torch.zeros(64, 2, 64, device="cuda", dtype=torch.bfloat16)

    def cache(sequences, width):
        shape = (sequences, 2, width * 16)
        return tg.PagedCache(rows.clone(), rows.clone(), torch.zeros(sequences, width, dtype=torch.int32, device="cuda"),
                             torch.zeros(sequences, dtype=torch.int32, device="cuda"), page_size=16,
                             weight=torch.zeros(shape, device="cuda"), seen=torch.zeros(sequences, dtype=torch.int32, device="cuda"),
                             position=torch.zeros(shape, dtype=torch.int32, device="cuda"))

    for sequences, width in ((0, 3), (0, 0), (2, 0)):
        source, target = cache(sequences, width), cache(sequences, width)
        source.evict(3, into=target)
        source.check()
        target.check()
        assert target.lengths.tolist() == [0] * sequences
    source = cache(2, 2)
    with pytest.raises(ValueError, match="of its own"):
        source.evict(3, into=tg.PagedCache(rows.clone(), rows.clone(), source.page_table.clone(), source.lengths, page_size=16))


def test_frequencies_with_a_gradient_are_taken_where_none_is_asked_for():
    """A model that keeps its frequencies as a parameter answers under no_grad; with gradients it is refused."""
    q = torch.randn(3, 2, 64, device="cuda")
    positions, frequencies = torch.arange(3, device="cuda"), tg.rotary_frequencies(64, device="cuda")
    parameter = torch.nn.Parameter(frequencies.clone())
    with pytest.raises(NotImplementedError, match="frequencies"):
        tg.norm_rotary(q, None, positions, parameter)
    want = tg.norm_rotary(q, None, positions, frequencies)
    with torch.no_grad():
        assert torch.equal(tg.norm_rotary(q, None, positions, parameter), want)
    with torch.inference_mode():
        assert torch.equal(tg.norm_rotary(q, None, positions, parameter), want)


@pytest.mark.parametrize("q_heads,heads,dim,dtype", (
    (10, 2, 80, torch.float16), (16, 1, 80, torch.bfloat16), (3, 3, 88, torch.bfloat16), (16, 1, 88, torch.float16),
    (8, 2, 96, torch.float16), (18, 2, 96, torch.bfloat16), (16, 1, 192, torch.bfloat16), (32, 2, 184, torch.float16),
    (1, 1, 256, torch.bfloat16), (4, 2, 248, torch.float16), (2, 2, 160, torch.float16), (12, 1, 136, torch.bfloat16)))
def test_every_layout_of_attention(q_heads, heads, dim, dtype):
    """Every width that the kernel is built for, with one and with two tiles of 8 queries, with and without columns
    that no row fills; a cluster per head and the split over all blocks."""
    plain.test_attention([1, 0, 47, 48, 49, 64, 333, 1500], q_heads, heads, dim, 24, dtype, "rows")


@pytest.mark.parametrize("lengths,budget,recent", (
    ([264, 257, 260] * 6 + [256, 0, 1], 256, 20), ([2049, 2056, 2048] + [9] * 17, 2048, 128),
    ([265, 900, 10] * 6 + [4000, 2100], 256, 0)))
@pytest.mark.parametrize("ties", (False, True))
def test_evict_more_heads_than_processors(lengths, budget, recent, ties):
    """160 (sequence, head) pairs: small blocks, and few places that go (at most 8) as well as many."""
    plain.test_evict(lengths, 8, 8, 64, budget, recent, max(lengths), ties)


@pytest.mark.parametrize("tokens", (6001, 40003))
@pytest.mark.parametrize("track", (False, True))
@pytest.mark.parametrize("strided", (False, True))
def test_append_of_long_runs(tokens, track, strided):
    """A warp takes 2 and 8 tokens in a row, the last warp fewer; runs end inside of a warp's share."""
    heads, dim, page = 2, 16, 24
    held = [3, 0, 24, 7, 50, 1]
    bounds = [2, 1003, 1003, 1004, 1020, tokens - 9, tokens - 1]          # one run empty, tokens before and behind the runs
    new = [b - a for a, b in zip(bounds, bounds[1:])]
    cache, gen = make(held, heads, dim, page, torch.bfloat16, tokens, track=track, capacity=tokens + 60, spare=0.0)
    key, value = cache.key.clone(), cache.value.clone()
    state = None if not track else (cache.weight.clone(), cache.position.clone())
    wide = torch.randn(tokens, 2, heads + strided, dim + 8 * strided, generator=gen, device="cuda").to(torch.bfloat16)
    rows = wide[:, 0, strided:, :dim], wide[:, 1, strided:, :dim]
    cache.append(*rows, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    cache.check()
    for b, count in enumerate(new):
        place = torch.arange(held[b], held[b] + count, device="cuda")
        at = cache.page_table[b].long()[place // page] * page + place % page
        key[at], value[at] = rows[0][bounds[b]:bounds[b + 1]], rows[1][bounds[b]:bounds[b + 1]]
        if track:
            state[0][b, :, held[b]:held[b] + count] = 0
            state[1][b, :, held[b]:held[b] + count] = place.to(torch.int32)
    want = [a + b for a, b in zip(held, new)]
    assert torch.equal(cache.key, key) and torch.equal(cache.value, value) and cache.lengths.tolist() == want
    if track:
        assert torch.equal(cache.weight, state[0]) and torch.equal(cache.position, state[1]) and cache.seen.tolist() == want


def test_a_default_device_changes_nothing(monkeypatch):
    """The first cache of a process, as after others have used up the words that faults are stored in."""
    import collections

    from tiga import cache as module

    monkeypatch.setattr(module._FaultWord, "_waiting", collections.deque())
    x = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    with torch.device("cuda"):
        cache = tg.PagedCache.empty(2, 32, 2, 64, track=True)
        q, k = tg.norm_rotary(x, x, torch.arange(2), tg.rotary_frequencies(64, sections=(32,))[0])
        cache.append(k, x)
        out = cache.attend(q, accumulate=True)
        cache.evict(1)
    cache.check()
    assert torch.equal(out, x) and cache.lengths.tolist() == [1, 1]
    assert [n.tolist() for n in cache.relation().resolve_csr()] == [[0, 1, 2], [0, 64]]


FAILED_LAUNCH = """
import sys
sys.path[:0] = {path!r}
import torch
import tiga as tg

class Sum(tg.MessagePassing):
    reducer = tg.sum()

    def edge(self, src, dst, edge):
        return src.x

rows = torch.tensor([0, 2, 3], device="cuda")
layer, graph = Sum(), tg.Graph.from_csr(rows, torch.tensor([0, 1, 1], device="cuda"), num_src=2)
x = torch.ones(2, 4, device="cuda")
want = layer(graph=graph, src={{"x": x}}, dst={{}})
cache = tg.PagedCache.empty(2, 8, 1, 8)
row = torch.ones(2, 1, 8, device="cuda", dtype=torch.bfloat16)
cache.append(row, row)
torch.cuda.synchronize()
stream, recording = torch.cuda.Stream(), torch.cuda.CUDAGraph()
failed = 0
with torch.cuda.stream(stream):
    recording.capture_begin()
    for call in (stream.synchronize, lambda: cache.append(row, row), recording.capture_end):
        try:
            call()
        except RuntimeError:
            failed += 1
assert failed == 3, failed
assert torch.equal(layer(graph=graph, src={{"x": x}}, dst={{}}), want)
cache.append(row, row)
cache.check()
assert cache.lengths.tolist() == [2, 2]
print("done")
"""


def test_a_launch_that_failed_is_reported_once():
    """Waiting for a stream while it is recorded spoils the recording, so that the launch after it fails.  The next call
    of another operator has nothing to do with that."""
    import subprocess
    import sys

    run = subprocess.run([sys.executable, "-c", FAILED_LAUNCH.format(path=sys.path)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stderr[-2000:]
