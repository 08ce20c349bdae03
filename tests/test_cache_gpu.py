"""Paged cache: append, attention of one token, accumulated weights and eviction, against plain
implementations in 64 bits.

Tolerance of attention (half = eps / 2 of the output's type, n places, D values a head):
* a score is a sum of D exact products, added in float32 by the matrix unit (2^-23 a step to allow for
  truncation): off by e = scale * D * 2^-23 * max sum |q k|, and by 2^-22 |score| for the scaling and the
  base-2 exponential's argument;
* a softmax weight is then off by a relative 2 e + 2^-21 (its own exponent and the denominator's), and by
  2^-15 where it is held as the sum of two bf16 values (cut down to 8 bits, off by 2^-7, and the rest rounded, 2^-8
  of it), 2^-21 as two of fp16;
* n weighted values are added in float32: n 2^-23 of the sum of absolute values; 64 pieces are joined by
  as many multiply-adds.
Append, eviction and everything in whole numbers is compared for equality."""
import math

import pytest
import torch

import tiga as tg

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


def make(lengths, heads, dim, page, dtype, seed, *, track=False, capacity=None, layout="rows", spare=float("nan")):
    """A cache with shuffled pages; `spare` fills every place that holds no token."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, width = len(lengths), -(-max(capacity or 0, max(lengths), 1) // page)
    pages = n * width + 2
    if layout == "rows":
        key, value = (torch.full((pages * page, heads, dim), spare, device="cuda", dtype=dtype) for _ in range(2))
    elif layout == "side-by-side":
        both = torch.full((pages * page, 2, heads, dim), spare, device="cuda", dtype=dtype)
        key, value = both[:, 0], both[:, 1]
    else:                                          # head-major, rows padded
        key, value = (torch.full((heads, pages * page, dim + 8), spare, device="cuda", dtype=dtype).transpose(0, 1)[:, :, :dim]
                      for _ in range(2))
    table = torch.randperm(pages, generator=gen, device="cuda")[:n * width].reshape(n, width).to(torch.int32)
    state = {}
    if track:
        shape = (n, heads, width * page)
        state = {"weight": torch.rand(shape, generator=gen, device="cuda"),
                 "position": torch.arange(shape[2], device="cuda", dtype=torch.int32).expand(shape).contiguous(),
                 "seen": torch.tensor(lengths, device="cuda", dtype=torch.int32)}
    cache = tg.PagedCache(key, value, table, torch.tensor(lengths, device="cuda", dtype=torch.int32), page_size=page, **state)
    for b, length in enumerate(lengths):
        rows = slots(cache, b, length)
        for t in (key, value):
            t[rows] = torch.randn(length, heads, dim, generator=gen, device="cuda").to(dtype)
    return cache, gen


def slots(cache, b, count, first=0):
    table = cache.page_table[b].tolist()
    return torch.tensor([table[t // cache.page_size] * cache.page_size + t % cache.page_size
                         for t in range(first, count)], dtype=torch.long, device="cuda")


def expected_attention(cache, query, scale):
    """(out, bound, [weights per sequence and head], their bounds) in 64 bits."""
    n, heads, dim = query.shape
    group = heads // cache.heads
    out, bound = torch.zeros(n, heads, dim, dtype=torch.float64, device="cuda"), None
    bound = torch.zeros_like(out)
    weight = torch.zeros(n, cache.heads, cache.capacity, dtype=torch.float64, device="cuda")
    weight_bound = torch.zeros_like(weight)
    half = HALF[query.dtype]
    split = 2.0 ** -15 if query.dtype == torch.bfloat16 else 2.0 ** -21
    for b, length in enumerate(cache.lengths.tolist()):
        if not length:
            continue
        rows = slots(cache, b, length)
        for h in range(cache.heads):
            q = query[b, h * group:(h + 1) * group].double()
            k, v = cache.key[rows, h].double(), cache.value[rows, h].double()
            score = q @ k.T * scale
            p = torch.softmax(score, dim=-1)
            e = abs(scale) * dim * 2.0 ** -23 * (q.abs() @ k.abs().T).max() + 2.0 ** -22 * score.abs().max()
            off = 2 * e + 2.0 ** -21 + split + (length + 64) * 2.0 ** -23
            o = p @ v
            out[b, h * group:(h + 1) * group] = o
            bound[b, h * group:(h + 1) * group] = half * o.abs() + off * (p @ v.abs()) + 2.0 ** -25
            weight[b, h, :length] = p.sum(0)
            weight_bound[b, h, :length] = (2 * e + 2.0 ** -20 + (length + 64 + group) * 2.0 ** -23) * p.sum(0)
    return out, bound, weight, weight_bound


def assert_within(got, want, bound):
    excess = (got.double() - want).abs() - bound
    assert bool((excess <= 0).all()), f"worst excess {excess.max().item()}"


CASES = (
    # lengths, q heads, heads, dim, page, dtype, layout
    ([1], 1, 1, 8, 1, torch.bfloat16, "rows"),
    ([0], 4, 2, 64, 16, torch.float16, "rows"),
    ([1, 15, 16, 17, 63, 64, 65, 0], 4, 4, 64, 16, torch.bfloat16, "rows"),
    ([127, 0, 0, 129, 1000], 8, 2, 128, 64, torch.bfloat16, "side-by-side"),
    ([300, 5], 6, 2, 40, 7, torch.float16, "padded"),
    ([77, 1024], 9, 1, 72, 24, torch.bfloat16, "rows"),               # nine queries on one key head: two tiles of 8
    ([513], 16, 1, 256, 64, torch.float16, "rows"),
    ([200, 90], 17, 1, 128, 48, torch.bfloat16, "side-by-side"),      # a second pass over the key head
    ([65, 64, 2], 40, 1, 64, 16, torch.float16, "rows"),
    ([5000], 8, 1, 128, 128, torch.float16, "rows"),
    ([20000, 3], 4, 4, 192, 256, torch.bfloat16, "rows"),
    ([7] * 200, 2, 2, 64, 8, torch.bfloat16, "rows"),                 # more sequences than threads of a block
    ([33] * 12, 32, 8, 128, 16, torch.bfloat16, "padded"),
)


@pytest.mark.parametrize("lengths,q_heads,heads,dim,page,dtype,layout", CASES)
def test_attention(lengths, q_heads, heads, dim, page, dtype, layout):
    cache, gen = make(lengths, heads, dim, page, dtype, len(lengths) + dim, layout=layout)
    query = torch.randn(len(lengths), q_heads, dim, generator=gen, device="cuda").to(dtype)
    scale = dim ** -0.5
    got = cache.attend(query)
    cache.check()
    want, bound, _, _ = expected_attention(cache, query, scale)
    assert got.dtype == dtype and got.is_contiguous()
    assert_within(got, want, bound)
    assert all(bool((got[b] == 0).all()) for b, length in enumerate(lengths) if not length)
    kernel = Attention()
    out = kernel(graph=cache.relation(), src={"key": cache.key, "value": cache.value}, dst={"query": query}, scale=scale)
    assert torch.equal(out, got) and kernel.last_variant.lowering == "b200-paged-cache-attention"
    assert torch.equal(cache.attend(query), got)                      # the same bits every time
    # the same tokens in a cache with room for many more: split over all blocks instead of a cluster per head. Table
    # entries that no length reaches are never looked at
    wide = torch.full((len(lengths), 200000 // page), -7, device="cuda", dtype=torch.int32)
    wide[:, :cache.page_table.shape[1]] = cache.page_table
    roomy = tg.PagedCache(cache.key, cache.value, wide, cache.lengths, page_size=page)
    split = roomy.attend(query)
    roomy.check()
    assert_within(split, want, bound)
    assert all(bool((split[b] == 0).all()) for b, length in enumerate(lengths) if not length)
    assert torch.equal(roomy.attend(query), split)
    packed = torch.randn(len(lengths), q_heads + 3, dim + 5, generator=gen, device="cuda").to(dtype)
    packed[:, 2:2 + q_heads, 1:1 + dim] = query
    assert torch.equal(cache.attend(packed[:, 2:2 + q_heads, 1:1 + dim]), got)      # an unaligned view


def test_scores_that_are_all_minus_infinity_give_zero():
    """The empty-row value of the online-softmax reducer: a denominator of 0 divides nothing."""
    cache, _ = make([5, 600], 1, 16, 16, torch.bfloat16, 5)
    for b, n in ((0, 5), (1, 600)):
        cache.key[slots(cache, b, n)] = -float("inf")
    query = torch.ones(2, 1, 16, device="cuda", dtype=torch.bfloat16)
    assert bool((cache.attend(query) == 0).all())
    cache.key[slots(cache, 1, 600)[300]] = 1                             # one place left: its value
    out = cache.attend(query)
    assert bool((out[0] == 0).all()) and torch.equal(out[1, 0], cache.value[slots(cache, 1, 600)[300], 0])
    cache.value[slots(cache, 1, 600)[300], 0, 3] = float("nan")
    assert bool(cache.attend(query)[1, 0, 3].isnan()) and int(cache.attend(query).isnan().sum()) == 1


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("places", (3, 700, 5000))
def test_infinite_values_stay_in_their_column(dtype, places):
    """An infinity among the values of a place that is looked at is the result of its column, with its sign; both signs
    in one column give NaN, and the other columns are what they are without it."""
    cache, gen = make([places, places], 2, 64, 16, dtype, places)
    query = torch.randn(2, 6, 64, generator=gen, device="cuda").to(dtype)
    clean = cache.attend(query)
    rows = slots(cache, 0, places)
    cache.value[rows[0], 1, 7] = float("inf")
    cache.value[rows[-1], 1, 9] = -float("inf")
    cache.value[rows[0], 1, 60], cache.value[rows[1], 1, 60] = float("inf"), -float("inf")
    got = cache.attend(query)
    want = clean.clone()
    want[0, 3:, 7], want[0, 3:, 9] = float("inf"), -float("inf")
    assert bool(got[0, 3:, 60].isnan().all())
    want[0, 3:, 60] = got[0, 3:, 60] = 0
    assert torch.equal(got, want)


def test_large_scores_and_a_dominating_place():
    cache, gen = make([400, 130], 2, 64, 16, torch.float16, 5)
    cache.key[slots(cache, 0, 400)] *= 30
    query = 8 * torch.randn(2, 4, 64, generator=gen, device="cuda").to(torch.float16)
    want, bound, _, _ = expected_attention(cache, query, 0.125)
    assert_within(cache.attend(query, 0.125), want, bound)
    # weights of 2^-20 next to one of 1: below fp16's normal numbers, they still count
    cache, _ = make([8192], 1, 16, 64, torch.float16, 6)
    rows = slots(cache, 0, 8192)
    cache.key[rows] = 0
    cache.key[rows[0], 0, 0] = 1
    cache.value[rows] = 1
    cache.value[rows[0]] = 0
    query = torch.zeros(1, 1, 16, device="cuda", dtype=torch.float16)
    query[0, 0, 0] = 1
    scale = 20 * math.log(2)
    share = 8191 * 2.0 ** -20 / (1 + 8191 * 2.0 ** -20)
    got = cache.attend(query, scale)
    assert bool(((got.double() - share).abs() <= share * (2.0 ** -11 + 8192 * 2.0 ** -23 + 2.0 ** -19)).all())


@pytest.mark.parametrize("lengths,q_heads,heads,dim,page", (
    ([1, 0, 64, 700], 8, 2, 128, 16), ([3000], 20, 1, 64, 64), ([90, 2000], 3, 3, 48, 7), ([5] * 40, 4, 4, 64, 8)))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_accumulated_weights(lengths, q_heads, heads, dim, page, dtype):
    cache, gen = make(lengths, heads, dim, page, dtype, dim, track=True, capacity=max(lengths) + 9)
    query = torch.randn(len(lengths), q_heads, dim, generator=gen, device="cuda").to(dtype)
    before = cache.weight.clone()
    out = cache.attend(query, accumulate=True)
    want, bound, weight, weight_bound = expected_attention(cache, query, dim ** -0.5)
    assert_within(out, want, bound)
    assert_within(cache.weight, before.double() + weight, weight_bound + 2.0 ** -23 * (before.double() + weight))
    held = torch.arange(cache.capacity, device="cuda") < cache.lengths[:, None, None]
    assert torch.equal(cache.weight.masked_fill(held, 0), before.masked_fill(held, 0))       # places behind: untouched
    again = cache.weight.clone()
    cache.weight.copy_(before)
    cache.attend(query, accumulate=True)
    assert torch.equal(cache.weight, again)


def test_far_offsets_of_a_large_cache():
    """The pages in use lie behind 2^31 values: offsets do not fit 32 bits."""
    heads, dim, page = 8, 128, 64
    pages = (2 ** 31 // (heads * dim) + 200 * page) // page
    key, value = (torch.empty(pages * page, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(pages - 8, pages, device="cuda", dtype=torch.int32).reshape(2, 4)
    cache = tg.PagedCache(key, value, table, torch.zeros(2, dtype=torch.int32, device="cuda"), page_size=page)
    gen = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.randn(2, 300, heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
    cache.append(rows[0], rows[1], cu_seqlens=torch.tensor([0, 200, 300], device="cuda", dtype=torch.int32))
    query = torch.randn(2, 16, dim, generator=gen, device="cuda").to(torch.bfloat16)
    got = cache.attend(query)
    cache.check()
    assert torch.equal(key[slots(cache, 0, 200)], rows[0, :200]) and torch.equal(value[slots(cache, 1, 100)], rows[1, 200:])
    want, bound, _, _ = expected_attention(cache, query, dim ** -0.5)
    assert_within(got, want, bound)


def test_layers_share_one_table():
    cache, gen = make([70, 9], 2, 64, 16, torch.bfloat16, 1)
    other_key, other_value = torch.randn_like(cache.key), torch.randn_like(cache.value)
    query = torch.randn(2, 2, 64, generator=gen, device="cuda").to(torch.bfloat16)
    out = Attention()(graph=cache.relation(), src={"key": other_key, "value": other_value}, dst={"query": query}, scale=0.1)
    second = cache.over(other_key, other_value)
    assert torch.equal(out, second.attend(query, 0.1)) and not torch.equal(out, cache.attend(query, 0.1))
    # a step of both layers: the first moves the lengths, the second writes at the place it had
    start = cache.lengths.clone()
    cache_room, row = 16 * cache.page_table.shape[1], torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    assert cache_room > 70
    cache.append(row, row)
    second.append(2 * row, 3 * row, start=start)
    assert cache.lengths.tolist() == [71, 10]
    at = torch.stack([slots(cache, 0, 71)[-1], slots(cache, 1, 10)[-1]])
    assert torch.equal(cache.key[at], row) and torch.equal(other_key[at], 2 * row) and torch.equal(other_value[at], 3 * row)


@pytest.mark.parametrize("heads,dim,page,dtype,layout", (
    (1, 8, 1, torch.bfloat16, "rows"), (8, 128, 64, torch.bfloat16, "rows"), (3, 72, 24, torch.float16, "side-by-side"),
    (2, 256, 16, torch.float16, "padded"), (40, 64, 5, torch.bfloat16, "rows")))
@pytest.mark.parametrize("track", (False, True))
def test_append(heads, dim, page, dtype, layout, track):
    lengths = [0, 3, 16, 31, 7]
    cache, gen = make(lengths, heads, dim, page, dtype, 4, track=track, capacity=80, layout=layout, spare=0.0)
    key, value = cache.key.clone(), cache.value.clone()

    def model(new_key, new_value, start, bounds):
        for b in range(5):
            count = bounds[b + 1] - bounds[b]
            if count > 0:
                rows = slots(cache, b, start[b] + count, start[b])
                key[rows], value[rows] = new_key[bounds[b]:bounds[b + 1]], new_value[bounds[b]:bounds[b + 1]]

    def rows(count):
        return torch.randn(count, heads, dim, generator=gen, device="cuda").to(dtype)

    def check(want):
        cache.check()
        assert cache.lengths.tolist() == want and torch.equal(cache.key, key) and torch.equal(cache.value, value)

    one = rows(5), rows(5)
    cache.append(*one)
    model(*one, lengths, range(6))
    check([1, 4, 17, 32, 8])
    # ragged runs, one empty; two tokens before the first run and four behind the last one are nobody's
    bounds = [2, 3, 3, 40, 60, 61]
    many = rows(65), rows(65)
    cache.append(*many, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    model(*many, [1, 4, 17, 32, 8], bounds)
    check([2, 4, 54, 52, 9])
    if track:
        assert cache.seen.tolist() == [2, 4, 54, 52, 9]
        for b, (first, last) in enumerate(zip(lengths, [2, 4, 54, 52, 9])):
            assert bool((cache.weight[b, :, first:last] == 0).all()) and bool((cache.weight[b, :, :first] > 0).all())
            assert cache.position[b, 0, first:last].tolist() == list(range(first, last))
    # drafted tokens taken back: five places of sequence 2 and all of sequence 4
    start = [2, 4, 49, 52, 0]
    packed = rows(5).new_zeros(5, 2 * heads, dim + 3)
    packed.normal_(generator=gen)
    new = packed[:, :heads, 3:], packed[:, heads:, :dim]               # unaligned and strided rows
    cache.append(*new, start=torch.tensor(start, dtype=torch.int32, device="cuda"))
    model(*new, start, range(6))
    check([3, 5, 50, 53, 1])
    if track:
        assert cache.seen.tolist() == [3, 5, 50, 53, 1] and cache.position[2, :, 49].tolist() == [49] * heads
    cache.append(rows(0), rows(0), cu_seqlens=torch.zeros(6, dtype=torch.int32, device="cuda"))
    check([3, 5, 50, 53, 1])


def test_contents_out_of_range_are_reported_and_never_followed():
    def fresh():
        cache, _ = make([10, 20], 2, 64, 16, torch.bfloat16, 3, capacity=32, track=True, spare=0.0)
        return cache, cache.key.clone()

    row = torch.ones(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    many = torch.ones(40, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache, key = fresh()
    cache.lengths[1] = 32
    cache.append(row, row)                                            # full: dropped
    with pytest.raises(RuntimeError, match="capacity"):
        cache.check()
    assert cache.lengths.tolist() == [11, 32]
    cache.append(many, many, cu_seqlens=torch.tensor([0, 40, 40], device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="capacity"):
        cache.check()
    assert cache.lengths.tolist() == [32, 32] and torch.equal(cache.key[slots(cache, 1, 32)], key[slots(cache, 1, 32)])
    for page in (-1, 10 ** 9, cache.key.shape[0] // 16):
        cache, key = fresh()
        table = cache.page_table.clone()
        cache.page_table[0, 0] = page
        cache.attend(row)
        with pytest.raises(RuntimeError, match="table"):
            cache.check()
        cache.append(row, row, start=torch.tensor([3, 20], device="cuda", dtype=torch.int32))
        with pytest.raises(RuntimeError, match="table"):
            cache.check()
        cache.evict(2)
        with pytest.raises(RuntimeError, match="table"):
            cache.check()
        cache.page_table.copy_(table)
        cache.attend(row)
        cache.check()                                                 # and the cache works again
    for length in (-1, 33, 2 ** 31 - 1, -(2 ** 31)):
        cache, key = fresh()
        cache.lengths[0] = length
        cache.attend(row, accumulate=True)
        with pytest.raises(RuntimeError, match="length"):
            cache.check()
        cache.evict(4)
        with pytest.raises(RuntimeError, match="length"):
            cache.check()
    for start in (-1, 11, 2 ** 31 - 1):
        cache, key = fresh()
        cache.append(row, row, start=torch.tensor([start, 20], device="cuda", dtype=torch.int32))
        with pytest.raises(RuntimeError, match="start"):
            cache.check()
    cache, key = fresh()                                              # bounds that run backwards or out of the tokens
    cache.append(many, many, cu_seqlens=torch.tensor([35, -5, 1000], device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError):
        cache.check()
    with pytest.raises(RuntimeError, match="length"):                 # the next call reports, too
        cache.lengths[0] = -4
        cache.attend(row)
        torch.cuda.synchronize()
        cache.attend(row)


def expected_eviction(cache, budget, recent):
    """Kept places, ascending, of every sequence and head: the definition by sorting."""
    kept = []
    for b, length in enumerate(cache.lengths.tolist()):
        for h in range(cache.heads):
            w, at = cache.weight[b, h, :length].tolist(), cache.position[b, h, :length].tolist()
            newest = int(cache.seen[b]) - recent
            order = sorted(range(length), key=lambda t: (at[t] < newest, math.isnan(w[t]) and at[t] < newest,
                                                         0.0 if math.isnan(w[t]) or at[t] >= newest else -w[t], t))
            kept.append(sorted(order[:budget]))
    return kept


def state_of(cache):
    return [t.clone() for t in (cache.key, cache.value, cache.weight, cache.position, cache.lengths, cache.seen)]


EVICTIONS = (
    # lengths, heads, dim, page, budget, recent, capacity
    ([0, 1, 5, 40], 1, 8, 1, 4, 0, 41), ([33, 64, 65], 2, 64, 16, 32, 5, 70), ([300, 17], 3, 72, 24, 16, 16, 320),
    ([5000, 2049, 9000], 2, 128, 64, 2048, 64, 9000), ([20], 4, 256, 8, 1, 1, 20), ([20], 4, 256, 8, 1, 0, 20),
    ([50000] + [10] * 79, 1, 8, 64, 20000, 7, 50000),                 # more ranks than a block keeps in shared memory
    ([30000, 24000], 2, 16, 16, 1500, 0, 30000),                      # a cluster of blocks per head
    ([90, 91], 1, 64, 64, 200, 3, 128), ([100], 2, 64, 16, 2 ** 31 - 1, 0, 112), ([20000], 1, 64, 64, 19999, 100, 20000),
)


@pytest.mark.parametrize("lengths,heads,dim,page,budget,recent,capacity", EVICTIONS)
@pytest.mark.parametrize("ties", (False, True))
def test_evict(lengths, heads, dim, page, budget, recent, capacity, ties):
    cache, gen = make(lengths, heads, dim, page, torch.bfloat16, dim + budget % 97, track=True, capacity=capacity, spare=0.0)
    if ties:
        cache.weight.mul_(4).floor_()
        cache.weight[:, :, ::7] = float("nan")
        cache.weight[:, :, 3::11] = -0.0
        cache.weight[:, :, 5::13] = float("inf")
        cache.weight[:, :, 6::17] = -float("inf")
        cache.position.copy_(cache.position.flip(2).sub(cache.capacity - max(lengths)))       # not in order of age
    kept = expected_eviction(cache, budget, recent)
    before = state_of(cache)
    places = min(budget, cache.capacity)
    target, _ = make([0] * len(lengths), heads, dim, page + 1, torch.bfloat16, 8, track=True, capacity=places, spare=0.0)
    untouched = state_of(target)
    cache.evict(budget, recent=recent, into=target)
    assert all(torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0)) for a, b in zip(before, state_of(cache)))
    for b, length in enumerate(lengths):
        for h in range(heads):
            keep = torch.tensor(kept[b * heads + h], dtype=torch.long, device="cuda")
            rows, to = slots(cache, b, length)[keep], slots(target, b, len(keep))
            for got, source in ((target.key, cache.key), (target.value, cache.value)):
                assert torch.equal(got[to, h], source[rows, h])
            for at, (got, source) in enumerate(((target.weight, cache.weight), (target.position, cache.position))):
                assert torch.equal(got[b, h, :len(keep)].nan_to_num(7.0), source[b, h, keep].nan_to_num(7.0))
                assert torch.equal(got[b, h, len(keep):], untouched[2 + at][b, h, len(keep):])
    want = [min(n, budget) for n in lengths]
    assert target.lengths.tolist() == want and torch.equal(target.seen, cache.seen)
    # in place: a kept place below the budget stays, the freed ones take the others in order
    cache.evict(budget, recent=recent)
    cache.check()
    assert cache.lengths.tolist() == want and torch.equal(cache.seen, before[5])
    expected = [t.clone() for t in before]
    for b, length in enumerate(lengths):
        for h in range(heads):
            keep = kept[b * heads + h]
            free = [t for t in range(min(length, budget)) if t not in set(keep)]
            rows = slots(cache, b, length)
            for to, source in zip(free, [t for t in keep if t >= budget]):
                for at in (0, 1):
                    expected[at][rows[to], h] = before[at][rows[source], h]
                for at in (2, 3):
                    expected[at][b, h, to] = before[at][b, h, source]
    for got, wanted in zip(state_of(cache)[:4], expected):
        assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(wanted, 7.0))


def test_evict_into_an_untracked_cache_of_the_same_pool():
    cache, gen = make([50, 8], 2, 64, 8, torch.float16, 2, track=True, capacity=64, spare=0.0)
    kept = expected_eviction(cache, 16, 4)
    pool = torch.cat([cache.key, torch.zeros(32, 2, 64, device="cuda", dtype=torch.float16)])
    values = torch.cat([cache.value, torch.zeros(32, 2, 64, device="cuda", dtype=torch.float16)])
    first = cache.key.shape[0] // 8
    source = tg.PagedCache(pool, values, cache.page_table, cache.lengths, page_size=8, weight=cache.weight,
                           position=cache.position, seen=cache.seen)
    target = tg.PagedCache(pool, values, torch.arange(first, first + 4, device="cuda", dtype=torch.int32).reshape(2, 2),
                           torch.zeros(2, device="cuda", dtype=torch.int32), page_size=8)
    source.evict(16, recent=4, into=target)
    for b in range(2):
        for h in range(2):
            keep = kept[2 * b + h]
            assert torch.equal(pool[slots(target, b, len(keep)), h], cache.key[slots(cache, b, 50)[keep] if b == 0 else slots(cache, 1, 8)[keep], h])
    assert target.lengths.tolist() == [16, 8]


def test_refusals():
    cache, _ = make([5, 6], 2, 64, 16, torch.bfloat16, 1, spare=0.0)
    other, _ = make([5, 6], 2, 64, 16, torch.bfloat16, 1, track=True, spare=0.0)
    row = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    index = torch.zeros(2, device="cuda", dtype=torch.int32)
    for call, error in (
        (lambda: cache.append(row[:1], row[:1]), ValueError), (lambda: cache.append(row, row.half()), ValueError),
        (lambda: cache.append(row, row[:, :1]), ValueError), (lambda: cache.append(row, row.cpu()), ValueError),
        (lambda: cache.append(row, row, cu_seqlens=index), ValueError),
        (lambda: cache.append(row, row, start=index.long()), ValueError),
        (lambda: cache.append(row, row, start=index.cpu()), ValueError),
        (lambda: cache.append(row.float().requires_grad_().bfloat16(), row), NotImplementedError),
        (lambda: cache.attend(row[:1]), ValueError), (lambda: cache.attend(row[:, :, :32]), ValueError),
        (lambda: cache.attend(row.half()), NotImplementedError),
        (lambda: cache.attend(row[:, :1].expand(2, 3, 64)), NotImplementedError),
        (lambda: cache.attend(row.float().requires_grad_().bfloat16()), NotImplementedError),
        (lambda: cache.attend(row, accumulate=True), ValueError), (lambda: cache.evict(4), ValueError),
        (lambda: other.evict(0), ValueError), (lambda: other.evict(4, recent=5), ValueError),
        (lambda: other.evict(4.0), ValueError), (lambda: other.evict(4, recent=-1), ValueError),
        (lambda: other.evict(17, into=tg.PagedCache.empty(2, 4, 2, 64, page_size=4)), ValueError),
        (lambda: other.evict(4, into=tg.PagedCache.empty(2, 4, 1, 64)), ValueError),
        (lambda: other.evict(4, into=other.over(other.key.clone(), other.value.clone())), ValueError),
        (lambda: other.evict(4, into=tg.PagedCache(other.key, other.value, other.page_table, other.lengths.clone(),
                                                   page_size=16)), ValueError),
    ):
        with pytest.raises(error):
            call()

    class Sum(tg.MessagePassing):
        reducer = tg.sum()

        def edge(self, src, dst, edge):
            return src.x

    with pytest.raises(NotImplementedError, match="paged cache"):
        Sum()(graph=cache.relation(), src={"x": torch.zeros(cache.key.shape[0], 4, device="cuda")}, dst={})
    q = torch.zeros(2, 2, 64, device="cuda")
    positions, frequencies = torch.zeros(2, device="cuda", dtype=torch.int64), tg.rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda")
    for arguments, error in (
        (dict(query=q.double()), NotImplementedError), (dict(query=q[0]), ValueError), (dict(key=q[:1]), ValueError),
        (dict(key=q.bfloat16()), ValueError), (dict(positions=positions.float()), ValueError),
        (dict(positions=positions[:1]), ValueError), (dict(positions=positions[:, None]), ValueError),
        (dict(positions=positions.cpu()), ValueError), (dict(frequencies=frequencies.double()), ValueError),
        (dict(frequencies=tg.rotary_frequencies(66, device="cuda")), ValueError),
        (dict(frequencies=frequencies.clone().requires_grad_()), NotImplementedError),
        (dict(frequencies=frequencies.expand(9, 32), positions=positions[:, None].expand(2, 9)), NotImplementedError),
        (dict(query_weight=w[:32]), ValueError), (dict(query_weight=w, eps=None), ValueError),
        (dict(query_weight=w.half()), ValueError), (dict(eps=-1.0), ValueError),
        (dict(key=None, key_weight=w), ValueError), (dict(query=torch.zeros(2, 1, 1025, device="cuda"), key=None), NotImplementedError),
    ):
        call = {"query": q, "key": q, "positions": positions, "frequencies": frequencies, **arguments}
        with pytest.raises(error):
            tg.norm_rotary(call.pop("query"), call.pop("key"), call.pop("positions"), call.pop("frequencies"), **call)


def test_a_captured_step_follows_table_and_lengths():
    def step(cache, row, query):
        cache.append(row, row)
        out = cache.attend(query, accumulate=True)
        cache.evict(24, recent=4)
        return out

    caches = [make([20, 3, 0], 2, 64, 8, torch.bfloat16, 7, track=True, capacity=40, spare=0.0)[0] for _ in range(2)]
    row = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    query = torch.randn(3, 4, 64, device="cuda").to(torch.bfloat16)
    saved = state_of(caches[0])
    step(caches[0], row, query)                                        # sets kernel attributes outside the capture
    for t, s in zip((caches[0].key, caches[0].value, caches[0].weight, caches[0].position, caches[0].lengths,
                     caches[0].seen), saved):
        t.copy_(s)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], row, query)
    with torch.cuda.graph(second):                                     # two graphs share no scratch
        out2 = step(caches[0], row, query)
    for i in range(8):
        row.normal_(generator=torch.Generator(device="cuda").manual_seed(i))
        query.normal_(generator=torch.Generator(device="cuda").manual_seed(100 + i))
        (graph, second)[i % 2].replay()
        want = step(caches[1], row, query)
        assert torch.equal((out, out2)[i % 2], want)
        assert all(torch.equal(a, b) for a, b in zip(state_of(caches[0]), state_of(caches[1])))
    assert caches[0].lengths.tolist() == [24, 11, 8] and caches[0].seen.tolist() == [28, 11, 8]
    caches[0].check()


def test_captured_branches_join_again():
    """Two layers' caches on two branches of one graph, mixed with other kernels on both sides of every call."""
    made = [[make([30 + i, 500], 2, 64, 16, torch.bfloat16, 7 + i, capacity=600)[0] for i in range(2)] for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 8, 64, generator=gen, device="cuda").to(torch.bfloat16)
    positions, frequencies = torch.tensor([3, 9], device="cuda"), tg.rotary_frequencies(64, device="cuda")

    def branch(cache, shift):
        q, k = tg.norm_rotary(x + shift, x[:, :2] * 2, positions, frequencies)
        cache.append(k, k + 1)
        return cache.attend(q) * 2

    def step(caches, side):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = branch(caches[1], 1)
        a = branch(caches[0], 0)
        here.wait_stream(side)
        return tg.norm_rotary(a + b, None, positions, frequencies) + 1

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = step(made[0], side)
    for i in range(12):
        x.normal_(generator=gen)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step(made[1], side))
    for a, b in zip(*made):
        assert torch.equal(a.lengths, b.lengths) and torch.equal(a.key.nan_to_num(9.0), b.key.nan_to_num(9.0))
    assert made[0][0].lengths.tolist() == [42, 512]


def test_calls_on_two_streams_do_not_disturb_each_other():
    caches = [make([900, 333], 2, 128, 16, torch.bfloat16, seed, track=True)[0] for seed in (1, 2)]
    queries = [torch.randn(2, 8, 128, device="cuda").to(torch.bfloat16) for _ in range(2)]
    want = [c.attend(q) for c, q in zip(caches, queries)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(caches[i].attend(queries[i]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_answering_token_by_token_equals_the_packed_sequence():
    """One attention layer: a packed batch at once (Graph.cu_seqlens), then prompt into the cache and the rest
    one token of every sequence at a time. Both are within one rounding of softmax weights and outputs (2^-8 each) of
    the 64-bit result, whose values are at most a few units."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    heads, kv_heads, dim, prompts, total = 8, 2, 128, [130, 64, 1], 140
    cu = torch.tensor([0, total, 2 * total, 3 * total], device="cuda", dtype=torch.int32)
    packed = torch.randn(3 * total, (heads + 2 * kv_heads) * dim, generator=gen, device="cuda").to(torch.bfloat16)
    q = packed[:, :heads * dim].view(-1, heads, dim)
    k = packed[:, heads * dim:(heads + kv_heads) * dim].view(-1, kv_heads, dim)
    v = packed[:, (heads + kv_heads) * dim:].view(-1, kv_heads, dim)
    weight, frequencies = 1 + 0.1 * torch.randn(dim, generator=gen, device="cuda"), tg.rotary_frequencies(dim, device="cuda")
    positions = torch.arange(total, device="cuda").repeat(3)
    layer, scale = Attention(), dim ** -0.5

    def heads_of(rows):
        return tg.norm_rotary(q[rows], k[rows], positions[rows], frequencies, query_weight=weight, key_weight=weight)

    everything = torch.arange(3 * total, device="cuda")
    full_q, full_k = heads_of(everything)
    whole = layer(graph=tg.Graph.cu_seqlens(cu), src={"key": full_k, "value": v}, dst={"query": full_q}, scale=scale)
    cache = tg.PagedCache.empty(3, total, kv_heads, dim, page_size=16)
    rows = torch.cat([everything[b * total:b * total + n] for b, n in enumerate(prompts)])
    bounds = torch.tensor([0, 130, 194, 195], device="cuda", dtype=torch.int32)
    _, prompt_key = heads_of(rows)
    cache.append(prompt_key, v[rows], cu_seqlens=bounds)
    answer, place = Attention(), torch.tensor(prompts, device="cuda")
    for _ in range(10):
        rows = torch.arange(3, device="cuda") * total + place
        step_q, step_k = heads_of(rows)
        cache.append(step_k, v[rows])
        out = answer(graph=cache.relation(), src={"key": cache.key, "value": cache.value}, dst={"query": step_q}, scale=scale)
        torch.testing.assert_close(out.float(), whole[rows].float(), rtol=3 * 2.0 ** -8, atol=2.0 ** -7)
        place += 1
    cache.check()
    # and the packed form trains: gradients reach the projection's output through the rotation
    leaf = packed.detach().requires_grad_()
    lq, lk, lv = leaf[:, :heads * dim], leaf[:, heads * dim:(heads + kv_heads) * dim], leaf[:, (heads + kv_heads) * dim:]
    tq, tk = tg.norm_rotary(lq.view(-1, heads, dim), lk.view(-1, kv_heads, dim), positions, frequencies)
    out = layer(graph=tg.Graph.cu_seqlens(cu), src={"key": tk, "value": lv.view(-1, kv_heads, dim)}, dst={"query": tq}, scale=scale)
    (grad,) = torch.autograd.grad(out.float().square().sum(), leaf)
    assert bool(torch.isfinite(grad).all()) and all(bool((part != 0).any()) for part in grad.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))


def test_the_first_calls_may_be_captured():
    """Sizes whose kernels nothing has launched yet in this process (a head size of 24, float16, 3 positions axes):
    attributes and modules are set up while the stream is captured."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache, _ = make([40, 700], 3, 24, 8, torch.float16, 9, track=True, capacity=800, spare=0.0)
    query, key = (torch.randn(2, 3, 24, generator=gen, device="cuda").to(torch.float16) for _ in range(2))
    positions = torch.randint(0, 50, (2, 3), generator=gen, device="cuda")
    frequencies = tg.rotary_frequencies(24, sections=(4, 4, 4), device="cuda")
    saved = state_of(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k = tg.norm_rotary(query, key, positions, frequencies, interleaved=True)
        cache.append(k, k)
        out = cache.attend(q, accumulate=True)
        cache.evict(600, recent=3)
    assert all(torch.equal(a, b) for a, b in zip(saved, state_of(cache)))       # capturing ran nothing
    graph.replay()
    got = [out.clone()] + state_of(cache)
    for t, s in zip((cache.key, cache.value, cache.weight, cache.position, cache.lengths, cache.seen), saved):
        t.copy_(s)
    q, k = tg.norm_rotary(query, key, positions, frequencies, interleaved=True)
    cache.append(k, k)
    want = [cache.attend(q, accumulate=True)]
    cache.evict(600, recent=3)
    assert all(torch.equal(a, b) for a, b in zip(got, want + state_of(cache)))


def test_attention_inside_a_program():
    cache, gen = make([70, 9], 2, 64, 16, torch.bfloat16, 1)
    query = torch.randn(2, 4, 64, generator=gen, device="cuda").to(torch.bfloat16)
    layer = Attention()

    @tg.program
    def answer(q):
        return layer(graph=cache.relation(), src={"key": cache.key, "value": cache.value}, dst={"query": q}, scale=0.125)

    assert torch.equal(answer(query).materialize(), cache.attend(query, 0.125))


def test_empty_batches_and_caches_without_room():
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    rows = torch.zeros(64, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache = tg.PagedCache(rows, rows.clone(), torch.zeros(0, 3, dtype=torch.int32, device="cuda"), none, page_size=16,
                          weight=torch.zeros(0, 2, 48, device="cuda"), seen=none.clone(),
                          position=torch.zeros(0, 2, 48, dtype=torch.int32, device="cuda"))
    cache.append(rows[:0], rows[:0])
    cache.append(rows[:5], rows[:5], cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert cache.attend(rows[:0]).shape == (0, 2, 64) and cache.attend(rows[:0], accumulate=True).shape == (0, 2, 64)
    cache.evict(3)
    cache.check()
    full = tg.PagedCache(rows, rows.clone(), torch.zeros(2, 0, dtype=torch.int32, device="cuda"),
                         torch.zeros(2, dtype=torch.int32, device="cuda"), page_size=16)
    assert full.capacity == 0 and bool((full.attend(rows[:2]) == 0).all())
    full.check()
    full.append(rows[:2], rows[:2])
    with pytest.raises(RuntimeError, match="capacity"):
        full.check()
    assert full.lengths.tolist() == [0, 0]
    full = tg.PagedCache(rows, rows.clone(), torch.zeros(2, 0, dtype=torch.int32, device="cuda"), full.lengths, page_size=16,
                         weight=torch.zeros(2, 2, 0, device="cuda"), seen=torch.zeros_like(full.lengths),
                         position=torch.zeros(2, 2, 0, dtype=torch.int32, device="cuda"))
    assert bool((full.attend(rows[:2], accumulate=True) == 0).all())
    full.evict(1)
    full.check()
