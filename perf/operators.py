"""Workloads of the token-by-token serving operators and of the query / key rotation, each in a plain
form (elementary torch operations) and through the package's entry points.

``own`` selects the side: False computes the plain form, True calls ``tiga``.  A case is a dict of plain
values; ``prepare`` makes its inputs from a seed, ``run`` is one pass, ``work`` the bytes and operations a
pass cannot do without, ``exact`` the result in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


def _tiga():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiga-lang_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import tiga

    return tiga


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a batch: a handful of rows, the launch is what costs
        {"name": "rotate-decode", "op": "rotate", "tokens": 32, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128,
         "axes": 1, "interleaved": False, "backward": False, "dtype": "bf16"},
        # the prompts of a serving batch, packed
        {"name": "rotate-prompt", "op": "rotate", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotated": 128, "axes": 1, "interleaved": False, "backward": False, "dtype": "bf16"},
        # a training step of one layer on packed sequences
        {"name": "rotate-train", "op": "rotate", "tokens": 8192, "heads": 16, "kv_heads": 16, "dim": 128,
         "rotated": 128, "axes": 1, "interleaved": False, "backward": True, "dtype": "bf16"},
        # training on video: (time, height, width) positions, adjacent pairs, an odd number of patches
        {"name": "rotate-video-train", "op": "rotate", "tokens": 9001, "heads": 24, "kv_heads": 8, "dim": 64,
         "rotated": 64, "axes": 3, "interleaved": True, "backward": True, "dtype": "fp16"},
        # the cache takes one token of every sequence of a decoding batch
        {"name": "append-decode", "op": "append", "sequences": 64, "longest": 4096, "new": 1, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # the cache takes ragged prompts
        {"name": "append-prompt", "op": "append", "sequences": 8, "longest": 1000, "new": 8192, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # one user, a short conversation
        {"name": "attend-short", "op": "attend", "sequences": 1, "longest": 1000, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "accumulate": False, "dtype": "bf16"},
        # a ragged decoding batch, one sequence of it idle
        {"name": "attend-batch", "op": "attend", "sequences": 64, "longest": 8192, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "accumulate": False, "dtype": "bf16"},
        # long contexts
        {"name": "attend-long", "op": "attend", "sequences": 16, "longest": 65536, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "accumulate": False, "dtype": "bf16"},
        # a cache held at a budget: every step adds the step's attention weights, one query head to a key head
        {"name": "attend-accumulate", "op": "attend", "sequences": 32, "longest": 2049, "ragged": False, "heads": 16,
         "kv_heads": 16, "dim": 128, "page": 16, "accumulate": True, "dtype": "fp16"},
        # prompts cut down to what their queries looked at, into a smaller cache
        {"name": "evict-prompt", "op": "evict", "sequences": 8, "longest": 16384, "budget": 2048, "recent": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a decoding step of a cache held at its budget: one token comes, one row of every head goes
        {"name": "evict-step", "op": "step", "sequences": 64, "budget": 2048, "recent": 128, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rotate", "rotate", "append", "attend", "attend", "attend", "evict", "step"))
    kv_heads, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 4, 5, 8, 16))
    dim, dtype, page = rng.choice((64, 80, 96, 128, 128, 192, 256)), rng.choice(("bf16", "fp16")), rng.choice((16, 24, 64, 128))
    if op == "rotate":
        heads = min(kv_heads * group, 64)
        heads -= heads % kv_heads
        rotated = rng.choice((dim, dim, dim // 2))
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        backward = rng.random() < 0.5
        most = 16384 * 40 * 128 * 2 // ((heads + kv_heads) * dim * _BYTES[dtype] * (3 if backward else 1))
        return {"op": op, "tokens": _log(rng, 1, max(1, min(16384, most))), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rotated": rotated, "axes": rng.choice((1, 1, 2, 3)), "interleaved": rng.random() < 0.5,
                "backward": backward, "dtype": dtype}
    if op == "append":
        sequences = _log(rng, 1, 128)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 65536 * 8 * 128 // (sequences * kv_heads * dim)))
        return {"op": op, "sequences": sequences, "longest": _log(rng, 1, 4096), "new": min(new, 8192),
                "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    if op == "attend":
        sequences = _log(rng, 1, 128)
        most = 16 * 65536 * 8 * 128 // (sequences * kv_heads * dim) // 4
        return {"op": op, "sequences": sequences, "longest": _log(rng, 1, max(1, min(65536, most))),
                "ragged": rng.random() < 0.7, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
                "accumulate": rng.random() < 0.3, "dtype": dtype}
    if op == "evict":
        longest = _log(rng, 64, 16384)
        budget = _log(rng, max(16, longest // 16), longest)
        return {"op": op, "sequences": _log(rng, 1, 8), "longest": longest, "budget": budget,
                "recent": rng.randint(0, budget // 2), "kv_heads": min(kv_heads, 8), "dim": min(dim, 128), "page": page,
                "dtype": dtype}
    budget = _log(rng, 16, 2048)
    return {"op": op, "sequences": _log(rng, 1, 64), "budget": budget, "recent": rng.randint(1, max(1, budget // 4)),
            "kv_heads": min(kv_heads, 8), "dim": min(dim, 128), "page": page, "dtype": dtype}


def _ragged(case, count, longest, ragged, what):
    """`count` lengths up to `longest`, the case's own; the last of eight or more ragged ones is 0."""
    if not ragged:
        return [longest] * count
    rng = random.Random("%s %d %d" % (what, count, longest))
    lengths = [longest] + [_log(rng, max(1, longest // 16), longest) for _ in range(count - 1)]
    if count >= 8:
        lengths[-1] = 0
    return lengths


def _lengths(case):
    """(tokens that each sequence holds, tokens that it takes)."""
    n = case["sequences"]
    if case["op"] == "append":
        new = _ragged(case, n, case["new"], case["new"] > 1, "new")
        return _ragged(case, n, case["longest"], True, "held"), new
    if case["op"] == "attend":
        return _ragged(case, n, case["longest"], case["ragged"], "held"), None
    if case["op"] == "evict":
        return _ragged(case, n, case["longest"], True, "held"), None
    return [case["budget"]] * n, [1] * n


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "rotate":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes, each = (5, 20) if case["backward"] else (2, 6)
        other = case["tokens"] * case["axes"] * 8 + case["axes"] * case["rotated"] * 2
        return {"bytes": passes * values * size + other, "flops": each * values}
    held, new = _lengths(case)
    row = case["kv_heads"] * case["dim"] * size
    if case["op"] == "append":
        return {"bytes": 4 * sum(new) * row + 8 * case["sequences"], "flops": 0}
    if case["op"] == "attend":
        queries = case["sequences"] * case["heads"] * case["dim"]
        tracked = 8 * sum(held) * case["kv_heads"] if case["accumulate"] else 0
        return {"bytes": 2 * sum(held) * row + 2 * queries * size + tracked,
                "flops": 4 * sum(held) * case["heads"] * case["dim"]}
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in held)
        return {"bytes": 4 * kept * row + (8 * sum(held) + 8 * kept) * case["kv_heads"], "flops": 0}
    n = case["sequences"]
    return {"bytes": 4 * n * row + 4 * n * row + 8 * n * (case["budget"] + 2) * case["kv_heads"], "flops": 0}


# --------------------------------------------------------------------------- inputs
def _cache(case, gen, held, capacity, tracked):
    """A paged cache whose pages lie in no order, as after some time of serving."""
    n, page, heads, dim = case["sequences"], case["page"], case["kv_heads"], case["dim"]
    width = -(-capacity // page)
    pages = n * width + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[: n * width].reshape(n, width).to(torch.int32)
    key, value = (torch.randn(pages * page, heads, dim, generator=gen, device="cuda", dtype=_TYPES[case["dtype"]])
                  for _ in range(2))
    state = {"key": key, "value": value, "table": table, "page": page,
             "lengths": torch.tensor(held, dtype=torch.int32, device="cuda")}
    if tracked:
        shape = (n, heads, width * page)
        # what a long run of queries leaves: a few slots with much of the weight
        state["weight"] = torch.randn(shape, generator=gen, device="cuda").exp()
        state["position"] = torch.arange(shape[2], device="cuda", dtype=torch.int32).expand(shape).contiguous()
        state["seen"] = state["lengths"].clone()
    if own:
        state["cache"] = _tiga().PagedCache(
            key, value, table, state["lengths"], page_size=page, weight=state.get("weight"),
            position=state.get("position"), seen=state.get("seen"))
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=kind)

    if case["op"] == "rotate":
        tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        packed = normal(tokens, (heads + 2 * kv_heads) * dim)       # the projection's output: queries, keys, values
        query = packed[:, :heads * dim].view(tokens, heads, dim)
        key = packed[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
        pairs, axes = case["rotated"] // 2, case["axes"]
        exponent = torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs
        frequencies = (10000.0 ** -exponent).to(torch.float32)
        if axes > 1:                                                # every axis owns a run of the pairs
            owner = torch.arange(pairs, device="cuda") * axes // pairs
            frequencies = frequencies * (owner == torch.arange(axes, device="cuda")[:, None])
        limit = 131072 if axes == 1 else 256
        positions = torch.randint(0, limit, (tokens, axes), generator=gen, device="cuda")
        state = {"query": query, "key": key, "positions": positions[:, 0].contiguous() if axes == 1 else positions,
                 "frequencies": frequencies, "interleaved": case["interleaved"],
                 "query_weight": 1 + 0.1 * normal(dim), "key_weight": 1 + 0.1 * normal(dim)}
        if case["backward"]:
            state["grads"] = [normal(tokens, heads, dim), normal(tokens, kv_heads, dim)]
            for name in ("query", "key", "query_weight", "key_weight"):
                state[name] = state[name].detach().requires_grad_()
        return {"op": "rotate", **state}
    held, new = _lengths(case)
    if case["op"] == "append":
        state = _cache(case, gen, held, max(a + b for a, b in zip(held, new)), False)
        total = sum(new)
        state["new_key"], state["new_value"] = (normal(total, case["kv_heads"], case["dim"]) for _ in range(2))
        state["start"] = state["lengths"].clone()
        state["bounds"] = None if case["new"] == 1 else torch.tensor(
            [sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    elif case["op"] == "attend":
        state = _cache(case, gen, held, case["longest"], case["accumulate"])
        state["query"] = normal(case["sequences"], case["heads"], case["dim"])
        state["accumulate"], state["scale"] = case["accumulate"], case["dim"] ** -0.5
        if own:
            tg = _tiga()

            class Attention(tg.MessagePassing):
                reducer = tg.online_softmax()

                def edge(self, src, dst, edge, scale):
                    return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)

            state["attention"] = Attention()
    elif case["op"] == "evict":
        state = _cache(case, gen, held, case["longest"], True)
        state["into"] = _cache(case, gen, [0] * case["sequences"], case["budget"], True)
        state["budget"], state["recent"] = case["budget"], case["recent"]
    else:
        state = _cache(case, gen, held, case["budget"] + 1, True)
        state["new_key"], state["new_value"] = (normal(case["sequences"], case["kv_heads"], case["dim"]) for _ in range(2))
        state["budget"], state["recent"] = case["budget"], case["recent"]
    return {"op": case["op"], **state}


# --------------------------------------------------------------------------- plain forms
def _angles(state):
    positions, frequencies = state["positions"].double(), state["frequencies"].double()
    if frequencies.ndim == 1:
        positions, frequencies = positions[:, None], frequencies[None]
    angle = (positions[:, :, None] * frequencies[None]).sum(1)
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _turn(x, cos, sin, interleaved):
    """Every pair of the first 2 * pairs values turned by its angle."""
    pairs = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * pairs:]), dim=-1)


def _plain_rotate(state):
    cos, sin = _angles(state)
    out, grads, weight_grads = [], [], []
    for at, name in enumerate(("query", "key")):
        x, w = state[name].detach().float(), state[name + "_weight"].detach().float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        unit = x * r
        out.append(_turn(unit * w, cos, sin, state["interleaved"]).to(state[name].dtype))
        if "grads" in state:
            dn = _turn(state["grads"][at].float(), cos, -sin, state["interleaved"])
            weight_grads.append((dn * unit).sum((0, 1)).to(state[name + "_weight"].dtype))
            g = dn * w
            grads.append((r * (g - unit * (g * unit).mean(-1, keepdim=True))).to(state[name].dtype))
    return out + grads + weight_grads


def _slots(state, sequence, place):
    """The cache's row of each sequence's `place`."""
    page = state["page"]
    return state["table"][sequence, place // page].long() * page + place % page


def _plain_append(state):
    rows = torch.arange(state["new_key"].shape[0], device="cuda")
    start = (state["start"] if "start" in state else state["lengths"]).long()
    if state.get("bounds") is None:
        sequence, rank, count = rows, torch.zeros_like(rows), 1
    else:
        bounds = state["bounds"].long()
        sequence = torch.searchsorted(bounds, rows, right=True) - 1
        rank, count = rows - bounds[sequence], bounds[1:] - bounds[:-1]
    place = start[sequence] + rank
    slots = _slots(state, sequence, place)
    state["key"].index_copy_(0, slots, state["new_key"])
    state["value"].index_copy_(0, slots, state["new_value"])
    if "seen" in state:
        state["weight"][sequence, :, place] = 0
        state["position"][sequence, :, place] = state["seen"][sequence][:, None]
        state["seen"].add_(count)
    state["lengths"].copy_(start + count)


def _plain_attend(state):
    lengths, table, query = state["lengths"], state["table"], state["query"]
    n, heads, dim = query.shape
    capacity = table.shape[1] * state["page"]
    place = torch.arange(capacity, device="cuda")
    slots = _slots(state, torch.arange(n, device="cuda")[:, None], place[None])
    kv_heads = state["key"].shape[1]
    q = query.float().view(n, kv_heads, heads // kv_heads, dim)
    there = place[None] < lengths[:, None]
    k = state["key"][slots].float().permute(0, 2, 3, 1)
    score = (q @ k) * state["scale"]
    del k
    score = score.masked_fill(~there[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    del score
    v = state["value"][slots].float().masked_fill(~there[:, :, None, None], 0.0).permute(0, 2, 1, 3)
    out = (p @ v).reshape(n, heads, dim).to(query.dtype)
    if not state["accumulate"]:
        return out
    state["weight"].add_(p.sum(2))
    return [out, state["weight"]]


def _kept(state):
    """Which slots of every (sequence, head) stay: [sequences, heads, capacity]."""
    lengths, weight = state["lengths"].long(), state["weight"]
    place = torch.arange(weight.shape[2], device="cuda")
    held = place[None, None] < lengths[:, None, None]
    newest = state["position"] >= (state["seen"] - state["recent"])[:, None, None]
    rank = weight.masked_fill(newest, math.inf).masked_fill(~held, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(held).expand(weight.shape).clone()
    kept.scatter_(2, order[..., :state["budget"]], True)
    return kept & held


def _move(state, target, sequence, head, source, place):
    """Rows of `state` at (sequence, head, source) go to `target` at (sequence, head, place)."""
    a, b = _slots(state, sequence, source), _slots(target, sequence, place)
    for name in ("key", "value"):
        target[name][b, head] = state[name][a, head]
    for name in ("weight", "position"):
        target[name][sequence, head, place] = state[name][sequence, head, source]


def _plain_evict(state):
    kept, target = _kept(state), state["into"]
    sequence, head, source = kept.nonzero(as_tuple=True)
    place = (kept.cumsum(-1) - 1)[sequence, head, source]
    _move(state, target, sequence, head, source, place)
    target["lengths"].copy_(state["lengths"].clamp(max=state["budget"]))
    target["seen"].copy_(state["seen"])
    return [target[name] for name in ("key", "value", "weight", "position", "lengths", "seen")]


def _plain_step(state):
    _plain_append(state)
    kept, budget = _kept(state), state["budget"]
    place = torch.arange(kept.shape[2], device="cuda")
    held = place[None, None] < state["lengths"][:, None, None]
    sequence, head, hole = (~kept & held & (place < budget)).nonzero(as_tuple=True)
    _, _, source = (kept & (place >= budget)).nonzero(as_tuple=True)
    _move(state, state, sequence, head, source, hole)
    state["lengths"].clamp_(max=budget)
    return [state[name] for name in ("key", "value", "weight", "position", "lengths", "seen")]


# --------------------------------------------------------------------------- one pass
def _own_rotate(state):
    out = _tiga().norm_rotary(state["query"], state["key"], state["positions"], state["frequencies"],
                              query_weight=state["query_weight"], key_weight=state["key_weight"], eps=_EPS,
                              interleaved=state["interleaved"])
    if "grads" not in state:
        return list(out)
    inputs = [state[name] for name in ("query", "key", "query_weight", "key_weight")]
    return [t.detach() for t in out] + list(torch.autograd.grad(out, inputs, state["grads"]))


def _own_attend(state):
    cache = state["cache"]
    if state["accumulate"]:
        return [cache.attend(state["query"], state["scale"], accumulate=True), cache.weight]
    return state["attention"](graph=cache.relation(), src={"key": cache.key, "value": cache.value},
                              dst={"query": state["query"]}, scale=state["scale"])


def run(state):
    op = state["op"]
    if op == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    if op == "append":
        if own:
            state["cache"].append(state["new_key"], state["new_value"], cu_seqlens=state["bounds"], start=state["start"])
        else:
            _plain_append(state)
        return [state["key"], state["value"], state["lengths"]]
    if op == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    if op == "evict":
        if not own:
            return _plain_evict(state)
        cache, target = state["cache"], state["into"]["cache"]
        cache.evict(state["budget"], recent=state["recent"], into=target)
        return [target.key, target.value, target.weight, target.position, target.lengths, target.seen]
    if not own:
        return _plain_step(state)
    cache = state["cache"]
    cache.append(state["new_key"], state["new_value"])
    cache.evict(state["budget"], recent=state["recent"])
    return [cache.key, cache.value, cache.weight, cache.position, cache.lengths, cache.seen]


# --------------------------------------------------------------------------- 64 bits
def _exact_rotate(state):
    """The definition with complex numbers; gradients by automatic differentiation of it."""
    positions = state["positions"].double().reshape(state["query"].shape[0], -1)
    frequencies = state["frequencies"].double().reshape(positions.shape[1], -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions @ frequencies)[:, None]
    pairs = turn.shape[-1]
    out, inputs = [], []
    for name in ("query", "key"):
        x, w = (state[n].detach().double().requires_grad_("grads" in state) for n in (name, name + "_weight"))
        n = torch.nn.functional.normalize(x, dim=-1, eps=0.0) * math.sqrt(x.shape[-1])
        square = x.square().mean(-1, keepdim=True)
        n = n * (square / (square + _EPS)).sqrt() * w
        front = n[..., :2 * pairs]
        front = front.unflatten(-1, (pairs, 2)) if state["interleaved"] else front.unflatten(-1, (2, pairs)).transpose(-1, -2)
        front = torch.view_as_real(torch.view_as_complex(front.contiguous()) * turn)
        front = front if state["interleaved"] else front.transpose(-1, -2)
        out.append(torch.cat((front.flatten(-2), n[..., 2 * pairs:]), dim=-1))
        inputs += [x, w]
    if "grads" not in state:
        return out
    dq, dwq, dk, dwk = torch.autograd.grad(out, inputs, [g.double() for g in state["grads"]])
    return [t.detach() for t in out] + [dq, dk, dwq, dwk]


def _rows(state, b, count):
    """Cache rows of the first `count` places of sequence b."""
    pages = state["table"][b].tolist()
    return torch.tensor([pages[t // state["page"]] * state["page"] + t % state["page"] for t in range(count)],
                        dtype=torch.long, device="cuda")


def _exact_append(state):
    for name in ("key", "value", "weight"):
        if name in state:
            state[name] = state[name].double()
    bounds = list(range(len(state["lengths"]) + 1)) if state.get("bounds") is None else state["bounds"].tolist()
    for b, length in enumerate(state["lengths"].tolist()):
        first, last = bounds[b], bounds[b + 1]
        rows = _rows(state, b, length + last - first)[length:]
        state["key"][rows] = state["new_key"][first:last].double()
        state["value"][rows] = state["new_value"][first:last].double()
        if "seen" in state:
            for t in range(last - first):
                state["weight"][b, :, length + t] = 0
                state["position"][b, :, length + t] = state["seen"][b] + t
            state["seen"][b] += last - first
        state["lengths"][b] += last - first
    return [state["key"], state["value"], state["lengths"]]


def _exact_attend(state):
    query = state["query"].double()
    n, heads, dim = query.shape
    kv_heads = state["key"].shape[1]
    out = torch.zeros_like(query)
    weight = state["weight"].double() if state["accumulate"] else None
    for b, length in enumerate(state["lengths"].tolist()):
        if not length:
            continue
        rows = _rows(state, b, length)
        for h in range(kv_heads):
            group = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            p = torch.softmax(query[b, group] @ state["key"][rows, h].double().T * state["scale"], dim=-1)
            out[b, group] = p @ state["value"][rows, h].double()
            if weight is not None:
                weight[b, h, :length] += p.sum(0)
    return out if weight is None else [out, weight]


def _exact_evict(state, target):
    """Slot by slot of the definition; `target` is `state` itself when rows are moved in place."""
    budget, names = state["budget"], ("key", "value", "weight", "position", "lengths", "seen")
    source = {name: state[name].clone() for name in ("key", "value", "weight", "position")}
    seen = state["seen"].tolist()
    for b, length in enumerate(state["lengths"].tolist()):
        rows = _rows(state, b, length)
        into = _rows(target, b, min(length, budget))
        for h in range(source["key"].shape[1]):
            newest = source["position"][b, h, :length] >= seen[b] - state["recent"]
            w = torch.where(newest, math.inf, source["weight"][b, h, :length].double())
            best = torch.argsort(-w, stable=True)[:budget].sort().values
            if target is not state:
                place = torch.arange(best.numel(), device="cuda")
            else:
                stays, comes = best[best < budget], best[best >= budget]
                free = torch.ones(min(length, budget), dtype=torch.bool, device="cuda")
                free[stays] = False
                place, best = free.nonzero()[:, 0][:comes.numel()], comes
            for name in ("key", "value"):
                target[name][into[place], h] = source[name][rows[best], h]
            for name in ("weight", "position"):
                target[name][b, h, place] = source[name][b, h, best]
    target["lengths"].copy_(state["lengths"].clamp(max=budget))
    target["seen"].copy_(state["seen"])
    return [target[name].double() if target[name].is_floating_point() else target[name] for name in names]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(state)
    if case["op"] == "append":
        return _exact_append(state)
    if case["op"] == "attend":
        return _exact_attend(state)
    if case["op"] == "evict":
        return _exact_evict(state, state["into"])
    _exact_append(state)
    return _exact_evict(state, state)
