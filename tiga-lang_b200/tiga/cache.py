"""Paged key/value cache: the source side of attention when a model answers token by token.

A cache is a relation whose destination rows are sequences and whose source rows are cache slots:
sequence i gathers from the first ``lengths[i]`` slots of its pages.  The online-softmax attention program
that runs over packed sequences (``Graph.cu_seqlens``) runs over ``cache.relation()`` too.  The reference
has no such relation; the nearest is its CSR over slots, which would be rebuilt for every token
(python/tiga/graph/core.py:157-217 of walkerchi/TIGA-lang).
"""
from __future__ import annotations

import collections
import ctypes

import torch

from . import _native
from .graph import Graph, GraphSchema
from .ops import current_device, forward_ad, raw_stream, refuse_tangents

_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}
_FAULTS = {
    1: "a page table entry lies outside the cache's pages",
    2: "tokens were appended beyond a sequence's capacity and dropped",
    3: "a length lies outside [0, capacity]",
    4: "a start lies outside [0, length]",
    5: "cu_seqlens run backwards or leave the tokens, and places that nothing was written to may count as held",
}


class _FaultWord:
    """A pinned word of one cache, and of those that ``over`` makes of it, that the kernels store a code into when a
    table, length, start or bound is out of range.  They skip the access, so the context stays usable; the cache's next
    call sees the code and raises.  (The kernels write host memory directly and only then: the good path has no copy
    and no extra launch.)

    The words are never given back, because kernels and recorded graphs may outlive the cache; a dropped cache's
    word is handed out again after the others that wait in line, a thousand at least."""

    _waiting: collections.deque = collections.deque()
    _chunks: list = []

    def __init__(self):
        if len(self._waiting) <= 1024:
            chunk = torch.zeros(4096, dtype=torch.int32, device="cpu").pin_memory()
            self._chunks.append(chunk)
            self._waiting.extend(range(chunk.data_ptr(), chunk.data_ptr() + 4 * chunk.numel(), 4))
        self.address = self._waiting.popleft()
        self.value = ctypes.c_int32.from_address(self.address)
        self.value.value = 0

    def __del__(self, waiting=_waiting):
        if hasattr(self, "address"):
            waiting.append(self.address)

    def raise_if_set(self, device):
        if self.value.value:
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.synchronize(device)      # the call at fault may still be storing its code
            code, self.value.value = self.value.value, 0
            raise RuntimeError("an earlier call on this paged cache met bad contents: "
                               f"{_FAULTS.get(code, f'code {code}')}; its results are incomplete")


def _same_memory(a, b) -> bool:
    """Tensors without elements all have the address 0."""
    return a.data_ptr() == b.data_ptr() and a.numel() > 0 and b.numel() > 0


class PagedCache:
    """Keys and values of many sequences in pages.

    ``key``, ``value``  [slots, H_kv, D] bfloat16 or float16 with ``slots`` a multiple of ``page_size``;
    any strides that keep every row of D values (a multiple of 8, at most 256) 16-byte aligned.
    ``page_table``  int32 [sequences, pages_per_sequence]; ``lengths``  int32 [sequences].  Place t of
    sequence i is slot ``page_table[i, t // page_size] * page_size + t % page_size``.

    ``weight`` (float32) and ``position`` (int32), both [sequences, H_kv, capacity], and ``seen`` (int32
    [sequences]) make the cache track what its places were looked at with, which ``evict`` needs; each
    head may then hold other tokens at a place.

    The tensors are the caller's and are read when a kernel runs: writing to ``page_table`` or ``lengths`` on the
    stream between two calls is how pages are handed out and taken back, and calls recorded in a CUDA graph read the
    contents of the replay. The kernels have the tensors' addresses: contents change in place, and assigning another
    tensor to an attribute raises (so must their storage stay: no ``.data =``, ``set_`` or ``resize_``). Sequences
    may share pages that nothing is appended to or evicted from. Calls on one cache are ordered by their stream;
    from several streams the caller orders them. Contents that lie outside their range are never followed: the
    access is skipped and the next call on the cache (or ``check()``) raises."""

    _FIXED = frozenset(("key", "value", "page_table", "lengths", "weight", "position", "seen", "page_size", "capacity",
                        "sequences", "heads", "dim", "device"))

    def __setattr__(self, name, value):
        # the same object may be assigned again: that is what `cache.lengths += 1` does after its in-place addition
        if name in self._FIXED and self.__dict__.get(name, value) is not value:
            raise AttributeError(f"{name} of a paged cache cannot be exchanged; write to its contents, or make another cache")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        if name in self._FIXED:
            raise AttributeError(f"{name} of a paged cache cannot be deleted")
        object.__delattr__(self, name)

    def __init__(self, key, value, page_table, lengths, *, page_size: int, weight=None, position=None, seen=None,
                 _fault: _FaultWord | None = None):
        if not isinstance(page_size, int) or page_size < 1:
            raise ValueError(f"page_size must be a positive number, got {page_size!r}")
        for name, t in (("key", key), ("value", value)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype not in _DTYPES:
                raise NotImplementedError(f"a paged cache holds bfloat16 or float16; {name} is {t.dtype}")
            if t.ndim != 3 or t.shape[0] < page_size or t.shape[0] % page_size:
                raise ValueError(f"{name} must have shape [pages * {page_size}, heads, dim], got {tuple(t.shape)}")
        if key.shape != value.shape or key.dtype != value.dtype or key.device != value.device:
            raise ValueError("key and value must share shape, dtype and device")
        slots, heads, dim = key.shape
        if heads < 1 or not 8 <= dim <= 256 or dim % 8:
            raise NotImplementedError(f"head sizes are multiples of 8 up to 256, got {heads} heads of {dim}")
        for name, t in (("key", key), ("value", value)):
            if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
                raise ValueError(f"{name} rows must be 16-byte aligned runs of {dim} values")
            if t.requires_grad:
                raise NotImplementedError("a paged cache has no gradients")
        if forward_ad._current_level >= 0:
            refuse_tangents("a paged cache", key, value, weight)
        device = key.device
        for name, t, ndim in (("page_table", page_table, 2), ("lengths", lengths, 1)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.ndim != ndim or not t.is_contiguous() \
                    or t.device != device:
                raise ValueError(f"{name} must be a contiguous int32 tensor of {ndim} dimension(s) on {device}")
        sequences, width = page_table.shape
        if lengths.shape[0] != sequences:
            raise ValueError(f"lengths must have {sequences} entries, got {lengths.shape[0]}")
        capacity = width * page_size
        if capacity > 1 << 30 or heads > 1 << 16 or sequences * heads > 1 << 30 or slots >= 1 << 31 \
                or max(key.stride(0), value.stride(0)) > 1 << 30:
            raise NotImplementedError("at most 2^30 places per sequence, 2^16 heads, 2^30 pairs of sequence and head, "
                                      "2^31 slots and 2^30 values from slot to slot")
        tracked = [t is not None for t in (weight, position, seen)]
        if any(tracked):
            if not all(tracked):
                raise ValueError("weight, position and seen come together")
            for name, t, kind, shape in (("weight", weight, torch.float32, (sequences, heads, capacity)),
                                         ("position", position, torch.int32, (sequences, heads, capacity)),
                                         ("seen", seen, torch.int32, (sequences,))):
                if t.dtype != kind or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
                    raise ValueError(f"{name} must be contiguous {kind} of shape {shape} on {device}")
        self.__dict__.update(key=key, value=value, page_table=page_table, lengths=lengths, weight=weight, position=position,
                             seen=seen, page_size=page_size, capacity=capacity, sequences=sequences, heads=heads, dim=dim,
                             device=device)
        self._index = device.index
        self._relation = self._block = self._address = self._fault = None
        self._scratch_bytes: dict = {}
        self._dtype, self._lib = key.dtype, None
        if device.type == "cuda":
            self._fault = _FaultWord() if _fault is None else _fault
            self._block = b = _native.PagedCacheArguments()
            b.key, b.value = key.data_ptr(), value.data_ptr()
            b.key_slot_stride, b.key_head_stride = key.stride(0), key.stride(1)
            b.value_slot_stride, b.value_head_stride = value.stride(0), value.stride(1)
            b.page_table, b.lengths = page_table.data_ptr(), lengths.data_ptr()
            if weight is not None:
                b.weight, b.position, b.seen = weight.data_ptr(), position.data_ptr(), seen.data_ptr()
            b.fault, b.num_pages = self._fault.address, slots // page_size
            b.sequences, b.pages_per_sequence, b.page_size = sequences, width, page_size
            b.heads, b.dim, b.dtype = heads, dim, _DTYPES[key.dtype]
            self._address = ctypes.addressof(b)

    @classmethod
    def empty(cls, sequences: int, capacity: int, heads: int, dim: int, *, page_size: int = 64,
              dtype=torch.bfloat16, device="cuda", track: bool = False) -> "PagedCache":
        """A cache of its own memory in which every sequence owns ``capacity`` places (rounded up to pages)."""
        if sequences < 1 or capacity < 1 or page_size < 1:
            raise ValueError("sequences, capacity and page_size must be positive")
        width = -(-capacity // page_size)
        key, value = (torch.zeros(sequences * width * page_size, heads, dim, dtype=dtype, device=device)
                      for _ in range(2))
        table = torch.arange(sequences * width, dtype=torch.int32, device=device).reshape(sequences, width)
        lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        state = {}
        if track:
            shape = (sequences, heads, width * page_size)
            state = {"weight": torch.zeros(shape, dtype=torch.float32, device=device),
                     "position": torch.zeros(shape, dtype=torch.int32, device=device), "seen": torch.zeros_like(lengths)}
        return cls(key, value, table, lengths, page_size=page_size, **state)

    @property
    def tracked(self) -> bool:
        return self.weight is not None

    def check(self) -> None:
        """Waits for the device and raises if a call met contents out of range."""
        if self._block is not None:
            torch.cuda.synchronize(self.device)
        self._ready()

    def _ready(self):
        """The address of the cache's descriptor, once earlier calls are known not to have failed."""
        if self._block is None:
            raise RuntimeError("a paged cache runs on CUDA tensors only (no CPU fallback)")
        if self._fault.value.value:
            self._fault.raise_if_set(self.device)
        if self._lib is None:
            self._lib = _native.lib()
        return self._address

    def _rows(self, name, t, rows):
        """New rows as the kernels read them: a tensor, its address and strides."""
        if not isinstance(t, torch.Tensor) or t.shape != (t.shape[0] if rows is None and t.ndim else rows, self.heads, self.dim) \
                or t.dtype is not self._dtype or t.get_device() != self._index:
            raise ValueError(f"{name} must be {self.key.dtype} of shape "
                             f"[{'tokens' if rows is None else rows}, {self.heads}, {self.dim}] on {self.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("a paged cache has no gradients; packed sequences (Graph.cu_seqlens) are the "
                                      "form to train with")
        token, head, value = t.stride()
        address = t.data_ptr()
        if value != 1 or (token | head) % 8 or address % 16:
            t = t.detach().clone(memory_format=torch.contiguous_format)
            (token, head, value), address = t.stride(), t.data_ptr()
        return t, address, token, head

    def _entries(self, name, t, count):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.shape != (count,) \
                or not t.is_contiguous() or t.get_device() != self._index:
            raise ValueError(f"{name} must be a contiguous int32 tensor of {count} entries on {self.device}")
        return t.data_ptr()

    def _launch(self, function, name, *arguments):
        if current_device() == self._index:
            status = function(*arguments)
        else:
            with torch.cuda.device(self._index):
                status = function(*arguments)
        if status:
            _native.check(status, name)

    def append(self, key, value, *, cu_seqlens=None, start=None) -> None:
        """Rows of new tokens, [tokens, H_kv, D], behind what each sequence holds.

        One token per sequence, or with ``cu_seqlens`` (int32 [sequences + 1]) the run ``cu_seqlens[i] :
        cu_seqlens[i + 1]`` for sequence i; tokens outside every run are ignored, bounds that run backwards or leave
        the tokens are reported. ``start`` (int32 [sequences], at most the length) puts a run at place ``start[i]``
        instead, dropping what was there and behind it: how drafted tokens are taken back. Tokens beyond the
        capacity are dropped and reported. In a tracking cache the new places have weight 0 and the tokens' numbers
        as positions; a start behind which an eviction has moved rows drops those rows, whichever tokens they
        are."""
        cache = self._ready()
        if forward_ad._current_level >= 0:
            refuse_tangents("a paged cache", key, value)
        key, key_address, key_token, key_head = self._rows("key", key, self.sequences if cu_seqlens is None else None)
        tokens = key.shape[0]
        value, value_address, value_token, value_head = self._rows("value", value, tokens)
        bounds = None if cu_seqlens is None else self._entries("cu_seqlens", cu_seqlens, self.sequences + 1)
        first = None if start is None else self._entries("start", start, self.sequences)
        self._launch(self._lib.tgb_cache_append, "tgb_cache_append", cache, key_address, value_address, key_token,
                     key_head, value_token, value_head, tokens, bounds, first, raw_stream(self._index))

    def relation(self) -> Graph:
        """The cache as a relation: ``num_src`` slots, one destination row per sequence.  Attention
        programs over it read table and lengths at every call; ``resolve_csr()`` is what they hold now."""
        relation = self._relation
        if relation is None:
            schema = GraphSchema(num_src=self.key.shape[0], num_dst=self.sequences, origin="paged_cache",
                                 lifecycle="dynamic", realization="paged_cache", index_dtype=torch.int64,
                                 sorted_by_dst=True)
            relation = Graph(schema, device=self.device)
            # the relation has a cache object of its own over the same tensors and fault word: this one keeps the
            # relation, and neither waits for the collector of reference cycles
            twin = object.__new__(type(self))
            twin.__dict__.update(self.__dict__)
            relation._cache, relation._cache_signature = twin, schema.specialization_key()
            self._relation = relation
        return relation

    def over(self, key, value) -> "PagedCache":
        """The cache of other keys and values under the same table and lengths: the layers of a model share
        one table.  (No tracked state: that belongs to the keys it was gathered from.)  Bad contents that a call on one of
        them meets are reported by whichever is called next."""
        if key is self.key and value is self.value:
            return self
        return PagedCache(key, value, self.page_table, self.lengths, page_size=self.page_size, _fault=self._fault)

    def resolve_csr(self):
        """(row_ptr, col_idx) of the slots that the sequences hold now.  Waits for the device, and raises where a length or
        a page that it reaches is out of range."""
        table, lengths = self.page_table.long(), self.lengths.long()
        if bool(((lengths < 0) | (lengths > self.capacity)).any()):
            raise RuntimeError(f"the paged cache has bad contents: {_FAULTS[3]}")
        first_place = torch.arange(table.shape[1], device=self.device) * self.page_size
        reached = first_place < lengths[:, None]
        if bool((reached & ((table < 0) | (table >= self.key.shape[0] // self.page_size))).any()):
            raise RuntimeError(f"the paged cache has bad contents: {_FAULTS[1]}")
        place = torch.arange(self.capacity, device=self.device)
        slots = table[:, place // self.page_size] * self.page_size + place % self.page_size
        row_ptr = torch.zeros(self.sequences + 1, dtype=torch.int64, device=self.device)
        torch.cumsum(lengths, 0, out=row_ptr[1:])
        return row_ptr, slots[place < lengths[:, None]]

    def attend(self, query, scale: float | None = None, *, accumulate: bool = False) -> torch.Tensor:
        """Attention of one query per sequence, [sequences, H, D] with H a multiple of H_kv, over the
        places that its sequence holds: ``softmax(scale * q . key) value`` (scale: 1 / sqrt(D) by default), 0 for a
        sequence without any. ``accumulate`` adds each place's softmax weights, summed over the query heads that
        share a key head, to ``weight``. Inference only: gradients are refused, forward-mode ones too. Scores of
        -inf alone give 0, as an empty row does, and nothing is read of places that hold no token; an infinite value
        is the result of its column unless its place's weight is below 2^-102 of the largest.
        ``accumulate`` takes scratch of 4 bytes per query head and place of the capacity for the call."""
        cache = self._ready()
        if not isinstance(query, torch.Tensor) or query.ndim != 3:
            raise ValueError(f"query must have shape [{self.sequences}, heads, {self.dim}]")
        sequences, heads, dim = query.shape
        if sequences != self.sequences or dim != self.dim or query.get_device() != self._index:
            raise ValueError(f"query must have shape [{self.sequences}, heads, {self.dim}] on {self.device}, got "
                             f"{tuple(query.shape)} on {query.device}")
        if query.dtype is not self._dtype:
            raise NotImplementedError(f"query and cache must share one dtype, got {query.dtype} and {self.key.dtype}")
        if heads < 1 or heads % self.heads:
            raise NotImplementedError(f"{heads} query heads are no multiple of the cache's {self.heads}")
        if heads > 1 << 16:
            raise NotImplementedError("at most 65536 query heads")
        if query.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("attention over a paged cache has no backward; packed sequences "
                                      "(Graph.cu_seqlens) are the form to train with")
        if forward_ad._current_level >= 0:
            refuse_tangents("attention over a paged cache", query)
        if accumulate and self.weight is None:
            raise ValueError("accumulate needs a cache that tracks attention weights")
        token, head, value = query.stride()
        address = query.data_ptr()
        if value != 1 or (token | head) % 2 or address % 4:
            query = query.detach().clone(memory_format=torch.contiguous_format)
            (token, head, value), address = query.stride(), query.data_ptr()
        lib = self._lib
        accumulate = bool(accumulate)
        size = self._scratch_bytes.get((heads, accumulate))
        if size is None:
            needed = ctypes.c_uint64()
            _native.check(lib.tgb_cache_attend_scratch_bytes(cache, heads, accumulate, ctypes.byref(needed)),
                          "tgb_cache_attend_scratch_bytes")
            size = self._scratch_bytes[(heads, accumulate)] = int(needed.value)
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None    # small caches need none
        self._launch(lib.tgb_cache_attend, "tgb_cache_attend", cache, address, token, head, out.data_ptr(), heads,
                     dim ** -0.5 if scale is None else scale, accumulate,
                     None if scratch is None else scratch.data_ptr(), size, raw_stream(self._index))
        return out

    def evict(self, budget: int, *, recent: int = 0, into: "PagedCache | None" = None) -> None:
        """At most ``budget`` places stay for every sequence and head: those of the newest ``recent``
        tokens, then those with the largest accumulated weight (of equal ones the lowest place; NaN counts as the
        smallest).  In place, the i-th place freed below the budget takes the i-th row kept at or above it,
        so that few rows move and the rest stay where they are; ``into`` another cache, which may read the same
        pool but owns pages of its own, the kept rows are written in the order of their places and this
        cache is left as it is: the form for pages that sequences share."""
        cache = self._ready()
        if not isinstance(budget, int) or not 1 <= budget < 1 << 31:
            raise ValueError(f"budget must be a positive number, got {budget!r}")
        if not isinstance(recent, int) or not 0 <= recent <= budget:
            raise ValueError(f"recent must lie in [0, {budget}], got {recent!r}")
        if self.weight is None:
            raise ValueError("evict needs a cache that tracks attention weights")
        target = None
        if into is not None and into is not self:
            if not isinstance(into, PagedCache) or into.sequences != self.sequences or into.heads != self.heads \
                    or into.dim != self.dim or into.key.dtype != self.key.dtype or into.device != self.device:
                raise ValueError("into must be a PagedCache of the same sequences, heads, dim, dtype and device")
            if into.capacity < min(budget, self.capacity):
                raise ValueError(f"into holds {into.capacity} places per sequence, fewer than the budget of {budget}")
            if _same_memory(into.lengths, self.lengths) or (
                    into.weight is not None and _same_memory(into.weight, self.weight)):
                raise ValueError("into must have lengths and tracked state of its own")
            if _same_memory(into.page_table, self.page_table) and _same_memory(into.key, self.key):
                raise ValueError("into must have pages of its own")
            target = into._ready()
        lib = self._lib
        size = self._scratch_bytes.get(budget)
        if size is None:
            needed = ctypes.c_uint64()
            _native.check(lib.tgb_cache_evict_scratch_bytes(cache, budget, ctypes.byref(needed)),
                          "tgb_cache_evict_scratch_bytes")
            size = self._scratch_bytes[budget] = max(int(needed.value), 8)
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device)
        self._launch(lib.tgb_cache_evict, "tgb_cache_evict", cache, target, budget, recent, scratch.data_ptr(), size,
                     raw_stream(self._index))


__all__ = ["PagedCache"]
