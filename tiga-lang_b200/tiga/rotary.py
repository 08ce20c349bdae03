"""Norm and rotation of query and key heads: what stands between a projection and attention.

``norm_rotary`` is one kernel for both fields (forward) and one more for the gradients, so the
positions of a token are turned into sines and cosines once for all of its heads.  The reference has no
counterpart; its attention programs take fields that are already positioned
(python/tiga/interop/torch/message_passing.py:1910-2020 of walkerchi/TIGA-lang).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .ops import _OnDevice, _stream

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}
_MAX_DIM, _MAX_AXES = 1024, 8


def rotary_frequencies(dim: int, *, base: float = 10000.0, sections=None, device=None) -> torch.Tensor:
    """Frequencies of the ``dim // 2`` pairs of a rotation over ``dim`` values: ``base ** (-j / pairs)``.

    ``sections`` gives each position axis its own run of the pairs (their counts must add up to
    ``dim // 2``); the result is then ``[axes, pairs]`` with zeros where an axis has no part in a pair,
    and ``[pairs]`` without sections.  Any other assignment is a matrix of the caller's own."""
    if not isinstance(dim, int) or dim < 2 or dim % 2:
        raise ValueError(f"dim must be a positive even number, got {dim!r}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base!r}")
    pairs = dim // 2
    exponent = torch.arange(pairs, dtype=torch.float64) / pairs
    frequencies = (float(base) ** -exponent).to(torch.float32)
    if sections is not None:
        sections = tuple(int(n) for n in sections)
        if not sections or min(sections) < 0 or sum(sections) != pairs:
            raise ValueError(f"sections must be counts that add up to {pairs} pairs, got {sections}")
        owner = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
        frequencies = frequencies * (owner == torch.arange(len(sections))[:, None])
    return frequencies.to(device) if device is not None else frequencies


def _check(query, key, positions, frequencies, query_weight, key_weight, eps):
    if not isinstance(query, torch.Tensor) or not query.is_cuda:
        raise RuntimeError("norm_rotary runs on CUDA tensors only (no CPU fallback)")
    if query.dtype not in _DTYPES:
        raise NotImplementedError(f"norm_rotary takes float32, bfloat16 or float16 fields; query is {query.dtype}")
    if query.ndim != 3:
        raise ValueError(f"query must have shape [tokens, heads, dim], got {tuple(query.shape)}")
    tokens, _, dim = query.shape
    device = query.device
    if not 1 <= dim <= _MAX_DIM:
        raise NotImplementedError(f"head sizes from 1 to {_MAX_DIM} are supported, got {dim}")
    if key is not None and (key.ndim != 3 or key.shape[0] != tokens or key.shape[2] != dim or key.dtype != query.dtype
                            or key.device != device):
        raise ValueError(f"key must have shape [{tokens}, heads, {dim}] and the query's dtype and device, got "
                         f"{tuple(key.shape)}, {key.dtype} on {key.device}")
    if frequencies.dtype != torch.float32 or frequencies.ndim not in (1, 2) or frequencies.device != device:
        raise ValueError(f"frequencies must be float32 [pairs] or [axes, pairs] on {device}")
    axes = 1 if frequencies.ndim == 1 else frequencies.shape[0]
    pairs = frequencies.shape[-1]
    if 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs do not fit into heads of {dim} values")
    if not 1 <= axes <= _MAX_AXES:
        raise NotImplementedError(f"1 to {_MAX_AXES} position axes are supported, got {axes}")
    shape = (tokens,) if frequencies.ndim == 1 else (tokens, axes)
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) != shape or positions.device != device:
        raise ValueError(f"positions must be int32 or int64 of shape {shape} on {device}, got "
                         f"{positions.dtype} {tuple(positions.shape)} on {positions.device}")
    if frequencies.requires_grad:
        raise NotImplementedError("frequencies have no gradient here")
    kind = None
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if w is None:
            continue
        if eps is None:
            raise ValueError(f"{name} belongs to the norm, which eps=None leaves out")
        if name == "key_weight" and key is None:
            raise ValueError("key_weight without a key")
        if tuple(w.shape) != (dim,) or w.device != device or w.dtype not in (torch.float32, query.dtype):
            raise ValueError(f"{name} must have shape ({dim},) on {device}, in float32 or the query's dtype; got "
                             f"{tuple(w.shape)}, {w.dtype} on {w.device}")
        if kind not in (None, w.dtype):
            raise ValueError("query_weight and key_weight must share one dtype")
        kind = w.dtype
    if eps is not None and not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps!r}")


def _rows(field):
    return field if field.stride(2) == 1 or field.shape[2] == 1 else field.contiguous()


def _arguments(fields, weights, positions, frequencies, eps, interleaved):
    """The argument block without its outputs; every tensor named in it must outlive the launch's enqueueing."""
    a = _native.NormRotary()
    first = fields[0]
    kind = None
    for side in (0, 1):
        x = fields[side]
        if x is None:
            continue
        a.x[side] = x.data_ptr()
        a.x_token_stride[side], a.x_head_stride[side] = x.stride(0), x.stride(1)
        a.heads[side] = x.shape[1]
        w = weights[side]
        if w is not None:
            a.weight[side] = w.data_ptr()
            kind = w.dtype
    a.tokens, a.dim = first.shape[0], first.shape[2]
    a.positions, a.position_bits = positions.data_ptr(), 64 if positions.dtype == torch.int64 else 32
    a.frequencies = frequencies.data_ptr()
    a.pairs, a.axes = frequencies.shape[-1], 1 if frequencies.ndim == 1 else frequencies.shape[0]
    a.dtype, a.weight_dtype = _DTYPES[first.dtype], _DTYPES[kind or first.dtype]
    a.normalise, a.eps = int(eps is not None), 0.0 if eps is None else eps
    a.interleaved = int(interleaved)
    return a


def _forward(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved):
    device = query.device
    a = _arguments((query, key), (query_weight, key_weight), positions, frequencies, eps, interleaved)
    out = [torch.empty(x.shape, dtype=x.dtype, device=device) if x is not None else None for x in (query, key)]
    for side in (0, 1):
        if out[side] is not None:
            a.out[side] = out[side].data_ptr()
    with _OnDevice(device):
        _native.check(_native.lib().tgb_norm_rotary_fwd(ctypes.addressof(a), _stream(device)), "tgb_norm_rotary_fwd")
    return out


class NormRotaryFunction(torch.autograd.Function):
    """Saves the inputs alone; the backward recomputes each head's norm."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, frequencies, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        query, key = _forward(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved)
        return query if key is None else (query, key)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        query, key, query_weight, key_weight, positions, frequencies = ctx.saved_tensors
        device, dim = query.device, query.shape[2]
        fields, weights = (query, key), (query_weight, key_weight)
        a = _arguments(fields, weights, positions, frequencies, ctx.eps, ctx.interleaved)
        kept, out, weight_grads = [], [None, None], [None, None]
        for side, x in enumerate(fields):
            if x is None:
                continue
            dy = _rows(grads[side].to(x.dtype))
            kept.append(dy)
            a.dy[side], a.dy_token_stride[side], a.dy_head_stride[side] = dy.data_ptr(), dy.stride(0), dy.stride(1)
            out[side] = torch.empty(x.shape, dtype=x.dtype, device=device)
            a.out[side] = out[side].data_ptr()
            if weights[side] is not None and ctx.needs_input_grad[2 + side]:
                weight_grads[side] = torch.empty_like(weights[side], memory_format=torch.contiguous_format)
        scratch = None
        lib = _native.lib()
        if any(w is not None for w in weight_grads):
            scratch = torch.empty(lib.tgb_norm_rotary_scratch_bytes(dim), dtype=torch.uint8, device=device)
        with _OnDevice(device):
            _native.check(lib.tgb_norm_rotary_bwd(
                ctypes.addressof(a), *(None if w is None else w.data_ptr() for w in weight_grads),
                None if scratch is None else scratch.data_ptr(), 0 if scratch is None else scratch.numel(),
                _stream(device)), "tgb_norm_rotary_bwd")
        needs = ctx.needs_input_grad
        return (out[0] if needs[0] else None, out[1] if needs[1] else None, weight_grads[0], weight_grads[1],
                None, None, None, None)


def norm_rotary(query, key, positions, frequencies, *, query_weight=None, key_weight=None, eps: float | None = 1e-6,
                interleaved: bool = False):
    """Query and key heads, each normalised by its root mean square and turned by its token's position.

    ``query`` [tokens, H, D] and ``key`` [tokens, H_kv, D] (or None) may be views into a packed projection.
    ``frequencies`` (float32) is ``[pairs]`` with ``positions`` [tokens], or ``[axes, pairs]`` with
    ``positions`` [tokens, axes]: pair j of a token turns by ``sum_a positions[a] * frequencies[a, j]``,
    formed in 64 bits.  Pair j is ``(j, j + pairs)``, or ``(2j, 2j + 1)`` with ``interleaved``; values from
    ``2 * pairs`` on are not turned.  ``eps=None`` leaves the norm out.  Returns contiguous
    ``(query, key)``, or the query alone when ``key`` is None; differentiable in fields and weights."""
    _check(query, key, positions, frequencies, query_weight, key_weight, eps)
    query, key = _rows(query), None if key is None else _rows(key)
    query_weight, key_weight = (None if w is None else w.contiguous() for w in (query_weight, key_weight))
    positions, frequencies = positions.contiguous(), frequencies.contiguous()
    arguments = (query, key, query_weight, key_weight, positions, frequencies, eps, bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in arguments[:4]):
        return NormRotaryFunction.apply(*arguments)
    query, key = _forward(*arguments)
    return query if key is None else (query, key)


__all__ = ["norm_rotary", "rotary_frequencies"]
