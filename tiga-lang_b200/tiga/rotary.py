"""Norm and rotation of query and key heads: what stands between a projection and attention.

``norm_rotary`` is one kernel for both fields (forward) and one more for the gradients, so the
positions of a token are turned into sines and cosines once for all of its heads.  The reference has no
counterpart; its attention programs take fields that are already positioned
(python/tiga/interop/torch/message_passing.py:1910-2020 of walkerchi/TIGA-lang).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .ops import current_device, forward_ad, raw_stream, refuse_tangents

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
    """Raises for arguments the kernels do not take.  Runs in every call: shapes and dtypes are compared as
    they are, and a message is formed only to be raised."""
    if not isinstance(query, torch.Tensor) or not query.is_cuda:
        raise RuntimeError("norm_rotary runs on CUDA tensors only (no CPU fallback)")
    kind, index = query.dtype, query.get_device()
    if kind not in _DTYPES:
        raise NotImplementedError(f"norm_rotary takes float32, bfloat16 or float16 fields; query is {kind}")
    if query.ndim != 3:
        raise ValueError(f"query must have shape [tokens, heads, dim], got {tuple(query.shape)}")
    tokens, _, dim = query.shape
    if not 1 <= dim <= _MAX_DIM:
        raise NotImplementedError(f"head sizes from 1 to {_MAX_DIM} are supported, got {dim}")
    if key is not None:
        shape = key.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or key.dtype is not kind or key.get_device() != index:
            raise ValueError(f"key must have shape [{tokens}, heads, {dim}] and the query's dtype and device, got "
                             f"{tuple(shape)}, {key.dtype} on {key.device}")
    shape = frequencies.shape
    if frequencies.dtype is not torch.float32 or len(shape) not in (1, 2) or frequencies.get_device() != index:
        raise ValueError(f"frequencies must be float32 [pairs] or [axes, pairs] on {query.device}")
    if 2 * shape[-1] > dim:
        raise ValueError(f"{shape[-1]} pairs do not fit into heads of {dim} values")
    if len(shape) == 2 and not 1 <= shape[0] <= _MAX_AXES:
        raise NotImplementedError(f"1 to {_MAX_AXES} position axes are supported, got {shape[0]}")
    wanted = (tokens,) if len(shape) == 1 else (tokens, shape[0])
    if positions.shape != wanted or positions.get_device() != index \
            or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"positions must be int32 or int64 of shape {wanted} on {query.device}, got "
                         f"{positions.dtype} {tuple(positions.shape)} on {positions.device}")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("frequencies have no gradient here")
    if query_weight is not None or key_weight is not None:
        _check_weights(query, key, query_weight, key_weight, eps)
    if eps is not None and not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps!r}")
    if forward_ad._current_level >= 0:
        refuse_tangents("norm_rotary", query, key, frequencies, query_weight, key_weight)


def _check_weights(query, key, query_weight, key_weight, eps):
    dim, index, kind = query.shape[2], query.get_device(), None
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if w is None:
            continue
        if eps is None:
            raise ValueError(f"{name} belongs to the norm, which eps=None leaves out")
        if w is key_weight and key is None:
            raise ValueError("key_weight without a key")
        if w.shape != (dim,) or w.get_device() != index or (w.dtype is not torch.float32 and w.dtype is not query.dtype):
            raise ValueError(f"{name} must have shape ({dim},) on {query.device}, in float32 or the query's dtype; got "
                             f"{tuple(w.shape)}, {w.dtype} on {w.device}")
        if kind is not None and kind is not w.dtype:
            raise ValueError("query_weight and key_weight must share one dtype")
        kind = w.dtype


def _rows(field):
    return field if field.stride(2) == 1 or field.shape[2] == 1 else field.contiguous()


def _pack(query, key, dy, out, query_weight, key_weight, positions, frequencies, eps, interleaved):
    """The argument block; every tensor named in it must outlive the launch's enqueueing."""
    tokens, heads, dim = query.shape
    token_stride, head_stride, _ = query.stride()
    key_address = key_heads = key_token_stride = key_head_stride = 0
    if key is not None:
        key_address, key_heads = key.data_ptr(), key.shape[1]
        key_token_stride, key_head_stride, _ = key.stride()
    dy_block = (0, 0, 0, 0, 0, 0)
    if dy is not None:
        first = dy[0].stride()
        second = dy[1].stride() if key is not None else (0, 0)
        dy_block = (dy[0].data_ptr(), dy[1].data_ptr() if key is not None else 0, first[0], second[0], first[1], second[1])
    weight = query_weight if query_weight is not None else key_weight
    return _native.NORM_ROTARY.pack(
        query.data_ptr(), key_address, dy_block[0], dy_block[1], out[0].data_ptr(),
        out[1].data_ptr() if key is not None else 0, query_weight.data_ptr() if query_weight is not None else 0,
        key_weight.data_ptr() if key_weight is not None else 0, positions.data_ptr(), frequencies.data_ptr(),
        token_stride, key_token_stride, head_stride, key_head_stride, *dy_block[2:], tokens,
        heads, key_heads, dim, frequencies.shape[-1], 1 if frequencies.ndim == 1 else frequencies.shape[0],
        64 if positions.dtype is torch.int64 else 32, _DTYPES[query.dtype],
        _DTYPES[query.dtype if weight is None else weight.dtype], eps is not None, interleaved,
        0.0 if eps is None else eps)


def _empty(x):
    """Uninitialised, contiguous, of the shape and dtype of x."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _forward(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved):
    index = query.get_device()
    out = (_empty(query), None if key is None else _empty(key))
    block = _pack(query, key, None, out, query_weight, key_weight, positions, frequencies, eps, interleaved)
    if current_device() == index:
        status = _native.lib().tgb_norm_rotary_fwd(block, raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = _native.lib().tgb_norm_rotary_fwd(block, raw_stream(index))
    if status:
        _native.check(status, "tgb_norm_rotary_fwd")
    return out


def _backward(ctx, *grads):
    query, key, query_weight, key_weight, positions, frequencies = ctx.saved_tensors
    index, needs = query.get_device(), ctx.needs_input_grad
    dy = [_rows(g if g.dtype is query.dtype else g.to(query.dtype)) for g in grads]
    out = (_empty(query), None if key is None else _empty(key))
    block = _pack(query, key, dy, out, query_weight, key_weight, positions, frequencies, ctx.eps, ctx.interleaved)
    lib = _native.lib()
    dwq = _empty(query_weight) if query_weight is not None and needs[2] else None
    dwk = _empty(key_weight) if key_weight is not None and needs[3] else None
    scratch, size = None, 0
    if dwq is not None or dwk is not None:
        size = lib.tgb_norm_rotary_scratch_bytes(query.shape[2])
        scratch = torch.empty(size, dtype=torch.uint8, device=query.device)
    arguments = (block, None if dwq is None else dwq.data_ptr(), None if dwk is None else dwk.data_ptr(),
                 None if scratch is None else scratch.data_ptr(), size, raw_stream(index))
    if current_device() == index:
        status = lib.tgb_norm_rotary_bwd(*arguments)
    else:
        with torch.cuda.device(index):
            status = lib.tgb_norm_rotary_bwd(*arguments)
    if status:
        _native.check(status, "tgb_norm_rotary_bwd")
    return out[0] if needs[0] else None, out[1] if needs[1] else None, dwq, dwk, None, None, None, None


_backward_once = once_differentiable(_backward)


class NormRotaryFunction(torch.autograd.Function):
    """Saves the inputs alone; the backward recomputes each head's norm."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, frequencies, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        out = _forward(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved)
        return out[0] if key is None else out

    @staticmethod
    def backward(ctx, *grads):
        # with create_graph the gradients are marked as not differentiable again
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def norm_rotary(query, key, positions, frequencies, *, query_weight=None, key_weight=None, eps: float | None = 1e-6,
                interleaved: bool = False):
    """Query and key heads, each normalised by its root mean square and turned by its token's position.

    ``query`` [tokens, H, D] and ``key`` [tokens, H_kv, D] (or None) may be views into a packed projection.
    ``frequencies`` (float32) is ``[pairs]`` with ``positions`` [tokens], or ``[axes, pairs]`` with
    ``positions`` [tokens, axes]: pair j of a token turns by ``sum_a positions[a] * frequencies[a, j]``,
    formed in 64 bits.  Pair j is ``(j, j + pairs)``, or ``(2j, 2j + 1)`` with ``interleaved``; values from
    ``2 * pairs`` on are not turned.  ``eps=None`` leaves the norm out.  Returns contiguous
    ``(query, key)``, or the query alone when ``key`` is None; differentiable in fields and
    weights, in reverse mode once: inputs that carry a forward-mode tangent are refused."""
    _check(query, key, positions, frequencies, query_weight, key_weight, eps)
    query, key = _rows(query), None if key is None else _rows(key)
    if not (positions.is_contiguous() and frequencies.is_contiguous()):
        positions, frequencies = positions.contiguous(), frequencies.contiguous()
    if query_weight is not None:
        query_weight = query_weight.contiguous()
    if key_weight is not None:
        key_weight = key_weight.contiguous()
    interleaved = bool(interleaved)
    if torch.is_grad_enabled() and (
            query.requires_grad or (key is not None and key.requires_grad)
            or (query_weight is not None and query_weight.requires_grad)
            or (key_weight is not None and key_weight.requires_grad)):
        return NormRotaryFunction.apply(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved)
    query, key = _forward(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved)
    return query if key is None else (query, key)


__all__ = ["norm_rotary", "rotary_frequencies"]
