"""Cache eviction by accumulated attention weight (no reference counterpart).

The segmented selection and compaction that a key/value cache of bounded size
needs, beside the segmented sort.  A serving loop calls, on one launch:

    device_attention_weight_add(launch, weights, scores, lengths)   # every step
    device_cache_select(launch, scores, lengths, kept, kept_lengths,
                        sinks=4, recent=64)                         # when full
    device_cache_compact(launch, kept, kept_lengths, [k, v, scores])  # in place

scores (batch, heads, capacity) float32 totals; lengths (batch,) int32
positions in use; kept (batch, heads, budget) int32.  All memory is the
caller's, every call is asynchronous on the launch's stream and reads nothing
back, so a step can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Sequence

import torch

from . import _lib
from .cub import Launch
from .errors import BadArgument, LengthMismatch
from .experts import _on, call, real_code


def _int32(role: str, t: torch.Tensor, *shape: int) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise BadArgument(f"{role} must be contiguous int32")
    if t.shape != shape:
        raise LengthMismatch(role, _count(shape), t.numel())


def _count(shape) -> int:
    return math.prod(shape)


_ROWS = struct.Struct("9N")  # rsort_cache_rows
assert _ROWS.size == ctypes.sizeof(_lib.CacheRows)


def _rows(t: torch.Tensor):
    """Address, shape, row width, element size and strides of a cache."""
    shape, strides, width = t.shape, t.stride(), 1
    if len(shape) == 4:
        width = shape[3]
        if width > 1 and strides[3] != 1 and t.numel():
            raise BadArgument("elements of a cache row must be neighbours")
    elif len(shape) != 3:
        raise BadArgument("caches must be (batch, heads, capacity[, width])")
    return t.data_ptr(), shape, width, t.element_size(), strides


def _scores(t: torch.Tensor) -> None:
    if t.dtype != torch.float32 or t.dim() != 3 or not (
            t.is_contiguous() or t.numel() == 0 or t.shape[2] == 1 or t.stride(2) == 1):
        raise BadArgument("cache scores must be (batch, heads, capacity) float32 with "
                          "neighbouring positions")


def device_attention_weight_add(launch: Launch, weights: torch.Tensor, scores: torch.Tensor,
                                lengths: Optional[torch.Tensor] = None, decay: float = 1.0,
                                causal: bool = False) -> None:
    """scores[b, h, s] = decay * scores[b, h, s] + the attention weights that
    position s got, summed in fp32 over the queries and over the query heads of
    cache head h, for s < lengths[b] (every position without lengths).

    weights (batch, query heads, queries, capacity), or (batch, query heads,
    capacity) for a single token: float32, float16 or bfloat16; query head
    h * group + g reads cache head h.  With causal the queries are the last
    ones of each sequence.  What is not seen, or lies behind a length, adds
    nothing whatever it holds, but may be read: nothing may write it meanwhile."""
    _on(launch, weights, scores, lengths)
    if weights.dim() == 3:
        weights = weights.unsqueeze(2)
    code = real_code(weights.dtype)
    _scores(scores)
    batch, heads, capacity = scores.shape
    shape, strides = weights.shape, weights.stride()
    if len(shape) != 4 or (strides[3] != 1 and capacity != 1 and weights.numel()):
        raise BadArgument("attention weights must be (batch, query heads[, queries], capacity) "
                          "with neighbouring positions")
    if shape[0] != batch:
        raise LengthMismatch("attention weight batch", batch, shape[0])
    if shape[3] != capacity:
        raise LengthMismatch("attention weight positions", capacity, shape[3])
    group = shape[1] // heads if heads else 1
    if group * heads != shape[1] or group < 1:
        raise LengthMismatch("attention weight heads", max(group, 1) * heads, shape[1])
    if lengths is not None:
        _int32("cache lengths", lengths, batch)
    score_b, score_h, _ = scores.stride()
    call(launch, _lib.lib().rsort_attention_weight_add, code, weights.data_ptr(), *strides[:3],
         batch, heads, group, shape[2], capacity,
         None if lengths is None else lengths.data_ptr(), decay, int(causal), scores.data_ptr(),
         score_b, score_h)


def device_cache_select(launch: Launch, scores: torch.Tensor, lengths: Optional[torch.Tensor],
                        kept: torch.Tensor, kept_lengths: torch.Tensor, sinks: int = 0,
                        recent: int = 0) -> None:
    """The positions of every head that stay: kept (batch, heads, budget)
    ascending, then -1; kept_lengths (batch,) = min(lengths, budget).  The first
    `sinks`, the last `recent` and the heaviest between stay; equal totals keep
    the lower position, NaN counts as -inf.  kept_lengths must not be lengths."""
    _on(launch, scores, lengths, kept, kept_lengths)
    _scores(scores)
    batch, heads, capacity = scores.shape
    if kept.dim() != 3:
        raise BadArgument("kept positions must be (batch, heads, budget)")
    budget = kept.shape[2]
    _int32("kept positions", kept, batch, heads, budget)
    _int32("kept lengths", kept_lengths, batch)
    if lengths is not None:
        _int32("cache lengths", lengths, batch)
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise BadArgument(f"{sinks} sinks, {recent} recent positions, budget {budget}")
    score_b, score_h, _ = scores.stride()
    call(launch, _lib.lib().rsort_cache_select, scores.data_ptr(), score_b, score_h,
         None if lengths is None else lengths.data_ptr(), batch, heads, capacity, budget, sinks,
         recent, kept.data_ptr(), kept_lengths.data_ptr())


def device_cache_compact(launch: Launch, kept: torch.Tensor, kept_lengths: torch.Tensor,
                         sources: Sequence[torch.Tensor],
                         destinations: Optional[Sequence[torch.Tensor]] = None) -> None:
    """destinations[i][b, h, j] = sources[i][b, h, kept[b, h, j]] for
    j < kept_lengths[b], all arrays in one launch; later rows are left as they
    are.  Arrays are (batch, heads, capacity) or (batch, heads, capacity, width)
    of any element type and any strides but neighbouring elements in a row
    (pass a transposed view of a (batch, capacity, heads, width) cache).
    Without destinations, or with the sources themselves, the cache is
    compacted in place by strictly ascending kept positions (as selected);
    otherwise they may be in any order and repeat."""
    if destinations is None:
        destinations = sources
    if len(sources) != len(destinations):
        raise LengthMismatch("compacted caches", len(sources), len(destinations))
    if len(sources) > _lib.MAX_CACHES:
        raise BadArgument(f"{len(sources)} caches (at most {_lib.MAX_CACHES})")
    in_place = destinations is sources
    _on(launch, kept, kept_lengths, *sources, *(() if in_place else destinations))
    if kept.dim() != 3:
        raise BadArgument("kept positions must be (batch, heads, budget)")
    batch, heads, budget = kept.shape
    _int32("kept positions", kept, batch, heads, budget)
    _int32("kept lengths", kept_lengths, batch)
    capacity = sources[0].shape[2] if sources and sources[0].dim() >= 3 else 0
    fewest = min(budget, capacity)  # no more rows than the capacity can be kept
    rows = (_lib.CacheRows * max(len(sources), 1))()
    for i, src in enumerate(sources):
        pointer, shape, width, size, strides = _rows(src)
        if shape[0] != batch or shape[1] != heads or shape[2] != capacity:
            raise LengthMismatch("cache", batch * heads * capacity, _count(shape[:3]))
        dst_pointer, dst_strides = pointer, strides
        dst = destinations[i]
        if dst is not src:
            if dst.dtype != src.dtype:
                raise BadArgument(f"cache of {src.dtype} into {dst.dtype}")
            dst_pointer, dst_shape, _, _, dst_strides = _rows(dst)
            if dst_shape[:2] != shape[:2] or dst_shape[3:] != shape[3:]:
                raise LengthMismatch("compacted cache", _count(shape[:2] + shape[3:]),
                                     _count(dst_shape[:2] + dst_shape[3:]))
            if dst_shape[2] < fewest:
                raise LengthMismatch("compacted cache positions", fewest, dst_shape[2])
        _ROWS.pack_into(rows, i * _ROWS.size, pointer, dst_pointer, width * size,
                        strides[0] * size, strides[1] * size, strides[2] * size,
                        dst_strides[0] * size, dst_strides[1] * size, dst_strides[2] * size)
    call(launch, _lib.lib().rsort_cache_compact, rows, len(sources), kept.data_ptr(),
         kept_lengths.data_ptr(), batch, heads, budget, capacity)
