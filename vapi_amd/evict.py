"""Eviction from the KV cache by running attention weight, host side.

accumulate_attention_weights adds what a step's queries attend to into a state
of one f32 per sequence, kv head and key; evict_kv moves the keys with the
largest sums (and the first and latest ones) of each sequence and kv head into
fewer blocks, whose attention then runs like any other's. Both work on 16-bit
PagedKvCaches and on 8-bit QuantKvCaches. The reference evicts whole cached
blocks only (crates/vapi-cache/src/pool.rs); this is the per-key counterpart.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch

from ._lib import Weights, check, lib
from .attention import PreparedAttention
from .cache import (HybridKvCache, _is_quantised, _per_layer, check_on_device, contiguous_on,
                    empty_on, keep_for, stream_handle)


def new_weights(rows: int, num_kv_heads: int, width: int, device="cuda") -> torch.Tensor:
    """A zeroed state for one layer: f32 [rows, num_kv_heads, width], a row per
    sequence (zero it before another sequence takes it) and a column per key."""
    return torch.zeros((rows, num_kv_heads, width), dtype=torch.float32, device=device)


def _state(weights: torch.Tensor, cache, index: torch.Tensor | None, batch: int, name: str):
    """vapi_kv_weights over a [rows, num_kv_heads, width] f32 tensor."""
    shape = weights.shape
    if len(shape) != 3 or shape[1] != cache.num_kv_heads:
        raise ValueError(f"{name} must be (rows, {cache.num_kv_heads}, width), "
                         f"got {tuple(shape)}")
    if weights.dtype != torch.float32:
        raise ValueError(f"{name} must be float32, not {weights.dtype}")
    rows, _, width = shape
    if rows == 0 or width == 0:
        raise ValueError(f"{name} is empty: {tuple(shape)}")
    row_stride, head_stride, last = weights.stride()
    if width > 1 and last != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if index is not None:
        if (index.dtype is not torch.int32 and index.dtype is not torch.uint32) or \
                index.dim() != 1 or index.shape[0] != batch or not index.is_contiguous():
            raise ValueError(f"rows must be {batch} contiguous 32-bit indices")
    elif batch > rows:
        raise ValueError(f"{batch} sequences but {rows} rows of {name}")
    return Weights(weights.data_ptr(), None if index is None else index.data_ptr(), row_stride,
                   head_stride, rows, width)


def _rows(rows, count: int, device) -> torch.Tensor | None:
    """Rows as a device index: a tensor as it is, host numbers checked first."""
    if rows is None or isinstance(rows, torch.Tensor):
        return rows
    rows = [int(r) for r in rows]
    if len(rows) != count:
        raise ValueError(f"{len(rows)} rows for {count} sequences")
    if len(set(rows)) != len(rows) or any(r < 0 for r in rows):
        raise ValueError("rows must be distinct and not negative")
    return torch.tensor(rows, dtype=torch.int32).to(device)


def accumulate_attention_weights(q: torch.Tensor, cache, layer: int, prepared: PreparedAttention,
                                 softmax_scale: float, weights: torch.Tensor, rows=None,
                                 last_queries: int = 0, decay: float = 1.0,
                                 window_size_left: int | None = None,
                                 window_size_right: int | None = 0, stream=None) -> torch.Tensor:
    """Adds the attention weights of a step's queries to a layer's state, in
    place (vapi_kv_attention_weights): per sequence, kv head and cached key

        weights = decay * weights + sum over the queries and the head's query
                  heads of softmax(scale q.k)

    q, prepared, softmax_scale and the windows as paged_attention_prepared,
    after whose cache write it runs. weights: f32 [rows, num_kv_heads, width]
    (new_weights), width at least prepared.max_seqlen_k. rows: the row of each
    sequence, as a device int32 tensor or host numbers, distinct (None:
    sequence i has row i). last_queries: only the last so many queries of a
    sequence count (0: all); with decay 0 that is the observation window at the
    end of a prompt, with decay 1 and single tokens the running sum of a
    generation. Returns weights."""
    held = cache.k[0]
    cache, layer = _per_layer(cache, layer)
    if getattr(cache, "has_v", True) is False:
        raise ValueError("a rows layer has no attention")
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        raise ValueError(f"q must be (tokens, heads, {cache.head_dim}), got {tuple(q.shape)}")
    if q.dtype != cache.dtype:
        raise ValueError(f"q is {q.dtype} but the cache is {cache.dtype}")
    if last_queries < 0:
        raise ValueError(f"last_queries must not be negative: {last_queries}")
    b = prepared.seqlens_q.shape[0] - 1
    index = _rows(rows, b, cache.device)
    state = _state(weights, cache, index, b, "weights")
    on = (weights, held, q, prepared.block_table, prepared.seqlens_q)
    check_on_device(*(on if index is None else on + (index,)))
    q = contiguous_on(stream, q)
    heads, max_q, max_k = q.shape[1], max(prepared.max_seqlen_q, 1), max(prepared.max_seqlen_k, 1)
    need = lib().vapi_kv_attention_weights_workspace_size(
        b, cache.num_kv_heads, heads, cache.head_dim, max_q, max_k, last_queries)
    ws = prepared.weights_workspace
    if need and (ws is None or ws.numel() < need):
        # Kept for the step's other layers, as the attention's; a smaller one stays
        # too (a captured graph may hold it).
        if ws is not None:
            prepared.weights_workspaces.append(ws)
        ws = empty_on(stream, q, need, torch.uint8)
        prepared.weights_workspace = ws
    quantised = _is_quantised(cache)
    fn = lib().vapi_kv_q8_attention_weights if quantised else lib().vapi_kv_attention_weights
    check(fn(cache.q8 if quantised else cache.pool, layer, q.data_ptr(),
             prepared.seqlens_q.data_ptr(), prepared.seqlens_k.data_ptr(),
             prepared.block_table.data_ptr(), b, prepared.block_table.shape[1], max_q, max_k,
             heads, float(softmax_scale), -1 if window_size_left is None else int(window_size_left),
             -1 if window_size_right is None else int(window_size_right), int(last_queries),
             float(decay), state, ws.data_ptr() if need else None, need, stream_handle(stream)))
    if stream is not None:
        prepared.keep_for(stream)
        keep_for(stream, q, weights, *([] if index is None else [index]), *([ws] if need else []))
    return weights


@dataclass
class EvictionPlan:
    """What one eviction of a batch needs on the device, built and checked once
    and used for every layer. lens[i]: keys of sequence i before, new_lens[i]
    after; its block table becomes the dst table."""
    lens: torch.Tensor
    src_table: torch.Tensor
    dst_table: torch.Tensor
    rows: torch.Tensor | None
    new_lens: list
    max_len: int
    max_keep: int
    budget: int
    sinks: int
    recent: int
    block_size: int
    top_block: int

    @classmethod
    def from_tables(cls, lens: Sequence[int], src_tables, dst_tables, budget: int, sinks: int,
                    recent: int, block_size: int, device, rows=None) -> "EvictionPlan":
        """lens: each sequence's keys; src_tables: the blocks that hold them;
        dst_tables: distinct blocks for the min(len, budget) kept ones, none of
        them a source (the sources may be shared with other sequences and stay
        as they are). Raises ValueError where a table is too short, a block is
        named twice, or the budget is below sinks + recent."""
        lens = [int(n) for n in lens]
        src = [[int(b) for b in t] for t in src_tables]
        dst = [[int(b) for b in t] for t in dst_tables]
        if not len(lens) == len(src) == len(dst):
            raise ValueError(f"{len(lens)} lengths, {len(src)} source and {len(dst)} new tables")
        if sinks < 0 or recent < 0 or budget < max(sinks + recent, 1):
            raise ValueError(f"a budget of {budget} keys for {sinks} first and {recent} last ones")
        new_lens = [min(n, budget) for n in lens]
        for n, new, s, d in zip(lens, new_lens, src, dst):
            if n < 0 or -(-n // block_size) > len(s) or -(-new // block_size) > len(d):
                raise ValueError(f"{n} keys (kept: {new}) need more blocks of {block_size} than "
                                 f"the {len(s)} given and {len(d)} new ones")
        flat = [b for t in dst for b in t]
        if len(set(flat)) != len(flat):
            raise ValueError("a new block is named twice")
        if not set(flat).isdisjoint(b for t in src for b in t):
            raise ValueError("a new block must not be a source")
        every = flat + [b for t in src for b in t]
        if any(b < 0 for b in every):
            raise ValueError("a block id is negative")
        if isinstance(rows, torch.Tensor):
            rows = rows.tolist()

        def table(tables):
            width = max([len(t) for t in tables] + [1])
            out = np.zeros((max(len(tables), 1), width), dtype=np.int32)
            for i, t in enumerate(tables):
                out[i, :len(t)] = t
            return torch.from_numpy(out).to(device)

        return cls(lens=torch.tensor(lens or [0], dtype=torch.int32).to(device),
                   src_table=table(src), dst_table=table(dst),
                   rows=_rows(rows, len(lens), device), new_lens=new_lens,
                   max_len=max(lens + [0]), max_keep=max(new_lens + [0]), budget=int(budget),
                   sinks=int(sinks), recent=int(recent), block_size=int(block_size),
                   top_block=max(every + [0]))


def _extent(t: torch.Tensor) -> tuple[int, int]:
    (r, h, w), (sr, sh, sw) = t.shape, t.stride()
    first = t.data_ptr()
    return first, first + 4 * ((r - 1) * sr + (h - 1) * sh + (w - 1) * sw + 1)


def evict_kv(cache, layer: int, weights: torch.Tensor, plan: EvictionPlan,
             weights_out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Moves one layer's kept keys into the plan's new blocks (vapi_kv_evict):
    of each sequence and kv head the first `sinks`, the last `recent` and of the
    others those with the largest weights, ties to the earlier key, in order of
    position. Returns their positions before, int32 [batch, num_kv_heads,
    max(plan.new_lens)], -1 past a sequence's new length.

    weights_out: a state whose rows plan.rows become the kept keys' weights,
    zeros after them; `weights` itself updates it in place. An 8-bit cache's
    kept codes get the scales of their new blocks."""
    held = cache.k[0]
    if isinstance(cache, HybridKvCache):
        if cache.layouts[layer][0] != "kv":
            raise ValueError("a rows layer has no attention weights to evict by")
        cache, layer = _per_layer(cache, layer)
    if plan.block_size != cache.block_size:
        raise ValueError(f"a plan for blocks of {plan.block_size}, a cache of {cache.block_size}")
    if plan.top_block >= max(cache.num_blocks, 1):
        raise ValueError(f"block {plan.top_block} of {cache.num_blocks}")
    b = len(plan.new_lens)
    src = _state(weights, cache, plan.rows, b, "weights")
    on = [weights, held, plan.lens, plan.src_table]
    dst = None
    if weights_out is weights:
        dst = src
    elif weights_out is not None:
        dst = _state(weights_out, cache, plan.rows, b, "weights_out")
        on.append(weights_out)
        if dst.data != src.data or weights_out.stride() != weights.stride():
            (a0, a1), (b0, b1) = _extent(weights), _extent(weights_out)
            if a0 < b1 and b0 < a1:
                raise ValueError("weights_out overlaps weights: give the same tensor or another")
    check_on_device(*on)
    kept = empty_on(stream, weights, (b, cache.num_kv_heads, plan.max_keep), torch.int32)
    quantised = _is_quantised(cache)
    fn = lib().vapi_kv_q8_evict if quantised else lib().vapi_kv_evict
    check(fn(cache.q8 if quantised else cache.pool, layer, src,
             None if dst is None else ctypes.byref(dst), plan.lens.data_ptr(),
             plan.src_table.data_ptr(), plan.src_table.shape[1], plan.dst_table.data_ptr(),
             plan.dst_table.shape[1], b, plan.max_len, plan.budget, plan.sinks, plan.recent,
             kept.data_ptr(), stream_handle(stream)))
    if stream is not None:
        keep_for(stream, kept, weights, plan.lens, plan.src_table, plan.dst_table,
                 *([] if plan.rows is None else [plan.rows]),
                 *([] if weights_out is None else [weights_out]))
    return kept
