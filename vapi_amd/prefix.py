"""Which sequences of a step share a prefix, host side.

The pool is content-addressed and refcounted (crates/vapi-cache/src/pool.rs:80-414):
forks of a prompt and requests behind one system prompt name the same blocks at the
front of their tables. PrefixPlan finds them in a step's block tables and holds the
device lists that vapi_paged_attention_shared takes, so that attention reads those
blocks once for all of them.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import Prefixes

# Sharing costs a fixed 15 to 25 us a layer against the ordinary call (tiles, partial
# results, their merge), which this many bytes of K and V take to read: 8 sequences
# over 2,000 keys (57 MB saved, 32 q / 8 kv heads) 29 us shared, 14 not; 32 over 1,000
# (126 MB) 33 and 34; 64 over 1,000 (256 MB) 41 and 55. In e4m3: 16 over 4,000 (123 MB)
# 33 and 34; 64 over 1,000 (128 MB) 38 and 36; 16 over 2,000 (32 kv heads, 246 MB) 30 and 56.
MIN_SAVED_BYTES = 128 << 20
# Rows (queries times query heads of a kv head) that a sequence brings to a group at
# most. More fill tiles by themselves, and read the prefix for many rows at once anyway:
# 16 sequences over 2,000 keys (32 kv heads), 64 queries each: 109 us shared, 147 not;
# 128 each: 182 and 151; 8 sequences (8 kv heads, 4 query heads each), 64: 72 and 40.
MAX_ROWS = 64


def find_shared_prefixes(block_tables, lens_q, lens_k, block_size: int,
                         max_queries: int) -> list[tuple[list[int], int]]:
    """Groups (members, shared keys) of sequences whose tables begin with the same
    blocks, each sequence in at most one: of all ways to group along the tree of
    common prefixes the one that saves the most key reads, (members - 1) * keys a
    group. Whole blocks within every member's context are shared. Sequences of more
    than `max_queries` queries are left out."""
    tables = [np.asarray(t)[:max(int(lk), 0) // block_size]
              for t, lk in zip(block_tables, lens_k)]
    live = [i for i, t in enumerate(tables) if len(t) and 1 <= lens_q[i] <= max_queries]

    def by_block(members, depth):
        """`members` by their table's entry `depth`; those whose table ends there in none."""
        out: dict[int, list[int]] = {}
        for i in members:
            if len(tables[i]) > depth:
                out.setdefault(int(tables[i][depth]), []).append(i)
        return list(out.values())

    def common(members, depth):
        """How many blocks the members, alike in the first `depth`, have in common."""
        first = tables[members[0]]
        same = min(len(tables[i]) for i in members)
        for i in members[1:]:
            differ = np.nonzero(tables[i][depth:same] != first[depth:same])[0]
            if differ.size:
                same = depth + int(differ[0])
        return same

    # Depth first, parents before children (without recursion: prefixes nest as deep as
    # there are sequences); then the better of each node and what its children found.
    nodes, todo = [], [(part, 0, -1) for part in by_block(live, 0) if len(part) > 1]
    while todo:
        members, depth, parent = todo.pop()
        same = common(members, depth)
        nodes.append([members, same, parent, 0, []])
        todo += [(part, same, len(nodes) - 1) for part in by_block(members, same) if len(part) > 1]
    groups = []
    for members, same, parent, saved, found in reversed(nodes):
        whole = (len(members) - 1) * same * block_size
        if whole >= saved:
            saved, found = whole, [(members, same * block_size)]
        if parent < 0:
            groups += found
        else:
            nodes[parent][3] += saved
            nodes[parent][4] = nodes[parent][4] + found
    return groups


class PrefixPlan:
    """The groups of a step and their device lists (vapi_kv_prefixes). `min_bytes`:
    the K and V bytes that sharing has to save in a layer."""

    def __init__(self, groups, cu_seqlens_q, cu_seqlens_k, device, min_bytes: int = 0):
        cq = np.asarray(cu_seqlens_q, dtype=np.int64)
        lens_k = np.diff(np.asarray(cu_seqlens_k, dtype=np.int64))
        batch = self.batch = len(lens_k)
        self.groups = [(list(map(int, m)), int(n)) for m, n in groups]
        self.min_bytes = min_bytes
        start = np.zeros(max(batch, 1), np.int64)
        rows, seqs, offsets = [], [], [0]
        for members, keys in self.groups:
            for s in members:
                if not 0 <= s < batch or start[s] or keys <= 0:
                    raise ValueError(f"sequence {s} of {batch} in a group of {keys} shared keys "
                                     "(each is in at most one group)")
                start[s] = keys
                rows += range(int(cq[s]), int(cq[s + 1]))
                seqs += [s] * int(cq[s + 1] - cq[s])
            offsets.append(len(rows))
        # Keys past the prefix, a member's on average: what of it a window leaves.
        self.past = [float(np.mean(lens_k[m])) - n if m else 0.0 for m, n in self.groups]
        keys = [n for _, n in self.groups]
        lists = [np.asarray(a or [0], dtype=np.int64) for a in (offsets, rows, seqs, keys)] + [start]
        sizes = np.cumsum([0] + [len(a) for a in lists])
        self.lists = torch.from_numpy(np.concatenate(lists).astype(np.uint32).view(np.int32)).to(device)
        at = [self.lists.data_ptr() + 4 * int(n) for n in sizes]
        self.arg = Prefixes(offsets=at[0], rows=at[1], seqs=at[2], keys=at[3], start=at[4],
                            n_groups=len(self.groups), n_rows=len(rows), max_keys=max(keys or [0]))
        self.ptr = ctypes.pointer(self.arg)

    def saved_keys(self, window_left: int | None = None) -> float:
        """Key reads that sharing saves a kv head, about (behind a left window only what
        it leaves of the prefix counts)."""
        total = 0.0
        for (members, keys), past in zip(self.groups, self.past):
            if window_left is not None and window_left >= 0:
                keys = min(max(window_left + 1 - past, 0.0), keys)
            total += (len(members) - 1) * keys
        return total

    def worth_it(self, cache, window_left: int | None = None) -> bool:
        size = 1 if getattr(cache, "fmt", None) else torch.empty((), dtype=cache.dtype).element_size()
        saved = self.saved_keys(window_left) * 2 * cache.num_kv_heads * cache.head_dim * size
        return saved >= self.min_bytes

    @classmethod
    def from_batch(cls, batch, cache, num_heads: int | None, device,
                   packed=None) -> "PrefixPlan | None":
        """The plan of a ForwardBatch over `cache`, for layers that it pays for; None
        where no two sequences share a block. Without `num_heads`, single queries are
        grouped only. `packed`: the batch's tables as rows of an array, if at hand (128
        tables of 2,068 entries take 15 ms as lists, 1 ms as rows)."""
        tables = batch.block_tables
        if packed is not None:
            tables = [row[:len(t)] for row, t in zip(packed, tables)]
        heads = getattr(cache, "num_kv_heads", None) or min(
            s[1] for s in cache.layouts if s[0] == "kv")
        queries = max(MAX_ROWS * heads // num_heads, 1) if num_heads else 1
        groups = find_shared_prefixes(tables, np.diff(batch.cu_seqlens_q),
                                      np.diff(batch.cu_seqlens_k), cache.block_size, queries)
        return cls(groups, batch.cu_seqlens_q, batch.cu_seqlens_k, device,
                   MIN_SAVED_BYTES) if groups else None
