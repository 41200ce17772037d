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

# Keys that need not be read again, times kv heads not counted, from which a group is
# worth its partial results; and the most queries a sequence brings to one (more fill
# tiles of their own).
MIN_SAVED_KEYS = 1024
MAX_QUERIES = 64


def find_shared_prefixes(block_tables, lens_q, lens_k, block_size: int,
                         min_saved: int = MIN_SAVED_KEYS,
                         max_queries: int = MAX_QUERIES) -> list[tuple[list[int], int]]:
    """Groups (members, shared keys) of sequences whose tables begin with the same
    blocks, each sequence in at most one: of all ways to group along the tree of
    common prefixes the one that saves the most key reads, (members - 1) * keys a
    group, counting groups of at least `min_saved`. Whole blocks within every
    member's context are shared. Sequences of more than `max_queries` queries are
    left out."""
    tables = [np.asarray(t, dtype=np.int64)[:max(int(lk), 0) // block_size]
              for t, lk in zip(block_tables, lens_k)]
    live = [i for i, t in enumerate(tables) if len(t) and 1 <= lens_q[i] <= max_queries]

    def by_block(members, depth):
        """`members` by their table's entry `depth`; those whose table ends there in none."""
        out: dict[int, list[int]] = {}
        for i in members:
            if len(tables[i]) > depth:
                out.setdefault(int(tables[i][depth]), []).append(i)
        return out

    def best(members, depth):
        """The saved keys and the groups of sequences that agree up to `depth` blocks."""
        if len(members) < 2:
            return 0, []
        first = tables[members[0]]
        same = min(len(tables[i]) for i in members)
        for i in members[1:]:
            differ = np.nonzero(tables[i][depth:same] != first[depth:same])[0]
            same = min(same, depth + int(differ[0]) if differ.size else same)
        saved, groups = 0, []
        for part in by_block(members, same).values():
            s, g = best(part, same)
            saved, groups = saved + s, groups + g
        whole = (len(members) - 1) * same * block_size
        if whole >= max(saved, min_saved, 1):
            return whole, [(members, same * block_size)]
        return saved, groups

    groups = []
    for part in by_block(live, 0).values():
        groups += best(part, 0)[1]
    return groups


class PrefixPlan:
    """The groups of a step and their device lists (vapi_kv_prefixes)."""

    def __init__(self, groups, cu_seqlens_q, batch: int, device):
        cq = np.asarray(cu_seqlens_q, dtype=np.int64)
        self.groups = [(list(map(int, m)), int(n)) for m, n in groups]
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
        keys = [n for _, n in self.groups]
        lists = [np.asarray(a or [0], dtype=np.int64) for a in (offsets, rows, seqs, keys)] + [start]
        sizes = np.cumsum([0] + [len(a) for a in lists])
        self.lists = torch.from_numpy(np.concatenate(lists).astype(np.uint32).view(np.int32)).to(device)
        at = [self.lists.data_ptr() + 4 * int(n) for n in sizes]
        self.arg = Prefixes(offsets=at[0], rows=at[1], seqs=at[2], keys=at[3], start=at[4],
                            n_groups=len(self.groups), n_rows=len(rows), max_keys=max(keys or [0]))
        self.ptr = ctypes.pointer(self.arg)

    @classmethod
    def from_batch(cls, batch, block_size: int, device, **limits) -> "PrefixPlan | None":
        """The plan of a ForwardBatch; None where sharing saves nothing. `limits`:
        find_shared_prefixes' min_saved and max_queries."""
        groups = find_shared_prefixes(batch.block_tables, np.diff(batch.cu_seqlens_q),
                                      np.diff(batch.cu_seqlens_k), block_size, **limits)
        return cls(groups, batch.cu_seqlens_q, batch.batch_size(), device) if groups else None
