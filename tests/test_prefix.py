"""Finding shared prefixes, and what calls with sinks or shared prefixes refuse, on the
CPU (nothing is launched)."""
import ctypes
import itertools

import numpy as np
import pytest

from test_abi import pool
from vapi_amd import _lib
from vapi_amd.attention import ForwardBatch, PreparedAttention, sinks_arg
from vapi_amd.cache import PagedKvCache
from vapi_amd.prefix import PrefixPlan, find_shared_prefixes


def saved(groups):
    return sum((len(m) - 1) * n for m, n in groups)


def test_groups_follow_the_tree_of_prefixes():
    find = find_shared_prefixes
    tables = [[1, 2, 3, 9], [1, 2, 3, 8], [1, 2, 7, 6], [5, 5], []]
    assert find(tables, [1] * 5, [64, 64, 60, 32, 0], 16, 8) == [([0, 1, 2], 32)]
    # A deep pair saves more than a shallow three.
    tables = [[1] + list(range(10, 20)), [1] + list(range(10, 20)), [1, 5]]
    assert find(tables, [1] * 3, [176, 176, 32], 16, 8) == [([0, 1], 176)]
    # Whole blocks of every member's context, few queries.
    assert find([[1, 2], [1, 2]], [1, 1], [31, 32], 16, 8) == [([0, 1], 16)]
    assert find([[1, 2], [1, 2]], [1, 9], [32, 32], 16, 8) == []
    assert find([[1, 2], [1, 2]], [1, 0], [32, 32], 16, 8) == []
    assert find([], [], [], 16, 8) == []


@pytest.mark.parametrize("seed", range(30))
def test_no_other_grouping_saves_more(seed):
    r = np.random.default_rng(seed)
    tables = [r.integers(0, 2, r.integers(0, 6)).tolist() for _ in range(6)]
    lens = [16 * len(t) for t in tables]
    got = find_shared_prefixes(tables, [1] * 6, lens, 16, 8)
    for members, keys in got:
        assert len({tuple(tables[i][:keys // 16]) for i in members}) == 1
    taken = [i for m, _ in got for i in m]
    assert len(taken) == len(set(taken))

    def most(left):
        """The most that groups among the sequences `left` save."""
        if not left:
            return 0
        best = most(left[1:])
        for n in range(1, len(left)):
            for others in itertools.combinations(left[1:], n):
                members = (left[0],) + others
                depth = 0
                while all(len(tables[i]) > depth and tables[i][depth] == tables[left[0]][depth]
                          for i in members):
                    depth += 1
                rest = [i for i in left if i not in members]
                best = max(best, n * depth * 16 + most(rest))
        return best

    assert saved(got) == most(list(range(6)))


def test_prefixes_as_deep_as_the_batch_is_wide():
    n = 3000
    tables = [list(range(i + 1)) for i in range(n)]
    groups = find_shared_prefixes(tables, [1] * n, [16 * (i + 1) for i in range(n)], 16, 8)
    assert saved(groups) >= max((n - i) * i for i in range(n)) * 16 - 16 * n


def batch_of(tables, lens_q, lens_k):
    return ForwardBatch(cu_seqlens_q=[0] + np.cumsum(lens_q).tolist(),
                        cu_seqlens_k=[0] + np.cumsum(lens_k).tolist(), block_tables=tables,
                        max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))


def test_a_plan_lists_every_query_of_its_members():
    batch = batch_of([[7, 1], [3], [7, 2]], [2, 1, 3], [20, 5, 30])
    plan = PrefixPlan([([0, 2], 16)], batch.cu_seqlens_q, batch.cu_seqlens_k, "cpu")
    words = plan.lists.numpy().view(np.uint32)
    a = plan.arg
    assert (a.n_groups, a.n_rows, a.max_keys) == (1, 5, 16)

    def at(p, n):
        i = (p - plan.lists.data_ptr()) // 4
        return words[i:i + n].tolist()

    assert at(a.offsets, 2) == [0, 5] and at(a.rows, 5) == [0, 1, 3, 4, 5]
    assert at(a.seqs, 5) == [0, 0, 2, 2, 2] and at(a.keys, 1) == [16]
    assert at(a.start, 3) == [16, 0, 16]
    assert plan.saved_keys() == 16 and plan.saved_keys(3) == 0 and plan.saved_keys(12) == 4
    for bad in ([([0, 0], 16)], [([0, 3], 16)], [([0], 16), ([0, 2], 16)], [([0, 2], 0)]):
        with pytest.raises(ValueError):
            PrefixPlan(bad, batch.cu_seqlens_q, batch.cu_seqlens_k, "cpu")


def test_sharing_is_for_layers_that_it_pays_for():
    cache = PagedKvCache(1, 8, 16, 8, 128, layout="HND", device="cpu")
    tables = [list(range(300)) + [400 + i] for i in range(40)]
    batch = batch_of(tables, [1] * 40, [4810] * 40)
    plan = PrefixPlan.from_batch(batch, cache, 32, "cpu")
    assert plan.groups == [(list(range(40)), 4800)]
    assert plan.worth_it(cache) and not plan.worth_it(cache, 100)
    narrow = PagedKvCache(1, 8, 16, 1, 64, layout="HND", device="cpu")
    assert not plan.worth_it(narrow)
    # Sequences of many queries are left out, and a step without shared blocks has none.
    assert PrefixPlan.from_batch(batch_of(tables, [17] * 40, [4810] * 40), cache, 32, "cpu") is None
    assert PrefixPlan.from_batch(batch_of(tables, [16] * 40, [4810] * 40), cache, 32, "cpu")
    alone = batch_of([[i] for i in range(4)], [1] * 4, [9] * 4)
    assert PrefixPlan.from_batch(alone, cache, 32, "cpu") is None
    with pytest.raises(ValueError):
        PreparedAttention.from_batch(alone, "cpu", share_prefixes=True)


def prefixes(**kw):
    p = dict(offsets=16, rows=16, seqs=16, keys=16, start=16, n_groups=2, n_rows=8, max_keys=64)
    p.update(kw)
    return ctypes.pointer(_lib.Prefixes(**p))


HEAD = [16, 16, 16, 16, 16, 4, 8]  # q, out, cu_q, cu_k, table, batch, max_blocks


def call(fn, p, prefix=None, head=HEAD, max_q=1, max_k=100, heads=8, sinks=3, flags=0, seqs=None,
         n_prefill=0, ws=(None, 0)):
    args = [*head, max_q, max_k, heads, 0.1, 9, 0, sinks, flags, seqs, n_prefill]
    return fn(p, 0, *args, *([] if prefix is None else [prefix]), *ws, None)


def q8_pool(**kw):
    p = dict(k=1 << 12, v=1 << 13, k_scale=1 << 14, v_scale=1 << 15, layer_stride_bytes=1 << 20,
             scale_layer_stride_bytes=1 << 16, scale_block_stride=2, num_layers=1, num_blocks=8,
             block_size=16, num_kv_heads=2, head_dim=64, dtype=_lib.BF16, format=_lib.Q8_E4M3,
             layout=_lib.LAYOUT_HND)
    p.update(kw)
    return _lib.Q8Pool(**p)


@pytest.mark.parametrize("q8", [False, True])
def test_calls_with_sinks_refuse_what_the_others_refuse(q8):
    L = _lib.lib()
    fn = L.vapi_kv_q8_attention_sinks if q8 else L.vapi_paged_attention_sinks
    make = q8_pool if q8 else pool
    assert call(fn, make(), heads=5) == _lib.EINVAL and b"multiple" in L.vapi_kv_last_error()
    assert call(fn, make(), flags=0x80) == _lib.EINVAL and b"flags" in L.vapi_kv_last_error()
    assert call(fn, make(), seqs=None, n_prefill=2) == _lib.EINVAL
    assert call(fn, make(), seqs=16, n_prefill=5) == _lib.EINVAL
    assert call(fn, make(), head=[24] + HEAD[1:]) == _lib.EINVAL
    assert call(fn, make(), head=HEAD[:6] + [0]) == _lib.EINVAL
    assert call(fn, make(num_blocks=0)) == _lib.EINVAL
    assert call(fn, make()) == _lib.ESPACE
    assert call(fn, make(), head=HEAD[:5] + [0, 8]) == _lib.OK  # nothing to do
    with pytest.raises(ValueError):
        sinks_arg(-1)
    assert sinks_arg(1 << 40) == 1 << 30


def test_a_write_with_sinks_is_refused_as_a_whole():
    L = _lib.lib()
    f = L.vapi_paged_attention_append_sinks

    def write(p, **kw):
        return call(lambda p_, layer, *a: f(p_, layer, 16, 16, 16, 4, *a), p, **kw)

    assert write(pool()) == _lib.ESPACE
    assert write(pool(), flags=0x10) == _lib.EINVAL
    assert write(pool(v=None)) == _lib.EINVAL
    assert write(pool(head_dim=512), ws=(16, 1 << 30)) == _lib.EUNSUP


@pytest.mark.parametrize("q8", [False, True])
def test_shared_prefixes_refuse(q8):
    L = _lib.lib()
    fn = L.vapi_kv_q8_attention_shared if q8 else L.vapi_paged_attention_shared
    size = (L.vapi_kv_q8_attention_shared_workspace_size if q8
            else L.vapi_paged_attention_shared_workspace_size)
    make = q8_pool if q8 else pool
    ok = prefixes()
    need = size(make(), 4, 0, 8, 1, 100, ok)
    assert need > 0
    assert call(fn, make(), ok) == _lib.ESPACE
    assert call(fn, make(), ok, ws=(16, need - 1)) == _lib.ESPACE
    for bad in (prefixes(start=None), prefixes(offsets=None), prefixes(rows=None),
                prefixes(max_keys=101)):
        assert call(fn, make(), bad) == _lib.EINVAL
        assert size(make(), 4, 0, 8, 1, 100, bad) == 0
    none = ctypes.POINTER(_lib.Prefixes)()
    assert call(fn, make(), none) == _lib.EINVAL and b"null prefixes" in L.vapi_kv_last_error()
    assert call(fn, make(), prefixes(n_groups=1001)) == _lib.EUNSUP
    assert call(fn, make(), prefixes(n_groups=1000)) == _lib.ESPACE
    big = HEAD[:5] + [5000, 8]
    assert call(fn, make(), ok, head=big) == _lib.EUNSUP
    assert call(fn, make(), prefixes(n_rows=1 << 31)) == _lib.EUNSUP
    if not q8:
        for p in (pool(dtype=_lib.F32), pool(head_dim=20), pool(block_size=8)):
            assert call(fn, p, ok) == _lib.EUNSUP
            assert size(p, 4, 0, 8, 1, 100, ok) == 0
    # A step that shares nothing, or has no groups, is an ordinary one.
    assert size(make(), 4, 0, 8, 1, 100, prefixes(n_groups=0, n_rows=0)) > 0


def test_a_plan_of_another_batch_is_refused():
    cache = PagedKvCache(1, 8, 16, 8, 128, layout="HND", device="cpu")
    batch = batch_of([[1, 2], [1, 3], [1, 4]], [1] * 3, [20] * 3)
    prep = PreparedAttention.from_batch(batch, "cpu")
    prep.prefixes = PrefixPlan([([0, 1], 16)], batch.cu_seqlens_q, batch.cu_seqlens_k, "cpu")
    assert prep.shared_bytes(cache, 32) > 0
    for n in (2, 4):
        cu = list(range(n + 1))
        prep.prefixes = PrefixPlan([([0, 1], 16)], cu, [20 * x for x in cu], "cpu")
        with pytest.raises(ValueError, match="sequences in a step of 3"):
            prep.shared_bytes(cache, 32)


def test_a_step_whose_plan_or_lengths_change_asks_again():
    cache = PagedKvCache(1, 8, 16, 8, 128, layout="HND", device="cpu")
    batch = batch_of([[1, 2]] * 40, [4] * 40, [20] * 40)
    prep = PreparedAttention.from_batch(batch, "cpu")

    def plan(n):
        return PrefixPlan([(list(range(n)), 16)], batch.cu_seqlens_q, batch.cu_seqlens_k, "cpu")

    prep.prefixes = plan(2)
    few = prep.shared_bytes(cache, 32)
    prep.prefixes = plan(40)
    many = prep.shared_bytes(cache, 32)
    assert 0 < few < many
    # (Without a decode row the call covers every sequence, whatever the list.)
    prep.flags, prep.n_prefill = 0, 1  # the others' queries have no tiles of their own
    assert 0 < prep.shared_bytes(cache, 32) < many
    prep.max_seqlen_k = 15  # fewer keys than the prefix: refused
    assert prep.shared_bytes(cache, 32) == 0
