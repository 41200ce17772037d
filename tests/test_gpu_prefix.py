"""Attention over shared prefixes on the GPU, against the definition in 64 bits.

Tolerances are those of test_gpu_sinks.py: probabilities and outputs rounded to the
pool's type (2 u max|v|), scores' f32 sums (2^-13 of it); joining partials adds f32
roundings only.
"""
import numpy as np
import pytest
import torch

from test_gpu_sinks import BF16, DEV, F16, F32, assert_close, reference
from vapi_amd._lib import VapiKvError, lib
from vapi_amd.attention import (ATTN_NO_DECODE_ROWS, ForwardBatch, PreparedAttention,
                                paged_attention_append_prepared, paged_attention_prepared)
from vapi_amd.cache import HybridKvCache, PagedKvCache, scatter_index
from vapi_amd.prefix import PrefixPlan
from vapi_amd.quant import QuantKvCache

pytestmark = pytest.mark.gpu


def make(groups, alone, heads, kvh, d, dtype, bs=16, layout="HND", fmt="none", seed=0,
         shuffle=True):
    """groups: (shared blocks, [(queries, keys past the prefix), ..]) each; alone:
    [(queries, keys), ..]. A cache of random rows, the step, its queries and the
    groups as (members, shared keys)."""
    gen = torch.Generator().manual_seed(seed + heads * d + len(groups))
    r = np.random.default_rng(seed + d)
    seqs = [(g, n, own, lq) for g, (n, members) in enumerate(groups) for lq, own in members]
    seqs += [(-1, 0, lk, lq) for lq, lk in alone]
    if shuffle:
        seqs = [seqs[i] for i in r.permutation(len(seqs))]
    need = [-(-own // bs) for _, _, own, _ in seqs]
    nb = sum(need) + sum(n for n, _ in groups) + 2
    args = (1, nb, bs, kvh, d, dtype)
    shape = (nb, kvh, bs, d) if layout == "HND" else (nb, bs, kvh, d)
    if fmt == "none":
        cache = PagedKvCache(*args, layout, DEV)
        cache.k[0].copy_(torch.randn(shape, generator=gen))
        cache.v[0].copy_(torch.randn(shape, generator=gen))
    else:
        cache = QuantKvCache(*args, fmt, layout, DEV)
        for c, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
            x = torch.randn(shape, generator=gen)
            c.copy_((x * 100).clamp(-127, 127).to(c.dtype))
            s.copy_(torch.exp2(torch.randint(-8, -5, s.shape, generator=gen).float()))
    perm, at, heads_of = r.permutation(nb).tolist(), 0, []
    for n, _ in groups:
        heads_of.append(perm[at:at + n])
        at += n
    tables = []
    for (g, _, _, _), n in zip(seqs, need):
        tables.append((heads_of[g] if g >= 0 else []) + perm[at:at + n])
        at += n
    lens_q = [lq for _, _, _, lq in seqs]
    lens_k = [n * bs + own for _, n, own, _ in seqs]
    batch = ForwardBatch(cu_seqlens_q=np.concatenate([[0], np.cumsum(lens_q)]).tolist(),
                         cu_seqlens_k=np.concatenate([[0], np.cumsum(lens_k)]).tolist(),
                         block_tables=tables, max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))
    q = torch.randn(sum(lens_q), heads, d, generator=gen).to(dtype).to(DEV)
    plan = [([i for i, s in enumerate(seqs) if s[0] == g], n * bs)
            for g, (n, members) in enumerate(groups) if n]
    return cache, q, batch, plan


def prepare(batch, cache, heads, plan, deterministic=False):
    prep = PreparedAttention.from_batch(batch, DEV, deterministic=deterministic)
    prep.prefixes = PrefixPlan(plan, batch.cu_seqlens_q, batch.cu_seqlens_k, DEV)
    return prep


def check(groups, alone, heads, kvh, d, dtype, left=None, sinks=0, right=0, scale=None, **kw):
    cache, q, batch, plan = make(groups, alone, heads, kvh, d, dtype, **kw)
    prep = prepare(batch, cache, heads, plan)
    assert prep.shared_bytes(cache, heads) > 0, lib().vapi_kv_last_error()
    scale = d ** -0.5 if scale is None else scale
    out = torch.full_like(q, float("nan"))
    got = paged_attention_prepared(q, cache, 0, prep, scale, left, right, out=out, sinks=sinks)
    assert_close(got, reference(q, cache, batch, scale, left, right, sinks), dtype)


def decode(n, lo, hi, seed):
    return [(1, int(x)) for x in np.random.default_rng(seed).integers(lo, hi + 1, n)]


GEOMETRIES = [(8, 2, 128, BF16, "none"), (4, 4, 64, F16, "none"), (6, 2, 256, BF16, "none"),
              (3, 1, 96, F16, "none"), (28, 4, 128, BF16, "none"), (71, 1, 64, BF16, "none"),
              (16, 1, 80, F16, "none"), (33, 1, 256, F16, "none"),
              (8, 2, 128, BF16, "e4m3"), (4, 4, 64, F16, "int8"), (40, 2, 80, BF16, "int8"),
              (6, 2, 256, F16, "e4m3")]


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", GEOMETRIES)
@pytest.mark.parametrize("groups,alone", [
    ([(3, decode(2, 1, 40, 0))], []),
    ([(1, decode(5, 1, 3, 1))], [(1, 1), (1, 200)]),
    ([(20, decode(9, 1, 300, 2)), (7, decode(3, 50, 90, 3)), (2, decode(2, 1, 20, 4))],
     decode(6, 1, 700, 5)),
    ([(64, decode(40, 1, 64, 6))], []),
])
def test_decode_rows(groups, alone, heads, kvh, d, dtype, fmt):
    check(groups, alone, heads, kvh, d, dtype, fmt=fmt)


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", GEOMETRIES)
def test_several_queries_and_mixed_steps(heads, kvh, d, dtype, fmt):
    check([(12, [(4, 30), (5, 5), (1, 77), (1, 1), (33, 33)])], [(1, 90), (70, 200), (2, 2)],
          heads, kvh, d, dtype, fmt=fmt, layout="NHD", bs=32)
    check([(30, [(3, 10), (8, 8)]), (5, [(2, 2), (2, 100)])], [(1, 5)], heads, kvh, d, dtype,
          fmt=fmt)


@pytest.mark.parametrize("left,sinks", [(20, 0), (20, 3), (130, 8), (300, 50), (40, 200), (1000, 1)])
@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", GEOMETRIES[:4] + GEOMETRIES[8:10])
def test_windows_and_sinks(left, sinks, heads, kvh, d, dtype, fmt):
    """Windows that hide some of the prefix, all of it, or part of it from some
    sequences; sinks that pass a short prefix."""
    check([(8, [(1, 20), (1, 150), (1, 7), (6, 90)]), (3, [(1, 1), (1, 400), (9, 9)])],
          [(1, 300), (20, 330)], heads, kvh, d, dtype, left, sinks, fmt=fmt)


def test_right_windows_and_negative_scales():
    shape = ([(8, [(1, 20), (6, 90), (1, 3)])], [(20, 60)], 8, 2, 64, BF16)
    for right in (None, 4):
        check(*shape, right=right)
    check(*shape, scale=-0.2)
    check(*shape, left=50, right=3, sinks=2)


def test_a_sequence_without_keys_of_its_own():
    """A group that shares everything a member has."""
    cache, q, batch, plan = make([(4, [(1, 5), (1, 9), (1, 30)])], [(1, 3)], 8, 2, 128, BF16,
                                 shuffle=False)
    batch.cu_seqlens_k = [0, 64, 133, 227, 230]  # the first ends with the prefix
    prep = prepare(batch, cache, 8, plan)
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), BF16)
    batch.cu_seqlens_k = [0, 40, 109, 203, 206]  # and inside it
    prep = prepare(batch, cache, 8, plan)
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), BF16)


def test_prefixes_that_end_inside_a_block():
    cache, q, batch, _ = make([(5, [(1, 5), (3, 9), (1, 30)])], [], 8, 2, 128, BF16)
    for keys in (1, 15, 33, 79):
        prep = prepare(batch, cache, 8, [([0, 1, 2], keys)])
        got = paged_attention_prepared(q, cache, 0, prep, 0.1)
        assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), BF16)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_long_prefixes_and_large_batches(dtype, d):
    check([(500, decode(60, 1, 600, 7)), (90, decode(30, 1, 50, 8))], decode(40, 1, 3000, 9), 16, 4,
          d, dtype)


@pytest.mark.parametrize("d,fmt", [(256, "none"), (256, "e4m3"), (64, "none")])
def test_as_many_groups_as_a_call_takes(d, fmt):
    check([(1, [(1, 1 + i % 7), (1, 2 + i % 5)]) for i in range(1000)], [(1, 40)], 2, 1, d, BF16,
          fmt=fmt)


def test_prompts_fill_many_tiles():
    """Long prompts beside a group: whole tiles, open ones and joined ones."""
    check([(40, [(1, 20), (200, 300), (64, 64)])], [(700, 900), (300, 300), (1, 2000)], 16, 4, 128,
          BF16)
    check([(4, [(1, 20), (1, 30)])], [(n, n) for n in range(30, 700, 23)], 8, 8, 64, F16)


def test_what_no_query_sees_does_not_matter():
    cache, q, batch, plan = make([(8, [(1, 20), (1, 150), (1, 7), (3, 90)])], [(1, 300)], 8, 2, 128,
                                 BF16)
    left, sinks, bs = 33, 10, 16
    want = reference(q, cache, batch, 0.1, left, 0, sinks)
    k, v = cache.reference_view(0, "k"), cache.reference_view(0, "v")
    cq, ck = batch.cu_seqlens_q, batch.cu_seqlens_k
    seen = set()
    for i, table in enumerate(batch.block_tables):
        lk = ck[i + 1] - ck[i]
        first = max(lk - (cq[i + 1] - cq[i]) - left, 0)
        seen |= {table[p // bs] * bs + p % bs for p in range(lk) if p < sinks or p >= first}
    for slot in range(cache.num_slots()):
        if slot not in seen:
            k[slot // bs, slot % bs] = float("nan")
            v[slot // bs, slot % bs] = float("inf") if slot % 2 else float("nan")
    got = paged_attention_prepared(q, cache, 0, prepare(batch, cache, 8, plan), 0.1, left, 0,
                                   sinks=sinks)
    assert_close(got, want, BF16)


def test_equal_calls_give_equal_bits():
    cache, q, batch, plan = make([(40, decode(20, 1, 200, 1))], decode(9, 1, 900, 2), 16, 4, 128,
                                 BF16)
    prep = prepare(batch, cache, 16, plan, deterministic=True)
    first = paged_attention_prepared(q, cache, 0, prep, 0.1).clone()
    for _ in range(3):
        assert torch.equal(first, paged_attention_prepared(q, cache, 0, prep, 0.1))


def test_the_step_finds_its_prefixes():
    cache, q, batch, plan = make([(200, decode(60, 1, 200, 1)), (70, decode(3, 1, 20, 2))],
                                 decode(3, 1, 400, 3), 8, 2, 128, F16)
    prep = PreparedAttention.from_batch(batch, DEV, cache, 8, share_prefixes=True)
    assert sorted((sorted(m), n) for m, n in prep.prefixes.groups) == sorted(
        (sorted(m), n) for m, n in plan)
    # 59 x 3,200 keys of 1 KiB are worth it; not behind a short window.
    assert prep.shared_bytes(cache, 8) > 0 and prep.shared_bytes(cache, 8, 100) == 0
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), F16)
    few = make([(40, decode(6, 1, 200, 1))], [], 8, 2, 128, F16)
    prep = PreparedAttention.from_batch(few[2], DEV, few[0], 8, share_prefixes=True)
    assert prep.prefixes is not None and prep.shared_bytes(few[0], 8) == 0
    got = paged_attention_prepared(few[1], few[0], 0, prep, 0.1)
    assert_close(got, reference(few[1], few[0], few[2], 0.1, None, 0, 0), F16)
    # Nothing to share: the ordinary call.
    lone = make([], decode(3, 1, 400, 3), 8, 2, 128, F16)
    assert PreparedAttention.from_batch(lone[2], DEV, lone[0], 8,
                                        share_prefixes=True).prefixes is None


def test_pools_that_take_no_prefixes_run_the_ordinary_call():
    cache, q, batch, plan = make([(70, decode(6, 1, 200, 1))], [(1, 30)], 8, 2, 64, F32)
    prep = PreparedAttention.from_batch(batch, DEV, cache, 8, share_prefixes=True)
    prep.prefixes.min_bytes = 0  # whatever it saves
    prep.sharing.clear()
    assert prep.shared_bytes(cache, 8) == 0 and b"16-bit" in lib().vapi_kv_last_error()
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), F32)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
def test_a_write_and_its_attention(fmt):
    cache, q, batch, plan = make([(20, [(1, 20), (1, 33), (4, 9)])], [(1, 50)], 8, 2, 64, BF16,
                                 fmt=fmt)
    cq, ck = batch.cu_seqlens_q, batch.cu_seqlens_k
    slots = [t[p // 16] * 16 + p % 16 for i, t in enumerate(batch.block_tables)
             for p in range(ck[i + 1] - ck[i] - (cq[i + 1] - cq[i]), ck[i + 1] - ck[i])]
    k, v = (torch.randn(len(slots), 2, 64, device=DEV).to(BF16) for _ in range(2))
    prep = prepare(batch, cache, 8, plan)
    got = paged_attention_append_prepared(q, k, v, scatter_index(np.array(slots), DEV), cache, 0,
                                          prep, 0.125)
    assert_close(got, reference(q, cache, batch, 0.125, None, 0, 0), BF16)
    # A refused call writes nothing.
    before = cache.k[0].clone()
    with pytest.raises(ValueError):
        paged_attention_append_prepared(q.view(-1)[1:1 + 6 * 8 * 64].view(6, 8, 64), k[:6], v[:6],
                                        scatter_index(np.array(slots[:6]), DEV), cache, 0, prep,
                                        0.125)
    assert torch.equal(before, cache.k[0])


def test_layers_of_different_geometry_in_one_step():
    cache = HybridKvCache([("kv", 2, 64), ("kv", 1, 128), ("kv", 2, 256)], 80, 16, BF16, device=DEV)
    for t in cache.k + cache.v:
        t.normal_()
    head = list(range(50))
    batch = ForwardBatch(cu_seqlens_q=[0, 1, 2, 3], cu_seqlens_k=[0, 810, 1640, 2490],
                         block_tables=[head + [50], head + [51, 52], head + [60, 61, 62, 63]],
                         max_seqlen_q=1, max_seqlen_k=850)
    prep = PreparedAttention.from_batch(batch, DEV, cache, 4, share_prefixes=True)
    assert prep.prefixes.groups == [([0, 1, 2], 800)]
    prep.prefixes.min_bytes = 0  # whatever it saves
    prep.sharing.clear()
    prep.reserve(cache, 4, DEV)
    assert all(prep.sharing.values())
    for layer, (kvh, d) in enumerate(((2, 64), (1, 128), (2, 256))):
        one = PagedKvCache(1, 80, 16, kvh, d, BF16)
        one.k[0].copy_(cache.k[layer])
        one.v[0].copy_(cache.v[layer])
        q = torch.randn(3, 4, d, device=DEV).to(BF16)
        for left, sinks in ((None, 0), (600, 4)):
            got = paged_attention_prepared(q, cache, layer, prep, 0.1, left, 0, sinks=sinks)
            assert_close(got, reference(q, one, batch, 0.1, left, 0, sinks), BF16)


def test_a_step_replays_from_a_graph_while_its_sequences_grow():
    """The plan stays while lengths on the device grow; other calls use the workspace
    between replays."""
    cache, q, batch, plan = make([(12, decode(7, 10, 40, 1))], decode(3, 10, 300, 2), 8, 2, 128,
                                 BF16, shuffle=False)
    for t in batch.block_tables:  # room to grow in blocks of the pool
        t.append(0)
    batch.max_seqlen_k += 8
    prep = prepare(batch, cache, 8, plan, deterministic=True)
    out = torch.empty_like(q)
    paged_attention_prepared(q, cache, 0, prep, 0.1, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attention_prepared(q, cache, 0, prep, 0.1, out=out)
    b = batch.batch_size()
    for step in range(4):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert_close(out, reference(q, cache, batch, 0.1, None, 0, 0), BF16)
        eager = paged_attention_prepared(q, cache, 0, prep, 0.1)
        assert torch.equal(out, eager)
        batch.cu_seqlens_k = [x + i for i, x in enumerate(batch.cu_seqlens_k)]
        prep.seqlens_k.copy_(torch.tensor(batch.cu_seqlens_k, dtype=torch.int32))
    assert b == 10


def test_other_streams():
    cache, q, batch, plan = make([(30, decode(20, 1, 200, 1))], decode(9, 1, 900, 2), 16, 4, 128,
                                 BF16)
    want = paged_attention_prepared(q, cache, 0, prepare(batch, cache, 16, plan, True), 0.1)
    side = torch.cuda.Stream()
    prep = prepare(batch, cache, 16, plan, True)
    side.wait_stream(torch.cuda.current_stream())
    got = paged_attention_prepared(q, cache, 0, prep, 0.1, stream=side)
    del prep
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [GEOMETRIES[0], GEOMETRIES[8], GEOMETRIES[11]])
def test_padded_batches(heads, kvh, d, dtype, fmt):
    """Members and others without queries, a group of none but those, rows past the last."""
    cache, q, batch, plan = make([(6, [(0, 5), (1, 9), (0, 30), (3, 8)]), (3, [(0, 1), (0, 7)])],
                                 [(0, 40), (1, 3), (0, 0), (5, 50)], heads, kvh, d, dtype, fmt=fmt)
    n = q.shape[0]
    q = torch.cat([q, torch.full_like(q[:4], float("nan"))])
    out = torch.full_like(q, 7.0)
    prep = prepare(batch, cache, heads, plan)
    assert prep.shared_bytes(cache, heads) > 0
    got = paged_attention_prepared(q, cache, 0, prep, 0.1, out=out)
    assert bool((got[n:] == 7.0).all())
    assert_close(got[:n], reference(q[:n], cache, batch, 0.1, None, 0, 0), dtype)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
def test_two_steps_at_once(fmt):
    """On two streams, each with its own prepared step."""
    work = [make([(40, decode(30, 1, 300, i)), (9, [(5, 9), (1, 80)])], decode(5, 1, 500, 7 + i),
                 8, 2, 128, BF16, fmt=fmt, seed=i) for i in range(2)]
    steps = [prepare(batch, cache, 8, plan, True) for cache, _, batch, plan in work]
    want = [paged_attention_prepared(q, cache, 0, p, 0.1)
            for (cache, q, _, _), p in zip(work, steps)]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, ((cache, q, _, _), p) in enumerate(zip(work, steps)):
            got[i].append(paged_attention_prepared(q, cache, 0, p, 0.1, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_call_that_covers_every_row_with_tiles():
    """ATTN_NO_DECODE_ROWS on a batch that has decode rows: they run as tiles too."""
    cache, q, batch, plan = make([(12, [(4, 30), (1, 77), (33, 33)])], [(1, 90), (70, 200)], 8, 2,
                                 128, BF16)
    prep = prepare(batch, cache, 8, plan)
    prep.flags |= ATTN_NO_DECODE_ROWS
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), BF16)


def test_blocks_past_32_bit_offsets():
    bs, kvh, d = 64, 8, 128
    nb = (5 << 30) // (bs * kvh * d * 2)
    cache = PagedKvCache(1, nb, bs, kvh, d, BF16)
    head = list(range(nb - 40, nb))
    tables = [head + [5], head + [nb - 41], head + [0, 7]]
    used = sorted({b for t in tables for b in t})
    small = PagedKvCache(1, len(used), bs, kvh, d, BF16)
    for i, b in enumerate(used):
        cache.k[0][b].normal_()
        cache.v[0][b].normal_()
        small.k[0][i].copy_(cache.k[0][b])
        small.v[0][i].copy_(cache.v[0][b])
    lens = [2560 + 9, 2560 + 64, 2560 + 70]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    batch = ForwardBatch(cu_seqlens_q=[0, 1, 2, 3], cu_seqlens_k=cu, block_tables=tables,
                         max_seqlen_q=1, max_seqlen_k=max(lens))
    local = ForwardBatch(cu_seqlens_q=[0, 1, 2, 3], cu_seqlens_k=cu, max_seqlen_q=1,
                         block_tables=[[used.index(b) for b in t] for t in tables],
                         max_seqlen_k=max(lens))
    q = torch.randn(3, 16, d, device=DEV).to(BF16)
    got = paged_attention_prepared(q, cache, 0, prepare(batch, cache, 16, [([0, 1, 2], 2560)]), 0.1)
    assert_close(got, reference(q, small, local, 0.1, None, 0, 0), BF16)


def test_refusals():
    cache, q, batch, plan = make([(4, [(1, 5), (1, 9)])], [], 8, 2, 64, BF16)
    with pytest.raises(ValueError):
        PreparedAttention.from_batch(batch, DEV, share_prefixes=True)
    for bad in ([([0, 0], 64)], [([0, 1], 64), ([1], 16)], [([0, 2], 64)], [([0, 1], 0)]):
        with pytest.raises(ValueError):
            PrefixPlan(bad, batch.cu_seqlens_q, batch.cu_seqlens_k, DEV)
    prep = prepare(batch, cache, 8, [([0, 1], 64)])
    prep.prefixes.arg.max_keys = 1 << 20
    assert prep.shared_bytes(cache, 8) == 0 and b"prefix" in lib().vapi_kv_last_error()
    prep = prepare(batch, cache, 8, plan)
    prep.flags = 0x80
    with pytest.raises(VapiKvError):
        paged_attention_prepared(q, cache, 0, prep, 0.1)


# Groups whose members all lie further past the prefix than the left window of 41 keys
# reaches, by one key or many, so that a tile of theirs sees its sinks only; prefixes of
# whole steps of 32 keys and not; one group beside another that is in reach.
PAST = [
    [(8, [(1, 42), (1, 150), (1, 77)])],
    [(9, [(1, 60), (4, 90), (1, 43), (2, 45), (30, 75)])],
    [(8, [(1, 100), (3, 47)]), (5, [(1, 3), (1, 300), (2, 41)])],
    [(3, [(1, 50 + 3 * i) for i in range(80)]), (12, [(5, 46 + i) for i in range(20)])],
]


@pytest.mark.parametrize("groups", PAST)
@pytest.mark.parametrize("sinks", [1, 5, 32, 40])
@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [
    (8, 8, 64, BF16, "none"), (8, 2, 128, F16, "none"), (4, 1, 256, BF16, "none"),
    (28, 1, 128, BF16, "none"), (71, 1, 64, F16, "none"), (6, 3, 96, BF16, "none"),
    (2, 2, 128, BF16, "e4m3"), (28, 1, 64, F16, "int8"), (71, 1, 256, BF16, "int8"),
    (4, 1, 256, F16, "e4m3")])
def test_sinks_of_a_prefix_that_no_window_reaches(groups, sinks, heads, kvh, d, dtype, fmt):
    check(groups, [(1, 200), (3, 30)], heads, kvh, d, dtype, 40, sinks, fmt=fmt)


def test_sinks_alone_behind_a_right_window():
    for right in (3, None):
        check(PAST[1], [], 8, 2, 128, BF16, 40, 5, right=right)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", BF16), ("int8", F16), ("none", F16)])
@pytest.mark.parametrize("heads,kvh,d", [(4, 1, 64), (2, 2, 64), (8, 8, 64), (32, 32, 96),
                                         (24, 12, 96), (8, 8, 80), (12, 3, 80), (34, 2, 80)])
def test_sinks_over_rows_that_share_cache_lines(heads, kvh, d, fmt, dtype):
    """Token-major pools, members (and others) whose own keys span several of the
    stream's ranges."""
    check([(70, decode(24, 1, 1500, d)), (4, [(1, 900), (3, 700), (1, 1)])], decode(8, 1, 2500, 3),
          heads, kvh, d, dtype, 1200, 20, fmt=fmt, layout="NHD")


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [
    (8, 2, 128, BF16, "e4m3"), (8, 2, 128, BF16, "int8"), (4, 4, 64, F16, "int8"),
    (6, 2, 256, F16, "e4m3")])
def test_what_no_query_sees_of_codes_does_not_matter(heads, kvh, d, dtype, fmt):
    """Codes that are NaN where no query looks, and scales of any value in blocks of those."""
    members = [(1, 20), (1, 150), (1, 7), (3, 90)]
    cache, q, batch, plan = make([(8, members), (9, [(1, 60), (1, 400)])], [(1, 300)], heads, kvh, d,
                                 dtype, fmt=fmt)
    left, sinks, bs = 33, 10, 16
    want = reference(q, cache, batch, 0.1, left, 0, sinks)
    cq, ck = batch.cu_seqlens_q, batch.cu_seqlens_k
    seen = set()
    for i, table in enumerate(batch.block_tables):
        lk = ck[i + 1] - ck[i]
        first = max(lk - (cq[i + 1] - cq[i]) - left, 0)
        seen |= {table[p // bs] * bs + p % bs for p in range(lk) if p < sinks or p >= first}
    hidden = torch.ones(cache.num_slots(), dtype=torch.bool)
    hidden[list(seen)] = False
    hidden = hidden.view(-1, bs).to(DEV)
    whole = hidden.all(dim=1)
    for c, s in ((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])):
        c.view(torch.uint8).masked_fill_(hidden[:, None, :, None], 0x7F)
        s.masked_fill_(whole[:, None], float("nan"))
    got = paged_attention_prepared(q, cache, 0, prepare(batch, cache, heads, plan), 0.1, left, 0,
                                   sinks=sinks)
    assert_close(got, want, dtype)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
@pytest.mark.parametrize("n_groups,n_rows", [(0, 8), (3, 0), (0, 0)])
def test_lists_of_nothing_are_not_read(n_groups, n_rows, fmt):
    """Rows without groups and groups without rows: the call takes null lists for them."""
    cache, q, batch, _ = make([], [(1, 300), (1, 20), (3, 90), (1, 2000)], 8, 2, 128, BF16, fmt=fmt)
    prep = prepare(batch, cache, 8, [])
    a = prep.prefixes.arg
    a.n_groups, a.n_rows, a.rows, a.seqs, a.keys = n_groups, n_rows, None, None, None
    assert prep.shared_bytes(cache, 8) > 0
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, reference(q, cache, batch, 0.1, None, 0, 0), BF16)


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [GEOMETRIES[0], GEOMETRIES[2], GEOMETRIES[9]])
@pytest.mark.parametrize("left_out", [0, 2, 4])
def test_sequences_that_the_prefill_list_leaves_out(left_out, heads, kvh, d, dtype, fmt):
    """They end with the shared keys, whatever an earlier call left in the workspace."""
    members = [(5, 40), (1, 60), (40, 300), (1, 5), (9, 9)]
    cache, q, batch, plan = make([(12, members)], [(30, 80), (1, 200)], heads, kvh, d, dtype, fmt=fmt,
                                 shuffle=False)
    prep = prepare(batch, cache, heads, plan)
    want, top = reference(q, cache, batch, 0.1, None, 0, 0)
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    assert_close(got, (want, top), dtype)
    prep.prefill_seqs = torch.tensor([s for s in (0, 2, 4, 5) if s != left_out], dtype=torch.int32,
                                     device=DEV)
    prep.n_prefill = 3
    got = paged_attention_prepared(q, cache, 0, prep, 0.1)
    lens = np.diff(batch.cu_seqlens_k)
    lens[left_out] = 12 * 16
    short = ForwardBatch(cu_seqlens_q=batch.cu_seqlens_q, block_tables=batch.block_tables,
                         cu_seqlens_k=np.concatenate([[0], np.cumsum(lens)]).tolist())
    rows = slice(batch.cu_seqlens_q[left_out], batch.cu_seqlens_q[left_out + 1])
    want[rows] = reference(q, cache, short, 0.1, None, None, 0)[0][rows]
    assert_close(got, (want, top), dtype)


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [GEOMETRIES[0], GEOMETRIES[5], GEOMETRIES[11]])
@pytest.mark.parametrize("members,many", [(3, 1), (150, 1), (5, 300), (1100, 1)])
def test_entries_that_name_no_query_are_left_out(members, many, heads, kvh, d, dtype, fmt):
    """The first of a group among them, and all of one: a sequence past the batch, one that
    has ended and whose table names nothing, a row that is not the sequence's."""
    if members * heads > 16000:
        heads = kvh  # (the reference's time)
    groups = [(6, [(1, 1 + i % 50) for i in range(members)])]
    groups += [(1, [(1, 1 + i % 9), (1, 3)]) for i in range(many)]
    cache, q, batch, plan = make(groups + [(3, [(0, 5), (0, 9)])], [(0, 0), (1, 40)], heads, kvh, d,
                                 dtype, fmt=fmt, shuffle=False)
    want = reference(q, cache, batch, 0.1, None, 0, 0)
    n, ended = len(batch.block_tables), members + 2 * many
    batch.block_tables[ended] = [0] * 4  # what a finished request leaves
    prep = prepare(batch, cache, heads, plan)
    a, words = prep.prefixes.arg, prep.prefixes.lists.cpu().numpy().view(np.uint32)

    def at(p, count):
        i = (p - prep.prefixes.lists.data_ptr()) // 4
        return words[i:i + count].tolist()

    offsets, rows, seqs = at(a.offsets, a.n_groups + 1), at(a.rows, a.n_rows), at(a.seqs, a.n_rows)
    dead = [(0, n), (0, ended), (0xFFFFFFFF, 0), (0, n - 1), (0xFFFFFFFF, 0xFFFFFFFF)]
    new = [[], [], [0]]
    for g in range(a.n_groups):
        front = dead * 30 if g == 0 else dead[g % 5:g % 5 + 1] * (g % 2)
        some = list(zip(rows, seqs))[offsets[g]:offsets[g + 1]]
        if not some:  # the group without queries: entries that name none
            front = dead * 2
        for row, seq in front + some[:2] + dead + some[2:]:
            new[0].append(row)
            new[1].append(seq)
        new[2].append(len(new[0]))
    lists = [new[2], new[0], new[1], at(a.keys, a.n_groups), at(a.start, n)]
    sizes = np.cumsum([0] + [len(x) for x in lists])
    prep.prefixes.lists = torch.from_numpy(
        np.concatenate(lists).astype(np.uint32).view(np.int32)).to(DEV)
    ptr = [prep.prefixes.lists.data_ptr() + 4 * int(x) for x in sizes]
    a.offsets, a.rows, a.seqs, a.keys, a.start = ptr[:5]
    a.n_rows = len(new[0])
    assert prep.shared_bytes(cache, heads) > 0
    out = torch.full_like(q, float("nan"))
    got = paged_attention_prepared(q, cache, 0, prep, 0.1, out=out)
    assert_close(got, want, dtype)


@pytest.mark.parametrize("heads,kvh,d,dtype,fmt", [
    (8, 2, 128, BF16, "none"), (4, 4, 64, F16, "none"), (6, 2, 256, BF16, "none"),
    (8, 2, 128, BF16, "e4m3"), (32, 32, 96, F16, "none")])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_a_nan_key_stays_with_the_rows_that_see_it(where, heads, kvh, d, dtype, fmt):
    """A NaN in the shared keys reaches every member's outputs, one in a member's own keys
    that member's."""
    members = [(1, 50), (1, 900), (4, 70), (1, 33), (30, 60)]
    cache, q, batch, plan = make([(40, members)], [(1, 200), (5, 90)], heads, kvh, d, dtype, fmt=fmt,
                                 shuffle=False)
    want, top = reference(q, cache, batch, 0.1, None, 0, 0)
    key = 300 if where == "prefix" else 640 + 5
    block = batch.block_tables[1][key // 16]
    if fmt == "none":
        cache.k[0][block, 0, key % 16] = float("nan")
    else:
        cache.k[0].view(torch.uint8)[block, 0, key % 16] = 0x7F
    got = paged_attention_prepared(q, cache, 0, prepare(batch, cache, heads, plan), 0.1)
    rows = slice(0, 37) if where == "prefix" else slice(1, 2)
    group = heads // kvh
    assert torch.isnan(got[rows, :group]).all()
    got[rows, :group] = 0.0
    want[rows, :group] = 0.0
    assert_close(got, (want, top), dtype)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
def test_a_plan_on_another_device_is_refused(fmt):
    cache, q, batch, plan = make([(4, [(1, 5), (1, 9)])], [], 8, 2, 64, BF16, fmt=fmt)
    prep = prepare(batch, cache, 8, plan)
    prep.prefixes = PrefixPlan(plan, batch.cu_seqlens_q, batch.cu_seqlens_k, "cpu")
    with pytest.raises(ValueError, match="cpu"):
        paged_attention_prepared(q, cache, 0, prep, 0.1)
    before = cache.k[0].clone()
    k = torch.zeros(2, 2, 64, device=DEV, dtype=BF16)
    with pytest.raises(ValueError, match="cpu"):
        paged_attention_append_prepared(q, k, k, scatter_index(np.array([0, 1]), DEV), cache, 0, prep,
                                        0.1)
    assert torch.equal(before.view(torch.uint8), cache.k[0].view(torch.uint8))


@pytest.mark.parametrize("fmt,layout", [("none", "HND"), ("e4m3", "NHD"), ("int8", "HND")])
def test_a_write_and_its_attention_behind_a_window_with_sinks(fmt, layout):
    """A layer's call of a windowed model over shared prefixes, members in and out of the
    prefix's reach."""
    members = [(1, 20), (1, 333), (4, 90), (1, 64), (9, 200)]
    cache, q, batch, plan = make([(20, members), (4, [(1, 300), (2, 400)])], [(1, 50), (3, 3)], 8, 2,
                                 64, BF16, fmt=fmt, layout=layout)
    cq, ck = batch.cu_seqlens_q, batch.cu_seqlens_k
    slots = [t[p // 16] * 16 + p % 16 for i, t in enumerate(batch.block_tables)
             for p in range(ck[i + 1] - ck[i] - (cq[i + 1] - cq[i]), ck[i + 1] - ck[i])]
    k, v = (torch.randn(len(slots), 2, 64, device=DEV).to(BF16) for _ in range(2))
    prep = prepare(batch, cache, 8, plan)
    got = paged_attention_append_prepared(q, k, v, scatter_index(np.array(slots), DEV), cache, 0,
                                          prep, 0.125, 63, 0, sinks=4)
    assert_close(got, reference(q, cache, batch, 0.125, 63, 0, 4), BF16)


@pytest.mark.parametrize("fmt", ["none", "int8"])
def test_a_graph_replays_while_windows_leave_the_prefix(fmt):
    """Two graphs over one workspace, a windowed layer with sinks and one without a window;
    the lengths on the device grow until no window reaches the prefix."""
    cache, q, batch, plan = make([(12, decode(5, 26, 30, 1))], decode(2, 10, 300, 2), 8, 2, 128,
                                 BF16, shuffle=False, fmt=fmt)
    spare = [b for b in range(cache.num_slots() // 16)
             if not any(b in t for t in batch.block_tables)]
    for i, t in enumerate(batch.block_tables):  # room to grow in blocks of the pool
        t.append(spare[i % len(spare)])
    batch.max_seqlen_k += 12
    prep = prepare(batch, cache, 8, plan, deterministic=True)
    calls = [(None, 0), (29, 3)]
    outs, graphs = [torch.empty_like(q) for _ in calls], []
    for out, (left, sinks) in zip(outs, calls):
        paged_attention_prepared(q, cache, 0, prep, 0.1, left, 0, out=out, sinks=sinks)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            paged_attention_prepared(q, cache, 0, prep, 0.1, left, 0, out=out, sinks=sinks)
    for step in range(4):
        for out, graph in zip(outs, graphs):
            out.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        for out, (left, sinks) in zip(outs, calls):
            assert_close(out, reference(q, cache, batch, 0.1, left, 0, sinks), BF16)
            assert torch.equal(out, paged_attention_prepared(q, cache, 0, prep, 0.1, left, 0,
                                                             sinks=sinks))
        torch.cuda.synchronize()
        batch.cu_seqlens_k = [x + 3 * i for i, x in enumerate(batch.cu_seqlens_k)]
        prep.seqlens_k.copy_(torch.tensor(batch.cu_seqlens_k, dtype=torch.int32))


@pytest.mark.parametrize("d,fmt", [(128, "none"), (64, "int8"), (256, "e4m3")])
def test_sinks_of_more_members_than_entries_in_lds(d, fmt):
    """Tiles past every window beside tiles in reach, their rows looked up one by one."""
    check([(3, [(1, 42 + i % 30) for i in range(700)] + [(1, 1 + i % 39) for i in range(500)])],
          [(1, 90)], 2, 1, d, BF16, 40, 5, fmt=fmt, shuffle=False)
