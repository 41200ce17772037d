"""The 8-bit paged KV cache on the GPU against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import quant_ref as ref
from vapi_amd._lib import SLOT_SKIP, VapiKvError, lib
from vapi_amd.attention import (ForwardBatch, PreparedAttention, paged_attention,
                                paged_attention_append_prepared, paged_attention_prepared)
from vapi_amd.backend import KvBlockBackend
from vapi_amd.cache import (PagedKvCache, gather_kv, scatter_index, write_kv_to_cache,
                            write_rows_indexed)
from vapi_amd.quant import QuantKvCache
from vapi_amd.spill import SpillStore, pinned_buffer, promote, spill_evicted

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rows(gen, n, kvh, d, dtype, spread=1.5):
    """Rows whose size differs from token to token and from channel to channel."""
    x = torch.randn(n, kvh, d, generator=gen)
    x = x * torch.exp2(spread * torch.randn(n, 1, 1, generator=gen))
    return (x * torch.exp2(torch.randn(1, kvh, d, generator=gen))).to(dtype)


def same(cache, layer, which, model):
    codes = (cache.k if which == "k" else cache.v)[layer].float().cpu().double()
    codes = codes if cache.layout == "HND" else codes.permute(0, 2, 1, 3)
    scale = (cache.k_scale if which == "k" else cache.v_scale)[layer].cpu().double()
    assert torch.equal(scale, torch.from_numpy(model.scale))
    assert torch.equal(codes, torch.from_numpy(model.codes))


def models(cache):
    args = (cache.num_blocks, cache.num_kv_heads, cache.block_size, cache.head_dim, cache.fmt,
            cache.dtype)
    return ref.Model(*args), ref.Model(*args)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,layout,bs,kvh,d", [
    (BF16, "HND", 16, 8, 128), (F16, "HND", 16, 2, 64), (BF16, "NHD", 32, 3, 80),
    (F16, "NHD", 16, 5, 96), (BF16, "HND", 64, 1, 16), (F16, "HND", 256, 2, 256),
    (BF16, "NHD", 128, 1, 240)])
def test_append_is_exact(fmt, dtype, layout, bs, kvh, d):
    gen = torch.Generator().manual_seed(bs * kvh + d)
    r = np.random.default_rng(bs + d)
    nb = 12
    cache = QuantKvCache(2, nb, bs, kvh, d, dtype, fmt, layout)
    mk, mv = models(cache)
    perm = r.permutation(nb)
    # Three sequences: a prompt, a few rows more, then single tokens; blocks are
    # started, added to, and filled over a step's end.
    at, tables = [0, 0, 0], [perm[:4], perm[4:8], perm[8:12]]
    for step, counts in enumerate([(2 * bs + 3, 5, bs), (1, 1, 1), (bs // 2, 3, 1), (1, 0, 1),
                                   (1, 1, 1)]):
        slots = [np.full(2, SLOT_SKIP)]
        for s, n in enumerate(counts):
            pos = np.arange(at[s], at[s] + n)
            slots += [tables[s][pos // bs] * bs + pos % bs, np.full(step % 2, SLOT_SKIP)]
            at[s] += n
        slots = np.concatenate(slots)
        k, v = rows(gen, len(slots), kvh, d, dtype), rows(gen, len(slots), kvh, d, dtype)
        write_kv_to_cache(cache, 1, k.cuda(), v.cuda(), slots)
        mk.append(k, slots)
        mv.append(v, slots)
        same(cache, 1, "k", mk)
        same(cache, 1, "v", mv)
    assert not cache.k_scale[0].any() and not cache.k[0].view(torch.uint8).any()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 513, 2000])
@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", F16)])
def test_append_of_many_single_tokens_and_runs(fmt, dtype, n):
    """Every kind of launch: a token per workgroup, and several."""
    gen = torch.Generator().manual_seed(n)
    r = np.random.default_rng(n)
    bs, kvh, d, nb = 16, 2, 64, n + 3
    cache = QuantKvCache(1, nb, bs, kvh, d, dtype, fmt)
    mk, mv = models(cache)
    perm = r.permutation(nb)
    for run in (5, 1, 40):
        slots, i, b = [], 0, 0
        while i < n:
            m = min(run, n - i)
            first = int(r.integers(0, bs))
            pos = np.arange(first, first + m)
            slots.append(perm[b + pos // bs] * bs + pos % bs)
            i, b = i + m, b + (first + m + bs - 1) // bs
            if b + 4 > nb:
                break
        slots = np.concatenate(slots)
        # Order within a block is free, and tokens may be skipped.
        slots[r.random(len(slots)) < 0.1] = SLOT_SKIP
        k, v = rows(gen, len(slots), kvh, d, dtype), rows(gen, len(slots), kvh, d, dtype)
        write_kv_to_cache(cache, 0, k.cuda(), v.cuda(), slots)
        mk.append(k, slots)
        mv.append(v, slots)
        same(cache, 0, "k", mk)
        same(cache, 0, "v", mv)


def test_append_long_skips_and_any_order_within_a_block():
    gen = torch.Generator().manual_seed(5)
    cache = QuantKvCache(1, 8, 16, 1, 64, BF16, "int8")
    mk, mv = models(cache)
    skip = [SLOT_SKIP] * 200
    # A block's tokens backwards with 200 skipped ones among them, and slots
    # past the pool, which are dropped.
    slots = skip + [47, 46] + skip + [33, 40] + skip + [9, 8, 10 ** 6, 128, 11] + skip
    k, v = rows(gen, len(slots), 1, 64, BF16), rows(gen, len(slots), 1, 64, BF16)
    write_rows_indexed(cache, 0, k.cuda(), v.cuda(), scatter_index(slots, "cuda"))
    mk.append(k, slots)
    mv.append(v, slots)
    same(cache, 0, "k", mk)
    same(cache, 0, "v", mv)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_of_extreme_rows(fmt, dtype):
    """Zeros, the dtype's largest and least values, infinities and NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    sub = float(torch.tensor(1, dtype=torch.int16).view(dtype))  # the least subnormal
    x = torch.zeros(6 * 16, 1, 16, dtype=dtype)
    x[16:32] = torch.linspace(-1, 1, 16).to(dtype) * big
    x[32:48] = torch.linspace(-40, 40, 16).to(dtype) * sub
    x[48, 0, 3], x[49, 0, 4], x[50, 0, 5] = float("inf"), float("nan"), float("-inf")
    x[51] = 1.0
    x[64:80] = float("nan")
    x[80:96] = torch.linspace(-1, 1, 16).to(dtype) * 300 * tiny
    cache = QuantKvCache(1, 6, 16, 1, 16, dtype, fmt)
    mk, mv = models(cache)
    write_kv_to_cache(cache, 0, x.cuda(), (-x).cuda(), np.arange(96))
    mk.append(x, np.arange(96))
    mv.append(-x, np.arange(96))
    same(cache, 0, "k", mk)
    same(cache, 0, "v", mv)
    got = gather_kv(cache, 0, list(range(6)), 96)
    assert torch.isfinite(got).all()
    # Codes times scales are values of the dtype.
    assert torch.equal(got.cpu().double().reshape(6, 16, 1, 16),
                       torch.from_numpy(mk.codes * mk.scale[:, :, None, None])
                       .permute(0, 2, 1, 3))


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("e4m3", F16), ("int8", BF16),
                                       ("int8", F16)])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_gather_gives_the_values(fmt, dtype, layout):
    gen = torch.Generator().manual_seed(3)
    cache = QuantKvCache(2, 9, 32, 3, 48, dtype, fmt, layout)
    table = [7, 2, 5, 0]
    slots = ref.slots_of(table, 100, 32)
    k, v = rows(gen, 100, 3, 48, dtype), rows(gen, 100, 3, 48, dtype)
    write_kv_to_cache(cache, 1, k.cuda(), v.cuda(), slots)
    for which in ("k", "v"):
        for n in (0, 1, 31, 32, 100):
            got = gather_kv(cache, 1, table, n, which)
            want = ref.values(cache, 1, which)[slots[:n]]
            assert got.dtype == dtype and torch.equal(got.cpu().double(), want)
    # A table entry past the pool reads nothing.
    assert not gather_kv(cache, 1, [7, 99], 40)[32:].any()


# ---- attention ------------------------------------------------------------------


def filled(lens_k, kvh, d, bs, fmt, dtype, layout, seed, layers=1, spare=2):
    """A cache whose sequences hold rows written by the append, and their tables."""
    gen = torch.Generator().manual_seed(seed)
    r = np.random.default_rng(seed)
    need = [-(-n // bs) for n in lens_k]
    nb = sum(need) + spare
    perm = r.permutation(nb).tolist()
    tables = []
    for n in need:
        tables.append([perm.pop() for _ in range(n)])
    cache = QuantKvCache(layers, nb, bs, kvh, d, dtype, fmt, layout)
    slots = np.concatenate([ref.slots_of(t, n, bs) for t, n in zip(tables, lens_k) if n])
    k, v = rows(gen, len(slots), kvh, d, dtype, 0.5), rows(gen, len(slots), kvh, d, dtype, 0.5)
    k = k / 4
    write_kv_to_cache(cache, layers - 1, k.cuda(), v.cuda(), slots)
    return cache, tables


def batch_of(lens_q, lens_k, tables):
    return ForwardBatch(cu_seqlens_q=np.concatenate([[0], np.cumsum(lens_q)]).tolist(),
                        cu_seqlens_k=np.concatenate([[0], np.cumsum(lens_k)]).tolist(),
                        block_tables=tables, max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))


def check_attention(lens_q, lens_k, heads, kvh, d, bs, fmt, dtype, layout, left=None, right=0,
                    scale=None, deterministic=False, seed=0):
    cache, tables = filled(lens_k, kvh, d, bs, fmt, dtype, layout, seed + sum(lens_k))
    gen = torch.Generator().manual_seed(seed + 1)
    n = sum(lens_q)
    q = torch.randn(n, heads, d, generator=gen).to(dtype)
    scale = d ** -0.5 if scale is None else scale
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda", cache, heads,
                                        deterministic)
    # Rows behind the last sequence stay as they were.
    out = torch.full((n + 3, heads, d), 7.0, dtype=dtype, device="cuda")
    first = None
    for _ in range(3):
        paged_attention_prepared(q.cuda(), cache, 0, prep, scale, left, right, out=out[:n])
        if deterministic:
            first = out.clone() if first is None else first
            assert torch.equal(out, first)
    assert torch.all(out[n:] == 7.0)
    want, bound = ref.attention(q, ref.values(cache, 0, "k"), ref.values(cache, 0, "v"), lens_q,
                                lens_k, tables, bs, scale, left, right)
    err = (out[:n].cpu().double() - want).abs()
    assert torch.all(err <= bound), f"{float((err / bound).max()):.3g} times the bound"


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("e4m3", F16), ("int8", BF16),
                                       ("int8", F16)])
@pytest.mark.parametrize("heads,kvh,d,bs,layout", [
    (8, 2, 128, 16, "HND"), (8, 8, 64, 32, "NHD"), (7, 1, 256, 16, "HND"),
    (10, 2, 80, 16, "NHD"), (4, 4, 96, 64, "HND"), (6, 3, 16, 16, "HND"),
    (17, 1, 128, 16, "HND"), (71, 1, 64, 16, "HND"), (40, 1, 208, 128, "NHD")])
def test_decode(fmt, dtype, heads, kvh, d, bs, layout):
    check_attention([1] * 8, [1, 2, 15, 16, 17, 64, 129, 700], heads, kvh, d, bs, fmt, dtype,
                    layout)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("e4m3", F16), ("int8", BF16),
                                       ("int8", F16)])
@pytest.mark.parametrize("heads,kvh,d,bs,layout,left", [
    (4, 2, 128, 16, "HND", None), (4, 4, 64, 32, "NHD", 50), (3, 1, 256, 16, "HND", None),
    (2, 2, 80, 16, "NHD", 70), (4, 4, 96, 64, "HND", 129), (3, 3, 16, 16, "HND", None),
    (34, 2, 128, 16, "HND", None), (71, 1, 64, 16, "HND", 40), (40, 1, 208, 128, "NHD", None)])
def test_decode_of_many_rows(fmt, dtype, heads, kvh, d, bs, layout, left):
    """More (sequence, kv head) pairs than the short-context kernel takes, rows of
    other lengths among them (the persistent stream)."""
    n = 260 // kvh + 3
    lens = [1 + (7 * i) % 150 + (400 if i % 41 == 7 else 0) for i in range(n)]
    check_attention([1 + 2 * (i == 5) for i in range(n)], [max(k, 3) for k in lens], heads, kvh,
                    d, bs, fmt, dtype, layout, left)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", F16), ("int8", BF16)])
@pytest.mark.parametrize("left", [0, 1, 15, 63, 64, 100, 5000])
def test_decode_window(fmt, dtype, left):
    check_attention([1] * 5, [1, 40, 64, 200, 1000], 8, 2, 128, 16, fmt, dtype, "HND", left)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("batch,len_k", [(1, 9000), (3, 3001), (300, 33)])
def test_decode_batches(fmt, batch, len_k):
    """One long sequence over many workgroups, and more rows than workgroups."""
    lens = [max(1, len_k - 7 * i % len_k) for i in range(batch)]
    check_attention([1] * batch, lens, 4, 1, 64, 16, fmt, BF16, "HND", deterministic=True)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", F16), ("int8", BF16),
                                       ("e4m3", F16)])
@pytest.mark.parametrize("heads,kvh,d,bs,layout,left,right", [
    (8, 2, 128, 16, "HND", None, 0), (4, 4, 64, 32, "NHD", 30, 0), (5, 1, 80, 16, "HND", None, None),
    (2, 1, 256, 64, "HND", 5, 3), (17, 1, 64, 16, "HND", 200, 0)])
def test_prefill_and_mixed_steps(fmt, dtype, heads, kvh, d, bs, layout, left, right):
    check_attention([1, 30, 1, 77, 2, 1, 130], [5, 30, 300, 500, 2, 64, 399], heads, kvh, d, bs,
                    fmt, dtype, layout, left, right)
    check_attention([40, 2, 130], [40, 300, 399], heads, kvh, d, bs, fmt, dtype, layout, left,
                    right)


def test_negative_and_zero_scales_and_empty_rows():
    check_attention([1, 20, 1], [50, 60, 3], 4, 2, 64, 16, "e4m3", BF16, "HND", scale=-0.2)
    check_attention([1, 20, 1], [50, 60, 3], 4, 2, 64, 16, "int8", F16, "HND", scale=0.0)
    check_attention([1, 0, 3, 0, 1], [9, 40, 60, 0, 3], 4, 2, 64, 16, "int8", BF16, "HND")


def test_what_lies_behind_the_keys_counts_for_nothing():
    """The slots past a sequence's last key, the spare blocks and the scales of
    blocks no table names hold NaN codes and scales."""
    lens = [5, 33, 64]
    cache, tables = filled(lens, 2, 128, 16, "e4m3", BF16, "HND", 1)
    q = torch.randn(6, 4, 128, device="cuda").to(BF16)
    for lens_q in ([1, 1, 1], [2, 1, 3]):
        prep = PreparedAttention.from_batch(batch_of(lens_q, lens, tables), "cuda", cache, 4)
        n = sum(lens_q)
        want = paged_attention_prepared(q[:n], cache, 0, prep, 0.1)
        saved = [t.clone() for t in (cache._codes, cache._scales)]
        used = torch.zeros(cache.num_slots(), dtype=torch.bool)
        for t, n_k in zip(tables, lens):
            used[ref.slots_of(t, n_k, 16)] = True
        dead = (~used.view(-1, 1, 16, 1).cuda()).expand(cache.k[0].shape)
        for c in (cache.k[0], cache.v[0]):
            c.view(torch.uint8)[dead] = 0x7F
        empty = (~used.view(-1, 16).any(dim=1)).cuda()
        cache.k_scale[0][empty] = float("nan")
        cache.v_scale[0][empty] = float("inf")
        assert torch.equal(paged_attention_prepared(q[:n], cache, 0, prep, 0.1), want)
        cache._codes.copy_(saved[0])
        cache._scales.copy_(saved[1])


def test_a_step_appends_then_attends():
    """The serving sequence: prompt, then decode steps through the one call."""
    gen = torch.Generator().manual_seed(11)
    kvh, heads, d, bs = 2, 8, 128, 16
    cache = QuantKvCache(1, 20, bs, kvh, d, BF16, "e4m3")
    mk, mv = models(cache)
    tables, lens = [[3, 9, 1, 7], [4, 11, 2, 12]], [0, 0]
    for lens_q in ([20, 33], [1, 1], [1, 1], [1, 7], [1, 1]):
        slots = []
        for s, n in enumerate(lens_q):
            slots.append(ref.slots_of(tables[s], lens[s] + n, bs)[lens[s]:])
            lens[s] += n
        slots = np.concatenate(slots)
        k, v = rows(gen, len(slots), kvh, d, BF16, .5), rows(gen, len(slots), kvh, d, BF16, .5)
        q = torch.randn(len(slots), heads, d, generator=gen).to(BF16)
        prep = PreparedAttention.from_batch(batch_of(lens_q, lens, tables), "cuda", cache, heads)
        out = paged_attention_append_prepared(q.cuda(), k.cuda(), v.cuda(),
                                              scatter_index(slots, "cuda"), cache, 0, prep, 0.1)
        mk.append(k, slots)
        mv.append(v, slots)
        same(cache, 0, "k", mk)
        same(cache, 0, "v", mv)
        want, bound = ref.attention(q, ref.values(cache, 0, "k"), ref.values(cache, 0, "v"),
                                    lens_q, lens, tables, bs, 0.1)
        assert torch.all((out.cpu().double() - want).abs() <= bound)


def test_blocks_copy_spill_and_come_back():
    """copy_blocks, export/import of codes and scales, in both layouts."""
    for layout, fmt, kvh in (("HND", "e4m3", 3), ("NHD", "int8", 20)):
        cache, tables = filled([100], kvh, 64, 16, fmt, BF16, layout, 2, layers=2, spare=20)
        be = KvBlockBackend(cache)
        free = [b for b in range(cache.num_blocks) if b not in tables[0]]
        q = torch.randn(1, kvh * 2, 64, device="cuda").to(BF16)
        want = paged_attention(q, cache, 1, batch_of([1], [100], tables), 0.1)
        copy = free[:len(tables[0])]
        be.copy_blocks(list(zip(tables[0], copy)))
        assert torch.equal(paged_attention(q, cache, 1, batch_of([1], [100], [copy]), 0.1), want)
        blobs = be.export_blocks(tables[0])
        assert blobs.numel() == len(copy) * cache.block_bytes()
        back = free[len(copy):2 * len(copy)]
        be.import_blocks(back, blobs)
        assert torch.equal(paged_attention(q, cache, 1, batch_of([1], [100], [back]), 0.1), want)


def test_captured_calls_replay():
    """Append and attention in one graph, replayed with eager work between."""
    gen = torch.Generator().manual_seed(4)
    kvh, heads, d, bs, lens = 2, 8, 128, 16, [40, 300]
    cache, tables = filled([n - 1 for n in lens], kvh, d, bs, "int8", BF16, "HND", 8)
    twin, _ = filled([n - 1 for n in lens], kvh, d, bs, "int8", BF16, "HND", 8)
    slots = scatter_index([t[(n - 1) // bs] * bs + (n - 1) % bs for t, n in zip(tables, lens)],
                          "cuda")
    prep = PreparedAttention.from_batch(batch_of([1, 1], lens, tables), "cuda", cache, heads,
                                        deterministic=True)
    q, k, v = (torch.zeros(2, h, d, dtype=BF16, device="cuda") for h in (heads, kvh, kvh))
    out = torch.zeros_like(q)

    def step(c, o):
        write_rows_indexed(c, 0, k, v, slots)
        paged_attention_prepared(q, c, 0, prep, 0.1, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(twin, out)
    torch.cuda.current_stream().wait_stream(side)
    twin, _ = filled([n - 1 for n in lens], kvh, d, bs, "int8", BF16, "HND", 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, out)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen))
        k.copy_(rows(gen, 2, kvh, d, BF16) * 2.0 ** i)
        v.copy_(rows(gen, 2, kvh, d, BF16) * 2.0 ** i)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(out)
        step(twin, want)
        assert torch.equal(out, want)
        assert torch.equal(cache._codes, twin._codes) and torch.equal(cache._scales, twin._scales)


def test_another_stream_and_layer():
    cache, tables = filled([70], 2, 64, 16, "e4m3", F16, "HND", 6, layers=3)
    q = torch.randn(1, 4, 64, device="cuda").to(F16)
    want = paged_attention(q, cache, 2, batch_of([1], [70], tables), 0.1)
    assert not paged_attention(q, cache, 0, batch_of([1], [70], tables), 0.1).any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prep = PreparedAttention.from_batch(batch_of([1], [70], tables), "cuda", cache, 4)
        got = paged_attention_prepared(q, cache, 2, prep, 0.1, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """Blocks whose codes lie past 4 GiB from the layer's base."""
    kvh, d, bs = 32, 256, 256
    nb = (1 << 32) // (kvh * d * bs) + 4
    gen = torch.Generator().manual_seed(1)
    cache = QuantKvCache(1, nb, bs, kvh, d, BF16, "int8")
    table = [nb - 1, nb - 3]
    slots = ref.slots_of(table, 300, bs)
    k, v = rows(gen, 300, kvh, d, BF16, .3) / 4, rows(gen, 300, kvh, d, BF16, .3)
    write_kv_to_cache(cache, 0, k.cuda(), v.cuda(), slots)
    kk = gather_kv(cache, 0, table, 300, "k").cpu().double()
    vv = gather_kv(cache, 0, table, 300, "v").cpu().double()
    assert float((kk - k.double()).abs().max()) < float(k.abs().max()) / 64
    small = [[0, 1]]
    for lens_q in ([1], [40]):
        q = torch.randn(lens_q[0], kvh, d, generator=gen).to(BF16)
        out = paged_attention(q.cuda(), cache, 0, batch_of(lens_q, [300], [table]), 1 / 16)
        want, bound = ref.attention(q, kk, vv, lens_q, [300], small, bs, 1 / 16)
        assert torch.all((out.cpu().double() - want).abs() <= bound)


def test_bad_tables_and_small_workspaces():
    """Table entries past the pool read its last block; a workspace too small is refused."""
    cache, tables = filled([40], 2, 64, 16, "e4m3", BF16, "HND", 6)
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    for lens_q in ([1], [3]):
        batch = batch_of(lens_q, [40], [[10 ** 6, 10 ** 6, 10 ** 6]])
        assert torch.isfinite(paged_attention(q[:lens_q[0]], cache, 0, batch, 0.1)).all()
    prep = PreparedAttention.from_batch(batch_of([3], [40], tables), "cuda")
    out = torch.full_like(q, 5.0)
    need = lib().vapi_kv_q8_attention_workspace_size(cache.q8, 1, 1, 4, 3, 40)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def call(flags, size):
        return lib().vapi_kv_q8_attention(
            cache.q8, 0, q.data_ptr(), out.data_ptr(), prep.seqlens_q.data_ptr(),
            prep.seqlens_k.data_ptr(), prep.block_table.data_ptr(), 1, 3, 3, 40, 4, 0.1, -1, 0,
            flags, None, 0, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)

    assert call(0, 100) == -4 and call(0x80, need) == -1
    torch.cuda.synchronize()
    assert torch.all(out == 5.0)
    assert call(0, need) == 0
    want = paged_attention(q, cache, 0, batch_of([3], [40], tables), 0.1)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with pytest.raises(VapiKvError):
        paged_attention_prepared(q, cache, 3, prep, 0.1)


def test_prefill_rows_without_any_key_are_written():
    """max_seqlen_k 0: zeros, as with a larger bound."""
    cache, tables = filled([40], 2, 64, 16, "e4m3", BF16, "HND", 6)
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    prep = PreparedAttention.from_batch(batch_of([3], [40], tables), "cuda")
    out, none = torch.full_like(q, 5.0), torch.zeros_like(prep.seqlens_k)
    need = lib().vapi_kv_q8_attention_workspace_size(cache.q8, 1, 1, 4, 3, 0)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    assert lib().vapi_kv_q8_attention(
        cache.q8, 0, q.data_ptr(), out.data_ptr(), prep.seqlens_q.data_ptr(), none.data_ptr(),
        prep.block_table.data_ptr(), 1, 3, 3, 0, 4, 0.1, -1, 0, 0, None, 0, ws.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert not out.any()


def test_a_refused_step_writes_nothing():
    """Whatever the attention of an append-and-attend call would refuse is refused
    before the rows are written."""
    cache, tables = filled([40], 2, 64, 16, "e4m3", BF16, "HND", 6)
    codes, scales = cache._codes.clone(), cache._scales.clone()
    k = torch.randn(3, 2, 64, device="cuda").to(BF16)
    slots = scatter_index(ref.slots_of(tables[0], 40, 16)[37:], "cuda")
    flat = torch.randn(3 * 4 * 64 + 8, device="cuda").to(BF16)
    q = flat[:3 * 4 * 64].view(3, 4, 64)

    def step(q=q, out=None, lens_q=(3,), heads=4, **fields):
        prep = PreparedAttention.from_batch(batch_of(lens_q, [40], tables), "cuda")
        for name, value in fields.items():
            setattr(prep, name, value)
        return paged_attention_append_prepared(q, k, k, slots, cache, 0, prep, 0.1, out=out)

    odd = flat[4:4 + 3 * 4 * 64].view(3, 4, 64)
    calls = [dict(q=odd), dict(out=odd), dict(q=q.cpu()), dict(out=q.cpu()),
             dict(q=q[:, :3].contiguous()), dict(q=q[:, :0].contiguous()),
             dict(max_seqlen_k=1 << 29), dict(flags=0x10),
             dict(block_table=torch.zeros(1, 0, dtype=torch.int32, device="cuda"))]
    for kw in calls:
        with pytest.raises((ValueError, VapiKvError)):
            step(**kw)
        torch.cuda.synchronize()
        assert torch.equal(cache._codes, codes) and torch.equal(cache._scales, scales), kw
    step()
    torch.cuda.synchronize()
    assert not torch.equal(cache._codes, codes)


@pytest.mark.parametrize("fmt", ["none", "f32", "valu", "e4m3", "int8"])
@pytest.mark.parametrize("lens_q", [[40, 1, 130], [300]])
def test_windows_near_2_to_the_31(fmt, lens_q):
    """They hide nothing, like no window: over 16-bit and 8-bit caches, f32 ones and
    head sizes that the vector unit serves."""
    lens_k = [n + 70 for n in lens_q]
    gen = torch.Generator().manual_seed(4)
    d, dtype = (72 if fmt == "valu" else 64), (torch.float32 if fmt in ("f32", "valu") else BF16)
    if fmt in ("e4m3", "int8"):
        cache, tables = filled(lens_k, 2, d, 16, fmt, dtype, "HND", 5)
    else:
        bs = 16 if fmt != "valu" else 8
        need = [-(-n // bs) for n in lens_k]
        cache = PagedKvCache(1, sum(need), bs, 2, d, dtype, "HND", "cuda")
        ends = np.cumsum(need)
        tables = [list(range(e - n, e)) for e, n in zip(ends, need)]
        slots = np.concatenate([ref.slots_of(t, n, bs) for t, n in zip(tables, lens_k)])
        k, v = (torch.randn(len(slots), 2, d, generator=gen).to(dtype).cuda() for _ in range(2))
        write_kv_to_cache(cache, 0, k, v, slots)
    q = torch.randn(sum(lens_q), 4, d, generator=gen).to(dtype).cuda()
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda", cache, 4,
                                        deterministic=True)
    far = 2 ** 31 - 1
    for near, left, right in ((0, far, 0), (None, None, far), (None, far, far), (0, far - 60, 0),
                              (None, far, far - 60)):
        want = paged_attention_prepared(q, cache, 0, prep, 0.1, None, near)
        got = paged_attention_prepared(q, cache, 0, prep, 0.1, left, right)
        assert torch.equal(got, want), (left, right)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", BF16), ("int8", F16)])
def test_shares_change_no_more_than_f32_sums(fmt, dtype):
    """Calls whose work is split at other keys, as the shares they measure move.

    P is rounded alike wherever a range of keys begins, so two calls add the same
    products in f32 in another order: sums of n ~ 1,000 terms, off by some 2^-22 of
    sum p |v|, which is about n ** 0.5 = 30 of the output here. An output's step is
    2^-8 (bf16) or 2^-11 of it, so some 30 * 2^-14 or 2^-11 of the outputs, 0.2 and
    1.5%, land on another side of a rounding border; rounding P anew moves 45%."""
    lens = [300 + 61 * i % 3000 for i in range(64)]
    cache, tables = filled(lens, 8, 128, 16, fmt, dtype, "HND", 3)
    q = torch.randn(64, 32, 128, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    prep = PreparedAttention.from_batch(batch_of([1] * 64, lens, tables), "cuda", cache, 32)
    # (Element by element the definition's bound: a p next to a rounding border goes
    # either way with the last bit of its exponent's f32 sum, by a step of its own.)
    want, bound = ref.attention(q, ref.values(cache, 0, "k"), ref.values(cache, 0, "v"), [1] * 64,
                                lens, tables, 16, 0.05)
    first = paged_attention_prepared(q, cache, 0, prep, 0.05)
    for _ in range(12):
        again = paged_attention_prepared(q, cache, 0, prep, 0.05)
        assert float((again != first).double().mean()) < 0.05
        assert torch.all((again.cpu().double() - want).abs() <= bound)


@pytest.mark.parametrize("layout,fmt,kvh", [("HND", "e4m3", 3), ("NHD", "int8", 20)])
def test_blocks_swap_and_come_back_from_the_store(layout, fmt, kvh):
    """Codes and scales through pinned host memory and through the spill tier."""
    cache, tables = filled([100], kvh, 64, 16, fmt, BF16, layout, 2, layers=2, spare=20)
    be, table = KvBlockBackend(cache), tables[0]
    free = [b for b in range(cache.num_blocks) if b not in table]
    q = torch.randn(1, kvh * 2, 64, device="cuda").to(BF16)
    want = paged_attention(q, cache, 1, batch_of([1], [100], tables), 0.1)

    def dev(ids):
        return torch.tensor(ids, dtype=torch.int32, device="cuda")

    def same_over(ids):
        assert torch.equal(paged_attention(q, cache, 1, batch_of([1], [100], [ids]), 0.1), want)

    n = len(table)
    size, back = n * cache.block_bytes(), free[:n]
    host = torch.empty(size, dtype=torch.uint8, pin_memory=True)
    staging = torch.empty(size, dtype=torch.uint8, device="cuda")
    be.swap_out(dev(table), host, staging)
    be.swap_in(dev(back), host, staging)
    same_over(back)
    store, pinned = SpillStore(None, 1 << 24, 0), pinned_buffer(cache, 3)
    hashes = [bytes([i]) * 32 for i in range(n)]
    assert spill_evicted(store, cache, zip(hashes, table), pinned) == n
    cache._codes.fill_(0x11)  # the blocks' next users
    cache._scales.fill_(3.0)
    back = free[n:2 * n]
    assert promote(store, cache, hashes, back, pinned) == n
    torch.cuda.synchronize()
    same_over(back)
    store.close()
