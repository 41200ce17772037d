"""Running attention weights and eviction on the GPU against their definitions."""
import numpy as np
import pytest
import torch

import quant_ref as ref
from test_gpu_quant import batch_of, rows as make_rows
from vapi_amd.attention import PreparedAttention, paged_attention_prepared
from vapi_amd.cache import HybridKvCache, PagedKvCache, scatter_index, write_kv_to_cache, \
    write_rows_indexed
from vapi_amd.evict import EvictionPlan, accumulate_attention_weights, evict_kv, new_weights
from vapi_amd.quant import QuantKvCache

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def new_cache(fmt, layers, nb, bs, kvh, d, dtype, layout):
    if fmt == "none":
        return PagedKvCache(layers, nb, bs, kvh, d, dtype, layout, "cuda")
    if fmt == "block_major":
        return PagedKvCache(layers, nb, bs, kvh, d, dtype, layout, "cuda", block_major=True)
    return QuantKvCache(layers, nb, bs, kvh, d, dtype, fmt, layout)


def filled(lens_k, kvh, d, bs, fmt, dtype, layout, seed, layers=1, spare=2):
    gen = torch.Generator().manual_seed(seed)
    r = np.random.default_rng(seed)
    need = [-(-n // bs) for n in lens_k]
    perm = r.permutation(sum(need) + spare).tolist()
    tables = [[perm.pop() for _ in range(n)] for n in need]
    cache = new_cache(fmt, layers, sum(need) + spare, bs, kvh, d, dtype, layout)
    slots = np.concatenate([ref.slots_of(t, n, bs) for t, n in zip(tables, lens_k)])
    k = make_rows(gen, len(slots), kvh, d, dtype, 0.5) / 4
    v = make_rows(gen, len(slots), kvh, d, dtype, 0.5)
    write_kv_to_cache(cache, layers - 1, k.cuda(), v.cuda(), slots)
    return cache, tables, perm


def weights_ref(q, k, lens_q, lens_k, tables, bs, scale, left, right, last, decay, old, rows):
    """(state, bound) in f64. A weight is a sum of p over queries and heads: p is
    off by at most twice 2^-24 ((d + 2) reach + the largest |lse|, itself at most
    reach + log2 len_k in log2 units, + len_k for the sum of its exponentials)
    + 2^-21 of itself (scores, their offset, exp2 and log2), the sum over n of
    them by n 2^-24, decay and the last addition by two roundings."""
    hq, d, kvh = q.shape[1], q.shape[2], k.shape[1]
    q = q.cpu().double()
    out, bound, first = old.double().clone(), torch.zeros_like(old, dtype=torch.float64), 0
    for i, (lq, lk, t) in enumerate(zip(lens_q, lens_k, tables)):
        first += lq
        n = min(lq, last) if last else lq
        if n == 0:
            continue
        at = torch.from_numpy(ref.slots_of(t, lk, bs))
        add, err = torch.zeros(kvh, lk, dtype=torch.float64), torch.zeros(kvh, lk,
                                                                          dtype=torch.float64)
        for h in range(hq):
            g = h * kvh // hq
            p, reach = ref.probabilities(q[first - n:first, h], k[at, g], n, scale, left, right)
            reach = reach * 1.4427
            each = 2 * 2.0 ** -24 * ((d + 3) * reach + np.log2(max(lk, 2)) + lk) + 2.0 ** -21
            add[g] += p.sum(dim=0)
            err[g] += p.sum(dim=0) * (each + n * hq * 2.0 ** -24)
        was = out[rows[i], :, :lk] * decay if decay else 0.0
        out[rows[i], :, :lk] = was + add
        bound[rows[i], :, :lk] = err + out[rows[i], :, :lk].abs() * 2.0 ** -22
    return out, bound


def check_weights(lens_q, lens_k, heads, kvh, d, bs, fmt, dtype, layout, left=None, right=0,
                  last=0, decay=1.0, scale=None, seed=0):
    cache, tables, _ = filled(lens_k, kvh, d, bs, fmt, dtype, layout, seed + sum(lens_k))
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lens_q), heads, d, generator=gen).to(dtype)
    scale = d ** -0.5 if scale is None else scale
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda")
    n_rows = len(lens_k) + 2
    rows = np.random.default_rng(seed).permutation(n_rows)[:len(lens_k)].tolist()
    old = torch.rand(n_rows, kvh, max(lens_k) + 5, generator=gen)
    if decay == 0:
        old[rows[0], 0, 0] = float("nan")  # replaced, whatever it held
    if sum(lens_k[0:1]):
        pass
    w = old.clone().cuda()
    out = accumulate_attention_weights(q.cuda(), cache, 0, prep, scale, w, rows=rows,
                                       last_queries=last, decay=decay, window_size_left=left,
                                       window_size_right=right)
    assert out is w
    k = ref.values(cache, 0, "k")
    want, bound = weights_ref(q, k, lens_q, lens_k, tables, bs, scale, left, right, last, decay,
                              old, rows)
    got = w.cpu().double()
    if decay == 0 and lens_q[0] == 0:
        got, want = torch.nan_to_num(got), torch.nan_to_num(want)
    err = (got - want).abs()
    assert torch.all(err <= bound), f"{float((err / bound.clamp_min(1e-300)).max()):.3g} bounds"
    # The same call on the same state gives the same bits.
    again = old.clone().cuda()
    accumulate_attention_weights(q.cuda(), cache, 0, prep, scale, again, rows=rows,
                                 last_queries=last, decay=decay, window_size_left=left,
                                 window_size_right=right)
    assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(w))


POOLS = [("none", BF16), ("none", F16), ("e4m3", BF16), ("int8", F16), ("int8", BF16),
         ("block_major", BF16)]


@pytest.mark.parametrize("fmt,dtype", POOLS)
@pytest.mark.parametrize("heads,kvh,d,bs,layout", [
    (8, 2, 128, 16, "HND"), (8, 8, 64, 32, "NHD"), (7, 1, 256, 16, "HND"),
    (10, 2, 80, 16, "NHD"), (6, 3, 16, 16, "HND"), (71, 1, 64, 16, "HND"),
    (40, 1, 208, 128, "NHD")])
def test_weights_of_single_tokens(fmt, dtype, heads, kvh, d, bs, layout):
    check_weights([1] * 8, [1, 2, 15, 16, 17, 64, 129, 1100], heads, kvh, d, bs, fmt, dtype,
                  layout)


@pytest.mark.parametrize("fmt,dtype", POOLS)
@pytest.mark.parametrize("heads,kvh,d,bs,layout,left,right,last,decay", [
    (8, 2, 128, 16, "HND", None, 0, 0, 1.0), (4, 4, 64, 32, "NHD", 30, 0, 0, 0.5),
    (5, 1, 80, 16, "HND", None, None, 7, 0.0), (2, 1, 256, 64, "HND", 5, 3, 0, 0.0),
    (17, 1, 64, 16, "HND", 200, 0, 32, 0.9), (4, 1, 128, 16, "HND", 0, 0, 0, 1.0)])
def test_weights_of_prompts_and_mixed_steps(fmt, dtype, heads, kvh, d, bs, layout, left, right,
                                            last, decay):
    check_weights([1, 30, 0, 77, 2, 1, 130], [5, 30, 300, 500, 2, 64, 399], heads, kvh, d, bs,
                  fmt, dtype, layout, left, right, last, decay)


@pytest.mark.parametrize("fmt,dtype", [("none", BF16), ("e4m3", F16)])
def test_weights_of_long_prompts(fmt, dtype):
    """More rows than a workgroup joins, and many chunks of keys."""
    check_weights([700, 1500], [700, 1600], 4, 2, 64, 16, fmt, dtype, "HND")
    check_weights([300], [5000], 4, 1, 128, 16, fmt, dtype, "HND", last=64, decay=0.0)
    check_weights([1], [20000], 4, 1, 64, 16, fmt, dtype, "HND")


@pytest.mark.parametrize("fmt,dtype,heads,kvh,d", [
    ("none", BF16, 4, 1, 128), ("int8", F16, 3, 1, 64), ("e4m3", BF16, 12, 4, 256)])
@pytest.mark.parametrize("left,right", [
    (0, 0), (50, 0), (333, 0), (50, 5), (None, 100), (20, None), (0, None), (1 << 30, 1 << 30),
    (2 ** 31 - 1, 2 ** 31 - 1)])
def test_weights_of_long_prompts_in_windows(fmt, dtype, heads, kvh, d, left, right):
    """Workgroups and waves whose keys no row, some rows or all rows see."""
    check_weights([700, 1, 90, 333], [900, 600, 1000, 333], heads, kvh, d, 16, fmt, dtype, "HND",
                  left, right, seed=2)


def test_weights_with_odd_scales_and_wide_batches():
    check_weights([1, 20], [50, 60], 4, 2, 64, 16, "none", BF16, "HND", scale=-0.2)
    check_weights([1, 20], [50, 60], 4, 2, 64, 16, "int8", F16, "HND", scale=0.0)
    check_weights([1] * 200, [1 + i % 70 for i in range(200)], 4, 2, 64, 16, "none", F16, "HND")


def test_weights_sum_to_the_queries():
    """Each query and head spreads a weight of one over the keys it sees."""
    cache, tables, _ = filled([300, 40], 2, 128, 16, "e4m3", BF16, "HND", 3)
    prep = PreparedAttention.from_batch(batch_of([50, 1], [300, 40], tables), "cuda")
    w = new_weights(2, 2, 300)
    q = torch.randn(51, 8, 128, device="cuda").to(BF16)
    for i in range(1, 4):
        accumulate_attention_weights(q, cache, 0, prep, 0.1, w)
        total = w.sum(dim=2).cpu()
        assert torch.allclose(total, torch.tensor([[200.0 * i] * 2, [4.0 * i] * 2]), rtol=1e-5)
    assert not w[1, :, 40:].any()


def test_nan_behind_the_mask_counts_for_nothing():
    """K past the last key and outside the window holds NaN and infinities."""
    cache, tables, _ = filled([70, 33], 1, 64, 16, "none", BF16, "HND", 4)
    q = torch.randn(6, 2, 64, device="cuda").to(BF16)
    prep = PreparedAttention.from_batch(batch_of([5, 1], [70, 33], tables), "cuda")

    def call():
        w = new_weights(2, 1, 80)
        return accumulate_attention_weights(q, cache, 0, prep, 0.1, w, window_size_left=20)

    want = call()
    used = torch.zeros(cache.num_slots(), dtype=torch.bool)
    for t, n, first in zip(tables, (70, 33), (65 - 20, 32 - 20)):
        used[ref.slots_of(t, n, 16)[first:]] = True
    dead = (~used).view(-1, 1, 16, 1).cuda().expand(cache.k[0].shape)
    cache.k[0][dead] = float("nan")
    assert torch.equal(call(), want)
    cache.k[0][dead] = float("inf")
    assert torch.equal(call(), want)


@pytest.mark.parametrize("fmt,dtype", [("none", BF16), ("none", F16), ("e4m3", BF16)])
@pytest.mark.parametrize("lens_q,heads,left,bad", [
    (400, 3, 20, (212, 213, 300)), (400, 4, 50, (243, 399)), (4, 4, None, (1, 2)),
    (5, 3, 7, (0, 4)), (1, 16, 30, (0,))])
def test_a_nan_query_reaches_only_the_keys_it_sees(fmt, dtype, lens_q, heads, left, bad):
    n = 400
    cache, tables, _ = filled([n], 1, 64, 16, fmt, dtype, "HND", 8)
    q = torch.randn(lens_q, heads, 64, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    prep = PreparedAttention.from_batch(batch_of([lens_q], [n], tables), "cuda")

    def call():
        return accumulate_attention_weights(q, cache, 0, prep, 0.1, new_weights(1, 1, n),
                                            window_size_left=left)[0, 0].cpu()

    want = call()
    for j in bad:
        q[j, 0] = float("nan")
        got, pos = call(), n - lens_q + j
        seen = torch.zeros(n, dtype=torch.bool)
        seen[0 if left is None else max(pos - left, 0):pos + 1] = True
        assert torch.equal(got[~seen], want[~seen])
        q[j, 0] = 1.0
        want = call()


def test_a_query_made_contiguous_waits_for_the_call_s_stream_alone():
    """A strided query or row is copied on the stream that the call is given."""
    cache, tables, _ = filled([200], 2, 64, 16, "e4m3", BF16, "HND", 5)
    prep = PreparedAttention.from_batch(batch_of([40], [200], tables), "cuda", cache, 4)
    wide = torch.randn(40, 4, 128, device="cuda").to(BF16)
    q, k = wide[:, :, ::2], wide[:, ::2, ::2]
    idx = scatter_index(ref.slots_of(tables[0], 200, 16)[160:], "cuda")

    def step(w, stream=None):
        write_rows_indexed(cache, 0, k, k, idx, stream=stream)
        out = paged_attention_prepared(q, cache, 0, prep, 0.1, stream=stream)
        accumulate_attention_weights(q, cache, 0, prep, 0.1, w, stream=stream)
        return out

    w = new_weights(1, 2, 200)
    step(new_weights(1, 2, 200))
    want = new_weights(1, 2, 200)
    first = step(want)
    junk = [torch.full((40, 4, 64), float("nan"), device="cuda", dtype=BF16) for _ in range(8)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    del junk
    torch.cuda._sleep(20_000_000)  # the current stream is behind, and not waited for
    out = step(w, side)
    side.synchronize()
    assert torch.equal(w, want) and torch.equal(out, first)


def test_rows_past_the_state_are_left_out_and_strided_states():
    cache, tables, _ = filled([30, 40], 2, 64, 16, "none", F16, "HND", 5)
    prep = PreparedAttention.from_batch(batch_of([1, 1], [30, 40], tables), "cuda")
    q = torch.randn(2, 4, 64, device="cuda").to(F16)
    want = accumulate_attention_weights(q, cache, 0, prep, 0.1, new_weights(2, 2, 40))
    big = torch.zeros(3, 4, 2, 50, device="cuda")
    view = big[:, 1]  # one layer's rows of a state that holds four
    bad = torch.tensor([2, 7], dtype=torch.int32, device="cuda")
    accumulate_attention_weights(q, cache, 0, prep, 0.1, view, rows=bad)
    assert torch.equal(view[2, :, :40], want[0])
    big[2, 1] = 0
    assert not big.any()


# ---- eviction ---------------------------------------------------------------------


def kept_ref(w, n, budget, sinks, recent):
    new = min(n, budget)
    held = [i for i in range(n) if i < sinks or i >= n - recent]
    rest = [i for i in range(n) if sinks <= i < n - recent]
    rank = [-np.inf if np.isnan(x) else x for x in w.tolist()]
    rest.sort(key=lambda i: (-rank[i], np.isnan(w[i]), i))
    return sorted((held + rest)[:new])


def check_evict(lens, kvh, d, bs, fmt, dtype, layout, budget, sinks, recent, weights,
                in_place=False, layers=1, hybrid=False):
    spare = sum(-(-min(n, budget) // bs) for n in lens) + 3
    cache, tables, free = filled(lens, kvh, d, bs, fmt, dtype, layout, sum(lens) + budget, layers,
                                 spare)
    layer = layers - 1
    dst = [[free.pop() for _ in range(-(-min(n, budget) // bs))] for n in lens]
    n_rows = len(lens) + 2
    rows = np.random.default_rng(1).permutation(n_rows)[:len(lens)].tolist()
    w = weights(n_rows, kvh, max(lens) + 3)
    state = w.cuda()
    kb, vb = ref.values(cache, layer, "k"), ref.values(cache, layer, "v")
    before = [t.clone() for t in ((cache._codes, cache._scales) if hasattr(cache, "q8")
                                  else (cache.k[layer], cache.v[layer]))]
    plan = EvictionPlan.from_tables(lens, tables, dst, budget, sinks, recent, bs, "cuda", rows)
    out = state if in_place else torch.full_like(state, 9.0)
    kept = evict_kv(cache, layer, state, plan, weights_out=out)
    if not in_place:
        assert torch.equal(torch.nan_to_num(state.cpu(), 5e5), torch.nan_to_num(w, 5e5))
    got_k, got_v = ref.values(cache, layer, "k"), ref.values(cache, layer, "v")
    out, kept = out.cpu(), kept.cpu()
    assert kept.shape == (len(lens), kvh, max(min(n, budget) for n in lens))
    touched = torch.zeros(cache.num_blocks, dtype=torch.bool)
    for i, n in enumerate(lens):
        new = min(n, budget)
        touched[dst[i]] = True
        to = torch.from_numpy(ref.slots_of(dst[i], new, bs))
        src_slots = ref.slots_of(tables[i], n, bs)
        for h in range(kvh):
            want = kept_ref(w[rows[i], h, :n].numpy(), n, budget, sinks, recent)
            assert kept[i, h, :new].tolist() == want
            assert torch.all(kept[i, h, new:] == -1)
            assert torch.equal(torch.nan_to_num(out[rows[i], h, :new], 5e5),
                               torch.nan_to_num(w[rows[i], h, want], 5e5))
            assert not out[rows[i], h, new:].any()
            src = torch.from_numpy(src_slots[want])
            for got, was in ((got_k, kb), (got_v, vb)):
                rows_of = was[src, h]
                if fmt not in ("e4m3", "int8"):
                    assert torch.equal(got[to, h], rows_of)
                    continue
                for b0 in range(0, new, bs):
                    block = rows_of[b0:b0 + bs].numpy()
                    s = ref.scale_of(float(np.abs(block).max()), fmt, dtype)
                    exact = ref.to_codes(block / s, fmt) * s if s else block * 0
                    assert torch.equal(got[to[b0:b0 + bs], h], torch.from_numpy(exact))
    if not in_place:
        other = [r for r in range(n_rows) if r not in rows]
        assert torch.all(out[other] == 9.0)
    # Blocks that are not new ones are as they were.
    after = (cache._codes, cache._scales) if hasattr(cache, "q8") else (cache.k[layer],
                                                                       cache.v[layer])
    if hasattr(cache, "q8"):
        for a, b in zip((cache.k[layer], cache.v[layer]),
                        (before[0][0, layer], before[0][1, layer])):
            size = a[0].numel()
            b = b[:cache.num_blocks * size].view(cache.num_blocks, size)
            a = a.view(torch.uint8).reshape(cache.num_blocks, size)
            assert torch.equal(a[~touched.cuda()], b[~touched.cuda()])
    else:
        for a, b in zip(after, before):
            assert torch.equal(a[~touched.cuda()], b[~touched.cuda()])


def plain_weights(n_rows, kvh, width):
    return torch.rand(n_rows, kvh, width, generator=torch.Generator().manual_seed(width))


def tied_weights(n_rows, kvh, width):
    w = plain_weights(n_rows, kvh, width)
    return (w * 4).round() / 4 * (w > 0.3)


@pytest.mark.parametrize("fmt,dtype", POOLS + [("none", F32)])
@pytest.mark.parametrize("kvh,d,bs,layout,budget,sinks,recent", [
    (2, 128, 16, "HND", 64, 4, 16), (1, 64, 32, "NHD", 33, 0, 0), (3, 80, 16, "HND", 100, 7, 93),
    (2, 256, 64, "HND", 1, 0, 1), (1, 16, 128, "NHD", 200, 1, 100), (5, 96, 16, "NHD", 17, 1, 0)])
def test_evict(fmt, dtype, kvh, d, bs, layout, budget, sinks, recent):
    if dtype == F32 and layout == "NHD":
        bs = 16
    check_evict([1, 16, 17, 64, 100, 101, 1500], kvh, d, bs, fmt, dtype, layout, budget, sinks,
                recent, plain_weights)


@pytest.mark.parametrize("fmt", ["none", "e4m3", "int8"])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_ties_and_whole_sequences(fmt, in_place):
    check_evict([5, 700, 1025, 3000], 2, 64, 16, fmt, BF16, "HND", 300, 4, 20, tied_weights,
                in_place)
    check_evict([5, 700], 2, 64, 16, fmt, BF16, "HND", 700, 4, 20, tied_weights, in_place, 2)
    check_evict([2500, 40], 1, 64, 16, fmt, BF16, "HND", 1100, 0, 0,
                lambda r, h, w: torch.zeros(r, h, w), in_place)


def test_evict_by_strange_weights():
    """NaN, infinities, negative numbers, both zeros and subnormal ones."""
    def strange(n_rows, kvh, width):
        w = plain_weights(n_rows, kvh, width) - 0.5
        pick = torch.arange(width)
        w[..., pick % 7 == 1] = float("nan")
        w[..., pick % 11 == 2] = float("inf")
        w[..., pick % 13 == 3] = -float("inf")
        w[..., pick % 5 == 4] = 0.0
        w[..., pick % 10 == 9] = -0.0
        w[..., pick % 17 == 5] = 1e-42
        return w

    for budget in (20, 60, 90, 130, 180, 195, 200):
        check_evict([200, 150], 2, 64, 16, "none", BF16, "HND", budget, 2, 5, strange)


def test_evict_other_row_sizes_and_pools():
    """Rows of 2, 4 and 8-byte pieces, odd block sizes, layers that differ."""
    for d, bs, dtype in ((3, 5, F16), (6, 7, BF16), (20, 24, F16), (1, 1, F32)):
        check_evict([30, 90], 2, d, bs, "none", dtype, "HND", 32, 2, 8, plain_weights, layers=3)
    cache = HybridKvCache([("rows", 64), ("kv", 2, 64)], 12, 16, BF16)
    k = torch.randn(100, 2, 64).to(BF16)
    write_kv_to_cache(cache, 1, k.cuda(), k.cuda(), np.arange(100))
    plan = EvictionPlan.from_tables([100], [list(range(7))], [[8, 9]], 32, 0, 32, 16, "cuda")
    kept = evict_kv(cache, 1, new_weights(1, 2, 100), plan)
    assert kept[0, 0].tolist() == list(range(68, 100))
    assert torch.equal(ref_rows(cache, 1)[8 * 16:10 * 16], k[68:])
    with pytest.raises(ValueError):
        evict_kv(cache, 0, new_weights(1, 1, 100), plan)


def ref_rows(cache, layer):
    x = cache.reference_view(layer, "k").cpu()
    return x.reshape(-1, *x.shape[2:])


@pytest.mark.parametrize("fmt", ["none", "int8"])
def test_prompt_eviction_and_generation(fmt):
    """As used: a prompt's weights from its last queries, an eviction, then
    decode steps that append, attend and go on accumulating over the new blocks."""
    gen = torch.Generator().manual_seed(7)
    kvh, heads, d, bs, layers, lens = 2, 8, 64, 16, 2, [200, 330]
    cache, tables, free = filled(lens, kvh, d, bs, fmt, BF16, "HND", 9, layers, spare=30)
    first = cache.k[0].clone()
    state = torch.zeros(layers, 2, kvh, 512, device="cuda")
    q = torch.randn(sum(lens), heads, d, generator=gen).to(BF16).cuda()
    prep = PreparedAttention.from_batch(batch_of(lens, lens, tables), "cuda")
    accumulate_attention_weights(q, cache, 1, prep, 0.125, state[1], last_queries=16, decay=0.0)
    new = [[free.pop() for _ in range(6)] for _ in lens]
    plan = EvictionPlan.from_tables(lens, tables, new, 80, 4, 16, bs, "cuda")
    kept = evict_kv(cache, 1, state[1], plan, weights_out=state[1])
    assert torch.equal(cache.k[0].view(torch.uint8), first.view(torch.uint8))
    lens, total = [80, 80], state[1].sum(dim=2).cpu()
    for _ in range(3):
        lens = [n + 1 for n in lens]
        slots = [t[(n - 1) // bs] * bs + (n - 1) % bs for t, n in zip(new, lens)]
        k, v = (make_rows(gen, 2, kvh, d, BF16, .3).cuda() for _ in range(2))
        write_rows_indexed(cache, 1, k, v, scatter_index(slots, "cuda"))
        q = torch.randn(2, heads, d, generator=gen).to(BF16)
        prep = PreparedAttention.from_batch(batch_of([1, 1], lens, new), "cuda", cache, heads)
        out = paged_attention_prepared(q.cuda(), cache, 1, prep, 0.125)
        accumulate_attention_weights(q.cuda(), cache, 1, prep, 0.125, state[1])
        want, bound = ref.attention(q, ref.values(cache, 1, "k"), ref.values(cache, 1, "v"),
                                    [1, 1], lens, new, bs, 0.125)
        assert torch.all((out.cpu().double() - want).abs() <= bound)
        now = state[1].sum(dim=2).cpu()
        assert torch.allclose(now, total + 4, rtol=1e-5)
        total = now
    assert not state[0].any() and kept.shape == (2, kvh, 80)


def test_another_stream():
    """Everything made for a call on a side stream outlives it: host rows, a query
    that has to be made contiguous, outputs dropped at once."""
    cache, tables, free = filled([300, 90], 2, 64, 16, "int8", BF16, "HND", 3, spare=20)
    dst = [[free.pop() for _ in range(4)] for _ in range(2)]
    plan = EvictionPlan.from_tables([300, 90], tables, dst, 60, 4, 10, 16, "cuda", [3, 1])
    prep = PreparedAttention.from_batch(batch_of([20, 1], [300, 90], tables), "cuda")
    wide = torch.randn(21, 4, 128, device="cuda").to(BF16)
    q = wide[:, :, ::2]
    want = accumulate_attention_weights(q, cache, 0, prep, 0.1, new_weights(4, 2, 300),
                                        rows=[3, 1])
    kept = evict_kv(cache, 0, want, plan)
    codes = cache._codes.clone()
    side = torch.cuda.Stream()
    w = new_weights(4, 2, 300)
    torch.cuda.synchronize()
    torch.cuda._sleep(10_000_000)  # the current stream is behind
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        accumulate_attention_weights(q, cache, 0, prep, 0.1, w, rows=[3, 1], decay=0.0,
                                     stream=side)
        got = evict_kv(cache, 0, w, plan, stream=side)
        junk = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (2, 21 * 256, 240)]
        del junk
    side.synchronize()
    assert torch.equal(w, want) and torch.equal(got, kept) and torch.equal(cache._codes, codes)


def test_states_of_two_sizes_share_a_step():
    """A call that needs a larger workspace leaves a captured one's alone."""
    cache, tables, _ = filled([300], 2, 64, 16, "none", BF16, "HND", 3)
    prep = PreparedAttention.from_batch(batch_of([200], [300], tables), "cuda")
    q = torch.randn(200, 4, 64, device="cuda").to(BF16)
    w, big = new_weights(1, 2, 300), new_weights(1, 2, 300)
    accumulate_attention_weights(q, cache, 0, prep, 0.1, w, last_queries=3, decay=0.0)
    want = w.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accumulate_attention_weights(q, cache, 0, prep, 0.1, w, last_queries=3, decay=0.0)
    accumulate_attention_weights(q, cache, 0, prep, 0.1, big)
    for _ in range(3):
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want)


def test_captured_weights_and_eviction_replay():
    cache, tables, free = filled([300, 90], 2, 64, 16, "e4m3", BF16, "HND", 3, spare=20)
    dst = [[free.pop() for _ in range(4)] for _ in range(2)]
    plan = EvictionPlan.from_tables([300, 90], tables, dst, 60, 4, 10, 16, "cuda")
    prep = PreparedAttention.from_batch(batch_of([20, 1], [300, 90], tables), "cuda")
    q = torch.randn(21, 4, 64, device="cuda").to(BF16)
    w, out = new_weights(2, 2, 300), new_weights(2, 2, 300)

    def step():
        accumulate_attention_weights(q, cache, 0, prep, 0.1, w)
        return evict_kv(cache, 0, w, plan, weights_out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    w.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for _ in range(4):
        q.copy_(torch.randn(q.shape))
        before = w.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (w, out, kept, cache._codes, cache._scales)]
        w.copy_(before)
        k2 = step()
        assert all(torch.equal(a, b) for a, b in zip(got, (w, out, k2, cache._codes,
                                                           cache._scales)))


@pytest.mark.parametrize("fmt,dtype", [("none", BF16), ("e4m3", F16)])
@pytest.mark.parametrize("left,max_k", [(None, 1 << 20), (None, 1 << 22), (300, 1 << 22)])
def test_weights_of_more_rows_than_a_workgroup_holds(fmt, dtype, left, max_k):
    """A bound on the keys that leaves room for few parts of the rows, or for one:
    each walks 512 rows at a time."""
    lens_q, lens_k, heads, kvh, d = [1300, 900], [1300, 1100], 4, 2, 64
    cache, tables, _ = filled(lens_k, kvh, d, 16, fmt, dtype, "HND", 12)
    q = torch.randn(sum(lens_q), heads, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda")
    prep.max_seqlen_k = max_k
    w = torch.zeros(2, kvh, max_k, device="cuda")
    accumulate_attention_weights(q.cuda(), cache, 0, prep, 0.125, w, window_size_left=left)
    n = max(lens_k) + 3
    assert not w[:, :, n:].any()
    old = torch.zeros(2, kvh, n)
    want, bound = weights_ref(q, ref.values(cache, 0, "k"), lens_q, lens_k, tables, 16, 0.125,
                              left, 0, 0, 1.0, old, [0, 1])
    err = (w[:, :, :n].cpu().double() - want).abs()
    assert torch.all(err <= bound), f"{float((err / bound.clamp_min(1e-300)).max()):.3g} bounds"


@pytest.mark.parametrize("fmt", ["none", "int8"])
@pytest.mark.parametrize("lens", [[0, 0], [0, 40]])
def test_sequences_without_keys_leave_zeros(fmt, lens):
    """The rows of a state that an eviction writes are zeros from a sequence's kept
    keys on, also where no sequence of the batch has any."""
    cache, tables, free = filled([40], 2, 64, 16, fmt, BF16, "HND", 3, spare=8)
    before = cache.k[0].clone()
    w = torch.rand(4, 2, 50, device="cuda")
    rows, held = [2, 0], w.clone()
    dst = [[], [free.pop(), free.pop()] if lens[1] else []]
    plan = EvictionPlan.from_tables(lens, [[], tables[0] if lens[1] else []], dst, 20, 2, 4, 16,
                                    "cuda", rows)
    out = torch.full_like(w, 9.0)
    for target in (out, w):
        kept = evict_kv(cache, 0, w, plan, weights_out=target)
        assert kept.shape == (2, 2, min(max(lens), 20)) and torch.all(kept[0] == -1)
        assert not target[2].any() and not target[0, :, min(lens[1], 20):].any()
    assert torch.all(out[[1, 3]] == 9.0) and torch.equal(w[[1, 3]], held[[1, 3]])
    assert evict_kv(cache, 0, held, plan).shape == kept.shape
    assert lens[1] or torch.equal(cache.k[0].view(torch.uint8), before.view(torch.uint8))


def tied_across(n_rows, kvh, width):
    """Few distinct weights, so the last kept ones are ties spread over the row."""
    return (plain_weights(n_rows, kvh, width) * 3).floor() / 4


@pytest.mark.parametrize("weights", [plain_weights, tied_across])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens", [[4097, 7], [12288, 300], [12289, 4096, 0], [30011, 12290, 100]])
def test_evict_long_sequences(lens, in_place, weights):
    """Past the keys that 256 threads take, and past those held in LDS at once, where
    a row is walked in tiles and what it keeps is written while later ones are read."""
    check_evict(lens, 1, 16, 16, "none", BF16, "HND", 2000, 4, 100, weights, in_place)
    check_evict(lens, 1, 16, 16, "none", BF16, "HND", lens[0] * 2 // 3, 0, 0, weights, in_place)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_evict_long_8_bit_sequences(fmt):
    check_evict([12289, 4100], 2, 32, 32, fmt, BF16, "NHD", 900, 4, 64, tied_across, True)
    check_evict([12289 + 4096], 1, 16, 16, fmt, F16, "HND", 13000, 4, 64, plain_weights)


def test_evict_long_sequences_of_one_weight():
    """Every key ties with every other, over three tiles."""
    check_evict([26000], 1, 16, 16, "none", F16, "HND", 13000, 10, 300,
                lambda r, h, w: torch.full((r, h, w), 0.5), True)


@pytest.mark.parametrize("lens_q", [[0, 3, 1], [2, 0, 40]])
def test_decay_0_replaces_nan_and_nothing_else(lens_q):
    """NaN in the rows of sequences with queries goes; other rows, and columns past a
    sequence's keys, keep theirs."""
    lens_k = [50, 64, 90]
    cache, tables, _ = filled(lens_k, 2, 64, 16, "none", BF16, "HND", 7)
    q = torch.randn(sum(lens_q), 4, 64, generator=torch.Generator().manual_seed(2)).to(BF16)
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda")
    old = torch.rand(5, 2, 100)
    old[:, :, ::7] = float("nan")
    rows = [4, 0, 2]
    w = old.cuda()
    accumulate_attention_weights(q.cuda(), cache, 0, prep, 0.125, w, rows=rows, decay=0.0)
    fresh = torch.zeros(5, 2, 100)
    want, bound = weights_ref(q, ref.values(cache, 0, "k"), lens_q, lens_k, tables, 16, 0.125,
                              None, 0, 0, 0.0, fresh, rows)
    written = torch.zeros(5, 2, 100, dtype=torch.bool)
    for r, lq, lk in zip(rows, lens_q, lens_k):
        written[r, :, :lk] = lq > 0
    got = w.cpu()
    assert torch.equal(got.isnan(), old.isnan() & ~written)
    assert torch.equal(torch.nan_to_num(got[~written], 5.0), torch.nan_to_num(old[~written], 5.0))
    assert torch.all((got.double() - want).abs()[written] <= bound[written])
