"""Attention with sinks behind a left window on the GPU, against the definition in
64 bits.

Tolerances. An output is a weighted mean of V with weights p_i / sum p. In a 16-bit
pool each p is rounded to the type (relative u: bf16 2^-8, f16 2^-11, half a step)
before it meets V and the sum stays f32, so the mean moves by at most u times the
mean of |v|; the output is rounded once more, by at most u of itself. Scores carry
f32 sums of d products: off by less than 2^-14 for these inputs, which moves weights
by as much of themselves. Together: 2 u max|v| over the visible keys, and 2^-13 of it
for the scores; f32 pools have u = 2^-24 and sums of up to 2^13 terms instead: 1e-5 of
max|v| as every f32 attention test here.
"""
import numpy as np
import pytest
import torch

from vapi_amd._lib import VapiKvError
from vapi_amd.attention import (ForwardBatch, PreparedAttention, paged_attention,
                                paged_attention_append_prepared, paged_attention_prepared)
from vapi_amd.cache import HybridKvCache, PagedKvCache, scatter_index
from vapi_amd.quant import QuantKvCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def make(lens_q, lens_k, heads, kvh, d, dtype, bs=16, layout="HND", fmt="none", seed=0):
    """A cache of random rows and a step over it."""
    gen = torch.Generator().manual_seed(seed + sum(lens_k) + heads * d)
    r = np.random.default_rng(seed + d)
    need = [max(-(-n // bs), 1) for n in lens_k]
    nb = sum(need) + 2
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
            c.copy_((x * 100).clamp(-127, 127).to(c.dtype))  # (past 448 e4m3 has NaN only)
            s.copy_(torch.exp2(torch.randint(-8, -5, s.shape, generator=gen).float()))
    perm = r.permutation(nb)
    ends = np.cumsum(need)
    tables = [perm[e - n:e].tolist() for e, n in zip(ends, need)]
    batch = ForwardBatch(cu_seqlens_q=np.concatenate([[0], np.cumsum(lens_q)]).tolist(),
                         cu_seqlens_k=np.concatenate([[0], np.cumsum(lens_k)]).tolist(),
                         block_tables=tables, max_seqlen_q=max(lens_q), max_seqlen_k=max(lens_k))
    q = torch.randn(sum(lens_q), heads, d, generator=gen).to(dtype).to(DEV)
    return cache, q, batch


def values(cache, which):
    """[block, token, head, d] in f64."""
    if isinstance(cache, QuantKvCache):
        return cache.values(0, which).cpu().double()
    return cache.reference_view(0, which).cpu().double()


def reference(q, cache, batch, scale, left, right, sinks):
    k, v = values(cache, "k"), values(cache, "v")
    bs, kvh = cache.block_size, cache.num_kv_heads
    qd = q.cpu().double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    top = torch.zeros(q.shape[:2], dtype=torch.float64)  # max|v| of the visible keys
    cq, ck = batch.cu_seqlens_q, batch.cu_seqlens_k
    for i, table in enumerate(batch.block_tables):
        lq, lk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
        if not lq:
            continue
        key = np.arange(lk)
        at = (torch.from_numpy(np.array(table)[key // bs]), torch.from_numpy(key % bs))
        p = np.arange(lk - lq, lk)[:, None]
        seen = np.ones((lq, lk), bool)
        if right is not None:
            seen &= key[None] <= p + right
        if left is not None:
            seen &= (key[None] >= p - left) | (key[None] < sinks)
        seen = torch.from_numpy(seen)
        for h in range(q.shape[1]):
            kk, vv = k[at][:, h * kvh // q.shape[1]], v[at][:, h * kvh // q.shape[1]]
            kk, vv = torch.nan_to_num(kk, 0, 0, 0), vv
            s = torch.where(seen, qd[cq[i]:cq[i + 1], h] @ kk.T * scale, -np.inf)
            w = torch.softmax(s, dim=1)
            any_seen = seen.any(dim=0)
            vv = torch.where(any_seen[:, None], vv, 0.0)
            out[cq[i]:cq[i + 1], h] = torch.nan_to_num(w) @ vv
            top[cq[i]:cq[i + 1], h] = vv.abs().max()
    return out, top


def assert_close(got, want, dtype):
    out, top = want
    err = (got.cpu().double() - out).abs().amax(dim=-1)
    tol = top * (1e-5 if dtype == F32 else 2 * HALF_STEP[dtype] + 2.0 ** -13)
    assert torch.isfinite(got).all()
    worst = (err / tol).max()
    assert worst <= 1, f"{float(worst)} of the tolerance"


def check(lens_q, lens_k, heads, kvh, d, dtype, left, sinks, right=0, scale=None, det=False, **kw):
    cache, q, batch = make(lens_q, lens_k, heads, kvh, d, dtype, **kw)
    scale = d ** -0.5 if scale is None else scale
    prep = PreparedAttention.from_batch(batch, DEV, cache, heads, deterministic=det)
    got = paged_attention_prepared(q, cache, 0, prep, scale, left, right, sinks=sinks)
    assert_close(got, reference(q, cache, batch, scale, left, right, sinks), dtype)
    return got


# Windows that start at every phase of a step, sinks that end before, in and past it.
LENS = [1, 2, 31, 33, 64, 100, 133, 150, 161, 190, 700, 1500]


@pytest.mark.parametrize("left,sinks", [(0, 1), (20, 4), (64, 16), (63, 33), (95, 64), (40, 65),
                                        (99, 200), (31, 5000), (2000, 4)])
@pytest.mark.parametrize("dtype,fmt,heads,kvh,d", [
    (BF16, "none", 8, 2, 128), (F16, "none", 4, 4, 64), (BF16, "none", 6, 2, 256),
    (F16, "none", 3, 1, 96), (F32, "none", 4, 2, 128), (F32, "none", 4, 1, 64),
    (BF16, "e4m3", 8, 2, 128), (F16, "int8", 3, 3, 80)])
def test_single_tokens(left, sinks, dtype, fmt, heads, kvh, d):
    check([1] * len(LENS), LENS, heads, kvh, d, dtype, left, sinks, fmt=fmt)


@pytest.mark.parametrize("dtype,fmt,d", [(BF16, "none", 128), (F16, "none", 64), (F32, "none", 128),
                                         (BF16, "none", 256), (F32, "none", 80), (F16, "none", 40),
                                         (BF16, "e4m3", 128), (BF16, "int8", 64)])
def test_a_full_batch_of_single_tokens(dtype, fmt, d):
    """The stream: more rows than the short-context kernel takes."""
    r = np.random.default_rng(d)
    lens = np.clip(np.exp(r.normal(np.log(900), 1.0, 70)), 1, 6000).astype(int).tolist()
    got = check([1] * 70, lens, 16, 4, d, dtype, 300, 37, fmt=fmt, layout="NHD", bs=32)
    again = check([1] * 70, lens, 16, 4, d, dtype, 300, 37, fmt=fmt, layout="NHD", bs=32, det=True)
    assert got.shape == again.shape


@pytest.mark.parametrize("dtype,fmt,heads,kvh,d", [
    (F16, "int8", 16, 16, 96), (BF16, "e4m3", 12, 6, 96), (BF16, "int8", 15, 15, 80),
    (F16, "e4m3", 8, 8, 48), (BF16, "e4m3", 4, 4, 160), (F16, "int8", 34, 2, 96),
    (BF16, "none", 8, 8, 80), (F16, "none", 12, 6, 96), (F32, "none", 9, 3, 80),
    (F32, "none", 8, 8, 16), (BF16, "none", 4, 4, 200), (F16, "none", 40, 2, 72)])
def test_rows_that_share_cache_lines(dtype, fmt, heads, kvh, d):
    """Token-major rows that are no whole lines: 1, 2, 3, 4 or 8 heads to a walk."""
    r = np.random.default_rng(d + heads)
    lens = r.integers(1, 700, 136).tolist() + [1, 2, 3, 900]
    got = check([1] * 140, lens, heads, kvh, d, dtype, 250, 20, fmt=fmt, layout="NHD", det=True)
    again = check([1] * 140, lens, heads, kvh, d, dtype, 250, 20, fmt=fmt, layout="NHD", det=True)
    assert torch.equal(got, again)


@pytest.mark.parametrize("left,sinks", [(0, 1), (20, 4), (63, 33), (64, 70), (300, 5), (31, 900)])
@pytest.mark.parametrize("dtype,fmt,heads,kvh,d", [
    (BF16, "none", 8, 2, 128), (F16, "none", 4, 4, 64), (BF16, "none", 2, 1, 256),
    (F16, "none", 6, 2, 96), (F32, "none", 4, 2, 128), (F32, "none", 4, 4, 64),
    (F32, "none", 8, 1, 112), (F16, "e4m3", 4, 1, 128)])
def test_prompts_and_chunks(left, sinks, dtype, fmt, heads, kvh, d):
    check([300, 77, 2, 500, 33], [300, 400, 90, 1200, 33], heads, kvh, d, dtype, left, sinks,
          fmt=fmt)


@pytest.mark.parametrize("dtype,fmt,d", [(BF16, "none", 128), (F16, "none", 64), (BF16, "none", 96),
                                         (BF16, "none", 256), (F32, "none", 128),
                                         (F16, "int8", 128)])
@pytest.mark.parametrize("block,layout", [(16, "HND"), (64, "NHD")])
def test_steps_of_both(dtype, fmt, d, block, layout):
    check([1, 1, 40, 1, 200, 1], [500, 3, 700, 2000, 260, 90], 8, 2, d, dtype, 100, 10, fmt=fmt,
          bs=block, layout=layout)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_chunks_fill_the_gpu(dtype):
    """Launches that are not split, ranges of equal work, and split ones."""
    for n, lq in ((40, 70), (3, 600), (1, 40)):
        r = np.random.default_rng(n)
        lens_q = r.integers(lq // 2, lq + 1, n).tolist()
        check(lens_q, [x + 300 for x in lens_q], 16, 4, 128, dtype, 128, 20)


@pytest.mark.parametrize("heads,kvh,d,dtype,bs", [
    (71, 1, 64, BF16, 16), (48, 1, 128, F16, 16),  # virtual kv heads
    (4, 2, 20, BF16, 16), (4, 2, 128, F16, 8),     # the VALU kernel
    (4, 2, 130, F32, 16), (4, 4, 16, F32, 4), (2, 2, 256, F32, 16)])
@pytest.mark.parametrize("left,sinks", [(50, 7), (700, 40), (10, 600)])
def test_other_geometries(heads, kvh, d, dtype, bs, left, sinks):
    check([1, 1, 1, 1], [30, 400, 1200, 1], heads, kvh, d, dtype, left, sinks, bs=bs)
    check([20, 1, 3], [600, 900, 3], heads, kvh, d, dtype, left, sinks, bs=bs)


def test_right_windows_and_negative_scales():
    for right in (None, 5):
        check([50, 1], [300, 200], 4, 2, 64, BF16, 20, 8, right=right)
    check([50, 1], [300, 200], 4, 2, 64, BF16, 20, 8, scale=-0.2)
    check([1] * 3, [300, 200, 20], 4, 2, 128, F16, 20, 8, scale=0.0)


def test_without_a_window_or_without_sinks_nothing_changes():
    for lens_q in ([1, 1], [40, 1]):
        cache, q, batch = make(lens_q, [300, 500], 8, 2, 128, BF16)
        for left in (None, 64):
            run = [paged_attention_prepared(
                q, cache, 0, PreparedAttention.from_batch(batch, DEV, deterministic=True), 0.1,
                left, 0, sinks=s) for s in ((0, 9) if left is None else (0, 0))]
            assert torch.equal(*run)
    # A sink count that no position passes: attention without a window.
    full = paged_attention(q, cache, 0, batch, 0.1)
    all_sinks = paged_attention(q, cache, 0, batch, 0.1, sliding_window=10, sinks=1 << 40)
    assert (full.float() - all_sinks.float()).abs().max() <= 2.0 ** -7 * full.float().abs().max()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 256), (F32, 128), (F32, 64), (BF16, 80),
                                     (F32, 130)])
@pytest.mark.parametrize("lens_q", [[1] * 6, [1] * 80, [5, 1, 1, 90, 1, 3]])
def test_what_no_query_sees_does_not_matter(dtype, d, lens_q):
    """NaN and infinities in K and V between the sinks and the windows, and table
    entries there that name any block."""
    lens_k = [40 + 37 * i % 900 + n for i, n in enumerate(lens_q)]
    cache, q, batch = make(lens_q, lens_k, 8, 2, d, dtype)
    left, sinks, bs = 33, 10, 16
    want = reference(q, cache, batch, 0.1, left, 0, sinks)
    k, v = cache.reference_view(0, "k"), cache.reference_view(0, "v")
    bad = [float("nan"), float("inf"), -float("inf")]
    for i, table in enumerate(batch.block_tables):
        first = max(lens_k[i] - lens_q[i] - left, 0)
        for key in range(sinks, first):
            k[table[key // bs], key % bs] = bad[key % 3]
            v[table[key // bs], key % bs] = bad[(key + i) % 3]
        for b in range(-(-sinks // bs) + 2, first // bs - 2):
            table[b] = 0xFFFFFFFF if b % 2 else 0
    got = paged_attention_prepared(q, cache, 0, PreparedAttention.from_batch(batch, DEV), 0.1, left,
                                   0, sinks=sinks)
    assert_close(got, want, dtype)


def test_a_write_and_its_attention():
    """paged_attention_append_prepared is the write and then the attention."""
    for dtype, fmt, lens_q in ((BF16, "none", [1, 1, 1]), (BF16, "none", [7, 1, 30]),
                               (F16, "e4m3", [1, 1, 1]), (F32, "none", [1, 1, 9])):
        cache, q, batch = make(lens_q, [100, 400, 333], 8, 2, 64, dtype, fmt=fmt)
        slots = []
        for t, lq, lk in zip(batch.block_tables, lens_q, [100, 400, 333]):
            slots += [t[p // 16] * 16 + p % 16 for p in range(lk - lq, lk)]
        k, v = (torch.randn(sum(lens_q), 2, 64, device=DEV).to(dtype) for _ in range(2))
        prep = PreparedAttention.from_batch(batch, DEV)
        got = paged_attention_append_prepared(q, k, v, scatter_index(np.array(slots), DEV), cache, 0,
                                              prep, 0.125, 50, 0, sinks=5)
        assert_close(got, reference(q, cache, batch, 0.125, 50, 0, 5), dtype)


def test_layers_of_a_hybrid_cache_with_and_without_sinks():
    """A model whose layers alternate: one workspace, full and windowed layers."""
    cache = HybridKvCache([("kv", 2, 64), ("kv", 1, 128)], 40, 16, BF16, device=DEV)
    for t in cache.k + cache.v:
        t.normal_()
    batch = ForwardBatch(cu_seqlens_q=[0, 1, 2], cu_seqlens_k=[0, 300, 520],
                         block_tables=[list(range(19)), list(range(20, 34))], max_seqlen_q=1,
                         max_seqlen_k=300)
    prep = PreparedAttention.from_batch(batch, DEV, cache, 4)
    for layer, (kvh, d) in enumerate(((2, 64), (1, 128))):
        one = PagedKvCache(1, 40, 16, kvh, d, BF16)
        one.k[0].copy_(cache.k[layer])
        one.v[0].copy_(cache.v[layer])
        q = torch.randn(2, 4, d, device=DEV).to(BF16)
        for left, sinks in ((None, 0), (60, 4)):
            got = paged_attention_prepared(q, cache, layer, prep, 0.1, left, 0, sinks=sinks)
            assert_close(got, reference(q, one, batch, 0.1, left, 0, sinks), BF16)


def test_calls_replay_from_graphs_and_run_on_other_streams():
    for dtype, fmt, lens_q in ((BF16, "none", [1] * 5), (F16, "int8", [1, 1, 1, 1, 60])):
        cache, q, batch = make(lens_q, [100, 900, 2000, 33, 700], 8, 2, 128, dtype, fmt=fmt)
        prep = PreparedAttention.from_batch(batch, DEV, cache, 8, deterministic=True)
        out = torch.empty_like(q)
        eager = paged_attention_prepared(q, cache, 0, prep, 0.1, 200, 0, sinks=4).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = paged_attention_prepared(q, cache, 0, prep, 0.1, 200, 0, stream=side, sinks=4)
        side.synchronize()
        assert torch.equal(got, eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_attention_prepared(q, cache, 0, prep, 0.1, 200, 0, out=out, sinks=4)
        q2 = q.flip(0).contiguous()
        keep = q.clone()
        for replay in range(3):
            q.copy_(keep if replay % 2 else q2)
            graph.replay()
            torch.cuda.synchronize()
            want = paged_attention_prepared(q, cache, 0, prep, 0.1, 200, 0, sinks=4)
            torch.cuda.synchronize()
            assert torch.equal(out, want), replay


def test_long_contexts_past_32_bit_offsets():
    """Blocks past 2^32 bytes of a layer: a small batch over a large pool."""
    bs, kvh, d = 64, 8, 128
    nb = (5 << 30) // (bs * kvh * d * 2)
    cache = PagedKvCache(1, nb, bs, kvh, d, BF16)
    lens = [7000, 130]
    tables = [list(range(nb - 110, nb)), [nb - 111, 0, 5]]
    for b in tables[0] + tables[1]:
        cache.k[0][b].normal_()
        cache.v[0][b].normal_()
    small = PagedKvCache(1, 113, bs, kvh, d, BF16)
    at = {b: i for i, b in enumerate(tables[0] + tables[1])}
    for b, i in at.items():
        small.k[0][i].copy_(cache.k[0][b])
        small.v[0][i].copy_(cache.v[0][b])
    batch = ForwardBatch(cu_seqlens_q=[0, 1, 2], cu_seqlens_k=[0, 7000, 7130], block_tables=tables,
                         max_seqlen_q=1, max_seqlen_k=7000)
    local = ForwardBatch(cu_seqlens_q=[0, 1, 2], cu_seqlens_k=[0, 7000, 7130],
                         block_tables=[[at[b] for b in t] for t in tables], max_seqlen_q=1,
                         max_seqlen_k=7000)
    q = torch.randn(2, 16, d, device=DEV).to(BF16)
    got = paged_attention(q, cache, 0, batch, 0.1, sliding_window=500, sinks=100)
    assert_close(got, reference(q, small, local, 0.1, 499, 0, 100), BF16)


def test_refusals():
    cache, q, batch = make([1, 1], [40, 50], 4, 2, 64, BF16)
    with pytest.raises(ValueError):
        paged_attention(q, cache, 0, batch, 0.1, sliding_window=9, sinks=-1)
    with pytest.raises(ValueError):
        paged_attention(q.half(), cache, 0, batch, 0.1, sliding_window=9, sinks=1)
    with pytest.raises(VapiKvError):
        paged_attention(torch.zeros(2, 3, 64, dtype=BF16, device=DEV), cache, 0, batch, 0.1,
                        sliding_window=9, sinks=1)


@pytest.mark.parametrize("dtype,fmt,heads,kvh,d,layout", [
    (BF16, "e4m3", 8, 2, 128, "HND"), (BF16, "int8", 8, 2, 128, "HND"),
    (F16, "e4m3", 4, 4, 64, "NHD"), (F16, "int8", 12, 4, 80, "NHD"),
    (BF16, "int8", 4, 2, 256, "NHD"), (F16, "e4m3", 6, 2, 256, "HND")])
@pytest.mark.parametrize("lens_q", [[1] * 6, [1] * 80, [5, 1, 1, 90, 1, 3]])
def test_what_no_query_sees_of_codes_does_not_matter(dtype, fmt, heads, kvh, d, layout, lens_q):
    """Codes that are NaN between the sinks and the windows, scales of any value in the
    blocks that lie there whole, and table entries there that name any block."""
    lens_k = [40 + 37 * i % 900 + n for i, n in enumerate(lens_q)]
    cache, q, batch = make(lens_q, lens_k, heads, kvh, d, dtype, fmt=fmt, layout=layout)
    left, sinks, bs = 33, 10, 16
    want = reference(q, cache, batch, 0.1, left, 0, sinks)
    bad = [float("nan"), float("inf"), -float("inf"), -1.0, 0.0]
    codes = [t[0].view(torch.uint8) for t in (cache.k, cache.v)]
    for i, table in enumerate(batch.block_tables):
        first = max(lens_k[i] - lens_q[i] - left, 0)
        for key in range(sinks, first):
            for c in codes:
                c.select(0, table[key // bs]).select(1 if layout == "HND" else 0,
                                                     key % bs).fill_(0x7F)
        for b in range(1, first // bs):
            cache.k_scale[0][table[b]] = bad[(i + b) % 5]
            cache.v_scale[0][table[b]] = bad[b % 5]
        # (64 keys a step: the next three blocks on either side may be read.)
        for b in range(1 + 3, first // bs - 3):
            table[b] = 0xFFFFFFFF if b % 2 else 0
    got = paged_attention_prepared(q, cache, 0, PreparedAttention.from_batch(batch, DEV), 0.1, left,
                                   0, sinks=sinks)
    assert_close(got, want, dtype)


@pytest.mark.parametrize("dtype,fmt,heads,kvh,d", [
    (BF16, "none", 8, 2, 128), (F16, "none", 4, 4, 64), (BF16, "none", 4, 1, 256),
    (F32, "none", 8, 2, 128), (BF16, "e4m3", 8, 2, 128), (F16, "none", 4, 2, 20)])
@pytest.mark.parametrize("lens_q", [[1, 1], [1] * 40, [3, 40], [300, 200, 100]])
@pytest.mark.parametrize("where", ["sink", "window"])
def test_a_nan_key_stays_with_the_rows_that_see_it(dtype, fmt, heads, kvh, d, lens_q, where):
    """However a row's keys are split over workgroups: NaN scores leave NaN, in no other row."""
    lens_k = [2500 + 11 * i for i in range(len(lens_q))]
    cache, q, batch = make(lens_q, lens_k, heads, kvh, d, dtype, fmt=fmt)
    left, sinks, bs = 1000, 3, 16
    want, top = reference(q, cache, batch, 0.1, left, 0, sinks)
    lq, lk, table = lens_q[1], lens_k[1], batch.block_tables[1]
    key = 1 if where == "sink" else lk - lq - 700  # every query of the sequence sees it
    if fmt == "none":
        cache.k[0][table[key // bs], 0, key % bs] = float("nan")
    else:
        cache.k[0].view(torch.uint8)[table[key // bs], 0, key % bs] = 0x7F
    got = paged_attention_prepared(q, cache, 0, PreparedAttention.from_batch(batch, DEV), 0.1, left,
                                   0, sinks=sinks)
    rows = slice(batch.cu_seqlens_q[1], batch.cu_seqlens_q[2])
    group = heads // kvh
    assert torch.isnan(got[rows, :group]).all()
    got[rows, :group] = 0.0
    want[rows, :group] = 0.0
    assert_close(got, (want, top), dtype)
