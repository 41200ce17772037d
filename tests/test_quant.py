"""The 8-bit cache, attention weights and eviction: what is refused, on the CPU.

Every call here is refused by the host before anything is launched, so the
pointers need not be device memory.
"""
import ctypes

import numpy as np
import pytest
import torch

import quant_ref as ref
from vapi_amd import _lib
from vapi_amd._lib import BF16, EINVAL, ESPACE, EUNSUP, F16, F32, Pool, Q8Pool, Weights, lib
from vapi_amd.attention import (ForwardBatch, PreparedAttention, _workspace,
                                workspace_bytes)
from vapi_amd.cache import (PagedKvCache, gather_kv, scatter_index, write_k_to_cache,
                            write_kv_to_cache, write_kv_to_cache_layers, write_rows_indexed,
                            write_v_rows_indexed)
from vapi_amd.evict import EvictionPlan, accumulate_attention_weights, evict_kv, new_weights
from vapi_amd.quant import QuantKvCache, check_block_runs

BASE = 1 << 20  # an aligned address that nothing reads


def q8_pool(**kw):
    p = dict(k=BASE, v=BASE, k_scale=BASE, v_scale=BASE, layer_stride_bytes=1 << 30,
             scale_layer_stride_bytes=1 << 30, scale_block_stride=16, num_layers=2, num_blocks=8,
             block_size=16, num_kv_heads=2, head_dim=64, dtype=BF16, format=0, layout=0)
    p.update(kw)
    return Q8Pool(**p)


def pool16(**kw):
    p = dict(k=BASE, v=BASE, layer_stride_bytes=1 << 30, num_layers=2, num_blocks=8,
             block_size=16, num_kv_heads=2, head_dim=64, dtype=BF16, layout=0)
    p.update(kw)
    return Pool(**p)


def state(**kw):
    p = dict(data=BASE, index=None, row_stride=200, head_stride=100, rows=4, width=100)
    p.update(kw)
    return Weights(**p)


def append(pool, layer=0, k=BASE, v=BASE, slots=BASE, n=4):
    return lib().vapi_kv_q8_append(pool, layer, k, v, slots, n, None)


def attend(pool, layer=0, q=BASE, out=BASE, batch=2, max_blocks=4, max_q=1, max_k=64, heads=4,
           flags=0, pf=None, n_pf=0, ws=BASE, ws_bytes=1 << 40):
    return lib().vapi_kv_q8_attention(pool, layer, q, out, BASE, BASE, BASE, batch, max_blocks,
                                      max_q, max_k, heads, 0.1, -1, 0, flags, pf, n_pf, ws,
                                      ws_bytes, None)


def weigh(pool, w, layer=0, q=BASE, batch=2, max_blocks=4, max_q=1, max_k=64, heads=4, last=0,
          decay=1.0, ws=BASE, ws_bytes=1 << 40):
    fn = (lib().vapi_kv_q8_attention_weights if isinstance(pool, Q8Pool)
          else lib().vapi_kv_attention_weights)
    return fn(pool, layer, q, BASE, BASE, BASE, batch, max_blocks, max_q, max_k, heads, 0.1, -1,
              0, last, decay, w, ws, ws_bytes, None)


def evict(pool, w, out=None, layer=0, lens=BASE, src=BASE, src_blocks=4, dst=BASE, dst_blocks=4,
          batch=2, max_len=64, budget=32, sinks=2, recent=8, kept=BASE):
    fn = lib().vapi_kv_q8_evict if isinstance(pool, Q8Pool) else lib().vapi_kv_evict
    return fn(pool, layer, w, None if out is None else ctypes.byref(out), lens, src, src_blocks,
              dst, dst_blocks, batch, max_len, budget, sinks, recent, kept, None)


BAD_POOLS = [
    (dict(format=2), EINVAL), (dict(dtype=9), EINVAL), (dict(dtype=F32), EUNSUP),
    (dict(layout=5), EINVAL), (dict(num_layers=0), EINVAL), (dict(head_dim=0), EINVAL),
    (dict(head_dim=72), EUNSUP), (dict(head_dim=272), EUNSUP), (dict(block_size=8), EUNSUP),
    (dict(block_size=48), EUNSUP), (dict(block_size=512), EUNSUP),
    (dict(num_blocks=1 << 28), EINVAL), (dict(scale_block_stride=1), EINVAL),
    (dict(layer_stride_bytes=100), EINVAL), (dict(scale_layer_stride_bytes=64), EINVAL),
    (dict(layer_stride_bytes=(1 << 30) + 8), EINVAL), (dict(k=BASE + 8), EINVAL),
    (dict(v=None), EINVAL), (dict(k_scale=None), EINVAL), (dict(v_scale=BASE + 2), EINVAL),
    (dict(num_kv_heads=70000, scale_block_stride=70000, layer_stride_bytes=1 << 40), EUNSUP)]


@pytest.mark.parametrize("change,code", BAD_POOLS)
def test_bad_pools_are_refused_everywhere(change, code):
    pool = q8_pool(**change)
    heads = 2 * pool.num_kv_heads
    assert append(pool) == code
    assert lib().vapi_kv_q8_gather(pool, 0, BASE, 1, 4, BASE, BASE, None) == code
    assert attend(pool, heads=heads) == code
    assert weigh(pool, state(), heads=heads) == code
    assert evict(pool, state()) == code
    assert lib().vapi_kv_q8_attention_workspace_size(pool, 2, 2, 4, 1, 64) == 0
    assert lib().vapi_kv_last_error()


def test_bad_calls_are_refused():
    pool = q8_pool()
    assert append(None) == EINVAL and append(pool, layer=2) == EINVAL
    assert append(pool, k=None) == EINVAL and append(pool, slots=None) == EINVAL
    assert append(pool, v=BASE + 4) == EINVAL and append(pool, n=1 << 31) == EUNSUP
    assert append(pool, n=0) == 0 and append(q8_pool(num_blocks=0), k=None) == 0
    gather = lib().vapi_kv_q8_gather
    assert gather(pool, 0, BASE, 2, 33, BASE, None, None) == EINVAL
    assert gather(pool, 0, None, 2, 32, BASE, None, None) == EINVAL
    assert gather(pool, 0, BASE, 2, 32, BASE + 8, None, None) == EINVAL
    assert gather(pool, 0, BASE, 2, 32, None, None, None) == 0
    assert attend(pool, layer=2) == EINVAL and attend(pool, heads=3) == EINVAL
    assert attend(pool, heads=2 * 257) == EUNSUP and attend(pool, q=None) == EINVAL
    assert attend(pool, out=BASE + 8) == EINVAL and attend(pool, max_blocks=0) == EINVAL
    assert attend(pool, flags=4) == EINVAL and attend(pool, n_pf=1) == EINVAL
    assert attend(pool, pf=BASE, n_pf=3) == EINVAL
    assert attend(q8_pool(num_blocks=0)) == EINVAL
    assert attend(pool, ws_bytes=64) == ESPACE and attend(pool, ws=None) == ESPACE
    assert attend(pool, batch=0) == 0 and attend(pool, max_q=0) == 0
    # A call with prefill rows needs room for their values.
    need = lib().vapi_kv_q8_attention_workspace_size(pool, 2, 1, 4, 8, 64)
    values = 2 * 64 * 2 * 64 * 2  # K and V of 64 keys, two kv heads of 64, two bytes
    decode = lib().vapi_kv_q8_attention_workspace_size(pool, 2, 0, 4, 8, 64)
    assert need >= decode + values
    assert attend(pool, max_q=8, pf=BASE, n_pf=1, ws_bytes=decode) == ESPACE
    assert attend(pool, max_q=8, ws_bytes=need) == ESPACE  # without a list: both sequences
    assert attend(pool, batch=70000, max_q=2, pf=BASE, n_pf=66000) == EUNSUP


@pytest.mark.parametrize("pool", [pool16(), pool16(dtype=F16, block_size=32), q8_pool()])
def test_bad_weights_calls_are_refused(pool):
    ok = state()
    assert weigh(pool, None) == EINVAL and weigh(pool, state(data=None)) == EINVAL
    assert weigh(pool, state(data=BASE + 2)) == EINVAL
    assert weigh(pool, state(index=BASE + 1)) == EINVAL
    assert weigh(pool, state(head_stride=99)) == EINVAL
    assert weigh(pool, state(row_stride=150)) == EINVAL
    assert weigh(pool, state(rows=1)) == EINVAL  # no index, two sequences
    assert weigh(pool, ok, max_k=101) == EINVAL and weigh(pool, ok, heads=3) == EINVAL
    assert weigh(pool, ok, decay=-1.0) == EINVAL
    assert weigh(pool, ok, decay=float("nan")) == EINVAL
    assert weigh(pool, ok, decay=float("inf")) == EINVAL
    assert weigh(pool, ok, q=BASE + 8) == EINVAL and weigh(pool, ok, q=None) == EINVAL
    assert weigh(pool, ok, max_blocks=0) == EINVAL and weigh(pool, ok, layer=2) == EINVAL
    size = lib().vapi_kv_attention_weights_workspace_size(2, 2, 4, 64, 1, 64, 0)
    assert size > 0 and weigh(pool, ok, ws_bytes=size - 1) == ESPACE
    assert weigh(pool, ok, ws=BASE + 8) == EINVAL
    assert weigh(pool, ok, batch=0) == 0 and weigh(pool, ok, max_k=0) == 0
    assert lib().vapi_kv_attention_weights_workspace_size(2, 3, 4, 64, 1, 64, 0) == 0


def test_weights_of_other_pools_are_refused():
    assert weigh(pool16(dtype=F32), state()) == EUNSUP
    assert weigh(pool16(head_dim=60), state()) == EUNSUP
    assert weigh(pool16(head_dim=264), state()) == EUNSUP
    assert weigh(pool16(block_size=24), state()) == EUNSUP
    assert weigh(pool16(v=None), state()) == EINVAL
    assert weigh(pool16(num_blocks=0, k=None), state()) == EINVAL


@pytest.mark.parametrize("pool", [pool16(), pool16(dtype=F32, head_dim=6, block_size=5), q8_pool()])
def test_bad_evictions_are_refused(pool):
    ok = state()
    assert evict(pool, None) == EINVAL and evict(pool, ok, layer=2) == EINVAL
    assert evict(pool, ok, out=state(data=None)) == EINVAL
    assert evict(pool, ok, budget=0, sinks=0, recent=0) == EINVAL
    assert evict(pool, ok, budget=9) == EINVAL
    assert evict(pool, ok, sinks=0xFFFFFFFF, recent=0xFFFFFFFF) == EINVAL
    assert evict(pool, ok, max_len=101) == EINVAL
    assert evict(pool, ok, out=state(width=31)) == EINVAL
    for name in ("lens", "src", "dst", "kept"):
        assert evict(pool, ok, **{name: None}) == EINVAL
    assert evict(pool, ok, src_blocks=0) == EINVAL and evict(pool, ok, dst_blocks=0) == EINVAL
    assert evict(pool, ok, batch=0) == 0 and evict(pool, ok, max_len=0) == 0
    assert evict(pool, state(rows=40000), batch=40000) == EUNSUP


def test_calls_past_a_grid_s_reach_are_refused():
    wide = state(head_stride=1 << 25, row_stride=1 << 27, width=1 << 25)
    most = 65535 * 192  # workgroups of 192 keys
    for pool in (pool16(), q8_pool()):
        assert weigh(pool, wide, max_k=most + 1) == EUNSUP
        assert weigh(pool, wide, max_k=most, ws_bytes=64) == ESPACE
        assert weigh(pool, state(index=BASE), batch=1 << 23) == EUNSUP
        assert weigh(pool, state(), heads=65538) == EUNSUP
    pool = q8_pool()
    assert append(pool, n=1 << 28) == EUNSUP
    assert attend(pool, max_q=2, max_k=1 << 28) == EUNSUP
    # (A size for no keys is that for one.)
    size = lib().vapi_kv_q8_attention_workspace_size
    assert size(pool, 2, 2, 4, 8, 0) == size(pool, 2, 2, 4, 8, 1)


def test_the_weights_workspace_of_long_prompts():
    """8 bytes a row and chunk, and at most 64 MiB of sums: not a sum for every key
    and 512 rows."""
    size = lib().vapi_kv_attention_weights_workspace_size
    for batch, kvh, heads, n in ((1, 8, 32, 32768), (4, 8, 32, 32768), (1, 8, 32, 131072),
                                 (1, 1, 16, 1 << 20), (64, 8, 32, 131072)):
        rows = batch * heads * n * 8
        assert rows <= size(batch, kvh, heads, 128, n, n, 0) <= rows + (64 << 20) + 4096


def test_sizes_that_are_refused_need_no_workspace():
    size, pool = lib().vapi_kv_q8_attention_workspace_size, q8_pool()
    for args in ((2, 2, 0, 1, 64), (2, 2, 3, 1, 64), (2, 2, 2 * 257, 1, 64),
                 (2, 2, 4, 2, 1 << 28), (70000, 66000, 4, 2, 64)):
        assert size(pool, *args) == 0 and lib().vapi_kv_last_error()
    assert size(pool, 70000, 66000, 4, 1, 64) > 0  # no prefill rows: the list counts for nothing


# ---- the Python side --------------------------------------------------------------


def cpu_cache(**kw):
    args = dict(num_layers=2, num_blocks=6, block_size=16, num_kv_heads=2, head_dim=64,
                device="cpu")
    args.update(kw)
    return QuantKvCache(**args)


@pytest.mark.parametrize("bad", [
    dict(layout="DHN"), dict(fmt="int4"), dict(dtype=torch.float32), dict(head_dim=40),
    dict(head_dim=288), dict(head_dim=0), dict(block_size=8), dict(block_size=24),
    dict(block_size=512), dict(num_layers=0), dict(num_kv_heads=0), dict(num_blocks=-1)])
def test_bad_caches_are_refused(bad):
    with pytest.raises(ValueError):
        cpu_cache(**bad)


@pytest.mark.parametrize("kvh", [2, 16, 20])
def test_a_block_holds_its_codes_and_scales(kvh):
    cache = cpu_cache(num_kv_heads=kvh)
    width = -(-kvh // 16) * 16
    assert cache.block_bytes() == 2 * 2 * (16 * kvh * 64 + 4 * width)
    assert cache.k_scale[1].shape == (6, kvh)
    assert cache.num_slots() == 96
    half = cpu_cache(num_kv_heads=kvh).k[0]
    assert half.element_size() == 1 and half.dtype == torch.float8_e4m3fn


def test_rows_that_do_not_fit_are_refused():
    cache = cpu_cache()
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    idx = scatter_index([0, 1, 2], "cpu")
    for rows, slots in ((k, [0, 1]), (k[:, :1], [0, 1, 2]), (k.half(), [0, 1, 2]),
                        (k, [0, 1, 96]), (k, [0, 1, 1]), (k, [0, 16, 1]), (k, [0, 1, 2])):
        with pytest.raises(ValueError):  # the last one: not on a GPU
            write_kv_to_cache(cache, 0, rows, rows, slots)
    for bad in (k.float(), k[:, :, :32], torch.zeros(3, 128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            write_rows_indexed(cache, 0, bad, bad, idx)
    with pytest.raises(ValueError):
        write_rows_indexed(cache, 0, k, None, idx)
    with pytest.raises(ValueError):
        write_v_rows_indexed(cache, 0, k, idx)
    with pytest.raises(ValueError):
        write_k_to_cache(cache, 0, k, [0, 1, 2])
    with pytest.raises(ValueError):
        write_kv_to_cache_layers(cache, 0, k[None], k[None], idx)
    with pytest.raises(ValueError):
        gather_kv(cache, 0, [0, 1], 20)


def test_block_runs():
    skip = _lib.SLOT_SKIP
    check_block_runs(np.array([3, 2, skip, 1, 40, skip, 16, 17], np.uint32), 16)
    check_block_runs(np.zeros(0, np.uint32), 16)
    for bad in ([0, 16, 1], [5, 5], [5, skip, 5], [32, 0, 47]):
        with pytest.raises(ValueError):
            check_block_runs(np.array(bad, np.uint32), 16)


def test_the_workspace_of_a_step():
    cache = cpu_cache()
    decode = workspace_bytes(cache, 2, 4, 1, 64)
    assert 0 < decode < workspace_bytes(cache, 2, 4, 8, 64, 1) < workspace_bytes(cache, 2, 4, 8, 64)
    # A prefill-only step covers the whole batch, whatever its list names.
    batch = ForwardBatch(cu_seqlens_q=[0, 3, 3], cu_seqlens_k=[0, 9, 20],
                         block_tables=[[0], [1]], max_seqlen_q=3, max_seqlen_k=11)
    prep = PreparedAttention.from_batch(batch, "cpu")
    assert prep.n_prefill_arg() == 1 and prep.n_prefill_arg(cache) is None


def test_a_larger_workspace_leaves_the_smaller_one_alone():
    """A captured graph, or a call on another stream, may still use it."""
    small, large = cpu_cache(), PagedKvCache(1, 6, 16, 2, 128, torch.bfloat16, "HND", "cpu")
    batch = ForwardBatch(cu_seqlens_q=[0, 1, 2], cu_seqlens_k=[0, 9, 20],
                         block_tables=[[0], [1]], max_seqlen_q=1, max_seqlen_k=11)
    prep = PreparedAttention.from_batch(batch, "cpu", small, 4)
    first = prep.workspace
    _workspace(large, prep, 2, 4, 1, 11, "cpu")
    second = prep.workspace
    assert second.numel() > first.numel()
    prep.reserve(cpu_cache(num_kv_heads=4, head_dim=256), 16, "cpu")
    assert prep.workspace.numel() > second.numel()
    assert prep.workspaces[0] is first and prep.workspaces[1] is second
    _workspace(small, prep, 2, 4, 1, 11, "cpu")
    assert len(prep.workspaces) == 2


def test_weights_states_that_do_not_fit_are_refused():
    cache = PagedKvCache(1, 6, 16, 2, 64, torch.bfloat16, "HND", "cpu")
    prep = PreparedAttention.from_batch(
        ForwardBatch(cu_seqlens_q=[0, 1, 2], cu_seqlens_k=[0, 9, 20], block_tables=[[0], [1]],
                     max_seqlen_q=1, max_seqlen_k=11), "cpu")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    w = new_weights(3, 2, 20, "cpu")

    def call(q=q, w=w, **kw):
        with pytest.raises(ValueError):
            accumulate_attention_weights(q, cache, 0, prep, 0.1, w, **kw)

    call(q=q.half())
    call(q=q[:, :, :32])
    call(w=w[:, :1])
    call(w=w.double())
    call(w=w[0])
    call(w=w[:1])
    call(w=w[:, :, ::2])
    call(w=w[:, :, :0])
    call(last_queries=-1)
    call(rows=[0, 0])
    call(rows=[0])
    call(rows=[0, -1])
    call(rows=torch.zeros(2, dtype=torch.int64))
    call(rows=torch.zeros(3, dtype=torch.int32))
    call()  # not on a GPU


def test_eviction_plans_that_do_not_fit_are_refused():
    def plan(lens=(40, 10), src=((0, 1, 2), (3,)), dst=((4, 5), (6,)), budget=20, sinks=2,
             recent=4, rows=None):
        return EvictionPlan.from_tables(lens, src, dst, budget, sinks, recent, 16, "cpu", rows)

    ok = plan()
    assert ok.new_lens == [20, 10] and ok.max_len == 40 and ok.max_keep == 20
    assert plan(lens=(40, 0), src=((0, 1, 2), ()), dst=((4, 5), ())).new_lens == [20, 0]
    for bad in (dict(budget=5), dict(budget=0, sinks=0, recent=0), dict(sinks=-1),
                dict(recent=-1), dict(lens=(40,)), dict(lens=(49, 10)), dict(lens=(40, -1)),
                dict(dst=((4,), (6,))), dict(dst=((4, 5), (5,))), dict(dst=((4, 0), (6,))),
                dict(src=((0, 1, -2), (3,))), dict(rows=[1, 1]), dict(rows=[1])):
        with pytest.raises(ValueError):
            plan(**bad)

    cache = PagedKvCache(1, 7, 16, 2, 64, torch.bfloat16, "HND", "cpu")
    w = new_weights(2, 2, 40, "cpu")
    for kw in (dict(cache=PagedKvCache(1, 7, 32, 2, 64, torch.bfloat16, "HND", "cpu")),
               dict(cache=PagedKvCache(1, 6, 16, 2, 64, torch.bfloat16, "HND", "cpu")),
               dict(w=w[:1]), dict(out=torch.zeros(1)), dict(out=w[:, :, 1:]), dict()):
        with pytest.raises(ValueError):
            evict_kv(kw.get("cache", cache), 0, kw.get("w", w), ok, weights_out=kw.get("out"))


# ---- the reference the GPU tests compare with ---------------------------------------


def test_rounding_of_the_reference():
    """The oracle's e4m3 is torch's, its int8 rounds ties to even."""
    x = torch.cat([torch.linspace(-470, 470, 4001), torch.linspace(-0.03, 0.03, 999),
                   torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 448.0])]).clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.to_codes(x.double().numpy(), "e4m3"), want)
    assert ref.to_codes([0.5, 1.5, -2.5, 126.6, 127.9], "int8").tolist() == [0, 2, -2, 127, 127]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_stored_values_are_near_and_of_the_dtype(fmt, dtype):
    """A value is off by at most half a step of its format (int8: a whole one at
    the block's largest), and codes times scales are values of the dtype."""
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 1, 32, generator=gen) * 3).to(dtype)
    m = ref.Model(4, 1, 16, 32, fmt, dtype)
    m.append(x, np.arange(64))
    got = torch.from_numpy(m.codes * m.scale[:, :, None, None]).permute(0, 2, 1, 3)
    got = got.reshape(64, 1, 32)
    assert torch.equal(got.to(dtype).double(), got)
    off = (got - x.double()).abs()
    if fmt == "e4m3":
        least = torch.from_numpy(m.scale).repeat_interleave(16, 0)[:, :, None] * 2.0 ** -10
        assert torch.all(off <= torch.maximum(x.double().abs() * 2.0 ** -4, least))
    else:
        step = torch.from_numpy(m.scale).repeat_interleave(16, 0)[:, :, None]
        assert torch.all(off <= step) and float((off / step).mean()) < 0.3
