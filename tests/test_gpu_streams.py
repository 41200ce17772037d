"""Calls on a stream of their own: their outputs' memory is not what work of the
current stream has yet to write, and what they read outlives them."""
import pytest
import torch

import quant_ref as ref
from test_gpu_evict import filled
from test_gpu_quant import batch_of
from vapi_amd.attention import (PreparedAttention, paged_attention_append_prepared,
                                paged_attention_prepared)
from vapi_amd.cache import scatter_index
from vapi_amd.evict import (EvictionPlan, accumulate_attention_weights, evict_kv,
                            new_weights)

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def behind(*outputs):
    """The current stream 20 ms behind, with fills of freed memory of these sizes
    still to come."""
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)
    for t in outputs:
        for _ in range(8):
            torch.full_like(t, -1)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
def test_an_output_is_not_memory_the_current_stream_still_writes(fmt):
    n, kvh, heads, d = 3000, 2, 8, 128
    cache, tables, free = filled([n], kvh, d, 16, fmt, BF16, "HND", 3, spare=80)
    prep = PreparedAttention.from_batch(batch_of([n], [n], tables), "cuda", cache, heads)
    q = torch.randn(n, heads, d, device="cuda").to(BF16)
    k = torch.randn(n, kvh, d, device="cuda").to(BF16)
    slots = scatter_index(ref.slots_of(tables[0], n, 16), "cuda")
    w = torch.rand(1, kvh, n, device="cuda")
    dst = [[free.pop() for _ in range(64)]]
    plan = EvictionPlan.from_tables([n], tables, dst, 1000, 4, 16, 16, "cuda")
    side = torch.cuda.Stream()

    calls = {
        "attention": lambda s: paged_attention_prepared(q, cache, 0, prep, 0.1, stream=s),
        "append": lambda s: paged_attention_append_prepared(q, k, k, slots, cache, 0, prep, 0.1,
                                                            stream=s),
        "evict": lambda s: evict_kv(cache, 0, w, plan, stream=s)}
    for name, call in calls.items():
        want = call(None)
        behind(want)
        got = call(side)
        torch.cuda.synchronize()
        assert torch.equal(got, want), name


def test_a_captured_call_names_its_stream():
    """stream= the stream that is captured: the output is the graph's."""
    cache, tables, _ = filled([200], 2, 64, 16, "e4m3", BF16, "HND", 5)
    prep = PreparedAttention.from_batch(batch_of([1], [200], tables), "cuda", cache, 4, True)
    q = torch.randn(1, 4, 64, device="cuda").to(BF16)
    paged_attention_prepared(q, cache, 0, prep, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention_prepared(q, cache, 0, prep, 0.1, stream=torch.cuda.current_stream())
    for _ in range(3):
        q.copy_(torch.randn(q.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_attention_prepared(q, cache, 0, prep, 0.1))


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
@pytest.mark.parametrize("lens_q", [[1, 1], [30, 1]])
def test_a_step_dropped_before_its_call_has_run(fmt, lens_q):
    """Its device arrays and workspace are not handed out while the call, on
    another stream, waits. (Zeros in their place would leave rows unwritten.)"""
    lens_k, heads, kvh, d = [300, 90], 4, 2, 64
    cache, tables, _ = filled(lens_k, kvh, d, 16, fmt, BF16, "HND", 3)
    q = torch.randn(sum(lens_q), heads, d, device="cuda").to(BF16)

    def step():
        return PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda", cache,
                                            heads, deterministic=True)

    w, want_w = new_weights(2, kvh, 300), new_weights(2, kvh, 300)
    prep = step()
    want = paged_attention_prepared(q, cache, 0, prep, 0.1)
    accumulate_attention_weights(q, cache, 0, prep, 0.1, want_w)
    prep, side = step(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
    got = paged_attention_prepared(q, cache, 0, prep, 0.1, stream=side)
    accumulate_attention_weights(q, cache, 0, prep, 0.1, w, stream=side)
    sizes = [t.numel() * t.element_size() for t in
             (prep.block_table, prep.seqlens_q, prep.seqlens_k, prep.prefill_seqs, prep.workspace,
              prep.weights_workspace)]
    del prep
    junk = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(w, want_w) and junk
