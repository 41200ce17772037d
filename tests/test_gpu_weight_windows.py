"""Attention weights of few rows under sliding windows: every key counts once,
whatever place in a chunk of keys the first visible one has."""
import pytest
import torch

import quant_ref as ref
from test_gpu_evict import filled, weights_ref
from test_gpu_quant import batch_of
from vapi_amd.attention import PreparedAttention
from vapi_amd.evict import accumulate_attention_weights

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def check(lens_q, lens_k, heads, kvh, d, fmt, dtype, left, last=0, max_k=0, layout="HND"):
    """Against the definition, and each row's weights against one: a weight of a row
    of n keys is off by the same part of itself as in weights_ref, so is their sum."""
    cache, tables, _ = filled(lens_k, kvh, d, 16, fmt, dtype, layout, sum(lens_k) + left)
    q = torch.randn(sum(lens_q), heads, d, generator=torch.Generator().manual_seed(left)).to(dtype)
    prep = PreparedAttention.from_batch(batch_of(lens_q, lens_k, tables), "cuda")
    prep.max_seqlen_k = max(max_k, prep.max_seqlen_k)
    scale, rows = d ** -0.5, list(range(len(lens_k)))
    old = torch.zeros(len(lens_k), kvh, max(max_k, max(lens_k)))
    w = old.cuda()
    accumulate_attention_weights(q.cuda(), cache, 0, prep, scale, w, last_queries=last,
                                 window_size_left=left)
    got = w.cpu().double()
    k = ref.values(cache, 0, "k")
    want, bound = weights_ref(q, k, lens_q, lens_k, tables, 16, scale, left, 0, last, 1.0, old,
                              rows)
    err = (got - want).abs()
    assert torch.all(err <= bound), f"{float((err / bound.clamp_min(1e-300)).max()):.3g} bounds"
    n = torch.tensor([min(lq, last) if last else lq for lq in lens_q], dtype=torch.float64)
    total = got.sum(dim=2)
    assert torch.all((total - n[:, None] * heads / kvh).abs() <= bound.sum(dim=2))


# The first visible key at every multiple of 16 (and off them) within a step of up
# to 64, contexts of many chunks of 256.
PHASES = [3000 + 16 * j + 3 * (j % 4) for j in range(8)]


@pytest.mark.parametrize("fmt,dtype", [("none", BF16), ("e4m3", BF16), ("int8", F16)])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("left", [519, 1024, 2047])
def test_single_tokens_in_windows(fmt, dtype, d, left):
    check([1] * 8, PHASES, 4, 2, d, fmt, dtype, left)


@pytest.mark.parametrize("fmt,dtype", [("none", F16), ("e4m3", F16), ("int8", BF16)])
@pytest.mark.parametrize("heads,kvh,last", [(4, 1, 4), (1, 1, 16), (16, 1, 1), (3, 1, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_last_queries_in_windows(fmt, dtype, heads, kvh, last, d):
    check([20] * 8, PHASES, heads, kvh, d, fmt, dtype, 700, last, layout="NHD")


@pytest.mark.parametrize("fmt", ["none", "e4m3", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_windows_over_longer_chunks(fmt, d):
    """Few sequences, and a batch whose long ones make the chunks longer."""
    check([1], [9016], 8, 2, d, fmt, BF16, 4036)
    check([1] * 64, [1 + 97 * i % 700 for i in range(63)] + [8990], 8, 4, d, fmt, BF16, 2500)


@pytest.mark.parametrize("fmt", ["none", "e4m3"])
@pytest.mark.parametrize("left", [1600, 2007, 2016])
def test_windows_where_scores_are_not_kept(fmt, left):
    """More scores than the call keeps between its passes."""
    check([1, 1], [9000, 8500], 32, 2, 64, fmt, BF16, left, max_k=1_100_000)
