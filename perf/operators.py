"""Cases of the 8-bit paged KV cache and of eviction by attention weight.

Four operators, each one call that a serving program makes per layer:

  append   K/V rows written into a cache of 8-bit codes with one scale for
           each (block, kv head) of K and of V
  attend   paged attention over such a cache: decode rows, prefill chunks, or
           a step of both
  weights  each cached key's attention weight from the step's queries, summed
           over the query heads of a kv head and added to a decayed running sum
  evict    of every sequence and kv head the keys with the largest running
           sums (and the first and the latest ones) moved into fewer blocks

A code c of a block with scale s stands for c * s; scales are powers of two, so
every step from rows to codes is exact but the one rounding, and two right
implementations hold the same values: a cache is returned as its codes (e4m3
numbers, or whole ones) and their scales.
With `own` false the operators are computed in their plain form.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SKIP = 0xFFFFFFFF
# Smallest scale, and the largest magnitude a row element is taken as, so that
# every code times its scale is a value of the rows' type.
SCALE_MIN = {("e4m3", "bf16"): 2.0 ** -117, ("e4m3", "f16"): 2.0 ** -15,
             ("int8", "bf16"): 2.0 ** -126, ("int8", "f16"): 2.0 ** -24}
LARGEST = {("e4m3", "bf16"): 1.875 * 2.0 ** 127, ("e4m3", "f16"): 1.875 * 2.0 ** 15,
           ("int8", "bf16"): 1.984375 * 2.0 ** 127, ("int8", "f16"): 1.984375 * 2.0 ** 15}


def _case(kind, **kw):
    case = {"kind": kind, "batch": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
            "dtype": "bf16", "fmt": "e4m3", "block": 16, "layout": "HND",
            # Keys of a sequence: log-normal (median, sigma) clipped to [lo, hi].
            "ctx_median": 2048, "ctx_sigma": 0.75, "ctx_lo": 256, "ctx_hi": 8192,
            # The last `chunks` sequences bring new_lo .. new_hi queries, the others one.
            "new_lo": 1, "new_hi": 1, "chunks": 0, "window": 0, "lens_seed": 1}
    case.update(kw)
    return case


def listed():
    return [
        # A decode step of 64 sequences: each row lands in a block that holds
        # earlier rows of its sequence already.
        {"name": "append_b64", "kind": "append", "tokens": 64, "run": 1, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "fmt": "e4m3", "block": 16, "layout": "HND",
         "blocks": 512, "pad": 0.0},
        # The rows of a 4,096-token step, 5% padding, sequences of any phase.
        {"name": "append_4096", "kind": "append", "tokens": 4096, "run": 256, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "fmt": "int8", "block": 16, "layout": "HND",
         "blocks": 1024, "pad": 0.05},
        # One user generating over a short context: all latency.
        {"name": "attend_b1", **_case("attend", ctx_median=1337, ctx_sigma=0.0)},
        # A full decode batch, contexts 256 to 8,192.
        {"name": "attend_b64", **_case("attend", batch=64, lens_seed=0x5EED0002)},
        # As many kv heads as query heads, head_dim 96, a sliding window of
        # 2,047 keys, int8 codes of f16 rows on [block, token, head, d] blocks of 32.
        {"name": "attend_b12_window",
         **_case("attend", batch=12, kv_heads=32, head_dim=96, dtype="f16", fmt="int8", block=32,
                 layout="NHD", window=2047, ctx_median=3000, lens_seed=12)},
        # Chunks of 300 to 512 new tokens over about 3,000 earlier keys.
        {"name": "attend_prefill_b4",
         **_case("attend", batch=4, chunks=4, new_lo=300, new_hi=512, ctx_median=3400,
                 ctx_sigma=0.2, lens_seed=4)},
        # A step of decode rows with one chunk of 256 tokens.
        {"name": "attend_mixed_b16",
         **_case("attend", batch=16, chunks=1, new_lo=256, new_hi=256, fmt="int8",
                 lens_seed=16)},
        # The running sums of a decode step over a 16-bit cache.
        {"name": "weights_b16",
         **_case("weights", batch=16, fmt="none", last=0, decay=1.0, lens_seed=161)},
        # At the end of a prompt: what its last 32 queries attended to, over an
        # 8-bit cache (28 q / 4 kv heads).
        {"name": "weights_last32_b2",
         **_case("weights", batch=2, q_heads=28, kv_heads=4, chunks=2, new_lo=400, new_hi=500,
                 ctx_median=6000, ctx_sigma=0.2, last=32, decay=0.0, lens_seed=21)},
        # All queries of fresh prompts, f16.
        {"name": "weights_prompt_b3",
         **_case("weights", batch=3, dtype="f16", fmt="none", chunks=3, new_lo=700, new_hi=2000,
                 ctx_median=0, last=0, decay=0.0, lens_seed=31)},
        # One sequence of an 8-bit cache back to 1,024 keys.
        {"name": "evict_b1",
         **_case("evict", ctx_median=1500, ctx_sigma=0.0, budget=1024, sinks=4, recent=128)},
        # Long sequences of a 16-bit cache back to 2,048 keys each.
        {"name": "evict_b16",
         **_case("evict", batch=16, fmt="none", ctx_median=6000, ctx_sigma=0.3, budget=2048,
                 sinks=4, recent=256, lens_seed=162)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "weights", "weights", "evict"])
    dtype, block = rng.choice(["bf16", "bf16", "f16"]), rng.choice([16, 16, 32, 64])
    layout = rng.choice(["HND", "HND", "NHD"])
    if kind == "append":
        case = {"kind": kind, "tokens": _log(rng, 1, 4096), "run": _log(rng, 1, 300),
                "kv_heads": rng.choice([1, 4, 5, 8]), "head_dim": rng.choice([64, 80, 96, 128, 256]),
                "dtype": dtype, "fmt": rng.choice(["e4m3", "int8"]), "block": block,
                "layout": layout, "pad": rng.choice([0.0, 0.05])}
        row = case["kv_heads"] * case["head_dim"]
        case["tokens"] = min(case["tokens"], 2 ** 22 // row)
        case["run"] = min(max(case["run"], case["tokens"] * block * row // 2 ** 25), 300)
        runs = -(-case["tokens"] // case["run"])
        case["blocks"] = runs * ((case["run"] + block - 2) // block + 1) + 4
        return case
    heads, kvh = rng.choice([(32, 8), (32, 8), (16, 8), (28, 4), (32, 32), (64, 8), (71, 1)])
    case = _case(kind, q_heads=heads, kv_heads=kvh, dtype=dtype, block=block, layout=layout,
                 head_dim=rng.choice([64, 80, 96, 128, 128, 128, 256]),
                 fmt=rng.choice(["e4m3", "int8"] if kind == "attend" else ["none", "e4m3", "int8"]),
                 ctx_median=_log(rng, 40, 4000), ctx_lo=1, lens_seed=rng.randrange(1 << 20))
    if kind == "evict":
        case.update(batch=_log(rng, 1, 16), sinks=rng.choice([0, 1, 4, 30]),
                    recent=_log(rng, 1, 300))
        case["budget"] = case["sinks"] + case["recent"] + _log(rng, 1, 2000)
        limit = 2.5e8
    else:
        if rng.random() < 0.25:
            case["window"] = _log(rng, 128, 4096)
        rows = rng.choice(["decode", "decode", "chunks", "mixed"])
        case["batch"] = _log(rng, 1, 64) if rows == "decode" else _log(rng, 1, 6)
        if rows != "decode":
            case["chunks"] = case["batch"]
            case["new_lo"] = _log(rng, 2, 200)
            case["new_hi"] = case["new_lo"] + _log(rng, 1, 700)
        if rows == "mixed":
            case["batch"] += _log(rng, 1, 20)
        if kind == "weights":
            case.update(last=rng.choice([0, 0, 8, 32]), decay=rng.choice([0.0, 0.9, 1.0]))
        limit = 3e8
    while True:  # no dearer than the listed cases
        w = work(case)
        if w["bytes"] <= limit and w["flops"] <= (9e10 if kind == "attend" else 2e10):
            return case
        if case["new_hi"] > 64:
            case["new_lo"] = max(case["new_lo"] // 2, 2)
            case["new_hi"] = max(case["new_hi"] // 2, case["new_lo"])
        case["ctx_median"] = max(case["ctx_median"] * 3 // 4, 1)
        case["ctx_hi"] = max(case["ctx_hi"] * 3 // 4, 64)


# ---- shapes -----------------------------------------------------------------


def _lens(case):
    """(len_q, len_k) of each sequence; len_k counts the new tokens."""
    r = np.random.default_rng(case["lens_seed"])
    b, c = case["batch"], case["chunks"]
    if case["ctx_median"] > 0:
        ctx = np.exp(r.normal(math.log(case["ctx_median"]), case["ctx_sigma"], size=b))
        ctx = np.clip(np.round(ctx), case["ctx_lo"], case["ctx_hi"]).astype(np.int64)
    else:
        ctx = np.zeros(b, np.int64)
    len_q = np.ones(b, np.int64)
    if c:
        len_q[b - c:] = r.integers(case["new_lo"], case["new_hi"] + 1, size=c)
    return len_q, np.maximum(ctx + np.where(len_q > 1, len_q, 0), len_q)


def _queries(case, len_q):
    """The queries of each sequence whose weights are taken."""
    return np.minimum(len_q, case["last"]) if case["last"] else len_q


def _pairs(case, n_q, len_k):
    """Visible (query, key) pairs of a sequence's last n_q queries, and the keys they see."""
    p = np.arange(len_k - n_q, len_k, dtype=np.int64)
    lo = np.maximum(0, p - (case["window"] - 1)) if case["window"] else np.zeros_like(p)
    return int((p - lo + 1).sum()), int(len_k - lo.min())


def _kept(case, len_k):
    return np.minimum(len_k, case["budget"])


def work(case):
    kvh, d, bs = case["kv_heads"], case["head_dim"], case["block"]
    code = 2.0 if case["fmt"] == "none" else 1.0
    if case["kind"] == "append":
        rows = case["tokens"] - int(round(case["pad"] * case["tokens"]))
        scales = 2 * 4.0 * kvh * (1 + rows // (bs if case["run"] >= bs else 1))
        return {"bytes": 2.0 * rows * kvh * d * (2 + code) + 4.0 * case["tokens"] + scales,
                "flops": 0.0}
    len_q, len_k = _lens(case)
    scale = 0.0 if case["fmt"] == "none" else 4.0 / bs  # bytes a key of one head
    if case["kind"] == "evict":
        new = _kept(case, len_k)
        moved = float(new.sum())
        return {"bytes": 2.0 * 2 * moved * kvh * (d * code + scale)      # K and V, read and written
                + 4.0 * kvh * (float(len_k.sum()) + 2 * moved), "flops": 0.0}  # sums in and out, kept keys
    pairs = keys = 0
    n_q = len_q if case["kind"] == "attend" else _queries(case, len_q)
    for lq, lk in zip(n_q, len_k):
        p, k = _pairs(case, int(lq), int(lk))
        pairs, keys = pairs + p, keys + k
    row = 2.0 * int(n_q.sum()) * case["q_heads"] * d
    tables = 4.0 * (int((-(-len_k // bs)).sum()) + 2 * (case["batch"] + 1))
    if case["kind"] == "attend":  # K and V, Q in and the output out
        return {"bytes": 2 * keys * kvh * (d * code + scale) + 2 * row + tables,
                "flops": 4.0 * d * case["q_heads"] * pairs}
    sums = 4.0 * kvh * int(len_k.sum()) * (2 if case["decay"] else 1)
    return {"bytes": keys * kvh * (d * code + scale) + row + tables + sums,
            "flops": 2.0 * d * case["q_heads"] * pairs}


# ---- inputs -----------------------------------------------------------------


def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _power(amax, fmt, dtype):
    """The scale of a block whose largest magnitude is amax (0 for none): the
    least power of two that takes it to at most 448, or below 128 for int8."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = e - 9 + (m > 0.875).to(e.dtype) if fmt == "e4m3" else e - 7
    s = ((e + 127).clamp(1, 254).to(torch.int32) << 23).view(torch.float32)  # 2^e
    s = s.clamp_min(SCALE_MIN[fmt, dtype])
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _finite(x, fmt, dtype):
    big = LARGEST[fmt, dtype]
    return torch.nan_to_num(x.float(), nan=0.0, posinf=big, neginf=-big).clamp(-big, big)


def _round(x, scale, fmt):
    """The codes of x under `scale` (0: all codes 0)."""
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)),
                    torch.zeros_like(x))
    return (y.clamp(-448, 448) if fmt == "e4m3" else y.round().clamp(-127, 127)).to(CODES[fmt])


def _by_head(x, layout):
    """A cache buffer as [block, head, token, d] (its own memory)."""
    return x if layout == "HND" else x.transpose(1, 2)


def _quantised(case, shape, gen):
    """A cache buffer of normal rows: codes in the case's layout and scales."""
    x = _finite(_normal(gen, shape, DTYPES[case["dtype"]]), case["fmt"], case["dtype"])
    s = _power(x.abs().amax(dim=(2, 3)), case["fmt"], case["dtype"])
    c = _round(x, s[:, :, None, None], case["fmt"])
    return (c if case["layout"] == "HND" else c.view(torch.int8).transpose(1, 2).contiguous()
            .view(CODES[case["fmt"]])), s


def _pool(case, blocks, gen):
    """One layer's K and V in the case's layout, scales too for 8-bit codes."""
    shape = (blocks, case["kv_heads"], case["block"], case["head_dim"])
    if case["fmt"] != "none":
        (k, ks), (v, vs) = _quantised(case, shape, gen), _quantised(case, shape, gen)
        return {"k": k, "v": v, "ks": ks, "vs": vs}
    if case["layout"] == "NHD":
        shape = (shape[0], shape[2], shape[1], shape[3])
    return {"k": _normal(gen, shape, DTYPES[case["dtype"]]),
            "v": _normal(gen, shape, DTYPES[case["dtype"]])}


def _tables(r, need, spare):
    """Block tables of need[i] distinct blocks each, and the pool's blocks."""
    nb = int(need.sum()) + spare
    perm = r.permutation(nb).astype(np.int64)
    ends = np.cumsum(need)
    return [perm[e - n:e] for n, e in zip(need, ends)], nb, perm[int(need.sum()):]


def _padded(tables):
    width = max([len(t) for t in tables] + [1])
    out = np.zeros((len(tables), width), np.int64)
    for i, t in enumerate(tables):
        out[i, :len(t)] = t
    return torch.from_numpy(out).to(DEV)


def _append_slots(case, r):
    """Runs of tokens in blocks of their own; single ones land anywhere in theirs."""
    n, bs, run = case["tokens"], case["block"], case["run"]
    perm, slots, at, done = r.permutation(case["blocks"]), [], 0, 0
    while done < n:
        m = min(run, n - done)
        first = int(r.integers(0, bs)) if run == 1 or r.random() < 0.5 else 0
        pos = np.arange(first, first + m)
        width = -(-(first + m) // bs)
        slots.append(perm[at:at + width][pos // bs] * bs + pos % bs)
        at, done = at + width, done + m
    slots = np.concatenate(slots).astype(np.int64)
    slots[r.choice(n, size=int(round(case["pad"] * n)), replace=False)] = SKIP
    return slots


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    r = np.random.default_rng(seed)
    state = {"case": case, "scale": case["head_dim"] ** -0.5}
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "append":
        state["blocks"] = case["blocks"]
        state.update(_pool(case, case["blocks"], gen))
        shape = (case["tokens"], case["kv_heads"], case["head_dim"])
        # Rows of different size, so that some blocks' scales have to grow.
        size = torch.exp2(_normal(gen, (case["tokens"], 1, 1)))
        state["k_new"] = (_normal(gen, shape) * size).to(dt)
        state["v_new"] = (_normal(gen, shape) * size).to(dt)
        state["slots"] = torch.from_numpy(_append_slots(case, r)).to(DEV)
        return _with_handles(state) if own else state
    len_q, len_k = _lens(case)
    bs, width = case["block"], int(len_k.max())
    spare = 3 if case["kind"] != "evict" else int((-(-_kept(case, len_k) // bs)).sum()) + 3
    tables, nb, rest = _tables(r, -(-len_k // bs), spare)
    state.update(_pool(case, nb, gen), blocks=nb, tables=tables, table=_padded(tables),
                 len_q=len_q, len_k=len_k, n_k=torch.from_numpy(len_k).to(DEV))
    if case["kind"] in ("weights", "evict"):
        # A state of three more rows than the step has sequences.
        shape = (case["batch"] + 3, case["kv_heads"], width)
        state["weights"] = torch.rand(shape, generator=gen, device=DEV) ** 4
        state["rows"] = torch.from_numpy(r.permutation(shape[0])[:case["batch"]]).to(DEV)
    if case["kind"] == "evict":
        new = _kept(case, len_k)
        at = np.cumsum(-(-new // bs))
        state["to"] = [rest[e - n:e] for n, e in zip(-(-new // bs), at)]
        state["to_table"], state["n_new"] = _padded(state["to"]), torch.from_numpy(new).to(DEV)
        # Ties among the sums, as keys that nothing attends to have.
        state["weights"][state["weights"] < 0.01] = 0.0
        state["weights_out"] = torch.zeros_like(state["weights"])
        return _with_handles(state) if own else state
    state["q"] = _normal(gen, (int(len_q.sum()), case["q_heads"], case["head_dim"]), dt)
    # Where the queries of the decode rows and of the chunks are among all rows.
    n_q = len_q if case["kind"] == "attend" else _queries(case, len_q)
    end = np.cumsum(len_q)
    state["parts"] = []
    for seqs in (np.nonzero(len_q == 1)[0], np.nonzero(len_q > 1)[0]):
        if len(seqs):
            most = int(n_q[seqs].max())
            j = np.arange(most)[None, :] - (most - n_q[seqs][:, None])  # aligned at the end
            at = np.where(j >= 0, (end[seqs] - n_q[seqs])[:, None] + j, -1)
            state["parts"].append({"seqs": torch.from_numpy(seqs).to(DEV),
                                   "at": torch.from_numpy(at).to(DEV),
                                   "keys": int(len_k[seqs].max())})
    return _with_handles(state) if own else state


def _with_handles(state):
    """The framework's cache with the same contents, and the plan of the step."""
    from vapi_amd.attention import ForwardBatch, PreparedAttention
    from vapi_amd.cache import PagedKvCache, scatter_index
    from vapi_amd.evict import EvictionPlan
    from vapi_amd.quant import QuantKvCache
    case = state["case"]
    args = (1, state["blocks"], case["block"], case["kv_heads"], case["head_dim"],
            DTYPES[case["dtype"]])
    if case["fmt"] == "none":
        cache = PagedKvCache(*args, case["layout"], DEV)
        cache.k[0].copy_(state["k"])
        cache.v[0].copy_(state["v"])
    else:
        cache = QuantKvCache(*args, case["fmt"], case["layout"], DEV)
        cache.k[0].view(torch.int8).copy_(state["k"].view(torch.int8))
        cache.v[0].view(torch.int8).copy_(state["v"].view(torch.int8))
        cache.k_scale[0].copy_(state["ks"])
        cache.v_scale[0].copy_(state["vs"])
    state["cache"] = cache
    state["k"] = state["v"] = None
    if case["kind"] == "append":
        state["slots"] = scatter_index(state["slots"].cpu().numpy(), DEV)
        return state
    if "rows" in state:
        state["rows"] = state["rows"].to(torch.int32)
    if case["kind"] == "evict":
        state["plan"] = EvictionPlan.from_tables(
            state["len_k"].tolist(), [t.tolist() for t in state["tables"]],
            [t.tolist() for t in state["to"]], case["budget"], case["sinks"], case["recent"],
            case["block"], DEV, rows=state["rows"].tolist())
        return state
    len_q, len_k = state["len_q"], state["len_k"]
    batch = ForwardBatch(
        cu_seqlens_q=np.concatenate([[0], np.cumsum(len_q)]).tolist(),
        cu_seqlens_k=np.concatenate([[0], np.cumsum(len_k)]).tolist(),
        block_tables=[t.tolist() for t in state["tables"]],
        max_seqlen_q=int(len_q.max()), max_seqlen_k=int(len_k.max()))
    state["left"] = case["window"] - 1 if case["window"] else None
    state["prepared"] = (PreparedAttention.from_batch(batch, DEV, cache, case["q_heads"])
                         if case["kind"] == "attend" else
                         PreparedAttention.from_batch(batch, DEV))
    return state


# ---- one pass -----------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"append": _append, "attend": _attend, "weights": _weights,
            "evict": _evict}[case["kind"]](state, case)


def _own(state, case):
    from vapi_amd.attention import paged_attention_prepared
    from vapi_amd.cache import write_rows_indexed
    from vapi_amd.evict import accumulate_attention_weights, evict_kv
    cache = state["cache"]
    if case["kind"] == "append":
        write_rows_indexed(cache, 0, state["k_new"], state["v_new"], state["slots"])
        return [cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0]]
    if case["kind"] == "attend":
        return [paged_attention_prepared(state["q"], cache, 0, state["prepared"], state["scale"],
                                         state["left"], 0)]
    if case["kind"] == "weights":
        accumulate_attention_weights(state["q"], cache, 0, state["prepared"], state["scale"],
                                     state["weights"], rows=state["rows"],
                                     last_queries=case["last"], decay=case["decay"],
                                     window_size_left=state["left"])
        return [state["weights"]]
    kept = evict_kv(cache, 0, state["weights"], state["plan"], weights_out=state["weights_out"])
    out = [kept, state["weights_out"], cache.k[0], cache.v[0]]
    return out + ([] if case["fmt"] == "none" else [cache.k_scale[0], cache.v_scale[0]])


def _values(state, name, slots, block, layout):
    """The f32 rows [.., kvh, d] that a buffer holds at `slots`."""
    x = state[name]
    raw = x.view(torch.int8) if x.element_size() == 1 else x
    x = _by_head(raw, layout)[slots // block, :, slots % block].view(x.dtype).float()
    return x * state[name + "s"][slots // block][..., None] if name + "s" in state else x


def _key_slots(state, case, table, keys):
    pos = torch.arange(keys, device=DEV)
    return table[:, pos // case["block"]] * case["block"] + pos % case["block"]


def _probabilities(state, case, part):
    """softmax(scale q.k) of one part's queries: [seq, kv head, query, group, key]."""
    at, seqs = part["at"], part["seqs"]
    slots = _key_slots(state, case, state["table"][seqs], part["keys"])
    k = _values(state, "k", slots, case["block"], case["layout"])
    kvh, d, (b, m) = case["kv_heads"], case["head_dim"], at.shape
    g = case["q_heads"] // kvh
    q = state["q"][at.clamp_min(0)].float().view(b, m, kvh, g, d).permute(0, 2, 1, 3, 4)
    s = torch.matmul(q.reshape(b, kvh, m * g, d), k.permute(0, 2, 3, 1)) * state["scale"]
    s = s.view(b, kvh, m, g, part["keys"])
    n_k = state["n_k"][seqs][:, None, None]
    pos = n_k - m + torch.arange(m, device=DEV)[None, :, None]
    key = torch.arange(part["keys"], device=DEV)
    hidden = (key > pos) | (at < 0)[:, :, None]
    if case["window"]:
        hidden = hidden | (key < pos - (case["window"] - 1))
    s = s.masked_fill(hidden[:, None, :, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(s - top)
    return e / e.sum(dim=-1, keepdim=True).clamp_min(1e-30), slots


def _attend(state, case):
    out = torch.empty(state["q"].shape, dtype=state["q"].dtype, device=DEV)
    for part in state["parts"]:  # the decode rows, the chunks
        p, slots = _probabilities(state, case, part)
        v = _values(state, "v", slots, case["block"], case["layout"]).permute(0, 2, 1, 3)
        b, kvh, m, g, keys = p.shape
        o = torch.matmul(p.view(b, kvh, m * g, keys), v).view(b, kvh, m, g, -1)
        o = o.permute(0, 2, 1, 3, 4).reshape(b, m, kvh * g, -1)
        live = part["at"] >= 0
        out[part["at"][live]] = o[live].to(out.dtype)
    return [out]


def _weights(state, case):
    w = state["weights"]
    for part in state["parts"]:
        p, _ = _probabilities(state, case, part)
        rows, n_k = state["rows"][part["seqs"]], state["n_k"][part["seqs"]]
        old = w[rows][:, :, :part["keys"]]
        live = torch.arange(part["keys"], device=DEV) < n_k[:, None, None]
        w[rows, :, :part["keys"]] = torch.where(live, old * case["decay"] + p.sum(dim=(2, 3)), old)
    return [w]


def _append(state, case):
    bs, d, kvh, nb = case["block"], case["head_dim"], case["kv_heads"], case["blocks"]
    fmt, dt = case["fmt"], case["dtype"]
    live = state["slots"] < nb * bs
    at = state["slots"][live]
    new = torch.zeros(nb * bs, dtype=torch.bool, device=DEV)
    new[at] = True
    new = new.view(nb, bs)
    touched, fresh = new.any(dim=1), new[:, 0]
    for name in ("k", "v"):
        x = torch.zeros((nb * bs, kvh, d), device=DEV)
        x[at] = _finite(state[name + "_new"][live], fmt, dt)
        x = x.view(nb, bs, kvh, d).transpose(1, 2)
        codes = _by_head(state[name], case["layout"])
        old = torch.where(fresh[:, None], 0.0, state[name + "s"])
        s = torch.maximum(old, _power(x.abs().amax(dim=(2, 3)), fmt, dt))
        x = torch.where(new[:, None, :, None], x, codes.float() * old[:, :, None, None])
        c = _round(x, s[:, :, None, None], fmt).view(torch.int8)
        was = codes.view(torch.int8)
        was.copy_(torch.where(touched[:, None, None, None], c, was))
        state[name + "s"].copy_(torch.where(touched[:, None], s, state[name + "s"]))
    return [state["k"], state["v"], state["ks"], state["vs"]]


def _evict(state, case):
    w = state["weights"][state["rows"]]
    b, kvh, width = w.shape
    n_k, n_new, most = state["n_k"], state["n_new"], min(case["budget"], width)
    key = torch.arange(width, device=DEV)
    held = (key < case["sinks"]) | (key >= n_k[:, None] - case["recent"])
    rank = torch.where(held[:, None], math.inf, w)
    rank = torch.where((key < n_k[:, None])[:, None], rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :, :most]
    live = (torch.arange(most, device=DEV) < n_new[:, None])[:, None]
    kept = torch.sort(torch.where(live, order, width), dim=-1).values
    kept = torch.where(live, kept, -1)
    out = torch.zeros((b, kvh, width), device=DEV)
    out[:, :, :most] = torch.where(live, torch.gather(w, 2, kept.clamp_min(0)), 0.0)
    state["weights_out"][state["rows"]] = out
    # The kept rows of each head into the new blocks, whole blocks at a time.
    bs, head = case["block"], torch.arange(kvh, device=DEV)[None, :, None]
    wide = -(-most // bs) * bs
    pos = torch.full((b, kvh, wide), -1, device=DEV)
    pos[:, :, :most] = kept
    src = torch.gather(state["table"], 1, (pos.clamp_min(0) // bs).view(b, -1)).view(pos.shape)
    there = (torch.arange(wide // bs, device=DEV) * bs < n_new[:, None])  # [seq, new block]
    to = state["to_table"][:, :wide // bs][there]
    for name in ("k", "v"):
        buf = state[name]
        raw = _by_head(buf.view(torch.int8) if buf.element_size() == 1 else buf, case["layout"])
        x = raw[src, head, pos.clamp_min(0) % bs]
        x = x.view(b, kvh, wide // bs, bs, -1).transpose(1, 2)[there]  # [new block, head, token, d]
        full = (pos >= 0).view(b, kvh, wide // bs, bs).transpose(1, 2)[there][..., None]
        if case["fmt"] == "none":
            raw[to] = torch.where(full, x, raw[to])
            continue
        s = state[name + "s"][src, head].view(b, kvh, wide // bs, bs).transpose(1, 2)[there]
        x = torch.where(full, x.view(buf.dtype).float() * s[..., None], 0.0)
        new_s = _power(x.abs().amax(dim=(2, 3)), case["fmt"], case["dtype"])
        raw[to] = _round(x, new_s[:, :, None, None], case["fmt"]).view(torch.int8)
        state[name + "s"][to] = new_s
    out = [kept.to(torch.int32), state["weights_out"], state["k"], state["v"]]
    return out + ([] if case["fmt"] == "none" else [state["ks"], state["vs"]])


# ---- the definitions in 64 bits -------------------------------------------------


def _grid64(x, fmt):
    """x rounded to the nearest code, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _scale64(amax, fmt, dtype):
    if amax == 0:
        return 0.0
    e = math.floor(math.log2(amax))
    top = amax / 2.0 ** e
    e = e - 6 if fmt == "int8" else e - 8 if top <= 1.75 else e - 7
    return max(2.0 ** e, SCALE_MIN[fmt, dtype])


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    return {"append": _append64, "attend": _attend64, "weights": _weights64,
            "evict": _evict64}[case["kind"]](state, case)


def _rows64(state, case, name, slots, h):
    x = state[name]
    raw = x.view(torch.int8) if x.element_size() == 1 else x
    blk, off = slots // case["block"], slots % case["block"]
    x = (raw[blk, h, off] if case["layout"] == "HND" else raw[blk, off, h]).view(x.dtype).double()
    return x * state[name + "s"][blk, h].double()[:, None] if case["fmt"] != "none" else x


def _weights_of(state, case, i, h, first, n_q):
    """Probabilities of sequence i's last n_q queries at query head h, and its key slots."""
    lk = int(state["len_k"][i])
    pos = np.arange(lk)
    slots = torch.from_numpy(state["tables"][i][pos // case["block"]] * case["block"]
                             + pos % case["block"]).to(DEV)
    kh = h // (case["q_heads"] // case["kv_heads"])
    q = state["q"][first:first + n_q, h].double()
    s = q @ _rows64(state, case, "k", slots, kh).T * case["head_dim"] ** -0.5
    p = torch.arange(lk - n_q, lk, device=DEV)[:, None]
    key = torch.arange(lk, device=DEV)[None, :]
    hidden = key > p
    if case["window"]:
        hidden |= key < p - (case["window"] - 1)
    return torch.softmax(s.masked_fill(hidden, -math.inf), dim=1), slots, kh


def _attend64(state, case):
    out, first = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEV), 0
    for i, lq in enumerate(state["len_q"].tolist()):
        for h in range(case["q_heads"]):
            p, slots, kh = _weights_of(state, case, i, h, first, lq)
            out[first:first + lq, h] = p @ _rows64(state, case, "v", slots, kh)
        first += lq
    return [out]


def _weights64(state, case):
    w, end = state["weights"].double(), 0
    for i, lq in enumerate(state["len_q"].tolist()):
        end += lq
        n_q, lk = int(_queries(case, np.array(lq))), int(state["len_k"][i])
        row = w[int(state["rows"][i])]
        row[:, :lk] *= case["decay"]
        for h in range(case["q_heads"]):
            p, _, kh = _weights_of(state, case, i, h, end - n_q, n_q)
            row[kh, :lk] += p.sum(dim=0)
    return [w]


def _append64(state, case):
    bs, slots = case["block"], state["slots"].cpu().numpy()
    blocks = {}
    for t, s in enumerate(slots.tolist()):
        if s < case["blocks"] * bs:
            blocks.setdefault(s // bs, []).append((s % bs, t))
    out = []
    for name in ("k", "v"):
        codes = _by_head(state[name].double(), case["layout"])
        scales = state[name + "s"].double()
        big = LARGEST[case["fmt"], case["dtype"]]
        rows = state[name + "_new"].double().nan_to_num(0.0, big, -big).clamp(-big, big)
        for blk, tokens in blocks.items():
            offs, ids = [o for o, _ in tokens], [t for _, t in tokens]
            fresh = 0 in offs
            most = rows[ids].abs().amax(dim=(0, 2)).tolist()
            s = torch.tensor([_scale64(a, case["fmt"], case["dtype"]) for a in most],
                             dtype=torch.float64, device=DEV)
            old = scales[blk] * (0.0 if fresh else 1.0)
            s = torch.maximum(s, old)
            by = torch.where(s > 0, s, 1.0)[:, None, None]
            held = _grid64(codes[blk] * old[:, None, None] / by, case["fmt"])
            held[:, offs] = _grid64(rows[ids].transpose(0, 1) / by, case["fmt"])
            codes[blk], scales[blk] = held, s
        out.append((codes if case["layout"] == "HND" else codes.transpose(1, 2), scales))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _evict64(state, case):
    """The kept keys are whole numbers, held to the plain form's; here the sums that go with them."""
    out = state["weights_out"].double()
    for i, (lk, new) in enumerate(zip(state["len_k"].tolist(), state["n_new"].tolist())):
        row = int(state["rows"][i])
        w = state["weights"][row].double().cpu().numpy()
        out[row] = 0.0
        for h in range(case["kv_heads"]):
            held = [k for k in range(lk) if k < case["sinks"] or k >= lk - case["recent"]]
            rest = [k for k in range(case["sinks"], lk - case["recent"])]
            rest.sort(key=lambda k: (-w[h, k], k))
            kept = sorted((held + rest)[:new])
            out[row, h, :new] = torch.from_numpy(w[h, kept]).to(DEV)
    return [None, out, None, None] + ([] if case["fmt"] == "none" else [None, None])
