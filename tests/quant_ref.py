"""The 8-bit cache and attention by their definitions, in 64 bits on the CPU."""
import math

import numpy as np
import torch

from vapi_amd._lib import SLOT_SKIP

MIN_EXP = {("e4m3", torch.bfloat16): -117, ("e4m3", torch.float16): -15,
           ("int8", torch.bfloat16): -126, ("int8", torch.float16): -24}
# Magnitudes a row element is taken as at most.
BIG = {("e4m3", torch.bfloat16): 1.875 * 2.0 ** 127, ("e4m3", torch.float16): 61440.0,
       ("int8", torch.bfloat16): 1.984375 * 2.0 ** 127, ("int8", torch.float16): 65024.0}


def scale_of(amax, fmt, dtype):
    """The least power of two (no smaller than the least scale) that takes amax
    to at most 448 (e4m3) or below 128 (int8)."""
    if amax == 0:
        return 0.0
    e = math.frexp(amax)[1] - 12
    fits = (lambda a: a <= 448.0) if fmt == "e4m3" else (lambda a: a < 128.0)
    while not fits(amax / 2.0 ** e):
        e += 1
    return 2.0 ** max(e, MIN_EXP[fmt, dtype])


def to_codes(x, fmt):
    """Numbers (f64, already divided by the scale) as codes' values."""
    x = np.asarray(x, np.float64)
    if fmt == "int8":
        return np.clip(np.rint(x), -127, 127)
    with np.errstate(divide="ignore"):
        e = np.maximum(np.floor(np.log2(np.abs(x))), -6.0)
    step = np.exp2(e - 3)
    return np.clip(np.rint(x / step) * step, -448.0, 448.0)


def finite(rows, fmt, dtype):
    """Row elements as they are stored: NaN as 0, magnitudes cut at BIG."""
    big = BIG[fmt, dtype]
    x = rows.double().numpy().copy()
    x[np.isnan(x)] = 0.0
    return np.clip(x, -big, big)


class Model:
    """One tensor (K or V) of a layer: code values [block, head, token, d] and
    scales [block, head], in f64."""

    def __init__(self, num_blocks, kvh, bs, d, fmt, dtype):
        self.fmt, self.dtype, self.bs = fmt, dtype, bs
        self.codes = np.zeros((num_blocks, kvh, bs, d))
        self.scale = np.zeros((num_blocks, kvh))

    def append(self, rows, slots):
        x = finite(rows, self.fmt, self.dtype)
        by_block = {}
        for t, s in enumerate(np.asarray(slots, np.int64).tolist()):
            if s != SLOT_SKIP and s < self.codes.shape[0] * self.bs:
                by_block.setdefault(s // self.bs, {})[s % self.bs] = t
        for b, at in by_block.items():
            for h in range(self.codes.shape[1]):
                old = 0.0 if 0 in at else self.scale[b, h]
                amax = max(float(np.abs(x[t, h]).max()) for t in at.values())
                s = max(old, scale_of(amax, self.fmt, self.dtype))
                for o in range(self.bs):
                    if o in at:
                        v = x[at[o], h]
                    else:
                        v = self.codes[b, h, o] * old
                    self.codes[b, h, o] = to_codes(v / s, self.fmt) if s > 0 else 0.0
                self.scale[b, h] = s


def values(cache, layer, which):
    """A QuantKvCache's (or PagedKvCache's) rows as f64 [slot, head, d]."""
    if hasattr(cache, "q8"):
        x = cache.values(layer, which).cpu().double()
    else:
        x = cache.reference_view(layer, which).cpu().double()
    return x.reshape(-1, cache.num_kv_heads, cache.head_dim)


def slots_of(table, n, bs):
    pos = np.arange(n)
    return np.asarray(table, np.int64)[pos // bs] * bs + pos % bs


def probabilities(q, k, len_q, scale, left, right):
    """softmax over keys of one head: q [len_q, d], k [len_k, d] in f64; rows
    that see nothing are 0. Also each row's score bound scale * sum |q||k|."""
    len_k = k.shape[0]
    if len_q == 0 or len_k == 0:
        return torch.zeros(len_q, len_k, dtype=torch.float64), 0.0
    s = (q @ k.T) * scale
    pos = torch.arange(len_k - len_q, len_k)[:, None]
    key = torch.arange(len_k)[None, :]
    hidden = torch.zeros(len_q, len_k, dtype=torch.bool)
    if right is not None:
        hidden |= key > pos + right
    if left is not None:
        hidden |= key < pos - left
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(dim=1, keepdim=True)
    p = torch.exp(s - top.clamp_min(-1e300))
    total = p.sum(dim=1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    reach = (q.abs() @ k.abs().T).amax() * abs(scale)
    return p, float(reach)


def attention(q, k, v, lens_q, lens_k, tables, bs, scale, left=None, right=0):
    """(out, bound): the definition's output in f64 and how far a right
    implementation in q's dtype may be from it, element by element.

    With u = eps / 2 of the dtype (half a step): P is rounded to the dtype (u of
    sum p |v|), the output once (u of itself). A score is a sum of d products
    and a scaling in f32, off by at most (d + 2) 2^-24 of scale * sum |q||k|,
    and exp2 by 2^-22: each p by twice that at most, numerator and denominator.
    The sum over keys is off by at most len_k 2^-24 of sum p |v|. A rounding of
    values below the dtype's least normal one is off by half its least step.
    """
    u = torch.finfo(q.dtype).eps / 2
    hq, d = q.shape[1], q.shape[2]
    kvh = k.shape[1]
    q = q.cpu().double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    first = 0
    for lq, lk, t in zip(lens_q, lens_k, tables):
        at = torch.from_numpy(slots_of(t, lk, bs))
        for h in range(hq):
            kk, vv = k[at, h * kvh // hq], v[at, h * kvh // hq]
            p, reach = probabilities(q[first:first + lq, h], kk, lq, scale, left, right)
            o = p @ vv
            pv = p @ vv.abs()
            soft = 2 * ((d + 2) * 2.0 ** -24 * reach + 2.0 ** -22) + lk * 2.0 ** -24
            out[first:first + lq, h] = o
            bound[first:first + lq, h] = pv * (u + soft) * (1 + u) + o.abs() * u
        first += lq
    return out, bound + 2.0 ** -25
