"""The paged KV pool held in 8 bits, host side.

QuantKvCache stands where a PagedKvCache does: write_kv_to_cache /
write_rows_indexed round rows into it, paged_attention* reads it, gather_kv
gives values back, and KvBlockBackend copies, spills and swaps its blocks. The
reference has no such cache (its pools hold the model's own dtype,
crates/vapi-backend-candle/src/cache.rs:12-118); include/vapi_kv.h states the
formats and the rounding.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import Pool, Q8Pool, lib
from .cache import _LAYOUTS, dtype_code

FORMATS = {"e4m3": (_lib.Q8_E4M3, torch.float8_e4m3fn), "int8": (_lib.Q8_INT8, torch.int8)}


class QuantKvCache:
    """Per-layer K and V pools of 8-bit codes with a scale for each (block, kv
    head): half the bytes of a 16-bit PagedKvCache.

    dtype: that of the rows written and gathered and of the queries (bfloat16
    or float16). fmt: "e4m3" (3 bits of mantissa: rows whose channels differ
    much in size) or "int8". layout as PagedKvCache. head_dim is a multiple of
    16 up to 256, block_size a power of two from 16 to 256.

    k[l], v[l]: codes (torch.float8_e4m3fn or torch.int8) in the layout;
    k_scale[l], v_scale[l]: f32 [num_blocks, num_kv_heads], powers of two. A
    code c of block b and head h stands for c * scale[b, h].

    pool describes the same memory to the block-level calls (copy_blocks,
    export/import, swap, the spill tier): codes as pairs of bytes, then the
    scales as rows of their own, chained. A block's blob holds both.
    """

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.bfloat16, fmt: str = "e4m3",
                 layout: str = "HND", device: str | torch.device = "cuda"):
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be HND or NHD, not {layout!r}")
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {', '.join(FORMATS)}, not {fmt!r}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"an 8-bit cache's rows are bfloat16 or float16, not {dtype}")
        if head_dim <= 0 or head_dim % 16 or head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 16 up to 256, not {head_dim}")
        if not 16 <= block_size <= 256 or block_size & (block_size - 1):
            raise ValueError(f"block_size must be a power of two from 16 to 256, not {block_size}")
        if num_layers <= 0 or num_kv_heads <= 0 or num_blocks < 0:
            raise ValueError(f"a cache of {num_layers} layers, {num_blocks} blocks and "
                             f"{num_kv_heads} kv heads")
        code, code_dtype = FORMATS[fmt]
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.fmt = fmt
        self.layout = layout
        self.device = torch.device(device)
        shape = ((num_blocks, num_kv_heads, block_size, head_dim) if layout == "HND"
                 else (num_blocks, block_size, num_kv_heads, head_dim))
        layer_bytes = num_blocks * block_size * num_kv_heads * head_dim
        stride = layer_bytes + -layer_bytes % 256
        slab = torch.zeros((2, num_layers, stride), dtype=torch.uint8, device=self.device)
        self._codes = slab
        self.k = [slab[0, i, :layer_bytes].view(code_dtype).view(shape) for i in range(num_layers)]
        self.v = [slab[1, i, :layer_bytes].view(code_dtype).view(shape) for i in range(num_layers)]
        # A block's scales as one row of `width` f32 per slot, enough for the heads.
        width = -(-num_kv_heads // block_size)
        row = block_size * width
        scales = torch.zeros((2, num_layers, num_blocks, row), dtype=torch.float32,
                             device=self.device)
        self._scales = scales
        self.k_scale = [scales[0, i, :, :num_kv_heads] for i in range(num_layers)]
        self.v_scale = [scales[1, i, :, :num_kv_heads] for i in range(num_layers)]

        def base(t):
            return t.data_ptr() if t.numel() else None

        geometry = dict(num_layers=num_layers, num_blocks=num_blocks, block_size=block_size)
        self.q8 = Q8Pool(
            k=base(slab[0]), v=base(slab[1]), k_scale=base(scales[0]), v_scale=base(scales[1]),
            layer_stride_bytes=stride, scale_layer_stride_bytes=num_blocks * row * 4,
            scale_block_stride=row, num_kv_heads=num_kv_heads, head_dim=head_dim,
            dtype=dtype_code(dtype), format=code, layout=_LAYOUTS[layout], **geometry)
        self._scale_pool = Pool(
            k=base(scales[0]), v=base(scales[1]), layer_stride_bytes=num_blocks * row * 4,
            num_kv_heads=1, head_dim=width, dtype=_lib.F32, layout=_lib.LAYOUT_HND, **geometry)
        self.pool = Pool(
            k=base(slab[0]), v=base(slab[1]), layer_stride_bytes=stride,
            num_kv_heads=num_kv_heads, head_dim=head_dim // 2, dtype=_lib.F16,
            layout=_LAYOUTS[layout], next=ctypes.addressof(self._scale_pool), **geometry)

    def num_slots(self) -> int:
        return self.num_blocks * self.block_size

    def block_bytes(self) -> int:
        """Bytes of one block's codes and scales across every layer, K and V."""
        return lib().vapi_kv_block_bytes(self.pool)

    def values(self, layer: int, which: str = "k") -> torch.Tensor:
        """What a layer's codes stand for, f32 [num_blocks, block_size, kv_heads,
        head_dim]: a view for inspection and tests, not a path of serving."""
        c = (self.k if which == "k" else self.v)[layer].float()
        s = (self.k_scale if which == "k" else self.v_scale)[layer]
        c = c.permute(0, 2, 1, 3) if self.layout == "HND" else c
        return c * s[:, None, :, None]


def check_block_runs(slots: np.ndarray, block_size: int) -> None:
    """Raises ValueError unless each block's tokens follow one another in
    `slots` (skipped ones aside) and no slot comes twice, as the append into an
    8-bit cache needs."""
    real = slots[slots != _lib.SLOT_SKIP].astype(np.int64)
    if np.unique(real).size != real.size:
        raise ValueError("a slot is written twice in one call")
    blocks = real // block_size
    runs = blocks[np.concatenate([[True], blocks[1:] != blocks[:-1]])] if blocks.size else blocks
    if np.unique(runs).size != runs.size:
        raise ValueError("the tokens of one block must follow one another in slot_mapping")
