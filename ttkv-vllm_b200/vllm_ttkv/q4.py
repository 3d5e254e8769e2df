"""A paged cache held in 4 bits: its layout, for layers that have no calibrated TT-KV decoder.

Keys and values are stored as the model gives them to its attention (keys after RoPE, so any rotary
scheme), each group of `group` lanes of a token and head as 4-bit codes with an fp16 scale and an
fp16 minimum: `d + 8 * d / group` bytes per token and KV head (136 at d = 128 and groups of 128,
against 512 in 16 bits), no fit and no state per request. No counterpart in the reference.

The cache of a layer is a uint8 tensor [num_blocks, H, block_size // 16, panel_bytes], one panel per
16 tokens of a head (the byte order is in `include/ttkv_b200.h`). Its slot ids are vLLM's flat
`block * block_size + offset`. The operators are `ops.q4_write_paged`, `ops.q4_read_paged`,
`ops.q4_decode_paged` and `ops.q4_prefill_paged`.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

PANEL_TOKENS = 16
LIMIT = 57344.0                  # values beyond it are stored as it


@dataclass(frozen=True)
class Q4Layout:
    """Geometry of one layer's 4-bit cache: H KV heads of d lanes in groups of `group`."""

    H: int
    d: int = 128
    group: int = 128

    def __post_init__(self):
        if self.H < 1:
            raise ValueError(f"a 4-bit cache needs at least one KV head, got H={self.H}")
        if self.d not in (64, 128):
            raise ValueError(f"head dim {self.d}: the 4-bit cache serves 64 and 128")
        if self.group not in (32, 64, 128) or self.group > self.d:
            raise ValueError(f"groups of {self.group} lanes: 32, 64 or 128, at most d={self.d}")
        # bytes of a panel: 16 tokens of one head
        object.__setattr__(self, "panel_bytes", PANEL_TOKENS * (self.d + 8 * (self.d // self.group)))
        # what the calls need of it
        object.__setattr__(self, "key", (self.H, self.d, self.group, self.panel_bytes))

    def bytes_per_token(self) -> int:
        """Cache bytes of one token over the layer's heads."""
        return self.H * self.panel_bytes // PANEL_TOKENS

    def ratio(self) -> float:
        """16-bit bytes over 4-bit bytes."""
        return 4 * self.H * self.d / self.bytes_per_token()

    def cache_shape(self, num_blocks: int, block_size: int) -> tuple[int, int, int, int]:
        if block_size < PANEL_TOKENS or block_size % PANEL_TOKENS:
            raise ValueError(f"block size {block_size} is not a multiple of {PANEL_TOKENS}")
        return num_blocks, self.H, block_size // PANEL_TOKENS, self.panel_bytes

    def new_cache(self, num_blocks: int, block_size: int, device="cuda") -> torch.Tensor:
        return torch.zeros(self.cache_shape(num_blocks, block_size), dtype=torch.uint8, device=device)

    def block_size(self, cache: torch.Tensor) -> int:
        """The block size of a cache tensor of this layout; raises if it is not one."""
        shape = cache.shape
        if cache.dtype != torch.uint8 or len(shape) != 4 or not cache.is_contiguous():
            raise ValueError(f"expected a contiguous uint8 [blocks, H, block_size/16, bytes] cache, got "
                             f"{tuple(shape)} {cache.dtype}")
        if shape[1] != self.H or shape[3] != self.panel_bytes or shape[2] < 1:
            raise ValueError(f"a cache of shape {tuple(shape)} does not hold H={self.H} heads in panels of "
                             f"{self.panel_bytes} bytes")
        return shape[2] * PANEL_TOKENS
