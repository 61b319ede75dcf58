"""A key / value cache held in 4 bits and attention over it (csrc/kv4.cuh, csrc/kv4_attn.cuh).

The bf16 caches of ``linear.attn_decode`` and its siblings (model.py:205-243 of Gu-J/TernaInfer) cost 512 bytes a token and
head; this one 144: 32 values along a head share an fp16 scale.  Sequences of a batch may have different lengths, heads 64 or 128
values.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .lib import load_host_call
from .rotary import RotaryTable

GROUP = 32                # values that share a scale
TILE = 64                 # the capacity is a multiple of this
MAX_BATCH = 65535         # sequences of a cache


@dataclass(frozen=True)
class KV4Cache:
    """Codes uint8 [B, Hkv, L, D / 2] and scales fp16 [B, Hkv, L, D / 32] of keys and values; the order of the codes in a row is
    that of the kernels (include/ternaspmm.h).  L is a multiple of 64."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self):
        B, H, L, half = self.k_codes.shape
        for t, dtype, n in ((self.k_codes, torch.uint8, half), (self.k_scales, torch.float16, half // 16), (self.v_codes, torch.uint8, half),
                            (self.v_scales, torch.float16, half // 16)):
            if t.dtype != dtype or tuple(t.shape) != (B, H, L, n) or not t.is_contiguous() or t.device != self.k_codes.device or t.data_ptr() % 16:
                raise ValueError("codes are contiguous uint8 [B, Hkv, L, D / 2], scales fp16 [B, Hkv, L, D / 32], all on one device")
        if half not in (32, 64) or L % TILE or L == 0 or H == 0 or not 0 < B <= MAX_BATCH:
            raise ValueError(f"heads have 64 or 128 values, the capacity is a multiple of {TILE} and there are 1 to {MAX_BATCH} sequences: not {2 * half}, {L}, {B}")

    @classmethod
    def empty(cls, batch: int, kv_heads: int, max_len: int, head_dim: int, device="cuda") -> "KV4Cache":
        """Room for ``max_len`` tokens in each sequence, rounded up to a multiple of 64."""
        L = -(-max_len // TILE) * TILE
        shape = (batch, kv_heads, L)
        return cls(*(torch.zeros((*shape, n), dtype=t, device=device)
                     for n, t in ((head_dim // 2, torch.uint8), (head_dim // GROUP, torch.float16)) * 2))

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def max_len(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]

    def _tensors(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, table: Optional[RotaryTable] = None) -> Optional[torch.Tensor]:
    """Writes T new tokens of every sequence: keys and values bf16 [B, T, Hkv, D] (strided views as they are) into rows start[b] .. of the
    cache, ``start`` int64 [B] or [1] on the device; of sequence b only the first counts[b], rows behind those stay as they were.  With ``table``
    keys - and queries bf16 [B, T, H, D], whose rotated form is returned - are turned by their positions first, in the same
    launch.  A sequence that does not fit into the cache, or has a token at a position that the table lacks, is not written at all,
    its queries come back as NaN, and the library's status is 1."""
    cos, sin, half = (None, None, False) if table is None else (table.cos, table.sin, table.layout == "half")
    return load_host_call().kv4_append(*cache._tensors(), k, v, start, counts, q, cos, sin, half)


def kv4_read(cache: KV4Cache, start: torch.Tensor, tokens: int, counts: Optional[torch.Tensor] = None):
    """The keys and values that rows start[b] .. start[b] + tokens - 1 stand for, bf16 [B, tokens, Hkv, D] each; zeros behind a sequence's
    counts[b]."""
    return load_host_call().kv4_read(*cache._tensors(), start, tokens, counts)


def kv4_attend(q: torch.Tensor, cache: KV4Cache, start: torch.Tensor, counts: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
    """Attention of T new tokens over the cache that holds them already: queries bf16 [B, T, H, D], rotated, H a multiple of Hkv; ``start``
    and ``counts`` as in ``kv4_append``.  The query of token t sees the keys up to position start[b] + t, below start[b] + counts[b],
    and with ``window`` only the last ``window`` of them; a query that sees none gives zeros.  ``scale`` of the scores: 1 / sqrt(D).  bf16
    [B, T, H, D].  A sequence outside of the cache gives NaN and status 1 of the library.  Scores beyond 2 x 10^7 in magnitude, where fp32 tells no
    differences of 1 apart, may give NaN.  Calls of several tokens may round the cache's keys and values to fp16: where they are beyond 65504 the
    rows that see them have NaN."""
    return load_host_call().kv4_attend(q, *cache._tensors(), start, counts, window, scale)
