"""A key / value cache held in 4 bits and attention over it (csrc/kv4.cuh, csrc/kv4_attn.cuh).

The bf16 caches of ``linear.attn_decode`` and its siblings (model.py:205-243 of Gu-J/TernaInfer) cost 512 bytes a token and
head; this one 144: 32 values along a head share an fp16 scale.  Sequences of a batch may have different lengths, heads 64 or 128
values.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from .lib import load_library
from .linear import _on, _stream
from .rotary import RotaryTable

GROUP = 32                # values that share a scale
TILE = 64                 # the capacity is a multiple of this


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
        if half not in (32, 64) or L % TILE or L == 0 or B == 0 or H == 0:
            raise ValueError(f"heads have 64 or 128 values and the capacity is a multiple of {TILE}: not {2 * half}, {L}")

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

    def _ptrs(self):
        return self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(), self.v_scales.data_ptr(), self.max_len


def _check(cache: KV4Cache, name: str, x: Optional[torch.Tensor], heads: Optional[int]):
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs CUDA tensors: the B200 library has no CPU path")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: the 4-bit cache has none")
    if (x.dim() != 4 or x.dtype != torch.bfloat16 or x.device != cache.k_codes.device or x.shape[0] != cache.batch or x.shape[3] != cache.head_dim
            or x.shape[2] == 0 or (heads is not None and x.shape[2] != heads)):
        raise ValueError(f"{name}: bf16 [{cache.batch}, T, {heads or 'heads'}, {cache.head_dim}] on {cache.k_codes.device} wanted, not {x.dtype} {list(x.shape)} on {x.device}")


def _check_places(cache: KV4Cache, start: torch.Tensor, counts: Optional[torch.Tensor]):
    for name, t, sizes in (("start", start, (1, cache.batch)), ("counts", counts, (cache.batch,))):
        if t is not None and (t.dtype != torch.int64 or t.dim() != 1 or t.shape[0] not in sizes or not t.is_contiguous() or t.device != cache.k_codes.device):
            raise ValueError(f"{name} is contiguous int64 [{cache.batch}] on {cache.k_codes.device}, not {t.dtype} {list(t.shape)}")


def _aligned(x: torch.Tensor, to: int):
    """x with contiguous heads whose rows start on multiples of ``to`` bytes."""
    ok = x.stride(3) == 1 and x.data_ptr() % to == 0 and all(s % (to // 2) == 0 for s in x.stride()[:3])
    return x if ok else x.contiguous()


def _strides(t: torch.Tensor):
    return (ctypes.c_longlong * 3)(*t.stride()[:3])


def _raise(status: int, name: str):
    if status:
        raise RuntimeError(f"{name}: status {status}")


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, table: Optional[RotaryTable] = None) -> Optional[torch.Tensor]:
    """Writes T new tokens of every sequence: keys and values bf16 [B, T, Hkv, D] (strided views as they are) into rows start[b] .. of the
    cache, ``start`` int64 [B] or [1] on the device; of sequence b only the first counts[b], rows behind those stay as they were.  With ``table``
    keys - and queries bf16 [B, T, H, D], whose rotated form is returned - are turned by their positions first, in the same
    launch.  A sequence that does not fit is not written, and the library's status is 1."""
    _check(cache, "k", k, cache.kv_heads)
    _check(cache, "v", v, cache.kv_heads)
    if v.shape != k.shape:
        raise ValueError(f"k and v have one shape, not {list(k.shape)} and {list(v.shape)}")
    _check_places(cache, start, counts)
    if table is not None and (table.rotary_dim > cache.head_dim or table.cos.device != k.device):
        raise ValueError(f"the table rotates {table.rotary_dim} values on {table.cos.device}, a head has {cache.head_dim} on {k.device}")
    B, T = k.shape[:2]
    out = None
    if q is not None:
        if table is None:
            raise ValueError("queries are only passed to be rotated: table is missing")
        _check(cache, "q", q, None)
        if q.shape[1] != T:
            raise ValueError(f"{q.shape[1]} queries beside {T} keys")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        q = _aligned(q, 8)
    if T == 0:
        return out
    k, v = _aligned(k, 8), _aligned(v, 8)
    with _on(k):
        _raise(load_library().ternaspmm_kv4_append(
            *cache._ptrs(), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), None if q is None else q.data_ptr(), None if q is None else _strides(q),
            None if q is None else out.data_ptr(), None if table is None else table.cos.data_ptr(), None if table is None else table.sin.data_ptr(),
            0 if table is None else table.max_len, 0 if table is None else table.rotary_dim, table is not None and table.layout == "half",
            start.data_ptr(), start.shape[0] > 1, None if counts is None else counts.data_ptr(), B, T, 0 if q is None else q.shape[2],
            cache.kv_heads, cache.head_dim, _stream()), "kv4_append")
    return out


def kv4_read(cache: KV4Cache, start: torch.Tensor, tokens: int, counts: Optional[torch.Tensor] = None):
    """The keys and values that rows start[b] .. start[b] + tokens - 1 stand for, bf16 [B, tokens, Hkv, D] each; zeros behind a sequence's
    counts[b]."""
    _check_places(cache, start, counts)
    if tokens < 0:
        raise ValueError(f"{tokens} tokens")
    if not cache.k_codes.is_cuda:
        raise RuntimeError("kv4_read needs CUDA tensors: the B200 library has no CPU path")
    k, v = (torch.empty((cache.batch, tokens, cache.kv_heads, cache.head_dim), dtype=torch.bfloat16, device=cache.k_codes.device) for _ in range(2))
    if tokens:
        with _on(k):
            _raise(load_library().ternaspmm_kv4_read(*cache._ptrs(), start.data_ptr(), start.shape[0] > 1, None if counts is None else counts.data_ptr(),
                                                     k.data_ptr(), v.data_ptr(), cache.batch, tokens, cache.kv_heads, cache.head_dim, _stream()), "kv4_read")
    return k, v


def kv4_attend(q: torch.Tensor, cache: KV4Cache, start: torch.Tensor, counts: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None) -> torch.Tensor:
    """Attention of T new tokens over the cache that holds them already: queries bf16 [B, T, H, D], rotated, H a multiple of Hkv; ``start``
    and ``counts`` as in ``kv4_append``.  The query of token t sees the keys up to position start[b] + t, below start[b] + counts[b],
    and with ``window`` only the last ``window`` of them; a query that sees none gives zeros.  ``scale`` of the scores: 1 / sqrt(D).  bf16
    [B, T, H, D].  A sequence outside of the cache gives NaN and status 1 of the library."""
    _check(cache, "q", q, None)
    _check_places(cache, start, counts)
    B, T, H, D = q.shape
    if H % cache.kv_heads:
        raise ValueError(f"{H} query heads over {cache.kv_heads} key heads")
    scale = D ** -0.5 if scale is None else float(scale)
    if window < 0 or window >= 1 << 31 or not 0 < scale <= 1e6:
        raise ValueError(f"window {window}, scale {scale}")
    out = torch.empty((B, T, H, D), dtype=torch.bfloat16, device=q.device)
    if T == 0:
        return out
    q = _aligned(q, 16)
    lib = load_library()
    with _on(q):
        need = lib.ternaspmm_kv4_attend_workspace(B, T, H, cache.kv_heads, D, cache.max_len)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        _raise(lib.ternaspmm_kv4_attend(q.data_ptr(), _strides(q), *cache._ptrs(), start.data_ptr(), start.shape[0] > 1,
                                        None if counts is None else counts.data_ptr(), window, scale, out.data_ptr(), B, T, H, cache.kv_heads, D,
                                        None if work is None else work.data_ptr(), max(need, 0), _stream()), "kv4_attend")
    return out
