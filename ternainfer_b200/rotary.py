"""Rotary positions: tables of the angles and the kernel that turns queries and keys by them.

``linear.rope`` and the attention kernels rotate adjacent pairs of a whole head of 128 by the reference's unscaled angles
(model.py:205-243 of Gu-J/TernaInfer).  Here are the other forms that checkpoints are trained with: pairs of the two halves, a
part of the head, and angles scaled for contexts longer than the trained ones.  Kernel: csrc/rotary.cuh; call site: csrc/host_operators.cpp.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from .lib import load_host_call

LAYOUTS = ("interleaved", "half")


@dataclass(frozen=True)
class RotaryTable:
    """cos, sin: fp32 [max_len, rotary_dim / 2], contiguous, on one device; pairs (2i, 2i+1) of a head's first rotary_dim values
    ("interleaved") or (i, i + rotary_dim / 2) ("half")."""
    cos: torch.Tensor
    sin: torch.Tensor
    layout: str = "interleaved"

    def __post_init__(self):
        if self.layout not in LAYOUTS:
            raise ValueError(f"layout is one of {LAYOUTS}, not {self.layout!r}")
        for t in (self.cos, self.sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape != self.cos.shape or not t.is_contiguous() or t.numel() == 0 or t.device != self.cos.device:
                raise ValueError("cos and sin are contiguous fp32 tensors [max_len, rotary_dim / 2] of one device")

    @property
    def rotary_dim(self) -> int:
        return 2 * self.cos.shape[1]

    @property
    def max_len(self) -> int:
        return self.cos.shape[0]


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None, device="cpu"):
    """(angle per position of every pair, float64 [rotary_dim / 2]; factor of cosines and sines).  ``scaling``:
    None, or a dict with "type" and "factor" (how many times longer the context is than the trained one):
      linear      every angle divided by factor
      ntk         theta raised so that the slowest pair turns `factor` times slower and the fastest as before
      yarn        pairs that turn more than beta_fast (32) times over original_len as before, those with fewer than beta_slow (1) turns divided
                  by factor, a ramp over the pairs between; cosines and sines times 0.1 ln(factor) + 1
      wavelength  pairs with more than `high` (4) turns over original_len as before, those with fewer than `low` (1) divided by factor,
                  mixed by their number of turns between."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim is even and at least 2, not {rotary_dim}")
    if not theta > 0:
        raise ValueError(f"theta is above 0, not {theta}")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    inv = theta ** (-2 * pair / rotary_dim)
    if scaling is None:
        return inv, 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 0))
    known = {"linear": (), "ntk": (), "yarn": ("original_len", "beta_fast", "beta_slow"), "wavelength": ("original_len", "low", "high")}
    if kind not in known or not factor > 0:
        raise ValueError(f"scaling has a type of {tuple(known)} and a factor above 0: {scaling}")
    if extra := set(scaling) - {"type", "factor", *known[kind]}:
        raise ValueError(f"{kind} scaling does not know {sorted(extra)}")
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        return (theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2 * pair / rotary_dim), 1.0
    if "original_len" not in scaling:
        raise ValueError(f"{kind} scaling needs original_len")
    length = float(scaling["original_len"])
    if not length > 0:
        raise ValueError(f"original_len is above 0, not {length}")
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not fast >= slow > 0 or theta == 1:
            raise ValueError(f"yarn scaling needs beta_fast >= beta_slow > 0 and a theta other than 1, not {fast}, {slow}, {theta}")

        def pair_with(turns):                # index of the pair that turns so often over the original length
            return rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair_with(fast)), 0), min(math.ceil(pair_with(slow)), rotary_dim - 1)
        ramp = ((pair - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
    if not high > low:
        raise ValueError("wavelength scaling needs high > low")
    keep = ((length * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return inv * keep + inv / factor * (1 - keep), 1.0


def rotary_table(head_dim: int, max_len: int, theta: float = 10000.0, *, rotary_dim: Optional[int] = None, layout: str = "interleaved",
                 scaling: Optional[dict] = None, device="cuda") -> RotaryTable:
    """Cosines and sines of positions 0 .. max_len - 1, computed in 64 bits (an fp32 angle of position 131072 is off by 0.004).
    ``rotary_dim``: how much of a head is rotated (all of it)."""
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    if rotary_dim > head_dim or max_len < 1:
        raise ValueError(f"rotary_dim {rotary_dim} of a head of {head_dim}, {max_len} positions")
    inv, factor = rotary_frequencies(rotary_dim, theta, scaling, device)
    angle = torch.arange(max_len, dtype=torch.float64, device=device)[:, None] * inv
    return RotaryTable((angle.cos() * factor).float(), (angle.sin() * factor).float(), layout)


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], table: RotaryTable, positions: torch.Tensor):
    """Queries [B, T, H, D] and keys [B, T, Hkv, D] (or None) turned by the angles of their positions, in one launch: (q, k) of the same type
    (bf16, fp16 or fp32), products in fp32, rounded once.  ``positions``: int64 [T] or [B, T] on the device.  Strided views are taken as
    they are.  Differentiable in q and k.  A position outside of the table gives NaN in its token and status 1 of the library."""
    return load_host_call().rotate(q, k, table.cos, table.sin, table.layout == "half", positions)
