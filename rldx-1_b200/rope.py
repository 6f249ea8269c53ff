"""Rotary positions of a decoder, planned once: which part of a head is turned, how its pairs lie, which axis of the
positions each takes, and the frequencies, scaled for contexts longer than the trained ones.

    rope = B200Rope(128, theta=1e6, sections=(24, 20, 20), interleaved_sections=True)   # three axes
    q, k = rope(q, k, positions)                     # rotated heads, no table
    cos, sin = rope.rows(positions)                  # the rows that ops.qkv_rope_append reads

Scaling is a dict: {"type": "linear", "factor": s} divides every frequency; {"type": "ntk", "factor": s} raises theta so
that the slowest pair is divided by s and the fastest kept; {"type": "yarn", "factor": s, "original": n} keeps pairs
that turn more than "beta_fast" (32) times within the original length, divides those of less than "beta_slow" (1) turns, blends
between them, and multiplies cos and sin by "attention_factor" (0.1 ln s + 1).
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import ops


def frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None):
    """float64 [rotary_dim / 2] radians a position on the CPU, and the factor on cos and sin."""
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    scaling = dict(scaling or {"type": None})
    kind, s = scaling.pop("type", None), scaling.pop("factor", None)
    if kind is None and s is not None:
        raise ValueError("a scaling's factor needs its type")
    s = 1.0 if s is None else float(s)
    if not (math.isfinite(theta) and theta > 0 and math.isfinite(s) and s > 0):
        raise ValueError("theta and the scaling's factor must be positive numbers")
    m = 1.0
    if kind is None or kind == "linear":
        f = theta ** (-i / rotary_dim) / s
    elif kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs more than one pair")
        f = (theta * s ** (rotary_dim / (rotary_dim - 2))) ** (-i / rotary_dim)
    elif kind == "yarn":
        original = scaling.pop("original", None)
        fast, slow = float(scaling.pop("beta_fast", 32.0)), float(scaling.pop("beta_slow", 1.0))
        if original is None or not original > 0 or not fast >= slow > 0 or theta <= 1.0:
            raise ValueError("yarn scaling needs the original length, beta_fast >= beta_slow > 0 and theta above 1")

        def pair_of(turns):  # (a real number) that turns so often within the original length
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        share = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)  # 0: kept, 1: divided
        if pair_of(slow) < 0:  # not even the fastest pair turns so often
            share = torch.ones_like(i)
        f = theta ** (-i / rotary_dim)
        f = f / s * share + f * (1 - share)
        m = float(scaling.pop("attention_factor", 0.1 * math.log(s) + 1.0 if s > 1 else 1.0))
    else:
        raise ValueError(f"scaling type {kind!r} is not 'linear', 'ntk' or 'yarn'")
    if scaling:
        raise ValueError(f"scaling has no {sorted(scaling)}")
    return f, m


class B200Rope:
    """The plan of a head's rotation on one device.  rotary_dim: the values of a head that are turned (its first; all by
    default); interleaved: pairs are neighbours, else halves; sections and interleaved_sections as ops.rope takes them;
    freqs: float64 [rotary_dim / 2] in place of theta and scaling."""

    def __init__(self, head_dim: int, *, theta: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 sections: Optional[Sequence[int]] = None, interleaved_sections: bool = False, scaling: Optional[dict] = None,
                 freqs: Optional[torch.Tensor] = None, factor: Optional[float] = None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 2 <= self.rotary_dim <= self.head_dim or self.rotary_dim % 2 or self.rotary_dim > 1024:
            raise ValueError(f"rotary_dim must be even, 2 to head_dim and 1024, got {self.rotary_dim} of {self.head_dim}")
        if freqs is None:
            f, m = frequencies(self.rotary_dim, float(theta), scaling)
        elif scaling is not None:
            raise ValueError("freqs are given as they are: no scaling goes with them")
        else:
            f, m = freqs.detach().to(torch.float64), 1.0
            if tuple(f.shape) != (self.rotary_dim // 2,):
                raise ValueError(f"freqs must be [{self.rotary_dim // 2}], got {tuple(f.shape)}")
        self.factor = m if factor is None else float(factor)
        self.interleaved, self.interleaved_sections = bool(interleaved), bool(interleaved_sections)
        self.sections = None if sections is None else tuple(int(n) for n in sections)
        if self.sections is not None and (not 1 <= len(self.sections) <= 4 or min(self.sections) < 0 or
                                          sum(self.sections) != self.rotary_dim // 2):
            raise ValueError(f"sections must be 1 to 4 counts that add up to {self.rotary_dim // 2} pairs, got {self.sections}")
        self.freqs = f.to(device).contiguous()

    @property
    def axes(self) -> int:
        return 1 if self.sections is None else len(self.sections)

    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, *, inverse: bool = False, out_q=None, out_k=None):
        """ops.rope with this plan: q and k (or None) turned."""
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"heads of {self.head_dim} values are turned, got {q.shape[-1]}")
        return ops.rope(q, k, positions, self.freqs, sections=self.sections, interleaved_sections=self.interleaved_sections,
                        interleaved=self.interleaved, factor=self.factor, inverse=inverse, out_q=out_q, out_k=out_k)

    def rows(self, positions: torch.Tensor, dtype=torch.float32):
        """cos and sin rows [tokens, rotary_dim] for a kernel that turns halves with a table."""
        if self.interleaved:
            raise ValueError("tables of cos and sin turn halves, this plan neighbours")
        return ops.rope_rows(positions, self.freqs, sections=self.sections, interleaved_sections=self.interleaved_sections,
                             factor=self.factor, dtype=dtype)
