"""Rotary positions on part of each head.

* ``rotary_frequencies(rot, ...)``: radians per position of each channel pair,
  plain, linearly stretched or stretched by wavelength ("yarn"), in float64;
  made once and kept.
* ``rotary(x, positions, freqs, ...)``: the rotated copy, differentiable in x in
  backward and forward mode.
* ``rotary_(x, positions, freqs, ...)``: in place, touching the rotated
  channels only; what a serving loop calls on its queries and, with
  ``inverse=True``, on the attention's output.

The cache rows are rotated where they are written: ``kv_cache.append``.
"""

from __future__ import annotations

import math

import torch

from . import ops


def rotary_frequencies(rot: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_len: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device=None) -> torch.Tensor:
    """float64 [rot/2] radians per position: ``base ** (-2i/rot)``.

    ``scaling="linear"`` divides every frequency by ``factor``.  ``"yarn"``
    divides by ``factor`` the pairs that turn less than ``beta_slow`` times in
    ``original_len`` positions, keeps those that turn more than ``beta_fast``
    times, and blends linearly over the pair index in between."""
    if rot <= 0 or rot % 2:
        raise ValueError("rot must be a positive even number of channels")
    if scaling not in ("none", "linear", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}: none, linear or yarn")
    if not base > 1 or not factor > 0:
        raise ValueError("base must be above 1 and factor above 0")
    pair = torch.arange(rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * pair / rot)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair_of(turns: float) -> float:  # the pair that turns so often in original_len positions
            return rot * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rot - 1)
        ramp = ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    return f.to(device if device is not None else "cuda")


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, interleaved: bool = True,
           offset: int | None = None, inverse: bool = False, amplitude: float = 1.0) -> torch.Tensor:
    """x [..., heads, dim] (bf16, fp16 or fp32, any strides) with the pairs of the
    ``2 * len(freqs)`` channels from ``offset`` on (default: the last ones)
    turned by ``positions * freqs``, times ``amplitude``; positions [...] (or flat)
    int32 or int64.  ``inverse`` turns back (the transposed map).  Differentiable in x,
    not in freqs."""
    return ops.load().rotary(x, positions, freqs, interleaved, offset, inverse, float(amplitude))


def rotary_(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, interleaved: bool = True,
            offset: int | None = None, inverse: bool = False, amplitude: float = 1.0) -> torch.Tensor:
    """``rotary`` in place on x (contiguous in its last dimension, not
    overlapping itself, no gradient); returns x."""
    ops.load().rotary_(x, positions, freqs, interleaved, offset, inverse, float(amplitude))
    return x
