"""Rotary positions (no reference module).

Dims f and f + r/2 of a head's first r dims (or 2f and 2f + 1, interleaved) are turned at
position t by the angle t * inv_freq[f] and scaled by a factor; the rest of the head is copied.

- ``rotary_frequencies`` computes the frequencies, as they are or stretched for contexts longer
  than the trained one;
- ``apply_rotary`` rotates dense Q and K, as the prefill entry points take them;
- ``paged_kv.append_paged_kv_rotary`` rotates the new tokens of a paged cache while it
  writes them.

The kernels (csrc/rotary.hip) form angles in 64 bits, so far positions keep their accuracy.
"""
from __future__ import annotations

import math

import torch

from . import _native as N


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, stretch=1.0, trained_len=None,
                       device="cuda"):
    """Returns (inv_freq, factor): float64 [rotary_dim / 2] on `device`, and a number.

    inv_freq[f] = base ** (-2 f / rotary_dim), and factor 1, unless `scaling` says otherwise;
    `stretch` (>= 1) is the ratio of the context to serve to the trained one:
      "linear"  every frequency divided by stretch (positions interpolated);
      "ntk"     base * stretch ** (r / (r - 2)): the last frequency is divided by stretch, the
                first keeps its value;
      "yarn"    frequencies that make fewer than 1 turn over trained_len positions are divided by
                stretch, those that make more than 32 are kept, between the two the mix is
                linear in the turns; factor 0.1 ln(stretch) + 1 (Peng et al. 2023, YaRN).
    """
    r = int(rotary_dim)
    if r <= 0 or r % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not base > 0 or not stretch >= 1:
        raise ValueError("base must be positive and stretch at least 1")
    f = torch.arange(r // 2, dtype=torch.float64)
    if scaling == "ntk":
        if r == 2:
            raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
        base = base * stretch ** (r / (r - 2))
    inv = float(base) ** (-2.0 * f / r)
    factor = 1.0
    if scaling == "linear":
        inv = inv / stretch
    elif scaling == "yarn":
        if trained_len is None or trained_len <= 0:
            raise ValueError("yarn scaling needs trained_len")
        keep = ((trained_len * inv / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        inv = inv * keep + inv / stretch * (1.0 - keep)
        factor = 0.1 * math.log(stretch) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f'scaling must be None, "linear", "ntk" or "yarn", got {scaling!r}')
    return inv.to(device), factor


def apply_rotary(Q, K, inv_freq, positions=None, interleaved=False, factor=1.0, transpose=False):
    """Returns (Q', K'): rotated contiguous copies of Q [B, Hq, S, D] and K [B, Hkv, S, D].

    Q and K are fp16 or bf16 (one type), in one launch; K may be None (K' is then None).
    inv_freq: float64 [rotary_dim / 2] on their device; positions: int32 or int64 [S] or [B, S],
    default 0 .. S - 1.  transpose=True applies the transposed map (negative angles, the same
    factor): it takes the gradient of Q' to that of Q, and undoes a rotation of factor 1.
    D is a multiple of 8 up to 1024.
    """
    return N.torch_ext().rotary(Q, K, inv_freq, positions=positions, interleaved=interleaved,
                                factor=factor, transpose=transpose)


__all__ = ["rotary_frequencies", "apply_rotary"]
