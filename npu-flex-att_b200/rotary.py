"""Rotary positions for queries and keys on hand-written sm_100a kernels.

``rotary_table`` builds the cos/sin table once (plain, or scaled for contexts
longer than a model was trained on); ``rotary_embedding`` turns q and k in one
kernel launch and is differentiable (any number of times). Layouts are the attention's [B, H, S, D]
with any strides, so a projection's [B, S, H, D] output goes in as a transposed
view. No counterpart in the reference, which takes q and k as given.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

import bfa_lib as _bfa
from npu_flash_attention import _CHECK_STATUS, check_device_status

__all__ = ["rotary_table", "rotary_embedding"]

_module = None


def _binding():
    global _module
    if _module is None:
        _module = _bfa.binding()
    return _module


def rotary_table(rotary_dim: int, positions: int, base: float = 10000.0, *, scaling: Optional[str] = None,
                 factor: float = 1.0, original_positions: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device=None):
    """(cos, sin), fp32 [positions, rotary_dim / 2], of position * frequency.

    Angles are formed in 64 bits: at position 10^6 a 32-bit product would be off
    by up to 0.06 rad. Pair i turns with frequency base^(-2i / rotary_dim).
    ``scaling`` stretches the table over ``factor`` times the trained length:
      "linear"  every frequency divided by factor (positions compressed);
      "ntk"     base raised so that the slowest pair is stretched by factor and
                the fastest stays as it is;
      "yarn"    by wavelength: pairs that turn more than beta_fast times within
                ``original_positions`` stay, those that turn less than beta_slow
                times are divided by factor, with a linear ramp between, and the
                table carries 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if positions < 0 or not base > 0 or not factor > 0:
        raise ValueError("positions must be >= 0, base and factor > 0")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r} (None, 'linear', 'ntk' or 'yarn')")
    if scaling == "yarn" and not beta_fast > beta_slow:
        raise ValueError("beta_fast must exceed beta_slow")
    m = 1.0
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / max(1, rotary_dim - 2))
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        turns = original_positions * freq / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        m = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return (angle.cos() * m).float().contiguous(), (angle.sin() * m).float().contiguous()


def rotary_embedding(query, key, cos, sin, positions=None, offsets=None, *, interleaved=False, out=None):
    """(query', key') with rotary positions applied; differentiable.

    query [B, Hq, S, D] and key [B, Hkv, S, D] (or None), any strides, one of
    fp32 / fp16 / bf16. cos, sin: fp32 [P, R/2], unit inner stride; R <= D dims
    turn, the rest is copied. Row s of sequence b stands at
    offsets[b] + positions[b, s]: ``positions`` int32/int64 [S] or [B, S]
    (default 0..S-1), ``offsets`` int32/int64 [B] (default 0; a decoding step's
    cached lengths). Pairs are (x[i], x[i + R/2]), or with ``interleaved``
    (x[2i], x[2i+1]). A position outside the table gives NaN rows and is
    reported by ``check_device_status``.

    ``out`` (a pair like (query, key), which may be the inputs themselves but may
    not overlap them, or itself, in another way) receives the results in place
    of new tensors; not differentiable.
    """
    pair = _binding().rotary_embedding(query, key, cos, sin, positions, offsets, bool(interleaved), out)
    if _CHECK_STATUS:
        check_device_status((query if query is not None else key).device)
    return pair
