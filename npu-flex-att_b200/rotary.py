"""Rotary positions for queries and keys on hand-written sm_100a kernels.

``rotary_table`` builds the cos/sin table once (plain, or scaled for contexts
longer than a model was trained on); ``rotary_embedding`` turns q and k in one
kernel launch and is differentiable. Layouts are the attention's [B, H, S, D]
with any strides, so a projection's [B, S, H, D] output goes in as a transposed
view. No counterpart in the reference, which takes q and k as given.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

import bfa_lib as _bfa

__all__ = ["rotary_table", "rotary_embedding", "RotaryEmbedding"]


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


def _integers(t, what):
    if t.dtype == torch.int32:
        return 4
    if t.dtype == torch.int64:
        return 8
    raise ValueError(f"{what} must be int32 or int64, got {t.dtype}")


def _launch(q, k, cos, sin, positions, offsets, interleaved, inverse, out=None):
    """One bfa_rope call; q or k may be None. Returns the outputs (None for None)."""
    some = q if q is not None else k
    dev = some.device
    B, _, S, D = some.shape
    if out is None:
        qo = torch.empty_like(q) if q is not None else None
        ko = torch.empty_like(k) if k is not None else None
    else:
        qo, ko = out
    pos = pos_bytes = pos_b = pos_s = 0
    if positions is not None:
        pos, pos_bytes = positions.data_ptr(), _integers(positions, "positions")
        pos_s = positions.stride(-1)
        pos_b = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    off = off_bytes = 0
    if offsets is not None:
        off, off_bytes = offsets.data_ptr(), _integers(offsets, "offsets")
    packed = _bfa.pack_rope(
        B, q.shape[1] if q is not None else 0, k.shape[1] if k is not None else 0, S, D, 2 * cos.shape[1],
        _bfa.bfa_dtype(some.dtype), 1 if interleaved else 0, 1 if inverse else 0,
        *(_bfa.flat(q)), *(_bfa.flat(k)), *(_bfa.flat(qo)), *(_bfa.flat(ko)),
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.stride(0), pos, pos_bytes, pos_b, pos_s, off, off_bytes,
        _bfa.status_ptr(dev))
    _bfa.launch("bfa_rope", packed, dev)
    return qo, ko


class RotaryEmbedding(torch.autograd.Function):
    """Autograd over two bfa_rope calls: the gradient of a rotation is the
    transposed rotation of the gradients, so only the table and the positions
    are saved. The table gets no gradient."""

    @staticmethod
    def forward(ctx, query, key, cos, sin, positions, offsets, interleaved):
        ctx.interleaved = interleaved
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, positions, offsets)
        return _launch(query, key, cos, sin, positions, offsets, interleaved, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        cos, sin, positions, offsets = ctx.saved_tensors
        gq = gk = None
        if dq is not None or dk is not None:
            gq, gk = _launch(dq, dk, cos, sin, positions, offsets, ctx.interleaved, True)
        return gq, gk, None, None, None, None, None


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

    ``out`` (a pair like (query, key), which may be the inputs themselves)
    receives the results in place of new tensors; not differentiable.
    """
    first = query if query is not None else key
    if first is None:
        raise ValueError("rotary_embedding needs query or key")
    assert first.dim() == 4, "query and key are [B, H, S, D]"
    B, _, S, D = first.shape
    if query is not None and key is not None:
        assert key.dim() == 4 and key.shape[0] == B and key.shape[2] == S and key.shape[3] == D, \
            "query and key must agree in batch, length and head dim"
        if key.dtype != query.dtype:
            raise RuntimeError("query and key must have one dtype")
    tensors = [t for t in (query, key, cos, sin, positions, offsets) if t is not None]
    _bfa.require_cuda("rotary_embedding", tensors)
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be fp32")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.stride() != sin.stride() or (cos.shape[1] > 1 and cos.stride(1) != 1):
        raise ValueError("cos and sin must be [positions, rotary_dim / 2] of one layout with unit inner stride")
    assert 0 < 2 * cos.shape[1] <= D, "rotary_dim must be in 2..head_dim"
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the rotary table is not differentiable here")
    if positions is not None and tuple(positions.shape) not in ((S,), (B, S), (1, S)):
        raise ValueError(f"positions must be [{S}] or [{B}, {S}], got {tuple(positions.shape)}")
    if offsets is not None and (tuple(offsets.shape) != (B,) or (B > 1 and offsets.stride(0) != 1)):
        raise ValueError(f"offsets must be a contiguous [{B}], got {tuple(offsets.shape)}")
    grads = torch.is_grad_enabled() and ((query is not None and query.requires_grad) or (key is not None and key.requires_grad))
    if out is not None:
        if grads:
            raise ValueError("out= is not differentiable; call it under torch.no_grad()")
        for name, t, o in (("query", query, out[0]), ("key", key, out[1])):
            if (t is None) != (o is None) or (t is not None and (o.shape != t.shape or o.dtype != t.dtype or o.device != t.device)):
                raise ValueError(f"out for {name} must match it in shape, dtype and device")
        return _launch(query, key, cos, sin, positions, offsets, interleaved, False, out)
    if grads:
        return RotaryEmbedding.apply(query, key, cos, sin, positions, offsets, interleaved)
    return _launch(query, key, cos, sin, positions, offsets, interleaved, False)
