"""Rotary positions, host side: the table and the refusals (CPU only)."""
import math

import pytest
import torch

import rotary


def test_table_is_formed_in_64_bits():
    cos, sin = rotary.rotary_table(64, 100001, base=10000.0)
    assert cos.shape == (100001, 32) and cos.dtype == torch.float32 and sin.is_contiguous()
    for t, i in ((0, 0), (1, 31), (77777, 0), (100000, 17)):
        angle = t * 10000.0 ** (-2 * i / 64)
        # One rounding to fp32 of a value of at most 1.
        assert abs(cos[t, i].item() - math.cos(angle)) <= 2 ** -24
        assert abs(sin[t, i].item() - math.sin(angle)) <= 2 ** -24


def _angles(**kw):
    """Position 1's angles: the frequencies (all below pi)."""
    cos, sin = rotary.rotary_table(32, 2, **kw)
    return torch.atan2(sin[1].double(), cos[1].double()), (cos[1].double() ** 2 + sin[1].double() ** 2).sqrt()


def test_scaled_tables():
    plain, _ = _angles()
    linear, _ = _angles(scaling="linear", factor=4.0)
    # atan2 of two fp32 values: relative error a few 2^-24.
    assert torch.allclose(linear, plain / 4, rtol=1e-6, atol=0)
    ntk, _ = _angles(scaling="ntk", factor=4.0)
    assert torch.allclose(ntk[:1], plain[:1], rtol=1e-6) and torch.allclose(ntk[-1:], plain[-1:] / 4, rtol=1e-6)
    yarn, size = _angles(scaling="yarn", factor=4.0, original_positions=64, beta_fast=8.0, beta_slow=1.0)
    turns = 64 * plain / (2 * math.pi)
    assert torch.allclose(yarn[turns > 8], plain[turns > 8], rtol=1e-6)
    assert torch.allclose(yarn[turns < 1], plain[turns < 1] / 4, rtol=1e-6)
    between = (turns > 1) & (turns < 8)
    assert between.any() and (yarn[between] < plain[between]).all() and (yarn[between] > plain[between] / 4).all()
    assert torch.allclose(size, torch.full_like(size, 0.1 * math.log(4.0) + 1.0), rtol=1e-6)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(positions=-1), dict(scaling="cubic"),
                                dict(base=0.0), dict(factor=0.0), dict(scaling="yarn", beta_fast=1.0, beta_slow=2.0)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        rotary.rotary_table(**dict(dict(rotary_dim=8, positions=4), **kw))


def test_cpu_tensors_are_refused():
    cos, sin = rotary.rotary_table(64, 16)
    q = torch.randn(1, 2, 16, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary.rotary_embedding(q, None, cos, sin)
    with pytest.raises(ValueError, match="query or key"):
        rotary.rotary_embedding(None, None, cos, sin)
    with pytest.raises(AssertionError):
        rotary.rotary_embedding(q, torch.randn(1, 2, 15, 64), cos, sin)


def test_tangents_are_refused():
    """Forward-mode differentiation would lose the tangent without a word."""
    import torch.autograd.forward_ad as fwd
    cos, sin = rotary.rotary_table(64, 16)
    q, k = torch.randn(1, 2, 16, 64), torch.randn(1, 1, 16, 64)
    with fwd.dual_level():
        for args in ((fwd.make_dual(q, torch.ones_like(q)), k, cos, sin), (None, fwd.make_dual(k, torch.ones_like(k)), cos, sin),
                     (q, k, fwd.make_dual(cos, torch.ones_like(cos)), sin)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                rotary.rotary_embedding(*args)
