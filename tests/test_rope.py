"""Rotary positions on the CPU: the frequencies and the argument rules; GPU parity is in test_gpu_rope.py."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import dsa_b200
from dsa_b200 import api, rope


def test_frequencies():
    f = dsa_b200.rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0
    assert math.isclose(f[31].item(), 10000.0 ** (-62 / 64), rel_tol=1e-14)
    assert torch.equal(dsa_b200.rotary_frequencies(64, scaling="linear", factor=8.0), f / 8.0)
    ntk = dsa_b200.rotary_frequencies(64, scaling="ntk", factor=8.0)
    # the fastest pair is kept, the slowest divided by the factor: theta'^(-62/64) = theta^(-62/64) / 8
    assert ntk[0] == 1.0 and math.isclose(ntk[31].item(), f[31].item() / 8.0, rel_tol=1e-12)
    yarn = dsa_b200.rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], f[turns > 40]) and torch.equal(yarn[turns < 0.7], f[turns < 0.7] / 40.0)
    assert bool(((yarn <= f) & (yarn >= f / 40.0)).all()) and bool((yarn[1:] < yarn[:-1]).all())


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=64, theta=1.0),
                                dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, scaling="other"),
                                dict(rotary_dim=64, scaling="yarn", factor=4.0),
                                dict(rotary_dim=2, scaling="ntk", factor=4.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        dsa_b200.rotary_frequencies(**kw)


def test_rotary_refusals(monkeypatch):
    monkeypatch.setattr(api, "DEVICE_TYPE", "meta")

    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    x, pos, freq = t(2, 3, 4, 64), t(2, 3, dtype=torch.int32), t(32, dtype=torch.float64)
    for args, kw, why in [
        ((t(2, 3), pos, freq), {}, "x must be"),
        ((t(2, 0, 4, 64), t(2, 0, dtype=torch.int32), freq), {}, "x must be"),
        ((t(2, 3, 4, 64, dtype=torch.float64), pos, freq), {}, "bfloat16, float16 or float32"),
        ((x, t(2, 4, dtype=torch.int32), freq), {}, "positions"),
        ((x, pos.float(), freq), {}, "positions"),
        ((x, pos, freq.float()), {}, "float64"),
        ((x, pos, t(33, dtype=torch.float64)), {}, "start"),
        ((x, pos, t(16, dtype=torch.float64)), dict(start=33), "start"),
        ((x, pos, t(16, dtype=torch.float64)), dict(start=-1), "start"),
        ((x, pos, t(0, dtype=torch.float64)), {}, "start"),
        ((t(2, 3, 4, 4098), pos, t(2049, dtype=torch.float64)), {}, "4096"),
        ((t(2, 3, 65537), pos, freq), {}, "65536"),
        ((x, pos, freq), dict(layout="other"), "layout"),
        ((x, pos, freq), dict(attention_factor=float("nan")), "attention_factor"),
        ((t(2, 3, 64, 4).transpose(2, 3), pos, freq), {}, "last dimension"),
        ((x, pos, freq), dict(out=t(2, 3, 4, 63)), "out must"),
        ((x, pos, freq), dict(out=t(2, 3, 1, 64).expand(2, 3, 4, 64)), "out must"),
        ((x, pos, t(32, dtype=torch.float64).requires_grad_()), {}, "gradient"),
    ]:
        with pytest.raises(ValueError, match=why):
            dsa_b200.rotary(*args, **kw)
    with pytest.raises(ValueError, match="CUDA device"):
        dsa_b200.rotary(torch.empty(2, 3, 4, 64, dtype=torch.bfloat16), pos, freq)
    with pytest.raises(ValueError, match="autograd"):
        dsa_b200.rotary(t(2, 3, 4, 64).requires_grad_(), pos, t(32, dtype=torch.float64), out=t(2, 3, 4, 64))


def test_out_tells_autograd(monkeypatch):
    """A tensor that was saved for a backward pass and then turned in place: torch's error, no gradient of other values."""
    monkeypatch.setattr(api, "DEVICE_TYPE", "cpu")
    monkeypatch.setattr(api, "enqueue", lambda *args: None)
    x, w = torch.randn(2, 3, 4, 64), torch.ones(64, requires_grad=True)
    pos, freq = torch.zeros(2, 3, dtype=torch.int32), dsa_b200.rotary_frequencies(64)
    y, part = x * w, x[:, :, :2]
    assert dsa_b200.rotary(part, pos, freq, out=part) is part and x._version == 1  # a view shares its base's
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    before = x._version
    dsa_b200.rotary(x, pos, freq)
    assert x._version == before
    with torch.inference_mode():
        z = torch.zeros(2, 3, 4, 64)
    dsa_b200.rotary(z, pos, freq, out=z)  # has no version


def _plain_launch(x, positions, inv_freq, out, number, start, factor, inverse):
    """The kernel's map, interleaved pairs of whole rows."""
    t = (positions.double()[..., None, None] * inv_freq).to(x.dtype) * (-1 if inverse else 1)
    a, b = x.detach()[..., 0::2], x.detach()[..., 1::2]
    return out.copy_(factor * torch.stack((a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()), -1).flatten(-2))


def test_forward_mode(monkeypatch):
    """The tangent is turned as the primal is, alone, with a graph of the tangent, and through the backward pass."""
    monkeypatch.setattr(api, "DEVICE_TYPE", "cpu")
    monkeypatch.setattr(rope, "_launch", _plain_launch)
    x, t, g = torch.randn(3, 2, 3, 4, 64).unbind(0)
    pos, freq = torch.arange(6, dtype=torch.int32).reshape(2, 3), dsa_b200.rotary_frequencies(64)

    def turn(x, **kw):
        return dsa_b200.rotary(x, pos, freq, attention_factor=1.5, **kw)

    with forward_ad.dual_level():
        for tangent in (t, t[..., :1].expand(2, 3, 4, 64), t.transpose(2, 3).contiguous().transpose(2, 3)):
            y = forward_ad.unpack_dual(turn(forward_ad.make_dual(x, tangent)))
            assert torch.equal(y.primal, turn(x)) and torch.equal(y.tangent, turn(tangent.contiguous()))
        with torch.no_grad():
            assert torch.equal(forward_ad.unpack_dual(turn(forward_ad.make_dual(x, t))).tangent, turn(t))
        assert forward_ad.unpack_dual(turn(x)).tangent is None
        with pytest.raises(ValueError, match="autograd"), torch.no_grad():
            dual = forward_ad.make_dual(x, t)
            turn(dual, out=dual)
        # the tangent's own graph
        t.requires_grad_()
        dot = forward_ad.unpack_dual(turn(forward_ad.make_dual(x, t))).tangent
        (gt,) = torch.autograd.grad(dot, t, g)
        assert torch.equal(gt, turn(g, inverse=True))
        # the gradient's tangent: that of its own input
        leaf = x.clone().requires_grad_()
        (gx,) = torch.autograd.grad(turn(leaf), leaf, forward_ad.make_dual(g, t.detach()))
        assert torch.equal(forward_ad.unpack_dual(gx).tangent, turn(t.detach(), inverse=True))
