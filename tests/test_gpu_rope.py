"""GPU parity of the rotary operator against its definition in FP64.

Tolerances: a cosine or sine is off by at most 1.0e-7 (polynomials of an angle
reduced exactly and rounded to 2^-24 of an eighth of a turn, see the kernel)
and by the factor's rounding, 2^-24, together below 2^-22; 2^-21 leaves room
for the FP64 reference's own angle at positions near 2^31 (2^31 * 2^-53 < 2^-21.9).
A result adds two products of FP32 rounding:
|error| <= f (|a| + |b|) (2^-21 + 3 * 2^-24) plus half a step of the type.
"""
import pytest
import torch

import dsa_b200

pytestmark = pytest.mark.gpu


def _reference(x, positions, inv_freq, layout, start, factor, sign=1.0):
    """The definition in FP64 and the sum |a| + |b| of every element's pair."""
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    d = 2 * inv_freq.shape[0]
    part = y[..., start:start + d]
    angle = sign * positions.double().reshape(positions.shape + (1,) * (x.dim() - 2)) * inv_freq
    cos, sin = angle.cos() * factor, angle.sin() * factor
    a, b = (slice(0, None, 2), slice(1, None, 2)) if layout == "interleaved" else (slice(0, d // 2), slice(d // 2, None))
    e0, e1 = part[..., a].clone(), part[..., b].clone()
    for place, value in ((a, e0 * cos - e1 * sin), (b, e1 * cos + e0 * sin)):
        y[..., start:start + d][..., place] = value
        size[..., start:start + d][..., place] = (e0.abs() + e1.abs()) * abs(factor)
    return y, size


def _check(got, x, positions, inv_freq, layout="interleaved", start=0, factor=1.0, sign=1.0):
    ref, size = _reference(x, positions, inv_freq, layout, start, factor, sign)
    tol = size * (2.0 ** -21 + 3 * 2.0 ** -24) + ref.abs() * torch.finfo(x.dtype).eps / 2 * (size > 0) + 1e-7 * (size > 0)
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (size > 0)  # half a step of the subnormal halves
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() - tol).max())


def _make(shape, dtype, seed, far=100000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype)
    return x, torch.randint(0, far, shape[:2], generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,rotary_dim,start", [
    ((1, 1, 1, 64), 64, 0), ((3, 5, 7, 64), 64, 0), ((1, 9, 64, 128), 64, 0), ((2, 3, 16, 192), 64, 128),
    ((2, 129, 2, 96), 32, 32), ((2, 3, 5, 11), 6, 3), ((1, 1, 1, 2), 2, 0), ((2, 2, 3, 30), 30, 0), ((2, 7, 576), 64, 512),
    ((1, 2, 300, 64), 64, 0), ((3, 7000, 1, 64), 64, 0), ((2, 3000, 128), 64, 0), ((5, 999, 1, 17), 10, 3), ((2, 5, 1, 4096), 64, 64), ((70, 130, 3, 72), 64, 8), ((1, 1, 1, 1024), 1024, 0), ((2, 3, 2, 4096), 4096, 0), ((1, 2, 3, 65536), 64, 65000), ((1, 1, 40000, 66), 66, 0), ((4, 40, 128, 24), 16, 8)])
def test_rotary(cuda_lib, shape, rotary_dim, start, dtype, layout):
    x, pos = _make(shape, dtype, sum(shape))
    freq = dsa_b200.rotary_frequencies(rotary_dim, device="cuda")
    _check(dsa_b200.rotary(x, pos, freq, layout=layout, start=start), x, pos, freq, layout, start)
    y = x.clone()
    assert dsa_b200.rotary(y, pos, freq, layout=layout, start=start, out=y) is y  # in place
    _check(y, x, pos, freq, layout, start)


def test_strides_types_and_far_positions(cuda_lib):
    """Slices, transposes, odd offsets, 64-bit and negative positions, positions near 2^31, factor and inverse."""
    g = torch.Generator(device="cuda").manual_seed(5)
    row = torch.randn((3, 4, 8, 203), generator=g, device="cuda").bfloat16()
    freq = dsa_b200.rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096, device="cuda")
    pos = torch.tensor([[0, 1, -1, 2 ** 31 - 1], [7, 10 ** 6, 123456789, -2 ** 31], [4, 4, 4, 4]], device="cuda")
    for x in (row[..., :64], row[..., 3:67], row[..., 8:200:1], row.transpose(1, 2)[:, :4, :4, 8:200]):
        for p in (pos, pos.int(), pos.int().t().contiguous().t()):
            for layout in ("interleaved", "half"):
                got = dsa_b200.rotary(x, p, freq, layout=layout, attention_factor=1.25, inverse=True)
                assert got.is_contiguous()
                _check(got, x, p, freq, layout, 0, 1.25, -1.0)
    big = torch.zeros((3, 4, 8, 256), device="cuda").bfloat16()
    out = big[..., 8:136]  # a strided destination; the rest stays
    dsa_b200.rotary(row[..., :128], pos, freq, start=32, out=out)
    _check(out, row[..., :128], pos, freq, "interleaved", 32)
    assert not bool(big[..., :8].any()) and not bool(big[..., 136:].any())


def test_special_values(cuda_lib):
    """Copied elements keep their bits, NaN and infinities included; a pair's go no further than the pair."""
    x, pos = _make((2, 3, 4, 128), torch.bfloat16, 3)
    x[0, 0, 0, 100], x[0, 0, 0, 101], x[0, 0, 1, 4] = float("nan"), float("inf"), float("nan")
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    y = dsa_b200.rotary(x, pos, freq)
    assert torch.equal(y[..., 64:].view(torch.int16), x[..., 64:].view(torch.int16))
    bad = torch.isnan(y[..., :64]).nonzero().tolist()
    assert bad == [[0, 0, 1, 4], [0, 0, 1, 5]]


def test_large_offsets(cuda_lib):
    """Rows behind 2^31 elements."""
    x = torch.zeros((2, 1100000, 1, 1024), dtype=torch.bfloat16, device="cuda")
    x[1, -1] = torch.randn((1, 1024), device="cuda").bfloat16()
    pos = torch.arange(1100000, dtype=torch.int32, device="cuda").expand(2, -1)
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    keep = x[1, -1:].clone()
    dsa_b200.rotary(x, pos, freq, start=960, out=x)
    _check(x[1:, -1:], keep[None], pos[1:, -1:], freq, "interleaved", 960)
    assert not bool(x[0, -3:].any())


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient(cuda_lib, layout):
    x, pos = _make((2, 5, 3, 80), torch.float32, 9, 1000)
    freq = dsa_b200.rotary_frequencies(32, device="cuda")
    g = torch.randn_like(x)
    x.requires_grad_()
    y = dsa_b200.rotary(x, pos, freq, layout=layout, start=16, attention_factor=0.75)
    (gx,) = torch.autograd.grad(y, x, g)
    _check(gx, g, pos, freq, layout, 16, 0.75, -1.0)  # the formula: the transposed map
    # differences: the map is linear, so a step of any size gives the derivative up to FP32 rounding
    d = torch.randn_like(x)
    with torch.no_grad():
        step = (dsa_b200.rotary(x + d, pos, freq, layout=layout, start=16, attention_factor=0.75) - y).double()
    lhs, rhs = float((step * g.double()).sum()), float((gx.double() * d.double()).sum())
    assert abs(lhs - rhs) <= x.numel() * 8 * 2.0 ** -22  # 2400 terms of size <= ~8, each off by < 2^-22 relative
    # an expanded gradient, a non-contiguous one, and one through another use of the leaf
    (gs,) = torch.autograd.grad(dsa_b200.rotary(x, pos, freq, layout=layout).sum(), x)
    _check(gs, torch.ones_like(x), pos, freq, layout, 0, 1.0, -1.0)
    gt = torch.randn((80, 3, 5, 2), device="cuda").permute(3, 2, 1, 0)
    (gn,) = torch.autograd.grad(dsa_b200.rotary(x, pos, freq, layout=layout), x, gt)
    _check(gn, gt, pos, freq, layout, 0, 1.0, -1.0)
    x.grad = None
    (dsa_b200.rotary(x, pos, freq, layout=layout).square().sum() / 2).backward()
    assert torch.allclose(x.grad, x.detach(), atol=1e-5)  # |R x| = |x|: four FP32 roundings of values below ~5


def test_second_derivative(cuda_lib):
    x, pos = _make((1, 2, 2, 8), torch.float32, 2, 50)
    freq = dsa_b200.rotary_frequencies(8, device="cuda")
    x.requires_grad_()
    g = torch.randn_like(x).requires_grad_()
    (gx,) = torch.autograd.grad(dsa_b200.rotary(x, pos, freq), x, g, create_graph=True)
    v = torch.randn_like(x)
    (gg,) = torch.autograd.grad(gx, g, v)
    _check(gg, v, pos, freq)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_forward_mode(cuda_lib, layout):
    """The tangent is turned as a tensor of its own would be, contiguous or not, and zero where it is known to be zero."""
    x, pos = _make((2, 5, 3, 80), torch.float32, 9, 1000)
    t = torch.randn_like(x)
    freq = dsa_b200.rotary_frequencies(32, device="cuda")

    def turn(x):
        return dsa_b200.rotary(x, pos, freq, layout=layout, start=16, attention_factor=0.75)

    with torch.autograd.forward_ad.dual_level():
        for tangent in (t, t.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)):
            y = torch.autograd.forward_ad.unpack_dual(turn(torch.autograd.forward_ad.make_dual(x, tangent)))
            assert torch.equal(y.primal, turn(x)) and torch.equal(y.tangent, turn(t))
        zero = torch._efficientzerotensor(x.shape, device="cuda")
        y = torch.autograd.forward_ad.unpack_dual(turn(torch.autograd.forward_ad.make_dual(x, zero)))
        assert torch.equal(y.primal, turn(x)) and (y.tangent is None or not bool(y.tangent.any()))


def test_captured_with_new_positions(cuda_lib):
    x, pos = _make((4, 1, 16, 64), torch.bfloat16, 1)
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    dsa_b200.rotary(x, pos, freq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dsa_b200.rotary(x, pos, freq)
    for k in range(3):
        pos += 17 * k
        x.mul_(0.5)
        graph.replay()
        _check(y, x, pos, freq)


def test_overlap_refused(cuda_lib):
    x = torch.randn((2, 3, 4, 128), device="cuda").bfloat16()
    pos = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        dsa_b200.rotary(x[..., :64], pos, freq, out=x[..., 32:96])
