"""Rotary positions of the rope parts and of the indexer's queries and keys.

``rotary(x, positions, inv_freq)`` turns pairs of elements of every head row
by the token's position; ``rotary_frequencies`` builds ``inv_freq``, plain or
scaled for long contexts. The reference takes ``q_rope`` and ``k_rope`` as
already turned (its forward only adds their product to the scores); these are
the tensors that a model makes with this operator.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _native, api

_POSITIONS = (torch.int32, torch.int64)
_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_FP16, torch.float32: _native.DTYPE_FP32}


def rotary_frequencies(rotary_dim, theta=10000.0, *, scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                       beta_slow=1.0, device=None):
    """FP64 ``[rotary_dim / 2]`` radians per position: ``theta ** (-2i / rotary_dim)``.

    ``scaling`` stretches them for contexts ``factor`` times as long:
    ``"linear"`` divides every frequency by ``factor``; ``"ntk"`` raises
    ``theta`` to ``theta * factor ** (d / (d - 2))``, which keeps the fastest
    frequency and divides the slowest by ``factor``; ``"yarn"`` (Peng et al.,
    2023) divides those that turn less than ``beta_slow`` times over
    ``original_length`` tokens, keeps those that turn more than ``beta_fast``
    times and blends linearly over the pair index in between. YaRN's factor on
    the cosines is ``rotary``'s ``attention_factor``.
    """
    if type(rotary_dim) is not int or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even int")
    if not (theta > 1.0 and math.isfinite(theta)) or not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("theta must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs rotary_dim of at least 4")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = theta ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_length is None or original_length <= 0 or not 0 < beta_slow < beta_fast:
            raise ValueError("yarn scaling needs original_length > 0 and 0 < beta_slow < beta_fast")

        def pair_index(turns):  # the (real-valued) pair that makes `turns` turns over original_length
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo = max(math.floor(pair_index(beta_fast)), 0)
        hi = min(math.ceil(pair_index(beta_slow)), rotary_dim - 1)
        stretched = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        freq = freq / factor * stretched + freq * (1.0 - stretched)
    return freq if device is None else freq.to(device)


def _overlaps_itself(t):
    """Whether two elements of ``t`` may share memory (a dimension's step does not clear the smaller ones)."""
    reach = 0
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


def _check_rope(positions, inv_freq, layout, attention_factor, lead, index):
    """The rope arguments of tokens of shape ``lead`` on device ``index``; the layout's number at the C ABI."""
    number = _native.ROPE_LAYOUTS.get(layout)
    if number is None:
        raise ValueError("layout must be 'interleaved' or 'half'")
    if not isinstance(attention_factor, (float, int)) or isinstance(attention_factor, bool) or not math.isfinite(attention_factor):
        raise ValueError("attention_factor must be a finite number")
    if positions.shape != lead or positions.dtype not in _POSITIONS:
        raise ValueError("positions must be int32 or int64 and have one entry per token")
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous 1-D float64 tensor (FP32 frequencies lose far positions)")
    if positions.get_device() != index or inv_freq.get_device() != index:
        raise ValueError("all inputs must be on the same CUDA device")
    if inv_freq.requires_grad:
        raise ValueError("inv_freq gets no gradient")
    return number


def _rows_like(x):
    """A contiguous tensor of the shape of ``x`` (half the host time of ``torch.empty``)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _launch(x, positions, inv_freq, out, number, start, factor, inverse):
    p0, p1 = positions.stride()
    if x.dim() == 4:
        batch, queries, heads, dim = x.shape
        x0, x1, x2, _ = x.stride()
        y0, y1, y2, _ = out.stride()
    else:
        batch, queries, dim = x.shape
        x0, x1, _ = x.stride()
        y0, y1, _ = out.stride()
        heads, x2, y2 = 1, 0, 0
    api.enqueue("dsa_rotary", _native.RotaryArgs(
        x.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), batch, queries, heads, dim,
        x0, x1, x2, y0, y1, y2, p0, p1, 2 * inv_freq.shape[0], start, _DTYPES[x.dtype],
        positions.dtype is torch.int64, number, inverse, factor), x.get_device())
    return out


def _followed(x):
    """Whether autograd follows what becomes of ``x``: backwards, or forwards as the primal of a dual tensor."""
    return ((x.requires_grad and torch.is_grad_enabled())
            or (forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None))


def _turn(x, positions, inv_freq, number, start, factor, inverse):
    """The rotation of ``x`` as a new tensor, with its derivatives where autograd follows it."""
    if _followed(x):
        return _Rotary.apply(x, (positions, inv_freq, number, start, factor, inverse))
    return _launch(x, positions, inv_freq, _rows_like(x), number, start, factor, inverse)


class _Rotary(torch.autograd.Function):
    """The rotation is linear with an orthogonal matrix times the factor: its gradient is the inverse rotation, its
    forward-mode derivative the rotation itself."""

    @staticmethod
    def forward(ctx, x, turn):  # one argument beside x: every further one costs the engine host time
        positions, inv_freq, *how = turn
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = how
        ctx.turn = turn if forward_ad._current_level >= 0 else None  # for jvp, which follows at once
        return _launch(x, positions, inv_freq, _rows_like(x), *how)

    @staticmethod
    def jvp(ctx, tangent, _):
        turn, ctx.turn = ctx.turn, None
        if tangent._is_zerotensor():  # no memory behind it
            return torch.zeros(tangent.shape, dtype=tangent.dtype, device=tangent.device)
        return _turn(tangent if tangent.stride(-1) == 1 else tangent.contiguous(), *turn)

    @staticmethod
    def backward(ctx, grad):
        positions, inv_freq = ctx.saved_tensors
        number, start, factor, inverse = ctx.how
        if grad.stride(-1) != 1:
            grad = grad.contiguous()
        return _turn(grad, positions, inv_freq, number, start, factor, not inverse), None


def rotary(x, positions, inv_freq, *, layout="interleaved", start=0, attention_factor=1.0, inverse=False, out=None):
    """Turn ``2 * len(inv_freq)`` elements of every row of ``x`` by its position.

    ``x`` is ``[B, S, H, D]`` (``q_rope``, the indexer's queries) or
    ``[B, S, D]`` (the indexer's keys), BF16, FP16 or FP32, of any strides
    with the last dimension contiguous; ``positions`` int32 or int64
    ``[B, S]``; ``inv_freq`` FP64 (``rotary_frequencies``). With
    ``t = position * inv_freq[i]`` each pair becomes
    ``f (a cos t - b sin t), f (b cos t + a sin t)``, ``f`` the
    ``attention_factor``: the pairs are elements ``start + 2i, start + 2i + 1``
    (``layout="interleaved"``) or ``start + i, start + i + len(inv_freq)``
    (``"half"``). Elements outside ``[start, start + 2 len(inv_freq))`` are
    copied. ``inverse`` turns back by ``-t`` (still times ``f``).

    Returns a new contiguous tensor, or ``out`` (same shape and type; ``x``
    itself for an update in place; autograd learns of the write, as of torch's
    own in-place operations). Without ``out`` the call is differentiable in
    ``x``, backwards and in forward mode; a derivative is one launch of the same
    kernel. Angles are reduced exactly (64-bit fractions of a turn), cosines and
    products are FP32, rounded once to the type of ``x``; frequencies and the
    factor are finite.
    """
    shape = x.shape
    if len(shape) not in (3, 4) or 0 in shape:
        raise ValueError("x must be [B,S,H,D] or [B,S,D] with positive sizes")
    if x.dtype not in _DTYPES:
        raise ValueError("x must be bfloat16, float16 or float32")
    device = x.device
    if device.type != api.DEVICE_TYPE:
        raise ValueError("all inputs must be on the same CUDA device")
    number = _check_rope(positions, inv_freq, layout, attention_factor, shape[:2], x.get_device())
    turned, dim = 2 * inv_freq.shape[0], shape[-1]
    if type(start) is not int or start < 0 or turned == 0 or start + turned > dim:
        raise ValueError("need 0 <= start and start + 2 * len(inv_freq) <= D")
    if turned > 4096 or dim > 65536:
        raise ValueError("at most 4096 turned elements of a row of at most 65536")
    if x.stride(-1) != 1:
        raise ValueError("the last dimension of x must be contiguous")
    inverse = bool(inverse)
    if out is None:
        return _turn(x, positions, inv_freq, number, start, attention_factor, inverse)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != device or out.stride(-1) != 1 or _overlaps_itself(out):
        raise ValueError("out must have the shape, type and device of x and rows that do not overlap")
    if _followed(x) or _followed(out):
        raise ValueError("out does not take part in autograd: leave it out, or call under torch.no_grad()")
    same = out.data_ptr() == x.data_ptr() and all(n == 1 or a == b for n, a, b in zip(x.shape, x.stride(), out.stride()))
    if not same and device.type == "cuda" and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr() \
            and not _apart(x, out):
        raise ValueError("out must be x itself or not overlap it")
    _launch(x, positions, inv_freq, out, number, start, attention_factor, inverse)
    torch.autograd.graph.increment_version(out)
    return out


def _apart(a, b):
    """Whether the address ranges of two tensors do not meet."""
    def ends(t):
        last = sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a1 <= b0 or b1 <= a0
