"""GPU parity of shared-prefix attention against its definition in FP64.

Tolerances, with W = sum_j w_j |v_j| over a row's normalised weights and
D = 2^-23 * 44 * max_j sum_i |q_i k_i| * scale, the bound of a score's error
(36 accumulations of the MMA, each cut to FP32, and a few roundings of the
scaling): a weight is off by a factor e^(+-2D) (its score and the maximum) and
by half a BF16 step, 2^-8, for the MMA; the sum by e^(+-2D); the output rounds
once more to BF16:
  |out - ref| <= W (2^-8 + 5 D + 2^-18) + 2^-8 |ref|   (2^-18: exponentials, joins)
  |max - ref| <= D + 2^-22 |ref|,  |sum - ref| <= ref (3 D + 2^-18)
"""
import ctypes

import pytest
import torch

import dsa_b200
from dsa_b200 import _native, shared_prefix
from oracle import sparse_mla as oracle

pytestmark = pytest.mark.gpu


def _reference(q, pk, qr, pr, kv, kr, ids, used, scale):
    """FP64, query by query: (out, max, sum, W, D)."""
    batch, queries, heads, _ = q.shape
    key = torch.cat((pk, pr), -1)[0, :used, 0].double()
    out = torch.zeros((batch, queries, heads, 512), dtype=torch.float64, device=q.device)
    top = torch.full((batch, queries, heads), -float("inf"), dtype=torch.float64, device=q.device)
    total, width, slack = torch.zeros_like(top), torch.zeros_like(out), torch.zeros_like(top)
    for b in range(batch):
        for s in range(queries):
            keys = key
            if ids is not None:
                i = ids[b, s, 0].long()
                i = i[(i >= 0) & (i < kv.shape[1])]
                keys = torch.cat((key, torch.cat((kv[b, i, 0], kr[b, i, 0]), -1).double()))
            if keys.shape[0] == 0:
                continue
            row = torch.cat((q[b, s], qr[b, s]), -1).double()
            z = row @ keys.T * scale
            top[b, s] = z.max(-1).values
            w = torch.exp(z - top[b, s, :, None])
            total[b, s] = w.sum(-1)
            out[b, s] = w @ keys[:, :512] / total[b, s, :, None]
            width[b, s] = w @ keys[:, :512].abs() / total[b, s, :, None]
            slack[b, s] = (row.abs() @ keys.abs().T).max(-1).values * scale * 44 * 2.0 ** -23
    return out, top, total, width, slack


def _check(got, args, used, scale=1 / 24):
    out, top, total, width, slack = _reference(*args, used, scale)
    o, m, l = got[0].double(), got[1].double()[:, 0], got[2].double()[:, 0]
    err = (o - out).abs() - (width * (2.0 ** -8 + 5 * slack[..., None] + 2.0 ** -18) + 2.0 ** -8 * out.abs())
    assert float(err.max()) <= 0, float(err.max())
    some = total > 0
    assert bool((m[~some] == -float("inf")).all()) and bool((l[~some] == 0).all())
    assert bool(((m - top).abs()[some] <= (slack + 2.0 ** -22 * top.abs())[some]).all())
    assert bool(((l - total).abs()[some] <= (total * (3 * slack + 2.0 ** -18))[some]).all())
    assert dsa_b200.device_status() == 0


def _make(batch, queries, heads, prefix, length, topk, seed=1, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g, device="cuda").bfloat16()

    q, qr = r(batch, queries, heads, 512) * gain, r(batch, queries, heads, 64) * gain
    if not topk:
        return q, r(1, prefix, 1, 512), qr, r(1, prefix, 1, 64), None, None, None
    ids = torch.randint(0, length, (batch, queries, 1, topk), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.rand(ids.shape, generator=g, device="cuda") < 0.1] = -1
    return q, r(1, prefix, 1, 512), qr, r(1, prefix, 1, 64), r(batch, length, 1, 512), r(batch, length, 1, 64), ids


@pytest.mark.parametrize("gain", [1.0, 12.0])  # flat weights, and a few keys that take all: rescales
@pytest.mark.parametrize("batch,queries,heads,prefix,length,topk", [
    (1, 1, 16, 1, 0, 0), (1, 1, 16, 64, 0, 0), (2, 1, 128, 65, 0, 0), (1, 3, 48, 1000, 0, 0), (3, 2, 16, 1000, 300, 77),
    (1, 1, 128, 129, 7, 1), (5, 7, 32, 4097, 50, 33), (64, 1, 16, 2048, 4096, 512), (9, 1, 128, 700, 2000, 2048),
    (80, 1, 128, 200, 100, 64), (160, 1, 128, 130, 0, 0), (1, 1, 16, 30000, 1, 1), (2, 1, 144, 3000, 40, 40)])
def test_parity(cuda_lib, batch, queries, heads, prefix, length, topk, gain):
    args = _make(batch, queries, heads, prefix, length, topk, gain=gain)
    _check(dsa_b200.forward_shared_prefix(*args), args, prefix)


@pytest.mark.parametrize("rows", [1, 2, 3, 160])  # row tiles: one MMA CTA, a pair, a pair and a half, without a split
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 128, 129, 300, 1100])
def test_lengths(cuda_lib, rows, prefix):
    args = _make(rows, 1, 128, prefix, 0, 0, seed=prefix)
    _check(dsa_b200.forward_shared_prefix(*args), args, prefix)


@pytest.mark.parametrize("topk", [0, 40])
def test_filled_part(cuda_lib, topk):
    """A buffer filled in part: lengths on every side of a tile's end, NaN and infinities behind the last key; one captured
    graph serves all of them."""
    args = _make(3, 2, 32, 700, 90, topk, seed=3)
    if topk:
        args[-1][1, 1] = -1  # a query without own keys
    args[1][0, 130:] = float("nan")
    args[3][0, 130:] = float("inf")
    length = torch.zeros(1, dtype=torch.int32, device="cuda")
    dsa_b200.forward_shared_prefix(*args, prefix_len=length)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dsa_b200.forward_shared_prefix(*args, prefix_len=length)
    for n in (0, 1, 63, 64, 65, 127, 128, 130, -5):
        length.fill_(n)
        graph.replay()
        _check(got, args, max(n, 0))
    args[1][0, 130:] = 1.0
    args[3][0, 130:] = -1.0
    for n in (131, 640, 699, 700, 100000):
        length.fill_(n)
        graph.replay()
        _check(got, args, min(n, 700))


def test_filled_part_without_partials(cuda_lib):
    """Rows enough for the kernel to write the output itself (no split, no own keys)."""
    args = _make(170, 1, 128, 130, 0, 0, seed=4)
    args[1][0, 70:] = float("nan")
    for n in (0, 1, 64, 70):
        _check(dsa_b200.forward_shared_prefix(*args, prefix_len=torch.tensor([n], dtype=torch.int32, device="cuda")), args, n)


def test_scale_and_repeat(cuda_lib):
    args = _make(4, 3, 64, 5000, 300, 200, seed=5)
    first = dsa_b200.forward_shared_prefix(*args, scale=0.11)
    _check(first, args, 5000, 0.11)
    again = dsa_b200.forward_shared_prefix(*args, scale=0.11)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_in_pieces(cuda_lib, monkeypatch):
    args = _make(3, 5, 16, 900, 60, 50, seed=6)
    monkeypatch.setattr(shared_prefix, "WORKSPACE_BUDGET", 1 << 20)
    _check(dsa_b200.forward_shared_prefix(*args), args, 900)


def test_against_forward(cuda_lib):
    """The same keys through ``forward``: prefix and own rows side by side, every index named."""
    q, pk, qr, pr, kv, kr, ids = _make(2, 2, 128, 500, 300, 64, seed=7)
    got = dsa_b200.forward_shared_prefix(q, pk, qr, pr, kv, kr, ids)
    both = torch.cat((pk.expand(2, -1, -1, -1), kv), 1).contiguous(), torch.cat((pr.expand(2, -1, -1, -1), kr), 1).contiguous()
    own = torch.where(ids >= 0, ids + 500, -1)
    every = torch.cat((torch.arange(500, dtype=torch.int32, device="cuda").expand(2, 2, 1, 500), own), -1).contiguous()
    ref = dsa_b200.forward(q, both[0], qr, both[1], every)
    # two results of the bound above: twice 2^-8 (W <= ~1 here) and two BF16 roundings
    assert float((got[0].float() - ref[0].float()).abs().max()) <= 4 * 2.0 ** -8
    assert torch.allclose(got[1], ref[1], rtol=1e-5, atol=1e-5) and torch.allclose(got[2], ref[2], rtol=1e-4)


def test_other_stream_and_unequal_calls_at_once(cuda_lib):
    a, b = _make(2, 1, 16, 3000, 100, 64, seed=8), _make(1, 2, 128, 1500, 0, 0, seed=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = dsa_b200.forward_shared_prefix(*a)
    second = dsa_b200.forward_shared_prefix(*b)
    torch.cuda.synchronize()
    _check(first, a, 3000)
    _check(second, b, 1500)


@pytest.mark.parametrize("heads", [16, 48, 128])
@pytest.mark.parametrize("where", ["own", "prefix", "one own key far below"])
def test_nan_in_live_keys(cuda_lib, heads, where):
    """A NaN score makes its row NaN whichever part of the keys it lies in; the rows without one stay as they are."""
    args = _make(2, 2, heads, 4097, 300, 77, seed=1)
    q, pk, qr, pr, kv, kr, ids = args
    ids[:, :, :, 0] = 7
    if where == "own":
        kv[1] = float("nan")  # every key of the part: it has no maximum
    elif where == "prefix":
        pk[0, :2048] = float("nan")
    else:  # row (1, 0, 0): 8 |q|^2 / 24 = 8 * 576 / 24 ~ 192 for its prefix key, 0 for its own keys: e^-192 is 0 in FP32
        kv[1], kr[1] = 0, 0
        kr[1, 7] = float("nan")
        pk[0, 9, 0], pr[0, 9, 0] = q[1, 0, 0] * 8, qr[1, 0, 0] * 8
    got = dsa_b200.forward_shared_prefix(*args)
    out, _, total = got
    assert bool(out[1].isnan().all()) and bool(total[1].isnan().all())
    if where == "prefix":
        assert bool(out.isnan().all()) and bool(total.isnan().all())
    else:
        _check([t[:1] for t in got], (q[:1], pk, qr[:1], pr, kv[:1], kr[:1], ids[:1]), 4097)


@pytest.mark.parametrize("batch,heads,prefix,topk", [(160, 128, 130, 0), (2, 128, 3000, 0), (2, 16, 500, 40), (2, 128, 500, 40)])
def test_statistics_of_nan_rows(cuda_lib, batch, heads, prefix, topk):
    """Maximum -inf and sum NaN, as ``forward`` gives, whether or not the kernel writes the output itself and whatever the
    other parts hold."""
    args = _make(batch, 1, heads, prefix, 90, topk, seed=2)
    args[0][0, 0, 5] = float("nan")
    _, top, total = dsa_b200.forward_shared_prefix(*args)
    row = torch.zeros_like(top, dtype=torch.bool)
    row[0, 0, 0, 5] = True
    assert torch.equal(total.isnan(), row) and torch.equal(top == -float("inf"), row)
    args[1][0, 3] = float("nan")
    _, top, total = dsa_b200.forward_shared_prefix(*args)
    assert bool(total.isnan().all()) and bool((top == -float("inf")).all())
    if topk:
        q, _, qr, _, kv, kr, ids = args
        _, top, total = dsa_b200.forward(q, kv, qr, kr, ids)
        assert torch.equal(total.isnan(), row) and torch.equal(top == -float("inf"), row)


@pytest.mark.parametrize("heads", [16, 48, 128])
def test_nan_behind_masked_indices(cuda_lib, heads):
    """Own rows that no valid index names may hold NaN: also the first and the last row, on which masked indices fall
    (negative ones, those past the end), alone in a tile or beside valid ones."""
    args = _make(3, 2, heads, 500, 90, 77, seed=3)
    kv, kr, ids = args[4:]
    ids[ids == 0], ids[ids == 89] = 1, 88
    ids[..., 5], ids[..., 6], ids[..., 40:72] = 90, 2 ** 31 - 1, -2 ** 31
    ids[0, 1, :, 32:] = -1
    ids[2, 0] = 90
    for row, value in ((0, float("nan")), (89, float("inf"))):
        kv[:, row], kr[:, row] = value, value
    _check(dsa_b200.forward_shared_prefix(*args), args, 500)


@pytest.mark.parametrize("batch,heads,prefix,topk", [
    (2, 16, 700, 0), (2, 16, 700, 40), (2, 128, 700, 40), (3, 48, 3000, 33), (160, 128, 130, 0), (70, 128, 65, 0)])
def test_exact_scores(cuda_lib, batch, heads, prefix, topk):
    """Small whole numbers, whose products and sums are exact in FP32 in any order: the maximum is the largest score's
    rounded quotient by 24, to the last bit, whichever set of keys it lies in. A key that is in both sets has one weight:
    with every prefix key among the own ones the sum doubles and the output stays, up to the exponentials' rounding."""
    g = torch.Generator(device="cuda").manual_seed(4)

    def r(*shape):
        return torch.randint(-1, 2, shape, generator=g, device="cuda").bfloat16()

    q, pk, qr, pr = r(batch, 1, heads, 512), r(1, prefix, 1, 512), r(batch, 1, heads, 64), r(1, prefix, 1, 64)
    own = [None, None, None]
    if topk:
        ids = torch.randint(0, 90, (batch, 1, 1, topk), generator=g, device="cuda", dtype=torch.int32)
        own = [r(batch, 90, 1, 512), r(batch, 90, 1, 64), ids]
    args = (q, pk, qr, pr, *own)
    got = dsa_b200.forward_shared_prefix(*args)
    _, top, total, _, _ = _reference(*args, prefix, 1.0)  # whole scores
    assert torch.equal(got[1][:, 0].cpu(), top.float().cpu() / 24.0)
    _, _, total, _, _ = _reference(*args, prefix, 1 / 24)
    # |score| < 8 (576 products of -1, 0, 1: a standard deviation of 16 / 24): exponents below 12 of FP32 rounding, 2^-20,
    # the exponential's 2^-22 and the sum's
    assert bool(((got[2][:, 0].double() - total).abs() <= total * 2.0 ** -18).all())
    if topk:
        every = torch.arange(prefix, device="cuda", dtype=torch.int32).expand(batch, 1, 1, prefix).contiguous()
        both = dsa_b200.forward_shared_prefix(q, pk, qr, pr, pk.expand(batch, -1, -1, -1).contiguous(),
                                              pr.expand(batch, -1, -1, -1).contiguous(), every)
        alone = dsa_b200.forward_shared_prefix(q, pk, qr, pr)
        assert torch.equal(both[1], alone[1])
        assert bool(((both[2] / 2 - alone[2]).abs() <= alone[2] * 2.0 ** -17).all())


def _plan(args):
    """(row tiles per item, prefix splits, own splits) of the call."""
    a, plan = _native.FwdArgs(), (ctypes.c_int32 * 3)()
    a.batch, a.queries, a.heads = args[0].shape[:3]
    if args[6] is not None:
        a.length, a.topk = args[4].shape[1], args[6].shape[-1]
    assert _native.load().dsa_fwd_prefix_plan(a, _native.PrefixKv(None, None, None, args[1].shape[1]), plan) == 0
    return tuple(plan)


# 74 row tiles fill the clusters of two SMs and overflow those of four; 37 tiles in two splits likewise
@pytest.mark.parametrize("batch,queries,heads,prefix,split,length,topk", [
    *((74, 1, 128, n, 1, 0, 0) for n in (1, 63, 64, 65, 128, 130, 1100)), (74, 8, 16, 300, 1, 0, 0),
    (37, 1, 128, 4097, 2, 0, 0), (37, 1, 128, 8191, 2, 0, 0), (74, 1, 128, 129, 1, 60, 40), (74, 8, 16, 129, 1, 60, 40),
    (37, 1, 128, 4097, 2, 90, 77), (37, 2, 64, 4100, 2, 90, 77)])
def test_one_row_tile_per_item(cuda_lib, batch, queries, heads, prefix, split, length, topk):
    args = _make(batch, queries, heads, prefix, length, topk, seed=prefix)
    assert _plan(args)[:2] == (1, split)
    _check(dsa_b200.forward_shared_prefix(*args), args, prefix)


def test_two_row_tiles_per_item(cuda_lib):
    for shape in ((1, 1, 16, 1, 0, 0), (64, 1, 16, 2048, 4096, 512), (160, 1, 128, 130, 0, 0)):  # of test_parity
        assert _plan(_make(*shape))[0] == 2


@pytest.mark.parametrize("batch,prefix,topk", [(74, 300, 0), (37, 4200, 0), (37, 4200, 40)])
def test_filled_part_of_one_row_tile_per_item(cuda_lib, batch, prefix, topk):
    """Lengths on every side of a tile's end, none and all of the buffer, NaN and infinities behind the last key."""
    args = _make(batch, 1, 128, prefix, 90, topk, seed=6)
    assert _plan(args)[0] == 1
    if topk:
        args[6][3] = -1
    for n in (0, 1, 63, 64, 65, 130, prefix - 1, prefix):
        pk, pr = args[1].clone(), args[3].clone()
        pk[0, n:], pr[0, n:] = float("nan"), float("inf")
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        _check(dsa_b200.forward_shared_prefix(args[0], pk, args[2], pr, *args[4:], prefix_len=length), args, n)


@pytest.mark.parametrize("batch,queries,heads,prefix,length,topk", [
    (3, 2, 16, 1000, 300, 77), (5, 7, 32, 4097, 50, 33), (9, 1, 128, 700, 2000, 2048), (160, 1, 128, 130, 0, 0),
    (74, 1, 128, 1100, 0, 0), (37, 1, 128, 4097, 90, 77), (64, 1, 16, 8192, 4096, 512)])
def test_framework_gate(cuda_lib, batch, queries, heads, prefix, length, topk):
    """The framework's requirement on the statistics of every forward, 1e-5, which is tighter than the bound above: each of
    a score's accumulations loses less than 2^-23 of the partial sum, 44 * 2^-23 = 5.2e-6 if that is the final one's size.
    The output's requirement, 5e-3 of its largest element, is no bound for rounding: an output of 1.4 with W = 0.8 is off
    by up to 2^-8 (half a BF16 step in [1, 2)) + 0.8 * 2^-8 = 7.03e-3 > 5e-3 * 1.4; _check has the output's."""
    args = _make(batch, queries, heads, prefix, length, topk, seed=12)
    got = [t.float().cpu() for t in dsa_b200.forward_shared_prefix(*args)]
    out, top, total, _, _ = _reference(*args, prefix, 1 / 24)
    metrics = oracle.accuracy(got, [t.float().cpu() for t in (out, top[:, None], total[:, None])])
    for name, gate in oracle.ELEMENT_GATES.items():
        assert metrics[name]["max_normalized"] <= gate and metrics[name]["max_relative"] <= gate, (name, metrics)
