"""Shared-prefix attention on the CPU: argument rules and workspace query; GPU parity is in test_gpu_shared_prefix.py."""
import ctypes

import pytest
import torch

import dsa_b200
from dsa_b200 import _native, api


def t(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_refusals(monkeypatch):
    monkeypatch.setattr(api, "DEVICE_TYPE", "meta")
    i32 = torch.int32
    q, qr, pk, pr = t(2, 3, 16, 512), t(2, 3, 16, 64), t(1, 50, 1, 512), t(1, 50, 1, 64)
    kv, kr, ids = t(2, 9, 1, 512), t(2, 9, 1, 64), t(2, 3, 1, 5, dtype=i32)
    for args, kw, why in [
        ((q[0], pk, qr, pr), {}, "4-D"), ((q, pk[0], qr, pr), {}, "4-D"),
        ((t(2, 3, 16, 256), pk, qr, pr), {}, "need q"), ((t(2, 0, 16, 512), pk, t(2, 0, 16, 64), pr), {}, "need q"),
        ((q, t(2, 50, 1, 512), qr, pr), {}, "need q"), ((q, pk, qr, t(1, 49, 1, 64)), {}, "need q"),
        ((q, t(1, 0, 1, 512), qr, t(1, 0, 1, 64)), {}, "need q"),
        ((t(2, 3, 8, 512), pk, t(2, 3, 8, 64), pr), {}, "multiple of 16"),
        ((q, pk, qr, pr, kv), {}, "go together"), ((q, pk, qr, pr, kv, kr), {}, "go together"),
        ((q, pk, qr, pr, t(3, 9, 1, 512), kr, ids), {}, "need kv"),
        ((q, pk, qr, pr, kv, kr, t(2, 3, 1, 0, dtype=i32)), {}, "need kv"),
        ((q, pk, qr, pr, kv, kr, t(2, 3, 1, 5, dtype=torch.int64)), {}, "int32"),
        ((q, pk, qr, pr), dict(prefix_len=t(2, dtype=i32)), "prefix_len"),
        ((q, pk, qr, pr), dict(prefix_len=t(1)), "prefix_len"),
        ((q, pk.half(), qr, pr), {}, "bfloat16"), ((q, pk, qr, pr, kv.float(), kr, ids), {}, "bfloat16"),
        ((t(3, 2, 16, 512).transpose(0, 1), pk, qr, pr), {}, "contiguous"),
        ((q, pk, qr, pr), dict(scale=0.75), "scale"),
        ((q, t(1, (1 << 26) + 1, 1, 512), qr, t(1, (1 << 26) + 1, 1, 64)), {}, "2\\^26"),
    ]:
        with pytest.raises(ValueError, match=why):
            dsa_b200.forward_shared_prefix(*args, **kw)


def test_workspace_bytes():
    lib, a = _native.load(), _native.FwdArgs()
    px = _native.PrefixKv(None, None, None, 32768)
    a.batch, a.queries, a.heads = 2, 1, 16
    alone = lib.dsa_fwd_prefix_workspace_bytes(ctypes.byref(a), ctypes.byref(px))
    assert alone % 256 == 0 and alone >= 2 * 128 * 514 * 4  # one row tile, split over the GPU
    a.length, a.topk = 100, 64
    assert lib.dsa_fwd_prefix_workspace_bytes(ctypes.byref(a), ctypes.byref(px)) >= alone + 2 * 16 * 514 * 4
    a.length = a.topk = 0
    a.batch = 4096  # rows enough for every SM: the kernel writes the output itself
    a.heads = 128
    assert lib.dsa_fwd_prefix_workspace_bytes(ctypes.byref(a), ctypes.byref(px)) == 0
    for field, value in (("heads", 24), ("batch", 0), ("topk", -1)):
        b = _native.FwdArgs()
        b.batch, b.queries, b.heads = 2, 1, 16
        setattr(b, field, value)
        assert lib.dsa_sparse_mla_fwd_prefix(ctypes.byref(b), ctypes.byref(px), None) == _native.STATUS_BAD_ARGUMENT


def test_plan():
    lib, a, plan = _native.load(), _native.FwdArgs(), (ctypes.c_int32 * 3)()
    px = _native.PrefixKv(None, None, None, 32768)
    a.batch, a.queries, a.heads = 64, 1, 16
    assert lib.dsa_fwd_prefix_plan(a, px, plan) == 0 and plan[0] in (1, 2) and plan[1] > 1 and plan[2] == 0
    a.length, a.topk = 100, 64
    assert lib.dsa_fwd_prefix_plan(a, px, plan) == 0 and plan[2] >= 1
    assert lib.dsa_fwd_prefix_plan(a, px, None) == _native.STATUS_BAD_ARGUMENT
    a.heads = 24
    assert lib.dsa_fwd_prefix_plan(a, px, plan) == _native.STATUS_BAD_ARGUMENT


def test_gradients_are_refused(monkeypatch):
    """The outputs have no graph: inputs that autograd follows, in either mode, are refused, not cut off."""
    monkeypatch.setattr(api, "DEVICE_TYPE", "cpu")
    monkeypatch.setattr(api, "enqueue", lambda *args: None)
    monkeypatch.setattr(api, "_status_words", {})
    shapes = (2, 3, 16, 512), (1, 50, 1, 512), (2, 3, 16, 64), (1, 50, 1, 64), (2, 9, 1, 512), (2, 9, 1, 64)
    ids = torch.zeros((2, 3, 1, 5), dtype=torch.int32)
    plain = [torch.zeros(s, dtype=torch.bfloat16) for s in shapes]
    for k in range(6):
        args = [t.clone().requires_grad_() if i == k else t for i, t in enumerate(plain)]
        with pytest.raises(ValueError, match="no gradient"):
            dsa_b200.forward_shared_prefix(*args, ids)
        with torch.no_grad():
            dsa_b200.forward_shared_prefix(*args, ids)
        dsa_b200.forward_shared_prefix(*(t.detach() for t in args), ids)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
            dual = torch.autograd.forward_ad.make_dual(plain[k], plain[k])
            dsa_b200.forward_shared_prefix(*(dual if i == k else t for i, t in enumerate(plain)), ids)
