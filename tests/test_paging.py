"""Page plans and cache appends on the CPU: the argument rules; GPU parity is in test_gpu_paging.py."""
import ctypes

import pytest
import torch

import dsa_b200
from dsa_b200 import _native, api


def t(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_plan_refusals(monkeypatch):
    monkeypatch.setattr(api, "DEVICE_TYPE", "meta")
    good = dict(block_table=t(4, 8), cached_lens=t(4), new_lens=t(4), free_blocks=t(32), free_count=t(1), block_size=16,
                queries=5)
    for change, why in [
        (dict(block_table=t(4)), "2-D"), (dict(block_size=0), "positive"), (dict(queries=0), "positive"),
        (dict(queries=2.0), "positive"), (dict(cached_lens=t(3)), "need block_table"),
        (dict(new_lens=t(4, 1)), "need block_table"), (dict(free_blocks=t(4, 8)), "need block_table"),
        (dict(free_blocks=t(0)), "need block_table"), (dict(free_count=t(2)), "need block_table"),
        (dict(reset=t(3, dtype=torch.bool)), "need block_table"), (dict(reset=t(4)), "reset bool"),
        (dict(block_table=t(4, 8, dtype=torch.int64)), "int32"), (dict(block_table=t(8, 4).t()), "contiguous"),
        (dict(block_size=1 << 30), "2\\^31"), (dict(queries=1 << 30), "2\\^31"),
    ]:
        with pytest.raises(ValueError, match=why):
            dsa_b200.plan_pages(**{**good, **change})


def test_plan_workspace_bytes():
    lib, a = _native.load(), _native.PlanPagesArgs()
    a.batch, a.queries, a.max_blocks, a.num_blocks, a.block_size = 5, 3, 8, 100, 64
    assert lib.dsa_plan_pages_workspace_bytes(ctypes.byref(a)) >= 5 * 16
    a.block_size = 1 << 30
    assert lib.dsa_plan_pages_workspace_bytes(ctypes.byref(a)) == 0


def test_append_refusals(monkeypatch):
    monkeypatch.setattr(api, "DEVICE_TYPE", "meta")
    bf, f64 = torch.bfloat16, torch.float64
    kv, kr, slots = t(2, 3, 1, 512, dtype=bf), t(2, 3, 1, 64, dtype=bf), t(2, 3)
    pool, rope = t(9, 16, 1, 512, dtype=bf), t(9, 16, 1, 64, dtype=bf)
    for args, kw, why in [
        ((t(2, 3, 512, dtype=bf), kr, slots, pool, rope), {}, "need kv"),
        ((kv, t(2, 3, 1, 32, dtype=bf), slots, pool, rope), {}, "need kv"),
        ((kv, kr, t(2, 4), pool, rope), {}, "slots"),
        ((kv, kr, t(2, 3, dtype=torch.int64), pool, rope), {}, "slots"),
        ((kv.float(), kr, slots, pool, rope), {}, "bfloat16"),
        ((kv, kr, slots, pool, t(9, 15, 1, 64, dtype=bf)), {}, "need kv_cache"),
        ((kv, kr, slots, pool.float(), rope), {}, "caches must be"),
        ((kv, kr, slots, pool, rope), dict(positions=t(2, 3)), "go together"),
        ((kv, kr, slots, pool, rope), dict(positions=t(2, 3), inv_freq=t(16, dtype=f64)), "32 entries"),
        ((kv, kr, slots, pool, rope), dict(positions=t(2, 3, dtype=torch.int64), inv_freq=t(32, dtype=f64)), "int32"),
        ((kv, kr, slots, pool, rope), dict(layout="other"), "layout"),
        ((kv, kr, slots, t(16, 9, 1, 512, dtype=bf).transpose(0, 1), rope), {}, "contiguous"),
    ]:
        with pytest.raises(ValueError, match=why):
            dsa_b200.append_kv(*args, **kw)
    for cache, why in [(t(9, 16, 1, 655, dtype=torch.uint8), "need cache"), (t(9, 16, 1, 656, dtype=torch.int8), "uint8")]:
        with pytest.raises(ValueError, match=why):
            dsa_b200.append_kv_fp8(kv, kr, slots, cache)


def test_writes_tell_autograd(monkeypatch):
    """Every tensor of the caller that a call writes counts as modified in place; the ones that it reads do not."""
    monkeypatch.setattr(api, "DEVICE_TYPE", "cpu")
    monkeypatch.setattr(api, "enqueue", lambda *args: None)

    def z(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype)

    table, cached, new, stack, count = z(4, 8), z(4), z(4), z(32), z(1)
    for inplace in (False, True):
        plan = dsa_b200.plan_pages(table, cached, new, stack, count, 16, 5, inplace=inplace)
        assert [t._version for t in (table, cached, new, stack, count)] == [int(inplace)] * 2 + [0] + [int(inplace)] * 2
    assert plan.block_table is table
    bf = torch.bfloat16
    kv, kr, slots = z(2, 3, 1, 512, dtype=bf), z(2, 3, 1, 64, dtype=bf), z(2, 3)
    pool, rope, rows = z(9, 16, 1, 512, dtype=bf), z(9, 16, 1, 64, dtype=bf), z(9, 16, 1, 656, dtype=torch.uint8)
    dsa_b200.append_kv(kv, kr, slots, pool, rope)
    dsa_b200.append_kv_fp8(kv, kr, slots, rows)
    assert [t._version for t in (kv, kr, slots, pool, rope, rows)] == [0, 0, 0, 1, 1, 1]
    w = torch.ones(512, dtype=bf, requires_grad=True)
    y = pool * w
    dsa_b200.append_kv(kv, kr, slots, pool, rope)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        pool, rope = z(9, 16, 1, 512, dtype=bf), z(9, 16, 1, 64, dtype=bf)
    dsa_b200.append_kv(kv, kr, slots, pool, rope)  # have no version


def test_append_refuses_gradients(monkeypatch):
    """No gradient goes through a cache: values and caches that autograd follows are refused outside torch.no_grad()."""
    monkeypatch.setattr(api, "DEVICE_TYPE", "cpu")
    monkeypatch.setattr(api, "enqueue", lambda *args: None)
    bf = torch.bfloat16
    plain = [torch.zeros(s, dtype=bf) for s in ((2, 3, 1, 512), (2, 3, 1, 64), (9, 16, 1, 512), (9, 16, 1, 64))]
    slots, rows = torch.zeros((2, 3), dtype=torch.int32), torch.zeros((9, 16, 1, 656), dtype=torch.uint8)
    for k in range(4):
        kv, kr, pool, rope = [t.clone().requires_grad_() if i == k else t for i, t in enumerate(plain)]
        with pytest.raises(ValueError, match="no gradient"):
            dsa_b200.append_kv(kv, kr, slots, pool, rope)
        if k < 2:
            with pytest.raises(ValueError, match="no gradient"):
                dsa_b200.append_kv_fp8(kv, kr, slots, rows)
        with torch.no_grad():
            dsa_b200.append_kv(kv, kr, slots, pool, rope)
            dsa_b200.append_kv_fp8(kv, kr, slots, rows)
