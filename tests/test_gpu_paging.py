"""GPU parity of page plans against a plain restatement on the host (whole numbers, equal), and of cache appends
against the definition in FP64 and ``quantize_kv_fp8``."""
import numpy as np
import pytest
import torch

import dsa_b200
from oracle import sparse_mla as oracle

pytestmark = pytest.mark.gpu


def plan_on_host(table, cached, new, stack, count, block, queries, reset):
    """One row after the other, one token after the other."""
    table, stack = table.copy(), stack.copy()
    batch, max_blocks = table.shape
    blocks, cap, top = len(stack), table.shape[1] * block, min(max(int(np.ravel(count)[0]), 0), len(stack))
    start = np.clip(cached, 0, cap)
    for b in range(batch):
        if reset[b]:
            for j in range(-(-start[b] // block)):
                if 0 <= table[b, j] < blocks and top < blocks:
                    stack[top] = table[b, j]
                    top += 1
            table[b], start[b] = -1, 0
    kept_stack, missing = stack.copy(), 0
    lens, positions, slots = start.copy(), np.full((batch, queries), -1, np.int32), np.full((batch, queries), -1, np.int32)
    for b in range(batch):
        for s in range(max(0, min(new[b], queries, cap - start[b]))):
            p = lens[b]
            j = p // block
            if p % block == 0:
                if top > 0:
                    top -= 1
                    table[b, j] = stack[top]
                else:
                    missing += 1
                    table[b, j] = -1
            positions[b, s] = p
            if 0 <= table[b, j] < blocks:
                slots[b, s] = table[b, j] * block + p % block
            lens[b] += 1
    return table, lens, positions, positions + 1, slots, kept_stack, np.array([top]), np.array([missing])


def make_state(batch, max_blocks, block, blocks, seed, fill=0.5):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, int(max_blocks * block * fill) + 1, batch)
    while sum(-(-c // block) for c in cached) > blocks:
        cached //= 2
    perm, table, at = rng.permutation(blocks), np.full((batch, max_blocks), -1), 0
    for b, c in enumerate(cached):
        n = -(-c // block)
        table[b, :n] = perm[at:at + n]
        at += n
    stack = np.full(blocks, -7)
    stack[:blocks - at] = perm[at:]
    return [x.astype(np.int32) for x in (table, cached, stack, np.array([blocks - at]))]


def run_plan(table, cached, new, stack, count, block, queries, reset, inplace=False):
    args = [torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda() for x in (table, cached, new, stack, count)]
    r = None if reset is None else torch.from_numpy(np.asarray(reset, dtype=bool)).cuda()
    got = dsa_b200.plan_pages(*args, block, queries, reset=r, inplace=inplace)
    if inplace:
        assert got.block_table is args[0] and got.seq_lens is args[1] and got.free_blocks is args[3] and got.free_count is args[4]
    else:
        for a, x in zip(args, (table, cached, new, stack, count)):
            assert np.array_equal(a.cpu().numpy(), x)  # the inputs stay
    return got


def same(got, ref):
    for name, g, r in zip(dsa_b200.PagePlan._fields, got, ref):
        assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), r), name


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("batch,max_blocks,block,blocks,queries", [
    (1, 1, 1, 1, 1), (1, 5, 16, 9, 1), (7, 6, 4, 40, 9), (64, 33, 64, 1500, 1), (33, 40, 1, 700, 21), (3, 7, 37, 30, 300),
    (1025, 4, 16, 4000, 5), (2100, 3, 8, 6000, 1), (5, 3000, 2, 9001, 2500), (200, 9, 16, 300, 64)])
def test_plan(cuda_lib, batch, max_blocks, block, blocks, queries, inplace):
    rng = np.random.default_rng(batch + queries)
    table, cached, stack, count = make_state(batch, max_blocks, block, blocks, batch)
    for resets in (0.0, 0.3, 1.0):
        new = rng.integers(0, queries + 1, batch).astype(np.int32)
        reset = rng.random(batch) < resets
        ref = plan_on_host(table, cached, new, stack, count, block, queries, reset)
        same(run_plan(table, cached, new, stack, count, block, queries, reset if resets else None, inplace), ref)


def test_plan_out_of_range(cuda_lib):
    """Lengths, counts and table entries out of range are clamped or name no page; an empty stack gives -1."""
    table, cached, stack, count = make_state(6, 4, 8, 20, 3)
    cached[:] = [-5, 1000, 8, 32, 17, 0]
    table[:] = -1
    table[1], table[2, 0], table[3], table[4, :3] = [3, 20, -1, 5], 7, [0, 1, 2, 4], [8, -2 ** 31, 2 ** 31 - 1]
    new = np.array([3, 5, -4, 9, 100, 2 ** 31 - 1], dtype=np.int32)
    for c in (-3, 0, 1, 5, 20, 99):
        for reset in ([0] * 6, [0, 1, 0, 1, 0, 0], [1] * 6):
            ref = plan_on_host(table, cached, new, stack, c, 8, 7, reset)
            same(run_plan(table, cached, new, stack, np.array([c], dtype=np.int32), 8, 7, reset), ref)


def test_plan_steps_keep_every_page_once(cuda_lib):
    """Many steps in place, in a captured graph: at every point each page is in one table or on the stack."""
    batch, max_blocks, block, blocks, queries = 40, 20, 8, 500, 30
    table, cached, stack, count = [torch.from_numpy(x).cuda() for x in make_state(batch, max_blocks, block, blocks, 1, 0.2)]
    new = torch.zeros(batch, dtype=torch.int32, device="cuda")
    reset = torch.zeros(batch, dtype=torch.bool, device="cuda")
    dsa_b200.plan_pages(table, cached, new, stack, count, block, queries, reset=reset, inplace=True)  # no tokens: no change
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = dsa_b200.plan_pages(table, cached, new, stack, count, block, queries, reset=reset, inplace=True)
    rng = np.random.default_rng(2)
    for _ in range(25):
        host = [x.cpu().numpy().copy() for x in (table, cached, stack, count)]
        n, r = rng.integers(0, queries + 1, batch).astype(np.int32), rng.random(batch) < 0.2
        new.copy_(torch.from_numpy(n))
        reset.copy_(torch.from_numpy(r))
        graph.replay()
        same(plan, plan_on_host(host[0], host[1], n, host[2], host[3], block, queries, r))
        if int(plan.missing) == 0:
            used = table[table >= 0].cpu().numpy()
            free = stack[:int(count)].cpu().numpy()
            assert sorted([*used, *free]) == list(range(blocks))
        else:
            break


@pytest.mark.parametrize("inplace", [False, True])
def test_plan_after_a_missing_page(cuda_lib, inplace):
    """A page that the stack could not give is reported by every step whose tokens would go on in it, also when the stack
    has pages again; no other row is counted, the next page is given, and a reset row starts anew."""
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[5, -1, -1, -1], [6, 7, -1, -1], [-1, -1, -1, -1]], **i32)
    lens, stack, count = torch.tensor([15, 20, 0], **i32), torch.zeros(8, **i32), torch.zeros(1, **i32)

    def step(new, reset=None):
        nonlocal table, lens, stack, count
        r = None if reset is None else torch.tensor(reset, device="cuda")
        plan = dsa_b200.plan_pages(table, lens, torch.tensor(new, **i32), stack, count, 16, 13, reset=r, inplace=inplace)
        table, lens, stack, count = plan.block_table, plan.seq_lens, plan.free_blocks, plan.free_count
        first = [[s for s, p in zip(*row) if p >= 0] for row in zip(plan.slots.tolist(), plan.positions.tolist())]
        return int(plan.missing), first

    assert step([2, 1, 0]) == (1, [[5 * 16 + 15, -1], [7 * 16 + 4], []])
    stack[:4], count[:] = torch.tensor([1, 2, 3, 4], **i32), 4
    assert step([1, 1, 0]) == (1, [[-1], [7 * 16 + 5], []])
    assert step([0, 1, 0]) == (0, [[], [7 * 16 + 6], []])  # nothing goes on in it
    # twelve tokens up to position 30, then the last of the missing page and the first of the next, which is there
    assert step([13, 0, 0]) == (1, [[-1] * 13, [], []])
    assert step([2, 0, 1]) == (1, [[-1, 4 * 16], [], [3 * 16]])
    assert step([1, 0, 0]) == (0, [[4 * 16 + 1], [], []])
    assert table.tolist() == [[5, -1, 4, -1], [6, 7, -1, -1], [3, -1, -1, -1]] and int(count) == 2
    assert step([2, 0, 0], [True, False, False]) == (0, [[4 * 16, 4 * 16 + 1], [], []])
    assert table.tolist()[0] == [4, -1, -1, -1] and stack[:int(count)].tolist() == [1, 2, 5]


def _tokens(batch, queries, seed, parts=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    row = torch.randn((batch, queries, 1, 576), generator=g, device="cuda").bfloat16() * 3
    return (row[..., :512], row[..., 512:]) if parts else (row[..., :512].contiguous(), row[..., 512:].contiguous())


def _slots(batch, queries, rows, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = torch.randperm(rows, generator=g, device="cuda")[:batch * queries].int().reshape(batch, queries)
    s[torch.rand(s.shape, generator=g, device="cuda") < 0.2] = -1
    return s


@pytest.mark.parametrize("parts", [False, True])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("batch,queries", [(1, 1), (5, 3), (2, 700)])
def test_append(cuda_lib, batch, queries, layout, parts):
    kv, kr = _tokens(batch, queries, 4, parts)
    rows = batch * queries + 13
    slots = _slots(batch, queries, rows, 5)
    if batch > 1:
        slots[0, 0], slots[1, 1] = rows, 2 ** 31 - 1  # outside the cache: not written
    pos = torch.randint(0, 100000, (batch, queries), device="cuda", dtype=torch.int32)
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    fill = torch.randn((rows, 1, 1, 512), device="cuda").bfloat16(), torch.randn((rows, 1, 1, 64), device="cuda").bfloat16()
    fill8 = torch.randint(0, 256, (rows, 1, 1, 656), device="cuda", dtype=torch.uint8)
    turned = dsa_b200.rotary(kr, pos, freq, layout=layout, attention_factor=1.5)
    real = ((slots >= 0) & (slots < rows)).flatten()
    to = slots.flatten()[real].long()
    for rope, kw in ((kr, {}), (turned, dict(positions=pos, inv_freq=freq, layout=layout, attention_factor=1.5))):
        want = [t.clone() for t in fill]
        want[0].view(rows, 512)[to] = kv.reshape(-1, 512)[real]
        want[1].view(rows, 64)[to] = rope.reshape(-1, 64)[real]
        got = [t.clone() for t in fill]
        dsa_b200.append_kv(kv, kr, slots, *got, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        want8 = fill8.clone()
        # on the host: torch's GPU division by the number 448 is a product with its rounded reciprocal
        want8.view(rows, 656)[to] = dsa_b200.quantize_kv_fp8(kv.cpu(), rope.cpu()).cuda().reshape(-1, 656)[real]
        got8 = fill8.clone()
        dsa_b200.append_kv_fp8(kv, kr, slots, got8, **kw)
        assert torch.equal(got8, want8)


def test_append_special_values(cuda_lib):
    """Blocks of zeros, one element, NaN, infinities, the smallest and largest numbers: as quantize_kv_fp8's values."""
    kv, kr = _tokens(1, 8, 6)
    kv[0, 0] = 0
    kv[0, 1, 0, 128:256] = 0
    kv[0, 1, 0, 200] = -3.0
    kv[0, 2, 0, 5] = float("nan")
    kv[0, 3, 0, 300], kv[0, 3, 0, 511] = float("inf"), float("-inf")
    kv[0, 4] = torch.finfo(torch.bfloat16).max
    kv[0, 5] = 1e-38
    kv[0, 6, 0, :128] = 2.0 ** -133  # the smallest subnormal
    slots = torch.arange(8, dtype=torch.int32, device="cuda").reshape(1, 8)
    cache = torch.zeros((1, 8, 1, 656), dtype=torch.uint8, device="cuda")
    dsa_b200.append_kv_fp8(kv, kr, slots, cache)
    want = dsa_b200.quantize_kv_fp8(kv.cpu(), kr.cpu()).cuda()
    for lo, hi, dtype in ((0, 512, torch.float8_e4m3fn), (512, 528, torch.float32), (528, 656, torch.bfloat16)):
        g, w = (c[..., lo:hi].contiguous().view(dtype).float() for c in (cache, want))
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(g.nan_to_num(7.0), w.nan_to_num(7.0)), lo


def test_append_signed_zeros_and_mixed_blocks(cuda_lib):
    """Bit for bit the host writer's rows: zeros of both signs, values that round to them, and blocks that hold a NaN next
    to infinities and the largest numbers (scale 1: those saturate)."""
    kv, kr = _tokens(1, 4, 9)
    kv[0, 0, 0, ::2] = -0.0
    kv[0, 0, 0, 128:256] = -0.0
    kv[0, 1] *= 2.0 ** torch.randint(-40, 2, (512,), device="cuda").float()
    kv[0, 2, 0, 7], kv[0, 2, 0, 8], kv[0, 2, 0, 9], kv[0, 2, 0, 10] = float("nan"), float("inf"), float("-inf"), 3e38
    slots = torch.arange(4, dtype=torch.int32, device="cuda").reshape(1, 4)
    cache = torch.zeros((1, 4, 1, 656), dtype=torch.uint8, device="cuda")
    dsa_b200.append_kv_fp8(kv, kr, slots, cache)
    want = dsa_b200.quantize_kv_fp8(kv.cpu(), kr.cpu()).cuda()
    nan = torch.isnan(want[..., :512].contiguous().view(torch.float8_e4m3fn).float())
    assert torch.equal(torch.isnan(cache[..., :512].contiguous().view(torch.float8_e4m3fn).float()), nan)
    assert torch.equal(cache[..., :512][~nan], want[..., :512][~nan]) and torch.equal(cache[..., 512:], want[..., 512:])


def test_append_every_mantissa(cuda_lib):
    """Bit for bit the host writer's rows for all pairs of a value's and a maximum's BF16 mantissa, at several exponents:
    scales and quotients are the rounded quotients, ties of the FP8 rounding among them."""
    top = (128 + torch.arange(128)).float().reshape(128, 1)                  # a block's maximum
    low = (128 + torch.arange(128)).float().reshape(1, 128) * 0.5            # 64 .. 127.5: below every maximum
    blocks = torch.cat([low * 2.0 ** -(torch.arange(128) % 9).float() * (1 - 2 * (torch.arange(128) % 2)), low, low / 16])
    blocks = torch.stack([b.expand(128, 128).clone() for b in blocks])       # [3, 128 maxima, 128 values]
    blocks[:, :, 0] = top.squeeze(1)
    blocks = torch.cat([blocks, blocks.roll(1, -1)])                         # mantissa 0 meets every maximum by its double
    kv = torch.stack([blocks, blocks * 2.0 ** -50, blocks * 2.0 ** 40]).reshape(1, -1, 1, 512).bfloat16().cuda()
    assert torch.equal(kv[0, :192].float().cpu().reshape(blocks.shape), blocks)
    tokens = kv.shape[1]
    kr = torch.zeros((1, tokens, 1, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda").reshape(1, tokens)
    cache = torch.zeros((1, tokens, 1, 656), dtype=torch.uint8, device="cuda")
    dsa_b200.append_kv_fp8(kv, kr, slots, cache)
    assert torch.equal(cache, dsa_b200.quantize_kv_fp8(kv.cpu(), kr.cpu()).cuda())


@pytest.mark.parametrize("batch,queries", [(3, 5), (5, 1), (1, 6), (2, 4)])
@pytest.mark.parametrize("gap", ["none", "kv", "rope", "both"])
def test_append_batch_strides(cuda_lib, batch, queries, gap):
    """Rows of a batch with and without a gap behind each row's tokens, for the latent and the rope values apart."""
    kv, kr = _tokens(batch, queries, 21)
    slots = torch.randperm(batch * queries + 7, device="cuda")[:batch * queries].int().reshape(batch, queries)
    pos = torch.randint(0, 9999, (batch, queries), dtype=torch.int32, device="cuda")
    kw = dict(positions=pos, inv_freq=dsa_b200.rotary_frequencies(64, device="cuda"))
    pad = lambda t: torch.cat([t, torch.full_like(t, 9.0)], 1)[:, :queries]
    got, want = [], []
    for out, x, y in ((want, kv, kr), (got, pad(kv) if gap in ("kv", "both") else kv, pad(kr) if gap in ("rope", "both") else kr)):
        for n, dtype in ((512, torch.bfloat16), (64, torch.bfloat16), (656, torch.uint8)):
            out.append(torch.zeros((batch * queries + 7, 1, 1, n), dtype=dtype, device="cuda"))
        dsa_b200.append_kv(x, y, slots, *out[:2], **kw)
        dsa_b200.append_kv_fp8(x, y, slots, out[2], **kw)
    to = slots.flatten().long()
    assert torch.equal(want[0][to], kv.reshape(-1, 1, 1, 512))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_append_far_rows(cuda_lib):
    """Rows behind 2^31 elements of the BF16 cache and 2^31 bytes of the FP8 cache; the rows around them stay."""
    kv, kr = _tokens(1, 2, 10)
    rows = (1 << 22) + 100
    slots = torch.tensor([[rows - 1, rows - 3]], dtype=torch.int32, device="cuda")
    pool = torch.zeros((rows, 1, 1, 512), dtype=torch.bfloat16, device="cuda")
    rope = torch.zeros((rows, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    dsa_b200.append_kv(kv, kr, slots, pool, rope)
    assert torch.equal(pool[-1], kv[0, :1]) and torch.equal(pool[-3], kv[0, 1:]) and torch.equal(rope[-3], kr[0, 1:])
    assert not bool(pool[-2].any()) and not bool(pool[:8].any())
    del pool
    cache = torch.zeros((rows, 1, 1, 656), dtype=torch.uint8, device="cuda")
    dsa_b200.append_kv_fp8(kv, kr, slots, cache)
    want = dsa_b200.quantize_kv_fp8(kv.cpu(), kr.cpu()).cuda()
    assert torch.equal(cache[-1], want[0, :1]) and torch.equal(cache[-3], want[0, 1:]) and not bool(cache[-2].any())


def test_captured_append_with_new_slots(cuda_lib):
    kv, kr = _tokens(3, 1, 11)
    slots, pos = torch.full((3, 1), -1, dtype=torch.int32, device="cuda"), torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    freq = dsa_b200.rotary_frequencies(64, device="cuda")
    pools = [torch.zeros((40, 1, 1, n), dtype=torch.bfloat16, device="cuda") for n in (512, 64)]
    dsa_b200.append_kv(kv, kr, slots, *pools, positions=pos, inv_freq=freq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dsa_b200.append_kv(kv, kr, slots, *pools, positions=pos, inv_freq=freq)
    want = [t.clone() for t in pools]
    for k in range(4):
        slots.copy_(torch.tensor([[k], [20 + k], [-1]]))
        pos.fill_(1000 * k)
        kv.neg_()
        graph.replay()
        want[0][[k, 20 + k], 0] = kv[:2, 0]
        want[1][[k, 20 + k], 0] = dsa_b200.rotary(kr, pos, freq)[:2, 0]
        assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])


def test_append_without_alignment(cuda_lib):
    """kv rows that start on no 16-byte boundary."""
    kv, kr = _tokens(2, 5, 8)
    wide = torch.zeros((2, 5, 1, 579), dtype=torch.bfloat16, device="cuda")
    wide[..., 1:513], wide[..., 513:577] = kv, kr
    slots = torch.randperm(10, device="cuda").int().reshape(2, 5)
    a = [torch.zeros((10, 1, 1, n), dtype=torch.bfloat16, device="cuda") for n in (512, 64, 512, 64)]
    dsa_b200.append_kv(kv, kr, slots, *a[:2])
    dsa_b200.append_kv(wide[..., 1:513], wide[..., 513:577], slots, *a[2:])
    assert torch.equal(a[0], a[2]) and torch.equal(a[1], a[3])
    c = [torch.zeros((10, 1, 1, 656), dtype=torch.uint8, device="cuda") for _ in range(2)]
    dsa_b200.append_kv_fp8(kv, kr, slots, c[0])
    dsa_b200.append_kv_fp8(wide[..., 1:513], wide[..., 513:577], slots, c[1])
    assert torch.equal(c[0], c[1])


def test_serving_step(cuda_lib):
    """Plan, rotary, append and forward_paged together, several steps of ragged requests, against the oracle on dense
    caches kept on the host."""
    batch, max_blocks, block, blocks, heads, topk = 3, 8, 16, 30, 16, 64
    length = max_blocks * block
    table = torch.full((batch, max_blocks), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    stack = torch.randperm(blocks, device="cuda").int()
    count = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    pool = torch.full((blocks, block, 1, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    rope_pool = torch.full((blocks, block, 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    freq = dsa_b200.rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096, device="cuda")
    dense_kv, dense_kr = torch.zeros((batch, length, 1, 512)), torch.zeros((batch, length, 1, 64))
    at = [0] * batch
    g = torch.Generator(device="cuda").manual_seed(3)
    for queries, new in ((40, [40, 1, 23]), (1, [1, 1, 1]), (5, [5, 0, 2]), (30, [0, 30, 30])):
        plan = dsa_b200.plan_pages(table, lens, torch.tensor(new, dtype=torch.int32, device="cuda"), stack, count, block,
                                   queries, inplace=True)
        kv, kr = _tokens(batch, queries, queries)
        q = torch.randn((batch, queries, heads, 512), generator=g, device="cuda").bfloat16()
        qr = torch.randn((batch, queries, heads, 64), generator=g, device="cuda").bfloat16()
        qr = dsa_b200.rotary(qr, plan.positions, freq)
        dsa_b200.append_kv(kv, kr, plan.slots, pool, rope_pool, positions=plan.positions, inv_freq=freq)
        qi = torch.randn((batch, queries, 16, 128), generator=g, device="cuda").bfloat16()
        ki = torch.randn((batch, length, 128), generator=g, device="cuda").bfloat16()
        w = torch.rand((batch, queries, 16), generator=g, device="cuda")
        ids = dsa_b200.indexer_topk(qi, ki, w, topk, lengths=plan.lengths)
        out = dsa_b200.forward_paged(q, pool.nan_to_num(0.0), qr, rope_pool.nan_to_num(0.0), plan.block_table, ids,
                                     seq_lens=plan.seq_lens)
        turned = dsa_b200.rotary(kr, plan.positions, freq).cpu()
        for b in range(batch):
            dense_kv[b, at[b]:at[b] + new[b]] = kv[b, :new[b]].cpu().float()
            dense_kr[b, at[b]:at[b] + new[b]] = turned[b, :new[b]].float()
            at[b] += new[b]
        assert plan.seq_lens.tolist() == at and int(plan.missing) == 0
        ref = oracle.reference_forward(q.cpu(), dense_kv.bfloat16(), qr.cpu(), dense_kr.bfloat16(), ids.cpu())
        real = (plan.positions >= 0).cpu()
        pick = lambda ts: [ts[0][real][None], *(t.reshape(batch, queries, heads)[real][None, None] for t in ts[1:])]  # noqa: E731
        metrics = oracle.accuracy(pick([t.float().cpu() for t in out]), pick([t.float() for t in ref]))
        assert oracle.passes(metrics), metrics
        assert not bool(out[0][~real.cuda()].any())  # padded queries select nothing
