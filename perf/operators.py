"""The cases of the serving operators around the sparse-MLA forward: rotary positions, page plans, cache appends
and attention over a shared prefix.

``listed()`` and ``draw()`` give cases, ``prepare()`` the tensors that a serving loop has in hand before the call,
``run()`` one pass (the framework's call where ``own`` is true, elementary torch operations in FP32 otherwise),
``exact()`` the same values in FP64 from the operator's definition and ``work()`` the bytes and operations that a
pass cannot do without.
"""
import math

import torch

own = False

DEVICE = "cuda"
LATENT, ROPE, ROW = 512, 64, 656
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- the cases --------------------------------------------------------------------------------------------


def _rotary(name, batch, queries, heads, dim, rotary_dim, start, layout, dtype, theta=10000.0, stretch=1.0, grad=False):
    return {"name": name, "op": "rotary", "batch": batch, "queries": queries, "heads": heads, "dim": dim,
            "rotary_dim": rotary_dim, "start": start, "layout": layout, "dtype": dtype, "theta": theta,
            "stretch": stretch, "grad": grad}


def _pages(name, batch, queries, max_blocks, block_size, resets):
    return {"name": name, "op": "pages", "batch": batch, "queries": queries, "max_blocks": max_blocks,
            "block_size": block_size, "resets": resets}


def _append(name, batch, queries, rows, block_size, fp8, layout):
    return {"name": name, "op": "append", "batch": batch, "queries": queries, "rows": rows, "block_size": block_size,
            "fp8": fp8, "layout": layout}


def _prefix(name, batch, queries, heads, prefix, filled, length, topk):
    return {"name": name, "op": "prefix", "batch": batch, "queries": queries, "heads": heads, "prefix": prefix,
            "filled": filled, "length": length, "topk": topk}


def listed():
    return [
        # the query rope part of one decode step of 64 requests: latency
        _rotary("rotary_decode", 64, 1, 128, 64, 64, 0, "interleaved", "bf16"),
        # the indexer's queries of a 4096-token prefill: half layout, the first 64 of 128 dims, stretched positions
        _rotary("rotary_indexer", 1, 4096, 64, 128, 64, 0, "half", "bf16", stretch=40.0),
        # a training step's query heads of 192 dims whose last 64 turn, forward and gradient, in FP32
        _rotary("rotary_grad", 2, 2048, 16, 192, 64, 128, "interleaved", "fp32", grad=True),
        # the query rope part of a batch of four 4096-token prompts: bandwidth
        _rotary("rotary_prefill", 4, 4096, 128, 64, 64, 0, "interleaved", "bf16"),
        # one token more for each of 64 requests of up to 65536 tokens, a few rows given to new requests
        _pages("pages_decode", 64, 1, 1024, 64, True),
        # a ragged chunk of prompts: up to 1021 tokens for each of 300 rows, small pages
        _pages("pages_prefill", 300, 1021, 515, 16, True),
        # the cache rows of one decode step of 64 requests, BF16 pages
        _append("append_decode", 64, 1, 65536, 64, False, "interleaved"),
        # the cache rows of four prompts of up to 4096 tokens, BF16 pages
        _append("append_prefill", 4, 4096, 32768, 64, False, "interleaved"),
        # the FP8 cache rows of eight prompts of up to 8192 tokens
        _append("append_fp8", 8, 8192, 98304, 128, True, "half"),
        # a handful of requests with a short common prompt
        _prefix("prefix_small", 3, 2, 16, 1000, 1000, 300, 77),
        # 64 samples of one 32768-token prompt on one of eight tensor-parallel ranks, 2048 own tokens selected
        _prefix("prefix_tp8", 64, 1, 16, 32768, 32768, 8192, 2048),
        # 32 samples of a prompt of 32003 tokens in a buffer of 32768, all 128 heads
        _prefix("prefix_h128", 32, 1, 128, 32768, 32003, 4096, 512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "pages", "append", "append", "prefix", "prefix"])
    if op == "rotary":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rotary_dim = rng.choice([32, 64, 64, 128, 6, 30])
        before, after = rng.choice([(0, 0), (0, 0), (0, 64), (128, 0), (3, 7), (8, 8)])
        heads = rng.choice([1, 1, 5, 16, 32, 64, 128])
        dim = before + rotary_dim + after
        batch = _log(rng, 1, 64)
        queries = _log(rng, 1, max(1, min(8192, 134217728 // (heads * dim * batch * 2))))
        return _rotary("", batch, queries, heads, dim, rotary_dim, before, rng.choice(["interleaved", "half"]), dtype,
                       rng.choice([10000.0, 500000.0]), rng.choice([1.0, 4.0, 40.0]), rng.random() < 0.4)
    if op == "pages":
        batch = _log(rng, 1, 1024)
        queries = _log(rng, 1, max(1, min(4096, 300000 // batch)))
        return _pages("", batch, queries, _log(rng, 1, 2048 if batch < 256 else 256),
                      rng.choice([1, 16, 37, 64, 64, 128]), rng.random() < 0.6)
    if op == "append":
        batch = _log(rng, 1, 64)
        queries = _log(rng, 1, max(1, 65536 // batch))
        block = rng.choice([1, 16, 48, 64, 128])
        rows = -(-(batch * queries + _log(rng, 1, 20000)) // block) * block
        return _append("", batch, queries, rows, block, rng.random() < 0.5, rng.choice(["interleaved", "half"]))
    heads = rng.choice([16, 16, 32, 64, 128])
    rows = _log(rng, 1, 4096 // heads)
    queries = rng.choice([q for q in (1, 1, 2, 3) if q <= rows])
    prefix = _log(rng, 1, 30000)
    topk = _log(rng, 1, 1024) if rng.random() < 0.8 else 0
    filled = prefix if rng.random() < 0.6 else rng.randint(0, prefix)
    return _prefix("", max(1, rows // queries), queries, heads, prefix, max(filled, 1) if not topk else filled,
                   topk + _log(rng, 1, 4096) if topk else 0, topk)


# ---- what a program has in hand ---------------------------------------------------------------------------


def _frequencies(rotary_dim, theta, stretch):
    """Angular frequencies in FP64, on the host: theta^(-2i/d), divided by `stretch` beyond one turn over 4096 tokens and left
    as they are beyond 32 turns, with a ramp in between."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = theta ** (-2.0 * i / rotary_dim)
    if stretch == 1.0:
        return freq
    turns = 4096.0 * freq / (2.0 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return freq / stretch * (1.0 - keep) + freq * keep


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEVICE, dtype=torch.int32)

    c, batch, queries = case, case["batch"], case["queries"]
    state = {"case": dict(case)}
    if c["op"] == "rotary":
        x = randn(batch, queries, c["heads"], c["dim"], dtype=TYPES[c["dtype"]])
        first = randint(0, int(4096 * c["stretch"]), batch, 1)
        state |= {"x": x.requires_grad_(c["grad"]),
                  "positions": first + torch.arange(queries, device=DEVICE, dtype=torch.int32),
                  "inv_freq": _frequencies(c["rotary_dim"], c["theta"], c["stretch"]).to(DEVICE),
                  "attention_factor": 0.1 * math.log(c["stretch"]) + 1.0}
        if c["grad"]:
            state["grad"] = randn(batch, queries, c["heads"], c["dim"], dtype=TYPES[c["dtype"]])
    elif c["op"] == "pages":
        max_blocks, block = c["max_blocks"], c["block_size"]
        blocks = -(-3 * batch * max_blocks // 4)  # a pool smaller than the tables could name
        cached = randint(0, max_blocks * block // 2 + 1, batch)
        had = (cached + block - 1) // block
        ends = had.cumsum(0)
        perm = torch.randperm(blocks, generator=g, device=DEVICE).int()
        j = torch.arange(max_blocks, device=DEVICE, dtype=torch.int32)
        at = (ends - had)[:, None] + j
        table = torch.where(j < had[:, None], perm[at.clamp(0, blocks - 1)], -1).int()
        i = torch.arange(blocks, device=DEVICE)
        left = blocks - ends[-1]
        free = torch.where(i < left, perm[(i + ends[-1]).clamp(0, blocks - 1)], -1).int()
        state |= {"block_table": table, "cached_lens": cached, "new_lens": randint(0, queries + 1, batch),
                  "free_blocks": free, "free_count": left.int().reshape(1),
                  "reset": torch.rand(batch, generator=g, device=DEVICE) < 0.05 if c["resets"] else None}
    elif c["op"] == "append":
        tokens = batch * queries
        lengths = randint(1, queries + 1, batch, 1) if queries > 1 else randint(1, 2, batch, 1)
        s = torch.arange(queries, device=DEVICE, dtype=torch.int32)
        blocks = c["rows"] // c["block_size"]
        # every request's tokens in pages of a shuffled pool, padding without a slot
        order = torch.randperm(blocks, generator=g, device=DEVICE).int()
        t = torch.arange(tokens, device=DEVICE, dtype=torch.int32).reshape(batch, queries)
        slots = order[(t // c["block_size"]).long()] * c["block_size"] + t % c["block_size"]
        real = s < lengths
        row = randn(batch, queries, LATENT + ROPE) * 2  # the projection's output: latent and rope part side by side
        state |= {"kv": row[..., None, :LATENT], "k_rope": row[..., None, LATENT:],
                  "slots": torch.where(real, slots, -1).int(),
                  "positions": torch.where(real, randint(0, 100000, batch, 1) + s, -1).int(),
                  "inv_freq": _frequencies(ROPE, 10000.0, 40.0).to(DEVICE), "attention_factor": 1.0}
        if c["fp8"]:
            state["cache"] = torch.zeros((blocks, c["block_size"], 1, ROW), dtype=torch.uint8, device=DEVICE)
        else:
            state["kv_cache"] = torch.zeros((blocks, c["block_size"], 1, LATENT), dtype=torch.bfloat16, device=DEVICE)
            state["k_rope_cache"] = torch.zeros((blocks, c["block_size"], 1, ROPE), dtype=torch.bfloat16, device=DEVICE)
    else:
        heads, prefix, topk = c["heads"], c["prefix"], c["topk"]
        state |= {"q": randn(batch, queries, heads, LATENT), "q_rope": randn(batch, queries, heads, ROPE),
                  "prefix_kv": randn(1, prefix, 1, LATENT), "prefix_k_rope": randn(1, prefix, 1, ROPE),
                  "prefix_len": None if c["filled"] == prefix else torch.full((1,), c["filled"], dtype=torch.int32, device=DEVICE),
                  "kv": None, "k_rope": None, "indices": None}
        if topk:
            length = c["length"]
            ids = torch.rand((batch * queries, length), generator=g, device=DEVICE).argsort(-1)[:, :topk].int()
            ids = torch.where(torch.rand(ids.shape, generator=g, device=DEVICE) < 0.02, -1, ids)  # a few empty places
            ids[:, 0] = ids[:, 0].clamp(min=0)
            state |= {"kv": randn(batch, length, 1, LATENT), "k_rope": randn(batch, length, 1, ROPE),
                      "indices": ids.reshape(batch, queries, 1, topk).int().contiguous()}
    return state


# ---- one pass ---------------------------------------------------------------------------------------------


def _turn(x, positions, inv_freq, layout, factor):
    """x [..., H, d] in FP32 turned by positions [...] (angles in FP64, cosines in FP32)."""
    angle = positions[..., None, None].double() * inv_freq
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_rotary(s):
    c, x = s["case"], s["x"]
    lo, hi = c["start"], c["start"] + c["rotary_dim"]
    turned = _turn(x[..., lo:hi].float(), s["positions"], s["inv_freq"], c["layout"], s["attention_factor"])
    return torch.cat((x[..., :lo], turned.to(x.dtype), x[..., hi:]), -1)


def _plain_pages(s):
    c = s["case"]
    batch, max_blocks = s["block_table"].shape
    block, queries, blocks = c["block_size"], c["queries"], s["free_blocks"].shape[0]
    cap = max_blocks * block
    reset = s["reset"] if s["reset"] is not None else torch.zeros(batch, dtype=torch.bool, device=DEVICE)
    cached = s["cached_lens"].long().clamp(0, cap)
    j = torch.arange(max_blocks, device=DEVICE)
    table = s["block_table"].long()
    # the pages of the rows that are given to new requests go back on the stack of free pages
    back = reset[:, None] & (j < ((cached + block - 1) // block)[:, None]) & (table >= 0) & (table < blocks)
    free_count = s["free_count"].long().clamp(0, blocks)
    at = free_count + back.flatten().cumsum(0) - 1
    at = torch.where(back.flatten() & (at < blocks), at, blocks)
    stack = torch.cat((s["free_blocks"].long(), s["free_blocks"].new_zeros(1).long()))
    stack[at] = table.flatten()
    stack = stack[:blocks]
    total = (free_count + back.sum()).clamp(max=blocks)
    # pages for the new tokens, from the top of the stack, in the order of the rows
    start = torch.where(reset, 0, cached)
    new = torch.minimum(s["new_lens"].long().clamp(0, queries), cap - start)
    lens = start + new
    kept = (start + block - 1) // block
    need = (lens + block - 1) // block - kept
    ends = need.cumsum(0)
    a = (ends - need)[:, None] + j - kept[:, None]
    got = torch.where(a < total, stack[(total - 1 - a).clamp(0, blocks - 1)], -1)
    fresh = (j >= kept[:, None]) & (j < (kept + need)[:, None])
    table = torch.where(fresh, got, torch.where(reset[:, None], -1, table))
    i = torch.arange(queries, device=DEVICE)
    positions = torch.where(i < new[:, None], start[:, None] + i, -1)
    page = table.gather(1, (positions.clamp(min=0) // block))
    slots = torch.where((positions >= 0) & (page >= 0) & (page < blocks), page * block + positions % block, -1)
    return {"block_table": table.int(), "seq_lens": lens.int(), "positions": positions.int(),
            "lengths": (positions + 1).int(), "slots": slots.int(), "free_blocks": stack.int(),
            "free_count": (total - ends[-1]).clamp(min=0).int(), "missing": (ends[-1] - total).clamp(min=0).int()}


def _plain_rows(s):
    """Cache rows of the tokens and where they go; a token without a slot repeats the row of one that has one."""
    slots = s["slots"].flatten().long()
    one = (slots >= 0).int().argmax()
    token = torch.where(slots >= 0, torch.arange(slots.numel(), device=DEVICE), one)
    rope = _turn(s["k_rope"].float(), s["positions"], s["inv_freq"], s["case"]["layout"], s["attention_factor"])
    return slots[token], token, s["kv"].reshape(-1, LATENT), rope.to(torch.bfloat16).reshape(-1, ROPE)


def _plain_append(s):
    to, token, kv, rope = _plain_rows(s)
    if not s["case"]["fp8"]:
        s["kv_cache"].view(-1, LATENT)[to] = kv[token]
        s["k_rope_cache"].view(-1, ROPE)[to] = rope[token]
        return
    blocks = kv.float().reshape(-1, 4, 128)
    amax = blocks.abs().amax(-1)
    scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    lat = (blocks / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(-1, LATENT)
    row = torch.cat((lat.view(torch.uint8), scale.view(torch.uint8), rope.view(torch.uint8)), -1)
    s["cache"].view(-1, ROW)[to] = row[token]


def _cache(s):
    """The cache as the values that it stands for."""
    if not s["case"]["fp8"]:
        return {"kv": s["kv_cache"], "k_rope": s["k_rope_cache"]}
    return {"latent": s["cache"][..., :LATENT].view(torch.float8_e4m3fn),
            "scales": s["cache"][..., LATENT:LATENT + 16].view(torch.float32),
            "k_rope": s["cache"][..., LATENT + 16:].view(torch.bfloat16)}


def _plain_prefix(s):
    q = torch.cat((s["q"], s["q_rope"]), -1).float()
    batch, queries, heads, _ = q.shape
    key = torch.cat((s["prefix_kv"], s["prefix_k_rope"]), -1).float().reshape(-1, LATENT + ROPE)
    value = key[:, :LATENT]
    if s["prefix_len"] is not None:
        hidden = torch.arange(key.shape[0], device=DEVICE) >= s["prefix_len"]
    score = (q.reshape(-1, LATENT + ROPE) @ key.T).reshape(batch, queries, heads, -1) / 24.0
    if s["prefix_len"] is not None:
        score.masked_fill_(hidden, -math.inf)
    if s["indices"] is not None:
        length = s["kv"].shape[1]
        ids = s["indices"].long().squeeze(2)
        bad = (ids < 0) | (ids >= length)
        row = torch.arange(batch, device=DEVICE)[:, None, None]
        at = ids.clamp(0, length - 1)
        own_key = torch.cat((s["kv"][row, at, 0], s["k_rope"][row, at, 0]), -1).float()
        mine = (q @ own_key.transpose(-1, -2) / 24.0).masked_fill(bad[:, :, None], -math.inf)
        score = torch.cat((score, mine), -1)
    top = score.amax(-1, keepdim=True)
    weight = (score - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    n = key.shape[0]
    out = (weight[..., :n].reshape(-1, n) @ value).reshape(batch, queries, heads, LATENT)
    if s["indices"] is not None:
        out = out + weight[..., n:] @ own_key[..., :LATENT]
    out = out / torch.where(total > 0, total, 1.0)
    return out.to(torch.bfloat16), top.reshape(batch, 1, queries, heads), total.reshape(batch, 1, queries, heads)


def run(s):
    c = s["case"]
    if own:
        import dsa_b200

        if c["op"] == "rotary":
            y = dsa_b200.rotary(s["x"], s["positions"], s["inv_freq"], layout=c["layout"], start=c["start"],
                                attention_factor=s["attention_factor"])
        elif c["op"] == "pages":
            return dsa_b200.plan_pages(s["block_table"], s["cached_lens"], s["new_lens"], s["free_blocks"],
                                       s["free_count"], c["block_size"], c["queries"], reset=s["reset"])._asdict()
        elif c["op"] == "append":
            rope = {"positions": s["positions"], "inv_freq": s["inv_freq"], "layout": c["layout"]}
            if c["fp8"]:
                dsa_b200.append_kv_fp8(s["kv"], s["k_rope"], s["slots"], s["cache"], **rope)
            else:
                dsa_b200.append_kv(s["kv"], s["k_rope"], s["slots"], s["kv_cache"], s["k_rope_cache"], **rope)
            return _cache(s)
        else:
            return dsa_b200.forward_shared_prefix(s["q"], s["prefix_kv"], s["q_rope"], s["prefix_k_rope"], s["kv"],
                                                  s["k_rope"], s["indices"], prefix_len=s["prefix_len"])
    elif c["op"] == "rotary":
        y = _plain_rotary(s)
    elif c["op"] == "pages":
        return _plain_pages(s)
    elif c["op"] == "append":
        _plain_append(s)
        return _cache(s)
    else:
        return _plain_prefix(s)
    if not c["grad"]:
        return y
    (gx,) = torch.autograd.grad(y, s["x"], s["grad"])
    return y.detach(), gx


# ---- the definition in 64 bits ----------------------------------------------------------------------------


def _rotation(x, positions, inv_freq, layout, factor, sign):
    """Each pair as a complex number times factor * exp(i * sign * position * frequency)."""
    d = x.shape[-1]
    pairs = x.reshape(*x.shape[:-1], d // 2, 2) if layout == "interleaved" else x.reshape(*x.shape[:-1], 2, d // 2).transpose(-1, -2)
    angle = sign * positions.double()[..., None, None] * inv_freq.double()
    z = torch.view_as_complex(pairs.double().contiguous()) * torch.polar(torch.full_like(angle, factor), angle)
    pairs = torch.view_as_real(z)
    return (pairs if layout == "interleaved" else pairs.transpose(-1, -2)).reshape(x.shape)


def _e4m3(y):
    """The nearest e4m3 number, ties to the even one, at most 448."""
    exponent = torch.frexp(y)[1].clamp(min=-5) - 1  # |y| in [2^e, 2^(e+1)), steps of 2^(e-3), subnormals from 2^-6 down
    step = torch.ldexp(torch.ones_like(y), exponent - 3)
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "pages":
        return None
    if c["op"] == "rotary":
        lo, hi = c["start"], c["start"] + c["rotary_dim"]

        def whole(x, sign):
            out = x.detach().double().clone()
            out[..., lo:hi] = _rotation(out[..., lo:hi], s["positions"], s["inv_freq"], c["layout"], s["attention_factor"], sign)
            return out

        return (whole(s["x"], 1.0), whole(s["grad"], -1.0)) if c["grad"] else whole(s["x"], 1.0)
    if c["op"] == "append":
        keep = s["slots"].flatten() >= 0
        to = s["slots"].flatten()[keep].long()
        kv = s["kv"].reshape(-1, LATENT)[keep].double()
        rope = _rotation(s["k_rope"], s["positions"], s["inv_freq"], c["layout"], 1.0, 1.0).reshape(-1, ROPE)[keep]
        shape = (c["rows"] // c["block_size"], c["block_size"], 1)

        def place(rows):
            out = torch.zeros((c["rows"], rows.shape[-1]), dtype=torch.float64, device=DEVICE)
            out[to] = rows
            return out.reshape(*shape, -1)

        if not c["fp8"]:
            return {"kv": place(kv), "k_rope": place(rope)}
        part = kv.reshape(-1, 4, 128)
        scale = part.abs().amax(-1) / 448.0
        scale[scale == 0] = 1.0
        lat = _e4m3(part / scale[..., None])
        return {"latent": place(lat.reshape(-1, LATENT)), "scales": place(scale), "k_rope": place(rope)}
    outs, tops, totals = [], [], []
    filled = c["filled"]
    common = torch.cat((s["prefix_kv"], s["prefix_k_rope"]), -1).reshape(-1, LATENT + ROPE)[:filled].double()
    for b in range(c["batch"]):
        for i in range(c["queries"]):
            keys = common
            if s["indices"] is not None:
                ids = s["indices"][b, i, 0].long()
                ids = ids[(ids >= 0) & (ids < c["length"])]
                keys = torch.cat((common, torch.cat((s["kv"][b, ids, 0], s["k_rope"][b, ids, 0]), -1).double()))
            z = torch.cat((s["q"][b, i], s["q_rope"][b, i]), -1).double() @ keys.T / 24.0
            top = z.max(-1).values
            w = torch.exp(z - top[:, None])
            total = w.sum(-1)
            outs.append(w @ keys[:, :LATENT] / total[:, None])
            tops.append(top)
            totals.append(total)
    shape = (c["batch"], 1, c["queries"], c["heads"])
    return (torch.stack(outs).reshape(c["batch"], c["queries"], c["heads"], LATENT), torch.stack(tops).reshape(shape),
            torch.stack(totals).reshape(shape))


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    c = case
    tokens = c["batch"] * c["queries"]
    if c["op"] == "rotary":
        passes = 2 if c["grad"] else 1
        n = tokens * c["heads"]
        return {"bytes": passes * 2 * n * c["dim"] * BYTES[c["dtype"]] + tokens * 4, "flops": passes * n * c["rotary_dim"] * 3}
    if c["op"] == "pages":
        blocks = -(-3 * c["batch"] * c["max_blocks"] // 4)
        return {"bytes": 8 * c["batch"] * c["max_blocks"] + 8 * blocks + 12 * tokens + 12 * c["batch"], "flops": 0}
    if c["op"] == "append":
        real = tokens if c["queries"] == 1 else tokens / 2  # prompts of every length up to the longest
        return {"bytes": real * (2 * (LATENT + ROPE) + (ROW if c["fp8"] else 2 * (LATENT + ROPE))) + 8 * tokens,
                "flops": real * (3 * ROPE + (2 * LATENT if c["fp8"] else 0))}
    rows = tokens * c["heads"]
    keys = c["filled"] + c["topk"]
    return {"bytes": rows * (4 * LATENT + 2 * ROPE + 8) + 2 * (LATENT + ROPE) * (c["filled"] + tokens * c["topk"]) + 4 * tokens * c["topk"],
            "flops": 2.0 * rows * keys * (2 * LATENT + ROPE)}
