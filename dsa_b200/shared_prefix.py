"""Attention of a batch over a prefix that its queries share, computed once for all of them.

Samples of one prompt, or requests behind one system prompt, attend to the
same leading keys. ``forward`` would gather those keys again for every query;
``forward_shared_prefix`` reads them once per 128 (query, head) rows as one
dense product and joins the result with each query's own selected keys. The
reference has no such call: its forward takes every key through a query's
index row (dsa/api.py:76-132).
"""
from __future__ import annotations

import torch

from . import _native, api

WORKSPACE_BUDGET = 1 << 31  # bytes of FP32 partials per library call
_AUTO = _native.Launch()  # family 0: the library's choice


def forward_shared_prefix(q, prefix_kv, q_rope, prefix_k_rope, kv=None, k_rope=None, indices=None, *, prefix_len=None,
                          scale=None):
    """``forward`` over ``[prefix keys, own selected keys]`` as one softmax.

    ``prefix_kv`` BF16 ``[1, P, 1, 512]`` and ``prefix_k_rope`` ``[1, P, 1, 64]``
    are attended to by every query in full (``prefix_len``, an int32 ``[1]``
    tensor on the device, limits them to the first ``prefix_len`` rows; the
    rows behind may hold anything). ``kv`` ``[B, L, 1, 512]``, ``k_rope``
    ``[B, L, 1, 64]`` and ``indices`` int32 ``[B, SQ, 1, K]`` are ``forward``'s
    for the keys of each batch row itself; without them the prefix is all
    there is. ``q`` ``[B, SQ, H, 512]`` and ``q_rope`` ``[B, SQ, H, 64]``, H a
    multiple of 16, are turned already, at positions behind the prefix.

    Returns ``(output, softmax_max, softmax_sum)`` as ``forward`` does, over
    both sets of keys: indices outside ``[0, L)`` are masked, duplicates keep
    their repeated weight, a row without any key gets output 0, maximum -inf
    and sum 0. Asynchronous on the current stream; partials are FP32, in
    pieces of whole queries that keep them under ``WORKSPACE_BUDGET`` bytes.
    """
    shape = q.shape
    if len(shape) != 4 or prefix_kv.dim() != 4:
        raise ValueError("q and prefix_kv must be 4-D tensors")
    batch, queries, heads, width = shape
    prefix = prefix_kv.shape[1]
    if (width != 512 or 0 in shape or prefix == 0 or q_rope.shape != (batch, queries, heads, 64)
            or prefix_kv.shape != (1, prefix, 1, 512) or prefix_k_rope.shape != (1, prefix, 1, 64)):
        raise ValueError("need q[B,SQ,H,512], q_rope[B,SQ,H,64], prefix_kv[1,P,1,512], prefix_k_rope[1,P,1,64]")
    if heads % 16:
        raise ValueError("the head count must be a multiple of 16")
    halves, ints = [q, q_rope, prefix_kv, prefix_k_rope], []
    length = topk = 0
    if kv is not None or k_rope is not None or indices is not None:
        if kv is None or k_rope is None or indices is None:
            raise ValueError("kv, k_rope and indices go together")
        if kv.dim() != 4 or indices.dim() != 4:
            raise ValueError("kv and indices must be 4-D tensors")
        length, topk = kv.shape[1], indices.shape[-1]
        if (kv.shape != (batch, length, 1, 512) or k_rope.shape != (batch, length, 1, 64)
                or indices.shape != (batch, queries, 1, topk) or length == 0 or topk == 0):
            raise ValueError("need kv[B,L,1,512], k_rope[B,L,1,64], indices[B,SQ,1,K]")
        halves += (kv, k_rope)
        ints.append(indices)
    if prefix_len is not None:
        if prefix_len.numel() != 1:
            raise ValueError("prefix_len must be an int32 tensor of one element")
        ints.append(prefix_len)
    device, index = q.device, q.get_device()
    if device.type != api.DEVICE_TYPE:
        raise ValueError("all inputs must be contiguous and on the same CUDA device")
    for tensors, dtype in ((halves, torch.bfloat16), (ints, torch.int32)):
        for t in tensors:
            if t.dtype != dtype:
                raise ValueError("q, q_rope, the prefix and kv/k_rope must be bfloat16, indices and prefix_len int32")
            if t.get_device() != index or not t.is_contiguous():
                raise ValueError("all inputs must be contiguous and on the same CUDA device")
    scale_arg = 0.0 if scale is None else api._check_scale(scale)
    if prefix > 1 << 30 or batch * queries > 0x7fffffff or batch * length > 0x7fffffff:
        raise ValueError("the prefix holds more than 2^30 rows, or the batch more than 2^31 - 1 queries or keys")
    output = torch.empty_like(q)
    maximum = torch.empty((batch, 1, queries, heads), device=device, dtype=torch.float32)
    denominator = torch.empty_like(maximum)
    lib = _native.load()
    px = _native.PrefixKv(prefix_kv.data_ptr(), prefix_k_rope.data_ptr(),
                          None if prefix_len is None else prefix_len.data_ptr(), prefix)
    bases = [t.data_ptr() for t in (q, q_rope, output, maximum, denominator)]
    own = (kv.data_ptr(), k_rope.data_ptr(), indices.data_ptr()) if topk else (None, None, None)
    status = api._status_word(device).data_ptr()

    def call(b0, b1, s0, s1):
        t0 = b0 * queries + s0
        rows = t0 * heads
        q_at, qr_at, out_at, max_at, sum_at = (at + rows * n for at, n in zip(bases, (1024, 128, 1024, 4, 4)))
        kv_at, kr_at, ids_at = own
        if topk and t0:
            kv_at, kr_at, ids_at = kv_at + b0 * length * 1024, kr_at + b0 * length * 128, ids_at + t0 * topk * 4
        a = _native.FwdArgs(q_at, kv_at, qr_at, kr_at, ids_at, out_at, max_at, sum_at, b1 - b0, s1 - s0, heads, length,
                            topk, _AUTO, None, 0, status, scale_arg)
        need = lib.dsa_fwd_prefix_workspace_bytes(a, px)
        if need > WORKSPACE_BUDGET and (b1 - b0) * (s1 - s0) > 1:
            return False
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), need
        api.enqueue("dsa_sparse_mla_fwd_prefix", a, index, px)
        return True

    pieces = [(0, batch, 0, queries)]
    while pieces:  # halves of what does not fit, in order
        b0, b1, s0, s1 = pieces.pop()
        if call(b0, b1, s0, s1):
            continue
        if b1 - b0 > 1:
            mid = (b0 + b1) // 2
            pieces += [(mid, b1, s0, s1), (b0, mid, s0, s1)]
        else:
            mid = (s0 + s1) // 2
            pieces += [(b0, b1, mid, s1), (b0, b1, s0, mid)]
    return output, maximum, denominator
