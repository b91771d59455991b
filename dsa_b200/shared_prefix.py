"""Attention of a batch over a prefix that its queries share, computed once for all of them.

Samples of one prompt, or requests behind one system prompt, attend to the
same leading keys. ``forward`` would gather those keys again for every query;
``forward_shared_prefix`` reads them once per 128 (query, head) rows as one
dense product and joins the result with each query's own selected keys. The
reference has no such call: its forward takes every key through a query's
index row (dsa/api.py:76-132).

The prefix is attended to in full, not by selection. That is dense MLA
attention (a model without an indexer, or its dense layers and warm-up), and
sparse attention as long as the whole prefix is among the selected keys, that
is up to the indexer's top-k. Beyond it a model with an indexer lets prefix and
own keys compete for the top-k: ``indexer_topk`` and ``forward`` over both.
"""
from __future__ import annotations

import torch

from . import _native, api
from .rope import _followed

WORKSPACE_BUDGET = 1 << 31  # bytes of FP32 partials per library call
_AUTO = _native.Launch()  # family 0: the library's choice


def forward_shared_prefix(q, prefix_kv, q_rope, prefix_k_rope, kv=None, k_rope=None, indices=None, *, prefix_len=None,
                          scale=None):
    """``forward`` over ``[prefix keys, own selected keys]`` as one softmax.

    ``prefix_kv`` BF16 ``[1, P, 1, 512]`` and ``prefix_k_rope`` ``[1, P, 1, 64]``
    are attended to by every query in full (``prefix_len``, an int32 ``[1]``
    tensor on the device, limits them to the first ``prefix_len`` rows; the
    rows behind may hold anything; the launch is planned for all ``P`` rows, so
    a buffer filled in small part is better cut to size where the host knows
    it). ``kv`` ``[B, L, 1, 512]``, ``k_rope`` ``[B, L, 1, 64]`` and ``indices``
    int32 ``[B, SQ, 1, K]`` are ``forward``'s for the keys of each batch row
    itself (rows that no valid index names may hold anything too); without them
    the prefix is all there is. ``q`` ``[B, SQ, H, 512]`` and ``q_rope`` ``[B, SQ, H, 64]``, H a
    multiple of 16, are turned already, at positions behind the prefix.

    Returns ``(output, softmax_max, softmax_sum)`` as ``forward`` does, over
    both sets of keys: indices outside ``[0, L)`` are masked, duplicates keep
    their repeated weight, a row without any key gets output 0, maximum -inf
    and sum 0, one with a NaN score NaN, -inf and NaN. The call has no gradient
    and refuses inputs that autograd follows. Asynchronous on the
    current stream; partials are FP32, in pieces of whole queries that keep
    them under ``WORKSPACE_BUDGET`` bytes.
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
    device, index, bf16, length, topk = q.device, q.get_device(), torch.bfloat16, 0, 0
    if device.type != api.DEVICE_TYPE:
        raise ValueError("all inputs must be contiguous and on the same CUDA device")
    tensors = (q, q_rope, prefix_kv, prefix_k_rope)
    if kv is not None or k_rope is not None or indices is not None:
        if kv is None or k_rope is None or indices is None:
            raise ValueError("kv, k_rope and indices go together")
        if kv.dim() != 4 or indices.dim() != 4:
            raise ValueError("kv and indices must be 4-D tensors")
        length, topk = kv.shape[1], indices.shape[-1]
        if (kv.shape != (batch, length, 1, 512) or k_rope.shape != (batch, length, 1, 64)
                or indices.shape != (batch, queries, 1, topk) or length == 0 or topk == 0):
            raise ValueError("need kv[B,L,1,512], k_rope[B,L,1,64], indices[B,SQ,1,K]")
        tensors = (q, q_rope, prefix_kv, prefix_k_rope, kv, k_rope)
    for t in tensors:
        if t.dtype is not bf16:
            raise ValueError("q, q_rope, the prefix and kv/k_rope must be bfloat16, indices and prefix_len int32")
        if t.get_device() != index or not t.is_contiguous():
            raise ValueError("all inputs must be contiguous and on the same CUDA device")
        if _followed(t):
            raise ValueError("forward_shared_prefix has no gradient: call it under torch.no_grad() or detach its inputs")
    if prefix_len is not None and prefix_len.numel() != 1:
        raise ValueError("prefix_len must be an int32 tensor of one element")
    for t in (indices, prefix_len):
        if t is None:
            continue
        if t.dtype is not torch.int32:
            raise ValueError("q, q_rope, the prefix and kv/k_rope must be bfloat16, indices and prefix_len int32")
        if t.get_device() != index or not t.is_contiguous():
            raise ValueError("all inputs must be contiguous and on the same CUDA device")
    scale_arg = 0.0 if scale is None else api._check_scale(scale)
    if prefix > 1 << 26 or batch * queries > 0x7fffffff or batch * length > 0x7fffffff:
        raise ValueError("the prefix holds more than 2^26 rows, or the batch more than 2^31 - 1 queries or keys")
    output = torch.empty_like(q)
    maximum = q.new_empty((batch, 1, queries, heads), dtype=torch.float32)
    denominator = torch.empty_like(maximum)
    px = _native.PrefixKv(prefix_kv.data_ptr(), prefix_k_rope.data_ptr(),
                          None if prefix_len is None else prefix_len.data_ptr(), prefix)
    args = _native.FwdArgs(
        q.data_ptr(), kv.data_ptr() if topk else None, q_rope.data_ptr(), k_rope.data_ptr() if topk else None,
        indices.data_ptr() if topk else None, output.data_ptr(), maximum.data_ptr(), denominator.data_ptr(), batch, queries,
        heads, length, topk, _AUTO, None, 0, api._status_word(device).data_ptr(), scale_arg)
    if not _enqueue(args, px, device, index):
        # halves of what does not fit the workspace budget, in order: batch rows, then queries of one row
        pieces = [(0, batch, 0, queries)]
        while pieces:
            b0, b1, s0, s1 = pieces.pop()
            if _enqueue(_piece(args, b0, b1, s0, s1), px, device, index):
                continue
            if b1 - b0 > 1:
                mid = (b0 + b1) // 2
                pieces += [(mid, b1, s0, s1), (b0, mid, s0, s1)]
            else:
                mid = (s0 + s1) // 2
                pieces += [(b0, b1, mid, s1), (b0, b1, s0, mid)]
    return output, maximum, denominator


def _enqueue(args, px, device, index):
    """Launch the call of ``args`` unless it takes more workspace than the budget and can be cut."""
    need = _native.load().dsa_fwd_prefix_workspace_bytes(args, px)
    if need:
        if need > WORKSPACE_BUDGET and args.batch * args.queries > 1:
            return False
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    api.enqueue("dsa_sparse_mla_fwd_prefix", args, index, px)
    return True


def _piece(args, b0, b1, s0, s1):
    """The arguments for batch rows ``[b0, b1)`` and queries ``[s0, s1)`` (all of them when there are several rows)."""
    t0 = b0 * args.queries + s0
    rows = t0 * args.heads
    piece = _native.FwdArgs.from_buffer_copy(args)
    piece.q, piece.q_rope, piece.output = args.q + rows * 1024, args.q_rope + rows * 128, args.output + rows * 1024
    piece.softmax_max, piece.softmax_sum = args.softmax_max + rows * 4, args.softmax_sum + rows * 4
    if args.topk:
        piece.kv, piece.k_rope = args.kv + b0 * args.length * 1024, args.k_rope + b0 * args.length * 128
        piece.indices = args.indices + t0 * args.topk * 4
    piece.batch, piece.queries = b1 - b0, s1 - s0
    return piece
