"""Page plans and cache appends: what a serving step does before ``forward_paged``.

``plan_pages`` builds, on the GPU, the block tables, token positions and cache
slots of a step from the requests' lengths; ``append_kv`` / ``append_kv_fp8``
write the new tokens' rows into the caches that ``forward_paged`` (or
``forward``) and ``forward_fp8`` read. The reference has no cache management
(README.md:19-20).

A dense cache ``[B, L, 1, 512]`` is the page pool of ``B`` blocks of ``L``
rows, so the slot of position ``p`` of row ``b`` is ``b * L + p``.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _native, api
from .rope import _check_rope, _followed

PagePlan = namedtuple("PagePlan", "block_table seq_lens positions lengths slots free_blocks free_count missing")


def plan_pages(block_table, cached_lens, new_lens, free_blocks, free_count, block_size, queries, *, reset=None,
               inplace=False):
    """Pages, positions and cache slots of ``new_lens[b]`` more tokens for every batch row.

    ``block_table`` int32 ``[B, MB]`` and ``cached_lens`` int32 ``[B]`` describe
    the cache so far; ``free_blocks`` int32 ``[NB]`` is a stack of
    ``free_count`` (int32 ``[1]``) page numbers; ``queries`` is the padded
    number of new tokens per row (``SQ`` of the step's tensors). ``reset``
    (bool ``[B]``) gives rows to new requests: their pages go back on the stack
    first and their cached length counts as 0 (with ``new_lens`` 0 the row is
    only released). Rows take pages from the top of the stack, in order.

    Returns a ``PagePlan`` of int32 tensors: the new ``block_table``,
    ``seq_lens`` ``[B]``, ``positions``, ``lengths`` (positions + 1, the
    indexer's key counts) and ``slots`` (cache rows, for ``append_kv``)
    ``[B, SQ]``, the stack ``free_blocks`` and ``free_count``, and ``missing``
    ``[1]``, the pages that the new tokens lack: their table entries and the
    slots of their tokens are -1, so that they are neither written nor read.
    They are the ones that the stack could not give now, and those of earlier
    steps (-1 in ``block_table``) in which new tokens go on: a page once missing
    is not asked for again, since its earlier tokens are lost. Rows with a
    position but no slot are the ones to ``reset`` and run again; their
    ``seq_lens`` count the lost tokens (a caller that would rather wait for
    pages keeps the inputs, without ``inplace``, and repeats the call). Padding
    has position and slot -1 and length 0. Lengths out of range are clamped (to
    ``[0, SQ]`` new tokens and to the table's room).

    New tensors are returned, unless ``inplace`` updates ``block_table``,
    ``cached_lens`` (to ``seq_lens``), ``free_blocks`` and ``free_count``; the
    call is asynchronous, allocates through torch and can be captured.
    """
    if type(block_size) is not int or type(queries) is not int or block_size <= 0 or queries <= 0 or block_table.dim() != 2:
        raise ValueError("block_table must be 2-D, block_size and queries positive ints")
    batch, max_blocks = block_table.shape
    num_blocks = free_blocks.numel()
    rows = cached_lens.shape
    if (not batch or not max_blocks or not num_blocks or free_blocks.dim() != 1 or rows != (batch,)
            or new_lens.shape != rows or free_count.numel() != 1 or (reset is not None and reset.shape != rows)):
        raise ValueError("need block_table[B,MB], cached_lens[B], new_lens[B], free_blocks[NB], free_count[1], reset[B]")
    device, index, int32 = block_table.device, block_table.get_device(), torch.int32
    if device.type != api.DEVICE_TYPE:
        raise ValueError("all inputs must be contiguous and on the same CUDA device")
    for t in (block_table, cached_lens, new_lens, free_blocks, free_count):
        if t.dtype is not int32:
            raise ValueError("block_table, lengths and free pages must be int32 and reset bool")
        if t.get_device() != index or not t.is_contiguous():
            raise ValueError("all inputs must be contiguous and on the same CUDA device")
    if reset is not None:
        if reset.dtype is not torch.bool:
            raise ValueError("block_table, lengths and free pages must be int32 and reset bool")
        if reset.get_device() != index or not reset.is_contiguous():
            raise ValueError("all inputs must be contiguous and on the same CUDA device")
    if (max_blocks * block_size > 0x7fffffff or num_blocks * block_size > 0x7fffffff or batch * queries > 0x7fffffff
            or batch * max_blocks > 0x7fffffff):
        raise ValueError("a table, the page pool or the step holds more than 2^31 - 1 entries")
    # few allocations and views: they cost more host time than the kernels take
    positions, lengths, slots = block_table.new_empty((3, batch, queries)).unbind(0)
    words = 4 * batch + 4
    if inplace:
        table, lens, stack, count = block_table, cached_lens, free_blocks, free_count
        work, missing = block_table.new_empty(words + 1).split_with_sizes((words, 1))
    else:
        table, stack = torch.empty_like(block_table), torch.empty_like(free_blocks)
        work, missing, count, lens = block_table.new_empty(words + 2 + batch).split_with_sizes((words, 1, 1, batch))
    api.enqueue("dsa_plan_pages", _native.PlanPagesArgs(
        block_table.data_ptr(), cached_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(),
        free_count.data_ptr(), None if reset is None else reset.data_ptr(), table.data_ptr(), lens.data_ptr(),
        positions.data_ptr(), lengths.data_ptr(), slots.data_ptr(), stack.data_ptr(), count.data_ptr(),
        missing.data_ptr(), batch, queries, max_blocks, num_blocks, block_size, work.data_ptr(), 4 * words), index)
    if inplace:
        torch.autograd.graph.increment_version((table, lens, stack, count))
    return PagePlan(table, lens, positions, lengths, slots, stack, count, missing)


def _append(kv, k_rope, slots, latent, rope, fp8, rows, positions, inv_freq, layout, attention_factor):
    """Checks and launch; the caches (``rows`` rows, shapes and types checked) are ``latent`` and ``rope``, or ``fp8``."""
    shape, index, bf16, int32 = kv.shape, kv.get_device(), torch.bfloat16, torch.int32
    if len(shape) != 4 or shape[2] != 1 or shape[3] != 512 or not shape[0] or not shape[1]:
        raise ValueError("need kv[B,S,1,512] and k_rope[B,S,1,64]")
    batch, queries, _, _ = shape
    if k_rope.shape != (batch, queries, 1, 64):
        raise ValueError("need kv[B,S,1,512] and k_rope[B,S,1,64]")
    lead = slots.shape
    if lead != (batch, queries) or slots.dtype is not int32:
        raise ValueError("slots must be int32 [B,S]")
    if kv.dtype is not bf16 or k_rope.dtype is not bf16:
        raise ValueError("kv and k_rope must be bfloat16")
    kv0, kv1, _, kv3 = kv.stride()
    kr0, kr1, _, kr3 = k_rope.stride()
    if kv3 != 1 or kr3 != 1:
        raise ValueError("the last dimension of kv and k_rope must be contiguous")
    first = latent if fp8 is None else fp8
    if (kv.device.type != api.DEVICE_TYPE or k_rope.get_device() != index or slots.get_device() != index
            or first.get_device() != index or (rope is not None and rope.get_device() != index)):
        raise ValueError("all inputs must be on the same CUDA device")
    if not slots.is_contiguous() or not first.is_contiguous() or (rope is not None and not rope.is_contiguous()):
        raise ValueError("slots and the cache must be contiguous")
    if _followed(kv) or _followed(k_rope) or _followed(first) or (rope is not None and _followed(rope)):
        raise ValueError("appends have no gradient: call them under torch.no_grad() or detach kv, k_rope and the cache")
    if inv_freq is not None and positions is not None:
        number = _check_rope(positions, inv_freq, layout, attention_factor, lead, index)
        if positions.dtype is not int32 or not positions.is_contiguous() or inv_freq.shape[0] != 32:
            raise ValueError("positions must be contiguous int32 [B,S] and inv_freq have 32 entries")
        pos_at, freq_at = positions.data_ptr(), inv_freq.data_ptr()
    elif inv_freq is not None or positions is not None:
        raise ValueError("positions and inv_freq go together")
    elif layout in _native.ROPE_LAYOUTS:
        number, attention_factor, pos_at, freq_at = 0, 1.0, None, None
    else:
        raise ValueError("layout must be 'interleaved' or 'half'")
    if rows > 0x7fffffff or batch * queries > 0x7fffffff:
        raise ValueError("the cache or the step holds more than 2^31 - 1 rows")
    if fp8 is None:
        caches = first.data_ptr(), rope.data_ptr(), None
    else:
        caches = None, None, first.data_ptr()
    api.enqueue("dsa_append_kv", _native.AppendKvArgs(
        kv.data_ptr(), k_rope.data_ptr(), slots.data_ptr(), pos_at, freq_at, *caches, batch, queries, rows,
        kv0, kv1, kr0, kr1, number, attention_factor), index)
    torch.autograd.graph.increment_version((first,) if rope is None else (first, rope))


def append_kv(kv, k_rope, slots, kv_cache, k_rope_cache, *, positions=None, inv_freq=None, layout="interleaved",
              attention_factor=1.0):
    """Write the new tokens' rows into a BF16 cache, in place.

    ``kv`` ``[B, S, 1, 512]`` and ``k_rope`` ``[B, S, 1, 64]`` BF16 (any
    strides with the last dimension contiguous: slices of the projection's
    output will do) go to the rows ``slots`` (int32 ``[B, S]``) of
    ``kv_cache`` ``[NB, BS, 1, 512]`` / ``k_rope_cache`` ``[NB, BS, 1, 64]``,
    flattened over the first two dimensions. A slot outside the cache writes
    nothing (padding is -1); the other rows keep what they hold. Slots of one
    call must be distinct (those of a plan are). With ``positions`` (int32
    ``[B, S]``) and ``inv_freq`` (FP64 ``[32]``) ``k_rope`` is turned first, as
    by ``rotary``; without them it is stored as given. ``kv`` and ``k_rope``
    share no memory with the cache. No gradient goes through a cache: tensors
    that autograd follows are refused.
    """
    shape = kv_cache.shape
    if len(shape) != 4 or shape[2] != 1 or shape[3] != 512 or not shape[0] or not shape[1]:
        raise ValueError("need kv_cache[NB,BS,1,512] and k_rope_cache[NB,BS,1,64]")
    blocks, block_size, _, _ = shape
    if k_rope_cache.shape != (blocks, block_size, 1, 64):
        raise ValueError("need kv_cache[NB,BS,1,512] and k_rope_cache[NB,BS,1,64]")
    if kv_cache.dtype is not torch.bfloat16 or k_rope_cache.dtype is not torch.bfloat16:
        raise ValueError("the caches must be bfloat16")
    _append(kv, k_rope, slots, kv_cache, k_rope_cache, None, blocks * block_size, positions, inv_freq, layout,
            attention_factor)


def append_kv_fp8(kv, k_rope, slots, cache, *, positions=None, inv_freq=None, layout="interleaved",
                  attention_factor=1.0):
    """``append_kv`` into the FP8 rows that ``forward_fp8`` reads.

    ``cache`` is uint8 ``[NB, BS, 1, 656]`` (``[B, L, 1, 656]`` for
    ``forward_fp8``). A row holds what ``quantize_kv_fp8`` makes of the same
    token on the host, bit for bit, with ``k_rope`` turned first when
    ``positions`` and ``inv_freq`` are given. (On the GPU that function's
    ``amax / 448`` is torch's product with the rounded 1 / 448, so its scales
    may be one FP32 step away.)
    """
    shape = cache.shape
    if len(shape) != 4 or shape[2] != 1 or shape[3] != _native.FP8_ROW_BYTES or not shape[0] or not shape[1]:
        raise ValueError("need cache[NB,BS,1,656]")
    if cache.dtype is not torch.uint8:
        raise ValueError("the FP8 cache must be uint8")
    _append(kv, k_rope, slots, None, None, cache, shape[0] * shape[1], positions, inv_freq, layout, attention_factor)
