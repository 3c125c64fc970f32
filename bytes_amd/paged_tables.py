"""Block tables, lengths and slot maps of a serving batch, kept on the GPU.

The tables are those of bytes_amd.paged: block_table [B, max_blocks] int32 (-1 where
there is no block) and context_lens [B] int32.  The blocks that nobody holds are a
ring: free_blocks [num_blocks] int32 and free_range = (head, count) int32, free being
free_blocks[(head + i) % num_blocks] for i < count.  All of it is device memory that a
step updates in place, without a synchronisation, so that a step can be captured
in a graph with the append and the attention that follow it.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _checks as C
from ._lib import call, native, ptr, size_query, stream_of


class Resized(NamedTuple):
    """What a step gives beside the tables: see paged_resize."""
    cu_seqlens: torch.Tensor
    granted: torch.Tensor
    seqs: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def paged_pool(num_blocks: int, B: int, max_blocks: int,
               device) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Empty tables of B sequences over a pool of num_blocks free blocks: block_table,
    context_lens, free_blocks, free_range."""
    if num_blocks < 1 or B < 1 or max_blocks < 1:
        raise ValueError(f"a pool has blocks, sequences and columns; got {num_blocks}, {B}, {max_blocks}")
    i32 = dict(dtype=torch.int32, device=device)
    return (torch.full((B, max_blocks), -1, **i32), torch.zeros(B, **i32), torch.arange(num_blocks, **i32),
            torch.tensor([0, num_blocks], **i32))


def _own(t: torch.Tensor, name: str, *shape: int) -> None:
    """int32 that is used (and written) in place."""
    C.dtype_in(t, name, torch.int32)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {list(shape)}; got {tuple(t.shape)}, strides {t.stride()}")


def paged_resize(block_table: torch.Tensor, context_lens: torch.Tensor, free_blocks: torch.Tensor,
                 free_range: torch.Tensor, new_lens: torch.Tensor, tokens: int, block_size: int, *,
                 keep: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0) -> Resized:
    """One step of a batch: tokens taken back, blocks returned and taken, lengths and the
    new tokens' places, in place and without a synchronisation.

    Of every sequence the first keep[b] tokens stay (int32 [B], more than it holds: all;
    0 ends it; None: all), so a row can take another request in the step in which its
    old one ends, and rejected draft tokens are taken back.  Blocks past them return to
    the pool.  With a window, so do the blocks whose tokens no position from keep[b]
    on sees (t > p - window or t < sinks), from the window's edge down to the first
    place without a block: attention with the same window does not read them, and the
    table holds -1 there.

    Then new_lens[b] tokens (int32 [B]; none if negative) are added.  They are granted
    in the order of the sequences, whole or not at all: where they fit the table's row,
    and where the blocks and the tokens that this and the earlier sequences ask for are
    at most those that were free and `tokens`.  (Blocks returned in a step can be had
    from the next one on.)  granted [B] int32 says how many; context_lens then counts
    them, as the paged operators take it.

    The rows of the step's tokens, `tokens` of them, hold the sequences one after
    another: cu_seqlens [B + 1] int32 as paged_kv_append and paged_prompt_attn take it, and
    for each row seqs, positions (int32) and slots (int64: block * block_size + row of
    the block, -1 where the table names no block); -1 in rows past cu_seqlens[B].

    block_table [B, max_blocks] (rows may be strided), context_lens, free_blocks and
    free_range are int32, written in place, and belong to one pool: each block is in one
    place of one table row, or in the ring.  A pool that is not is answered wrongly,
    but nothing is read or written outside these tensors."""
    if window is not None:
        if int(window) < 1 or int(sinks) < 0:
            raise ValueError(f"window={window}, sinks={sinks}: a window has at least one token, sinks are none or more")
        w, s = min(int(window), 2 ** 30), min(int(sinks), 2 ** 30)
    elif int(sinks) != 0:
        raise ValueError(f"sinks={sinks}: without a window no block is returned")
    else:
        w = s = 0
    out = native().paged_resize(block_table, context_lens, free_blocks, free_range, new_lens, keep, tokens, block_size, w, s)
    if out is not None:
        return Resized(*out)
    C.cuda_tensors(block_table, context_lens, free_blocks, free_range, new_lens, *((keep,) if keep is not None else ()))
    C.ndim(block_table, 2, "block_table"), C.ndim(free_blocks, 1, "free_blocks")
    C.dtype_in(block_table, "block_table", torch.int32)
    B, W = block_table.shape
    N, T, bs = free_blocks.shape[0], int(tokens), int(block_size)
    if B == 0 or W == 0 or N == 0:
        raise ValueError(f"empty block_table {tuple(block_table.shape)} or free_blocks [{N}]")
    if (W > 1 and block_table.stride(1) != 1) or (B > 1 and block_table.stride(0) < W):
        raise ValueError(f"block_table is written: rows of unit stride apart from each other; got strides "
                         f"{block_table.stride()}")
    if T < 0 or bs < 1:
        raise ValueError(f"tokens={tokens}, block_size={block_size}: not negative, and at least 1")
    if W * bs > 2 ** 30 or T > 2 ** 30 or N > 2 ** 30 or B > 2 ** 24:
        raise ValueError("more than 2^30 positions in a row, tokens or blocks, or 2^24 sequences")
    _own(context_lens, "context_lens", B), _own(free_blocks, "free_blocks", N), _own(free_range, "free_range", 2)
    C.dtype_in(new_lens, "new_lens", torch.int32)
    if keep is not None:
        C.dtype_in(keep, "keep", torch.int32)
    for t, n in ((new_lens, "new_lens"), (keep, "keep")):
        if t is not None and tuple(t.shape) != (B,):
            raise ValueError(f"{n} must be [B] = [{B}]; got {tuple(t.shape)}")
    mine = (block_table, context_lens, free_blocks, free_range)
    if len({t.data_ptr() for t in mine}) < len(mine) or any(
            t is not None and any(t.data_ptr() == o.data_ptr() for o in mine) for t in (new_lens, keep)):
        raise ValueError("what a step writes must be memory of its own")
    new_lens = new_lens.contiguous()
    keep = keep.contiguous() if keep is not None else None
    dev = block_table.device
    with torch.cuda.device(dev):
        i32 = dict(dtype=torch.int32, device=dev)
        cu, granted = torch.empty(B + 1, **i32), torch.empty(B, **i32)
        seqs, positions = torch.empty(T, **i32), torch.empty(T, **i32)
        slots = torch.empty(T, dtype=torch.int64, device=dev)
        n = size_query("bytes_paged_resize_workspace_size", B)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
        call("bytes_paged_resize", ptr(block_table), block_table.stride(0), ptr(context_lens), ptr(free_blocks),
             ptr(free_range), ptr(keep) if keep is not None else None, ptr(new_lens), ptr(cu), ptr(granted), ptr(seqs),
             ptr(positions), ptr(slots), B, W, N, T, bs, w, s, ptr(ws), ws.numel(), stream_of(block_table))
    return Resized(cu, granted, seqs, positions, slots)
