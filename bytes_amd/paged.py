"""Paged dense KV caches: append with rotation, decode, page-sparse decode.

A cache is a pair k_paged, v_paged [num_blocks, H_k, block_size, D] of bf16, or
of float8_e4m3fn whose values stand for value * k_scale (v_scale): the layout of
the paged product-quantized operators (src/attention_kernels.py:588-622,
:858-906), with dense rows.  Any strides are taken as long as rows have unit
stride along D and start on 16-byte boundaries (a [.., block_size, H_k, D]
storage as well); caches are never copied, other layouts are refused.  Token p of
sequence b is row p % block_size of block block_table[b, p // block_size].

`context_lens[b]` is the number of tokens of sequence b in the cache, in every
operator here: the append takes it with the new tokens counted, so one tensor
serves a whole decode step.  Lengths, block tables and cu_seqlens stay on the
device; nothing here synchronises, and every call can be captured in a graph
(lengths and tables are read at replay).  The decodes hold lengths to 0 .. max_blocks *
block_size; the append takes them as they are, and new tokens at positions outside
that range are not written.  A block id outside [0, num_blocks) names no block (-1 past a
sequence's blocks, or a hole where a block was evicted): nothing is written for
its tokens and they take no part in attention.  A sequence none of whose tokens
take part (length 0, as in the padding rows of a batch) gets zeros.

Results carry no autograd graph.  H_q must be a multiple of H_k and D 64 or 128.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _checks as C
from ._lib import call, native, ptr, size_query, stream_of
from .sparse import _topk

_F8 = torch.float8_e4m3fn
Meta = Tuple[torch.Tensor, torch.Tensor]


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """A tensor that is used in place: unit stride along D, 16-byte rows."""
    es = t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(t.size(d) > 1 and t.stride(d) * es % 16 for d in range(t.dim() - 1)):
        raise ValueError(f"{name} needs unit stride in D and 16-byte-aligned rows (no copy is made); got strides "
                         f"{tuple(t.stride())}")
    return t


def _cache(k_paged: torch.Tensor, v_paged: torch.Tensor, k_scale: float, v_scale: float):
    """-> (num_blocks, H_k, block_size, D, the cache is fp8)."""
    C.ndim(k_paged, 4, "k_paged"), C.ndim(v_paged, 4, "v_paged")
    C.dtype_in(k_paged, "k_paged", torch.bfloat16, _F8)
    C.dtype_in(v_paged, "v_paged", k_paged.dtype)
    if tuple(v_paged.shape) != tuple(k_paged.shape):
        raise ValueError(f"shape mismatch: k_paged {tuple(k_paged.shape)}, v_paged {tuple(v_paged.shape)}")
    N, Hk, bs, D = k_paged.shape
    if N == 0 or Hk == 0 or bs == 0:
        raise ValueError(f"empty paged cache {tuple(k_paged.shape)}")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} not supported (64 or 128)")
    _rows(k_paged, "k_paged"), _rows(v_paged, "v_paged")
    fp8 = k_paged.dtype == _F8
    for s, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if not 0.0 < float(s) < float("inf"):
            raise ValueError(f"{n}={s} must be a positive finite number")
        if not fp8 and float(s) != 1.0:
            raise ValueError(f"{n}={s}: a bf16 cache has no scale (1.0)")
    return N, Hk, bs, D, fp8


def _int32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype == torch.int64:                   # values past int32 stay out of range
        return t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    C.dtype_in(t, name, torch.int32)
    return t


def _tables(block_table: torch.Tensor, context_lens: torch.Tensor, B: int, bs: int):
    if block_table.dim() != 2 or block_table.shape[0] != B or tuple(context_lens.shape) != (B,):
        raise ValueError(f"block_table must be [B, max_blocks] and context_lens [B] with B={B}; got "
                         f"{tuple(block_table.shape)}, {tuple(context_lens.shape)}")
    if block_table.shape[1] == 0:
        raise ValueError("block_table has no columns")
    if block_table.shape[1] * bs > 2 ** 30:
        raise ValueError(f"block_table names {block_table.shape[1]} blocks of {bs} tokens: more than 2^30 positions")
    bt = _int32(block_table, "block_table")
    if bt.stride(-1) != 1 and bt.shape[1] > 1:
        bt = bt.contiguous()
    return bt, _int32(context_lens, "context_lens").contiguous()


def _meta(meta: Meta, N: int, Hk: int, D: int) -> Meta:
    kmin, kmax = meta
    for t, n in ((kmin, "kmin"), (kmax, "kmax")):
        C.dtype_in(t, n, torch.bfloat16)
        if tuple(t.shape) != (N, Hk, D) or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{n} must be contiguous [num_blocks, H_k, D] = {(N, Hk, D)}; got {tuple(t.shape)}")
    return kmin, kmax


def _written(a: torch.Tensor, b: torch.Tensor, names: Tuple[str, str]) -> None:
    """Refuses two tensors that are written if two of their elements are in one place."""
    for t, n in zip((a, b), names):
        if any(t.size(d) > 1 and t.stride(d) == 0 for d in range(t.dim())):
            raise ValueError(f"{n} is written: an expanded view, with several elements in one place, is not supported")
    if a.data_ptr() == b.data_ptr():
        raise ValueError(f"{names[0]} and {names[1]} are written and must not be the same memory")


def _query(q: torch.Tensor, Hk: int, D: int):
    C.ndim(q, 4, "q")
    C.dtype_in(q, "q", torch.bfloat16)
    B, Hq, one, Dq = q.shape
    if one != 1 or Dq != D or B == 0 or Hq == 0:
        raise ValueError(f"q must be [B, H_q, 1, D] with D={D}; got {tuple(q.shape)}")
    if Hq % Hk != 0:
        raise ValueError(f"H_q={Hq} is not a multiple of H_k={Hk}")
    return C.rows16(q.squeeze(2)), B, Hq


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_paged: torch.Tensor, v_paged: torch.Tensor,
                    block_table: torch.Tensor, context_lens: torch.Tensor, *,
                    cu_seqlens: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                    cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, interleaved: bool = False,
                    meta: Optional[Meta] = None, k_scale: float = 1.0,
                    v_scale: float = 1.0) -> Optional[torch.Tensor]:
    """Write new tokens' keys and values into the cache, keys rotated by their
    position, in place.

    k, v [T, H_k, D] bf16 hold the new tokens of all sequences one after another
    (views of a fused projection are fine): sequence b's are rows cu_seqlens[b] ..
    cu_seqlens[b+1] (int32 [B+1], ascending from 0), or row b alone without
    cu_seqlens (T = B, the decode step).  Its n new tokens end at context_lens[b]:
    token i has position context_lens[b] - n + i.  Tokens without a position in
    0 .. max_blocks * block_size, and rows past cu_seqlens[B], are not written;
    cache rows that no new token names keep their bytes.

    cos, sin [P, R/2] fp32 (P >= max_blocks * block_size, R a multiple of 16, at
    most D): the first R dims of keys (and queries) are rotated in pairs (x0, x1)
    -> (x0 cos - x1 sin, x1 cos + x0 sin), pairs (j, j + R/2), or (2j, 2j + 1) if
    interleaved.
    fp8 caches store k / k_scale and v / v_scale, values beyond the format's range
    (infinities too) as its largest ones.

    meta (kmin, kmax), each [num_blocks, H_k, D] bf16: the elementwise min / max of
    every block's stored keys, kept for paged_quest_decode.  A block that a
    sequence enters at its first row starts anew, others are folded into: rows
    written again (after a rollback) widen them until then, so they stay bounds.
    (For a cache filled otherwise, quest_page_minmax(k_paged, block_size) gives
    them where all blocks are full.)

    q [T, H_q, D] bf16: returned rotated, [T, H_q, D] bf16 (with T = B,
    q_rot.unsqueeze(2) is paged_decode_attn's query); zeros in rows that have no
    position.  Without q the result is None.

    Blocks that receive tokens must belong to one sequence each, and be named once
    in its table row (blocks of a shared prefix are only read).  The caches and
    min / max must be memory of their own, without expanded dims."""
    kmin, kmax = meta if meta is not None else (None, None)
    out = native().paged_append(k, v, k_paged, v_paged, block_table, context_lens, cu_seqlens, q, cos, sin,
                                bool(interleaved), kmin, kmax, k_scale, v_scale)
    if out is not None:
        return out if q is not None else None
    C.cuda_tensors(k, v, k_paged, v_paged, block_table, context_lens,
                   *(t for t in (cu_seqlens, q, cos, sin, *(meta or ())) if t is not None))
    N, Hk, bs, D, fp8 = _cache(k_paged, v_paged, k_scale, v_scale)
    C.ndim(k, 3, "k"), C.ndim(v, 3, "v")
    C.dtype_in(k, "k", torch.bfloat16), C.dtype_in(v, "v", torch.bfloat16)
    T = k.shape[0]
    if tuple(k.shape) != (T, Hk, D) or tuple(v.shape) != (T, Hk, D):
        raise ValueError(f"k, v must be [T, H_k, D] with H_k={Hk}, D={D}; got {tuple(k.shape)}, {tuple(v.shape)}")
    B = block_table.shape[0] if block_table.dim() == 2 else 0
    bt, cl = _tables(block_table, context_lens, B, bs)
    if cu_seqlens is not None:
        if tuple(cu_seqlens.shape) != (B + 1,):
            raise ValueError(f"cu_seqlens must be [B + 1] = [{B + 1}]; got {tuple(cu_seqlens.shape)}")
        cu_seqlens = _int32(cu_seqlens, "cu_seqlens").contiguous()
    elif T != B:
        raise ValueError(f"{T} new tokens for {B} sequences need cu_seqlens")
    Hq = 0
    if q is not None:
        C.ndim(q, 3, "q")
        C.dtype_in(q, "q", torch.bfloat16)
        Hq = q.shape[1]
        if tuple(q.shape) != (T, Hq, D) or Hq == 0:
            raise ValueError(f"q must be [T, H_q, D] = [{T}, H_q, {D}]; got {tuple(q.shape)}")
    rot = P = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        for t, n in ((cos, "cos"), (sin, "sin")):
            C.ndim(t, 2, n)
            C.dtype_in(t, n, torch.float32)
        P, rot = cos.shape[0], 2 * cos.shape[1]
        if tuple(sin.shape) != tuple(cos.shape) or rot == 0 or rot % 16 or rot > D:
            raise ValueError(f"cos, sin must both be [P, R/2] with R a multiple of 16, at most D={D}; got "
                             f"{tuple(cos.shape)}, {tuple(sin.shape)}")
        if P < bt.shape[1] * bs:
            raise ValueError(f"cos, sin hold {P} positions, the block table {bt.shape[1] * bs}")
        cos, sin = C.rows16(cos), C.rows16(sin)
    _written(k_paged, v_paged, ("k_paged", "v_paged"))
    if meta is not None:
        kmin, kmax = _meta(meta, N, Hk, D)
        _written(kmin, kmax, ("kmin", "kmax"))
    k, v = C.rows16(k), C.rows16(v)
    out = None
    if q is not None:
        q = C.rows16(q)
        out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=q.device)
    if T == 0 or B == 0:
        return out.zero_() if out is not None else None
    z = lambda t, i: t.stride(i) if t is not None else 0    # noqa: E731
    p = lambda t: ptr(t) if t is not None else None          # noqa: E731
    with torch.cuda.device(k_paged.device):
        call("bytes_paged_kv_append", ptr(k), k.stride(0), k.stride(1), ptr(v), v.stride(0), v.stride(1),
             p(q), z(q, 0), z(q, 1), p(out), z(out, 0), z(out, 1),
             ptr(k_paged), k_paged.stride(0), k_paged.stride(1), k_paged.stride(2),
             ptr(v_paged), v_paged.stride(0), v_paged.stride(1), v_paged.stride(2), int(fp8), p(kmin), p(kmax),
             ptr(bt), bt.stride(0), ptr(cl), p(cu_seqlens), p(cos), z(cos, 0), p(sin), z(sin, 0), int(P), int(rot),
             int(bool(interleaved)), float(k_scale), float(v_scale), T, B, Hq, Hk, D, bs, N, bt.shape[1],
             stream_of(k_paged))
    return out


def paged_decode_attn(q: torch.Tensor, k_paged: torch.Tensor, v_paged: torch.Tensor, block_table: torch.Tensor,
                      context_lens: torch.Tensor, scale: float = 1.0, *, k_scale: float = 1.0,
                      v_scale: float = 1.0) -> torch.Tensor:
    """softmax(scale * q.K^T) V of one new token per sequence over the cache.

    q [B,H_q,1,D] bf16; `scale` as in decode_attn_bf16 (default 1.0; pass
    1/sqrt(D) for standard attention).  For fp8 caches the rows stand for
    k * k_scale and v * v_scale.  fp32 scores, softmax and sums.  An infinite value
    that takes part gives that infinity, unless its weight underflows fp32 (below
    2^-100 of the row's largest it may give NaN).  Returns [B,H_q,1,D] bf16."""
    out = native().paged_decode(q, k_paged, v_paged, block_table, context_lens, scale, k_scale, v_scale)
    if out is not None:
        return out
    C.cuda_tensors(q, k_paged, v_paged, block_table, context_lens)
    N, Hk, bs, D, fp8 = _cache(k_paged, v_paged, k_scale, v_scale)
    qs, B, Hq = _query(q, Hk, D)
    bt, cl = _tables(block_table, context_lens, B, bs)
    W = bt.shape[1]
    with torch.cuda.device(q.device):
        out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=q.device)
        n = size_query("bytes_paged_decode_workspace_size", B, Hq, Hk, D, int(fp8), bs, W)
        # the call's own: calls on other streams share nothing
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)
        call("bytes_paged_decode_attn", ptr(qs), qs.stride(0), qs.stride(1),
             ptr(k_paged), k_paged.stride(0), k_paged.stride(1), k_paged.stride(2),
             ptr(v_paged), v_paged.stride(0), v_paged.stride(1), v_paged.stride(2), int(fp8), ptr(bt), bt.stride(0),
             ptr(cl), ptr(out), out.stride(0), out.stride(1), B, Hq, Hk, D, bs, N, W, float(scale) * float(k_scale),
             float(v_scale), ptr(ws), ws.numel(), stream_of(q))
    return out.unsqueeze(2)


def paged_page_scores(q: torch.Tensor, meta: Meta, block_table: torch.Tensor, context_lens: torch.Tensor,
                      block_size: int, scaling: float = 1.0, *, local_w: int = 0) -> torch.Tensor:
    """bound[b,h,j] = scaling * sum_d q_d * (q_d >= 0 ? kmax_d : kmin_d) over the
    min / max of block block_table[b, j]: the largest score that a key of the block
    can have (the bound of quest_page_scores, benchmarks/sparse_attention.py:342-345).
    The sum is taken in 64 bits, so no order of it moves a selection, and rounded
    to fp32 once.  -inf for blocks that hold no token that takes part, +inf for those
    that reach into the sequence's last local_w tokens (:346-355).  q [B,H_q,1,D]
    bf16; meta as paged_kv_append keeps it.  Returns [B,H_q,max_blocks] fp32."""
    C.cuda_tensors(q, *meta, block_table, context_lens)
    C.ndim(meta[0], 3, "kmin")
    N, Hk, D = meta[0].shape
    if N == 0 or Hk == 0 or int(block_size) < 1:
        raise ValueError(f"bad metadata / block_size: {tuple(meta[0].shape)}, {block_size}")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} not supported (64 or 128)")
    kmin, kmax = _meta(meta, N, Hk, D)
    qs, B, Hq = _query(q, Hk, D)
    bt, cl = _tables(block_table, context_lens, B, int(block_size))
    return _page_scores(qs, kmin, kmax, bt, cl, int(block_size), float(scaling), local_w, -1)


def _page_scores(qs, kmin, kmax, bt, cl, bs: int, scale: float, local_w: int, skip: int) -> torch.Tensor:
    if int(local_w) < 0:
        raise ValueError(f"local_w={local_w} is negative")
    (B, Hq, D), (N, Hk, _), W = qs.shape, kmin.shape, bt.shape[1]
    with torch.cuda.device(qs.device):
        # rows that a kernel reads on are whole 16-byte chunks
        bound = torch.empty((B, Hq, W if skip < 0 else (W + 3) // 4 * 4), dtype=torch.float32, device=qs.device)
        call("bytes_paged_page_scores", ptr(qs), qs.stride(0), qs.stride(1), ptr(kmin), ptr(kmax), ptr(bt), bt.stride(0),
             ptr(cl), ptr(bound), bound.stride(0), bound.stride(1), B, Hq, Hk, D, bs, N, W, min(int(local_w), 2 ** 30),
             skip, scale, stream_of(qs))
    return bound


_SELECT_MAX = 16384        # blocks of a sequence that bytes_paged_quest_attn selects from


def paged_quest_decode(q: torch.Tensor, k_paged: torch.Tensor, v_paged: torch.Tensor, meta: Meta,
                       block_table: torch.Tensor, context_lens: torch.Tensor, kb: int, scaling: float, *,
                       local_w: int = 0, k_scale: float = 1.0, v_scale: float = 1.0, return_pages: bool = False):
    """quest_decode over a paged cache whose blocks are the pages: the
    ceil(kb / block_size) blocks of the highest bounds per query head
    (paged_page_scores; the lowest block first on equal bounds), exact attention over
    their tokens.  A sequence of fewer blocks is attended over whole.  The blocks of
    the last local_w tokens are all equally best, so a window of more blocks than are
    picked loses its newest ones, as in quest_decode: take kb of at least local_w +
    block_size.  q [B,H_q,1,D] bf16; meta as paged_kv_append keeps it.  Returns out
    [B,H_q,1,D] bf16 (and the selected blocks' places in the table, int32
    [B,H_q,min(ceil(kb / block_size), max_blocks)] ascending, if return_pages;
    places past a short sequence's blocks stand for nothing)."""
    if not return_pages:
        out = native().paged_quest(q, k_paged, v_paged, *meta, block_table, context_lens, kb, scaling, local_w, k_scale,
                                   v_scale)
        if out is not None:
            return out
    C.cuda_tensors(q, k_paged, v_paged, *meta, block_table, context_lens)
    N, Hk, bs, D, fp8 = _cache(k_paged, v_paged, k_scale, v_scale)
    if kb < 1:
        raise ValueError(f"kb={kb} must be at least 1")
    qs, B, Hq = _query(q, Hk, D)
    bt, cl = _tables(block_table, context_lens, B, bs)
    kmin, kmax = _meta(meta, N, Hk, D)
    W = bt.shape[1]
    npick = min((int(kb) + bs - 1) // bs, W)
    scale = float(scaling) * float(k_scale)
    listed = return_pages or W > _SELECT_MAX
    bound = _page_scores(qs, kmin, kmax, bt, cl, bs, scale, local_w, -1 if listed else npick)
    with torch.cuda.device(q.device):
        pages = None
        if listed:                               # with a top-k workspace of the call's own, as all else here
            n = size_query("bytes_topk_workspace_size", B * Hq, W, npick)
            pages = _topk(bound, npick, sorted=False, ws=torch.zeros(max(n, 16), dtype=torch.uint8, device=q.device))
        out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=q.device)
        n = size_query("bytes_paged_quest_workspace_size", B, Hq, Hk, D, int(fp8), bs, W, npick)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)
        call("bytes_paged_quest_attn", ptr(qs), qs.stride(0), qs.stride(1),
             ptr(k_paged), k_paged.stride(0), k_paged.stride(1), k_paged.stride(2),
             ptr(v_paged), v_paged.stride(0), v_paged.stride(1), v_paged.stride(2), int(fp8),
             None if listed else ptr(bound), bound.stride(0), bound.stride(1),
             ptr(pages) if listed else None, pages.stride(0) if listed else 0, pages.stride(1) if listed else 0, npick,
             ptr(bt), bt.stride(0), ptr(cl), ptr(out), out.stride(0), out.stride(1), B, Hq, Hk, D, bs, N, W, scale,
             float(v_scale), ptr(ws), ws.numel(), stream_of(q))
    return (out.unsqueeze(2), pages) if return_pages else out.unsqueeze(2)
