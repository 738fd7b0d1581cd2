"""Eviction from the 8-bit block cache: a conversation that grows without end keeps a budget of entries, the ones that
its queries have attended to most, with the first and the most recent positions among them.

    cache = BlockKVCache(..., evicting=True)                        # with weights and positions per entry
    plan = cache.plan(seqs, counts, n_tokens)
    for layer: q, k = cache.rotate(plan, q, k, inv_freq, scale)     # positions go on where entries were evicted
               cache.append(layer, plan, k, v)
               out = cache.decode(layer, plan, q)
               cache.weigh_decode(layer, plan, q)                   # kvt_block_weigh: the attention weight of each entry
    cache.evict(seqs, budget, recent, sinks)                        # kvt_block_keep and _evict per layer, kvt_block_trim

Every KV head keeps its own entries, all of them the same number, so the heads and layers share one block table.  Entries
that stay below the budget stay where they are, and those from behind it fill the places that become free: a cache's
entries are in no order of positions after that, which attention does not ask for.  All of it happens on the device,
without host lengths, and captures into a graph.  The functions take the buffers themselves:

    weights fp32 [rows, H, width]      accumulated attention weight of each entry
    pos int32 [rows, H, width], held int32 [rows], evicted int32 [rows]
                                       entry e of a table row sits at position pos[e] of its conversation if e < held,
                                       else (it was never moved) at e + evicted
with width >= max_blocks * block.  The reference has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .block_kv import BLOCKS, CODE, FREE_OVER, _apart, _grown, _i32, _overlap, _pool, _rows16, _stream

# Workgroups of the launches.  One query per request: of the scores (at most 256 splits of a pair, whose maxima and sums
# every workgroup of the sums reads; us per call with 512 / 1,024 / 2,048 / 4,096: 32 requests x 2 heads, D 256, up to
# 16,384 positions 49 / 43 / 45 / 42, int8 64 x 8, D 128, up to 8,191 133 / 96 / 84 / 77) and of their sums.
_ROW_BLOCKS = 4096
# Chunks: this many where the work allows pieces of 512 positions (rows) at least (1,024 / 2,048 / 4,096 / 8,192: a prompt
# of 10,001, D 256, 1,071 / 890 / 867 / 890; 8 x 64 queries, D 128, 148 / 143 / 136 / 135), and as many as fit the CUs
# where it does not (61 queries x 12 heads over 60,000 positions, D 128: 256 64.4, 512 53.5, 768 50.1, 1,024 53.2).
# (D 64: four workgroups a CU, three with int8 codes and fp16 queries, where 8 x 64 queries x 64 / 8 heads over 12,000
# positions take 183 / 181 / 183 us with 512 / 768 / 1,024.)
_CHUNK_BLOCKS = 4096
_CHUNK_FIT = {64: 1024, 128: 768, 256: 512}
_SUMS = 1 << 26          # partial sums of a call at most (256 MB)
# Scores of a call's requests at once (4 GB; of one request at least).  256 requests x 64 / 8 heads that hold 4,160 entries,
# D 128, in tables of 262,144: 486 us in turns of 1 GB, 373 of 4 GB, 369 all at once (17 GB).
_SCORES = 1 << 30


@dataclass
class BlockTrim:
    """What a trim leaves: kv_lens int32 [n] (the requests' lengths after it), next_head int32 [1] (of the free list)."""
    kv_lens: torch.Tensor
    next_head: torch.Tensor


def _per_entry(name: str, x: torch.Tensor, dtype: torch.dtype, rows: int, H: int, width: int) -> None:
    assert x.dtype == dtype and x.dim() == 3 and x.stride(2) == 1, f"{name} must be {dtype} [rows, H, width], unit last stride"
    if x.shape[0] < rows or x.shape[1] != H or x.shape[2] < width:
        raise ValueError(f"{name} of {tuple(x.shape)} for {rows} rows x {H} heads x {width} entries")


def kvt_block_weigh(q: torch.Tensor, k8: torch.Tensor, ks: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                    weights: torch.Tensor, cu_q: Optional[torch.Tensor] = None, seqs: Optional[torch.Tensor] = None,
                    since: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[dict] = None) -> torch.Tensor:
    """Add to each entry's weight the attention that the step's queries pay it: softmax(scale q K^T), summed over the
    queries that see the entry and the q heads of its KV head.

    q [rows, Hq, D] (bf16 / fp16).  cu_q None: one query per request, which sees all kv_lens[j] entries.  cu_q (int32 [n + 1]):
    request j owns rows cu_q[j] .. cu_q[j + 1]; they are its last positions and each sees the entries up to its own, as in
    kvt_block_prefill.  They may be the end of a longer chunk: its last queries alone, as a sample of all.
    Entries from since[j] on (int32 [n]; default: the call's own positions) start from zero, whatever `weights` holds there;
    since = 0 weighs anew.  (So a step that is not weighed leaves its entries' weights undefined: weigh every step, or give
    since.)  The sums go to `out` (default: weights itself; else a tensor of its own: a step that may be
    taken back), entries behind kv_lens[j] are left as they are.  A query that sees nothing adds nothing; one that sees a
    NaN, or a block whose scale is not finite, makes NaN of every entry that it sees.  Rows of seqs have to be distinct.
    scale: > 0, default D ** -0.5.  workspace as in kvt_block_decode: its buffers follow from the table's width (one query
    per request: 4 * Hq bytes per entry of every request, up to 4 GB, where requests go in turns)."""
    n = kv_lens.numel()
    nb, H, B, D = _pool(k8, k8, ks, ks, block_table, n, seqs)
    assert q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float16), "queries are bf16 or fp16 [rows, Hq, D]"
    rows, Hq, d = q.shape
    assert d == D, f"queries of {d} channels over blocks of {D}"
    if H == 0 or Hq == 0 or Hq % H or Hq // H > 16:
        raise ValueError(f"{Hq} q heads over {H} KV heads: a multiple, at most 16 each, is served")
    _i32("kv_lens", kv_lens, n)
    if cu_q is not None:
        _i32("cu_q", cu_q, n + 1)
    elif rows != n:
        raise ValueError(f"{rows} queries for {n} requests")
    if since is not None:
        _i32("since", since, n)
    max_blocks = block_table.shape[1]
    cap = max_blocks * B
    _per_entry("weights", weights, torch.float32, block_table.shape[0], H, cap)
    if out is None:
        out = weights
    elif out is not weights:
        _per_entry("out", out, torch.float32, block_table.shape[0], H, cap)
        if _overlap(out, weights) and (out.data_ptr() != weights.data_ptr() or out.stride() != weights.stride()):
            raise ValueError("out overlaps weights: pass weights itself, or other memory")
    _apart(out)
    if n == 0:
        return out
    st = _stream(q, k8, ks, block_table, kv_lens, weights, cu_q, seqs, since, out)
    q, qp, qn, qh = _rows16(q, 8)
    gs, pairs = Hq // H, n * H
    row_splits, fit = 1, 0
    if cu_q is None:
        at_once = min(n, max(1, _SCORES // (Hq * cap))) if cap else n   # (the others follow, launch after launch)
        splits = max(1, min(256, _ROW_BLOCKS // (at_once * H), -(-cap // 256)))
        groups = max(1, min(_ROW_BLOCKS // (at_once * H), -(-cap // 1024)))
        need = at_once * (Hq * cap + H * splits * 32)
    else:
        # (the most that there may be: the kernels divide each request by its own lengths)
        items, fit = rows * gs // 256 + n, _CHUNK_FIT[D]
        splits = max(1, min(max(fit, _CHUNK_BLOCKS) // (items * H), cap // 128, 1024))
        groups = max(1, _CHUNK_BLOCKS // pairs)
        tiles = -(-cap // 256)
        # Splits of the rows need another launch, of 4 to 10 us: for requests that may have 8,192 rows, more than 512 on
        # average, or more than 128 and tiles that do not fill the CUs (8 x 64 queries x 8 heads over 12,000 positions 138 us
        # with it, 127 without; 32 x 12 over 4,000 32 with it, 40 without).
        row_splits = 1
        if rows * gs >= 8192 or rows * gs > 512 * n or rows * gs > 128 * n and fit >= 2 * pairs * tiles:
            row_splits = max(1, min(groups, -(-rows * gs // 128), _SUMS // (pairs * cap), 1024))
        groups = min(groups, tiles * row_splits)
        need = rows * Hq * 2 * (splits + 1) + (row_splits * pairs * cap if row_splits > 1 else 0)
    ws = {} if workspace is None else workspace             # (held until the launch)
    work = _grown(ws, "weigh", need, q)
    _lib.call("kvt_block_weigh", qp, qn, qh, _lib.DTYPE_CODE[q.dtype], _lib.ptr(cu_q), rows, kv_lens.data_ptr(), n, H, Hq, D,
              CODE[k8.dtype], k8.data_ptr(), ks.data_ptr(), nb, B, block_table.data_ptr(), block_table.stride(0),
              *block_table.shape, _lib.ptr(seqs), D ** -0.5 if scale is None else float(scale), _lib.ptr(since),
              weights.data_ptr(), weights.stride(0), weights.stride(1), out.data_ptr(), out.stride(0), out.stride(1), splits,
              row_splits, groups, fit, _CHUNK_BLOCKS, work.data_ptr(), need, st)
    return out


def _cut(budget: int, block: int) -> None:
    if block not in BLOCKS:
        raise ValueError(f"blocks of {block} tokens: {BLOCKS} are served")
    if budget < block or budget % block:
        raise ValueError(f"a budget of {budget} entries: a multiple of the block size {block} is served")


def kvt_block_keep(weights: torch.Tensor, kv_lens: torch.Tensor, budget: int, seqs: Optional[torch.Tensor] = None,
                   recent: int = 0, sinks: int = 0, pos: Optional[torch.Tensor] = None,
                   held: Optional[torch.Tensor] = None, evicted: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, workspace: Optional[dict] = None) -> torch.Tensor:
    """Choose the `budget` entries that each request and KV head keeps: entries below `sinks`, those at its last `recent`
    positions, and the heaviest of the others; equal weights by the lower entry, NaN below all.

    Returns src int32 [n, H, budget] (or writes `out`): the entry that goes to place e.  It is e itself where that stays;
    entries from behind the budget, in ascending order, go to the places that become free, in ascending order.  A request of
    no more than `budget` entries keeps all: src is e up to its length, -1 behind.  pos, held and evicted (together; see the
    module) say which positions moved entries have: without them, entry e sits at position e."""
    assert weights.dtype == torch.float32 and weights.dim() == 3 and weights.stride(2) == 1
    rows, H, width = weights.shape
    n = kv_lens.numel()
    _i32("kv_lens", kv_lens, n)
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"a budget of {budget} entries with {sinks} first and {recent} recent ones")
    if seqs is not None:
        _i32("seqs", seqs, n)
    elif rows < n:
        raise ValueError(f"{n} requests, but weights has {rows} rows")
    if (pos is None) != (held is None) or (pos is None) != (evicted is None):
        raise ValueError("pos, held and evicted go together")
    if pos is not None:
        _per_entry("pos", pos, torch.int32, rows, H, width)
        _i32("held", held, rows)
        _i32("evicted", evicted, rows)
    if out is None:
        out = torch.empty(n, H, budget, dtype=torch.int32, device=weights.device)
    else:
        assert out.dtype == torch.int32 and out.shape == (n, H, budget) and out.is_contiguous()
    if n == 0 or H == 0:
        return out
    if width == 0:
        raise ValueError("weights of no entries")
    st = _stream(weights, kv_lens, seqs, pos, held, evicted, out)
    ws = {} if workspace is None else workspace             # (held until the launch)
    work, need = None, 0
    if width > 32768 and width > budget:                    # (shorter ones are one workgroup's, in registers)
        chunks = max(1, min(256, -(-width // 4096), 1024 // (n * H)))
        need = n * H * (6144 + 4 * chunks + 12 + 2 * (budget + budget % 2))
        work = _grown(ws, "keep", need, weights, torch.int32).data_ptr()
    sp = (0, 0) if pos is None else (pos.stride(0), pos.stride(1))
    _lib.call("kvt_block_keep", weights.data_ptr(), weights.stride(0), weights.stride(1), kv_lens.data_ptr(), n, H, rows,
              _lib.ptr(seqs), width, budget, recent, sinks, _lib.ptr(pos), *sp, _lib.ptr(held), _lib.ptr(evicted),
              out.data_ptr(), work, need, st)
    return out


def kvt_block_evict(src: torch.Tensor, kv_lens: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, ks: torch.Tensor,
                    vs: torch.Tensor, block_table: torch.Tensor, seqs: Optional[torch.Tensor] = None,
                    weights: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None,
                    held: Optional[torch.Tensor] = None, evicted: Optional[torch.Tensor] = None) -> None:
    """Move the entries of one layer to where src (int32 [n, H, budget], as kvt_block_keep gives it) has them: codes,
    weights and positions of request j's entries below the budget, a multiple of the block size.  Requests of no more than
    `budget` entries (kv_lens) are left as they are.

    A block that gets no other entry is left as it is.  Another one's scales become the smallest powers of two that hold
    its rows, as if their values were stored anew: exact for e4m3 codes but for those that become subnormal, int8 codes are
    rounded to a scale that grew.  Where a row's scale is not finite, the block's becomes NaN.  An entry of src that is
    neither its own place nor behind the budget and within the length stays where it is.  weights and pos are optional; pos
    takes held and evicted with it, which kvt_block_trim updates once all layers are done.  Rows of seqs have to be
    distinct (kv_lens of a row that is listed again: 0), and a block may be in one row of the table only."""
    n = kv_lens.numel()
    nb, H, B, D = _pool(k8, v8, ks, vs, block_table, n, seqs)
    assert src.dtype == torch.int32 and src.dim() == 3 and src.is_contiguous(), "src is a contiguous int32 [n, H, budget]"
    if src.shape[:2] != (n, H):
        raise ValueError(f"src of {tuple(src.shape)} for {n} requests x {H} heads")
    budget = src.shape[2]
    _cut(budget, B)
    _i32("kv_lens", kv_lens, n)
    rows, max_blocks = block_table.shape
    if weights is not None:
        _per_entry("weights", weights, torch.float32, rows, H, max_blocks * B)
        _apart(weights)
    if pos is not None:
        _apart(pos)
        if held is None or evicted is None:
            raise ValueError("pos goes with held and evicted")
        _per_entry("pos", pos, torch.int32, rows, H, max_blocks * B)
        _i32("held", held, rows)
        _i32("evicted", evicted, rows)
    if n == 0 or H == 0 or budget > max_blocks * B:          # (no request can be over its budget)
        return
    st = _stream(src, kv_lens, k8, v8, ks, vs, block_table, seqs, weights, pos, held, evicted)
    sw = (0, 0) if weights is None else (weights.stride(0), weights.stride(1))
    sp = (0, 0) if pos is None else (pos.stride(0), pos.stride(1))
    _lib.call("kvt_block_evict", src.data_ptr(), kv_lens.data_ptr(), n, H, D, CODE[k8.dtype], k8.data_ptr(), v8.data_ptr(),
              ks.data_ptr(), vs.data_ptr(), nb, B, block_table.data_ptr(), block_table.stride(0), rows, max_blocks,
              _lib.ptr(seqs), budget, _lib.ptr(weights), *sw, _lib.ptr(pos), *sp, _lib.ptr(held), _lib.ptr(evicted), st)


def kvt_block_trim(seqs: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, free_list: torch.Tensor,
                   free_head: torch.Tensor, budget: int, block: int = 64, held: Optional[torch.Tensor] = None,
                   evicted: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None,
                   commit: bool = True) -> BlockTrim:
    """Cut the table rows seqs[j] to `budget` entries, once their entries have been moved in every layer: the counterpart
    of kvt_block_plan.  The blocks behind the budget go back in front of free_list[free_head[0]], in request order; their
    table entries become -1, seq_lens[row] the budget, and held and evicted (int32 [rows]) say how many entries have
    positions of their own and how many positions are gone.  Rows of no more entries are left as they are.

    commit=False writes the free list's entries, which are nobody's until its head moves, and leaves everything else as it
    is.  status (int32 [1]): bits BAD_ROW (a row out of range, or listed twice: the first one counts) and FREE_OVER (more
    blocks come back than were handed out; those over are lost) are or-ed in.  At most 1,024 requests."""
    n = seqs.numel()
    _i32("seqs", seqs, n)
    _i32("seq_lens", seq_lens, 1)
    _i32("free_list", free_list, 0)
    _i32("free_head", free_head, 1)
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1
    rows = block_table.shape[0]
    _cut(budget, block)
    if (held is None) != (evicted is None):
        raise ValueError("held and evicted go together")
    for name, x in (("seq_lens", seq_lens), ("held", held), ("evicted", evicted)):
        if x is not None:
            _i32(name, x, rows)
    if status is not None:
        _i32("status", status, 1)
    st = _stream(seqs, seq_lens, block_table, free_list, free_head, held, evicted, status)
    if n == 0:
        return BlockTrim(seqs.new_empty(0), free_head[:1].clamp(0, free_list.numel()))
    work, kv_lens, next_head = seqs.new_empty(5 * n + 5).split_with_sizes((4 * n + 4, n, 1))       # (one allocation)
    _lib.call("kvt_block_trim", n, seqs.data_ptr(), seq_lens.data_ptr(), rows, block_table.data_ptr(), block_table.stride(0),
              block_table.shape[1], free_list.data_ptr(), free_list.numel(), free_head.data_ptr(), block, budget,
              _lib.ptr(held), _lib.ptr(evicted), kv_lens.data_ptr(), next_head.data_ptr(), _lib.ptr(status),
              int(bool(commit)), work.data_ptr(), st)
    return BlockTrim(kv_lens, next_head)
