"""8-bit paged KV cache with one scale per block of tokens and KV head, and its operators.

The slot pools of this package keep a scale per token and channel group; here a block of 16, 32 or 64 tokens of one KV head
shares one power-of-two fp32 scale for K and one for V, over e4m3 or int8 codes: H * D * 2 bytes per token and 8 * H bytes
per block.  The step of a serving program is four calls, all on the device (no host lengths, capturable):

    cache = BlockKVCache(layers, H, D, n_blocks, max_seqs, max_blocks, device)
    s = cache.add_seq()
    plan = cache.plan(seqs, counts, n_tokens)            # kvt_block_plan: blocks, slots, lengths
    for layer: cache.append(layer, plan, k, v)           # kvt_block_store
               out = cache.decode(layer, plan, q)        # kvt_block_decode, one query per request
               out = cache.prefill(layer, plan, q)       # kvt_block_prefill, the step's tokens as queries

The functions take the buffers themselves.  k8 / v8: float8_e4m3fn or int8 [n_blocks, H, block, D]; ks / vs: fp32
[n_blocks, H]; block_table: int32 [rows, max_blocks], -1 where there is no block; seqs: the table row of each request
(default: its number).  The reference has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import torch

from . import _lib

CODE = {torch.float8_e4m3fn: 0, torch.int8: 1}
_I32, _F32 = torch.int32, torch.float32
BLOCKS = (16, 32, 64)
HEAD_DIMS = (64, 128, 256)
POOL_SHORT, ROW_FULL, TOKENS_OVER, BAD_ROW = 1, 2, 4, 8   # status bits of a plan
# Decode.  Few requests: a number of splits for each (request, KV head) pair.  From _SHARE_REQUESTS on, over long
# tables: equal shares of all positions.  Measured, device us per call with the merge, caches cold, best splits against
# shares, up to 8,191 positions ragged: 8 requests x 8 heads (D 128) 19.7 / 22.7; 32 x 2 (D 256, up to 16,384) 65.7 /
# 52.9; 64 x 2 (D 256) 50.2 / 44.9; 16 x 20 (D 64) 40.0 / 37.6; 64 x 8 (D 128) 117 / 98; up to 1,000 positions, 64 x 2
# 17.9 / 20.5.  Both this choice and the number of splits follow from the table's width, since the lengths stay on the
# device: in a table that is much wider than its requests they are those of long requests (one of 777 positions in a
# table of 262,144 14.0 - 15.4 us against 12.1 - 12.8 in one of its own width, 8 up to 2,000 16.4 against 14.2; 32 up
# to 1,000 14.8 against 16.6, 24 / 2 heads, D 256).
_SHARE_REQUESTS, _SHARE_CAP = 16, 2048
# Workgroups of a launch in equal shares, and of one request's splits (D 256: one per CU, whose four wavefronts keep
# enough loads in flight: 52.9 us for 32 x 2 against 57.9 with two; D 128: 98 against 113 with one and 103 with three),
# and of chunks of few rows (4 queries a request: 8 x 8, D 128, up to 4,000 positions 19.9 with 8 splits, 24.7 with 16;
# 32 x 2, D 256, up to 1,000 21.1 with 4, 32.6 with 8).  (Two workgroups a CU are what the kernel of equal shares has
# registers for: at D 64 and 128 the merge inside the launch takes the most of them, 239 and 255 where
# block_rows_kernel, with the same loop, has 96 and 135.)
_DECODE_BLOCKS = {64: 512, 128: 512, 256: 256}
# Splits of a pair that a launch with a kept workspace merges itself.  us per call, merged by a second launch / by
# itself: 8 requests x 2 heads (D 256, up to 2,000 positions, 16 splits) 15.4 / 12.4; one x 8 (D 128, 2,000, 16 splits)
# 12.7 / 8.6; 8 x 8 (D 128, up to 4,000, 12 splits) 18.7 / 15.5; chunks of four queries over the same (8 splits) 22.1 /
# 19.9; but two of 300 positions x 2 heads (24 q heads) 11.5 / 12.1.  Past 16 the second launch's many workgroups read
# the parts faster than the last one does.  (Equal shares: the entry point decides.)
_MERGE_SPLITS = 16
_TILE_ROWS = 128         # (query, q head) rows of a workgroup of the query-tile kernel
# Workgroups of a split launch of it for one request, us per call (merge included): D 256, 16 items x 30,000 positions
# 256 workgroups 150, 512 110; D 128, 6 x 60,000 258 59.7, 384 57.9, 510 63.5; D 64, 20 x 30,000 320 86, 480 77, 640 65.
# Half as many again for several, whose lengths differ: 4 x 8 heads (D 128), 64 queries, up to 6,000 positions 75 / 58,
# 8 x 20 heads (D 64) up to 1,500 52.5 / 45.5, 8 x 2 (D 256) up to 4,000 124 / 110, 8 x 8 (D 128) up to 3,000 53 / 55.
_TILE_BLOCKS = {64: 768, 128: 384, 256: 512}
# Positions of a split at least: its part of 128 rows is 512 D bytes written and read again.  Half of it where those
# splits would leave half of the CUs idle: 5 query tiles (D 128) behind 1,758 positions 26.0 us with 512, 20.7 with 256,
# 19.3 with 128; 24 (D 256) behind 1,000 42 / 34 / 33; but 34 (D 256) behind 3,428 49 / 51 / 80, 44 (D 64) behind 4,000
# 36 / 35 / 47.
_TILE_LEAST = 512
# Rows per request and KV head (on average) from which it serves a call.  us per call against the 16-row kernel's, one
# request behind 30,000 positions: D 128, 64 rows 41 / 42, 128 rows 66 / 64, 256 rows 72 / 102; D 64, 128 rows 78 / 79,
# 256 rows 116 / 143; D 256, 128 rows 59 / 44, 256 rows 60 / 61, 512 rows 82 / 90.  Eight ragged requests behind 4,000:
# D 128, 116 rows 54 / 45, 230 rows 70 / 77.
_TILE_MIN = {64: 128, 128: 128, 256: 256}


@dataclass
class BlockPlan:
    """A step: cu int32 [n + 1] (prefix sums of the token counts), slots int32 [n_tokens] (block * block size + row of every
    token, -1 for none), kv_lens int32 [n] (lengths with the step's tokens), next_head int32 [1] (the free list's next
    entry after the step), seqs int32 [n] (table rows)."""
    seqs: torch.Tensor
    cu: torch.Tensor
    slots: torch.Tensor
    kv_lens: torch.Tensor
    next_head: torch.Tensor


def _stream(*tensors: Optional[torch.Tensor]) -> int:
    """The current stream of the tensors' device, which has to be the current one (launches go there)."""
    cur = torch.cuda.current_device() if tensors[0].is_cuda else -1
    for t in tensors:
        if t is not None and t.get_device() != cur or cur < 0:
            _lib.require_device(*tensors)
            raise ValueError(f"tensor on {t.device}, but the current device is cuda:{cur}")
    return _lib.stream(cur)


def _i32(name: str, t: torch.Tensor, n: int) -> None:
    assert t.dtype == _I32 and t.dim() == 1 and t.is_contiguous(), f"{name} must be a contiguous int32 vector"
    if t.numel() < n:
        raise ValueError(f"{name} has {t.numel()} entries, {n} are needed")


def _pool(k8, v8, ks, vs, block_table, n, seqs):
    """Checks of a layer's buffers; (n_blocks, H, block, D)."""
    shape, dtype = k8.shape, k8.dtype
    assert dtype in CODE and v8.dtype == dtype, "block codes are float8_e4m3fn or int8"
    assert len(shape) == 4 and v8.shape == shape and k8.is_contiguous() and v8.is_contiguous()
    nb, H, B, D = shape
    assert ks.dtype == vs.dtype == _F32 and ks.is_contiguous() and vs.is_contiguous()
    assert ks.shape == vs.shape == (nb, H)
    assert block_table.dtype == _I32 and block_table.dim() == 2 and block_table.stride(1) == 1
    if B not in BLOCKS or D not in HEAD_DIMS:
        raise ValueError(f"blocks of {B} tokens x {D} channels: {BLOCKS} tokens and {HEAD_DIMS} channels are served")
    if seqs is not None:
        _i32("seqs", seqs, n)
    elif block_table.shape[0] < n:
        raise ValueError(f"{n} requests, but the block table has {block_table.shape[0]} rows")
    return nb, H, B, D


def kvt_block_plan(seqs: torch.Tensor, counts: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
                   free_list: torch.Tensor, free_head: torch.Tensor, n_tokens: int, block: int = 64,
                   status: Optional[torch.Tensor] = None, req_to_token: Optional[torch.Tensor] = None,
                   commit: bool = True) -> BlockPlan:
    """Plan a step on the device: request j appends counts[j] tokens to table row seqs[j], whose length is seq_lens[row].

    The blocks that the requests open come from free_list (int32 [n_blocks], read from free_head[0] on) in request order
    and are written into block_table; every token gets its slot (block * block size + row: a location of the slot-indexed
    pools too), and with req_to_token (int32 [rows, context]) the slot of every position is recorded there.  n_tokens:
    the length of `slots`, a host int >= the counts' sum (slots behind that are -1).  commit=False leaves seq_lens and
    free_head as they are, to look at a plan (its status, its next_head) before it is taken: the next plan starts from the same state.
    status (int32 [1]): bits POOL_SHORT, ROW_FULL, TOKENS_OVER, BAD_ROW (a row out of range, or listed twice: the later
    request appends nothing) are or-ed in.  At most 1,024 requests; of none, the plan is empty."""
    n = seqs.numel()
    _i32("seqs", seqs, n)
    _i32("counts", counts, n)
    _i32("seq_lens", seq_lens, 1)
    _i32("free_list", free_list, 0)
    _i32("free_head", free_head, 1)
    assert block_table.dtype == _I32 and block_table.dim() == 2 and block_table.stride(1) == 1
    rows = block_table.shape[0]
    if seq_lens.numel() < rows:
        raise ValueError(f"seq_lens has {seq_lens.numel()} entries for {rows} table rows")
    if status is not None:
        _i32("status", status, 1)
    rtt, rtt_stride, rtt_cols = None, 0, 0
    if req_to_token is not None:
        assert req_to_token.dtype == torch.int32 and req_to_token.dim() == 2 and req_to_token.stride(1) == 1
        if req_to_token.shape[0] < rows:
            raise ValueError(f"req_to_token has {req_to_token.shape[0]} rows, the block table {rows}")
        rtt, rtt_stride, rtt_cols = req_to_token.data_ptr(), req_to_token.stride(0), req_to_token.shape[1]
    st = _stream(seqs, counts, seq_lens, block_table, free_list, free_head, status, req_to_token)
    if n == 0:                                             # (an idle step: no slots, and the state as it is)
        zero = seqs.new_zeros(1)
        return BlockPlan(seqs, zero, seqs.new_full((n_tokens,), -1), zero[:0], free_head[:1].clamp(0, free_list.numel()))
    one = seqs.new_empty(n_tokens + 2 * n + 2)              # (one allocation)
    slots, cu, kv_lens, next_head = one.split_with_sizes((n_tokens, n + 1, n, 1))
    _lib.call("kvt_block_plan", n, seqs.data_ptr(), counts.data_ptr(), seq_lens.data_ptr(), rows, block_table.data_ptr(),
              block_table.stride(0), block_table.shape[1], free_list.data_ptr(), free_list.numel(), free_head.data_ptr(),
              block, n_tokens, cu.data_ptr(), slots.data_ptr(), kv_lens.data_ptr(), next_head.data_ptr(),
              _lib.ptr(status), rtt, rtt_stride, rtt_cols, int(commit), st)
    return BlockPlan(seqs, cu, slots, kv_lens, next_head)


def _strides(x: torch.Tensor):
    """Strides of token and head; 0 for a dimension of one entry, whose stride may be anything."""
    (n, h, _), (a, b, _) = x.shape, x.stride()
    return a if n > 1 else 0, b if h > 1 else 0


def _rows16(x: torch.Tensor, per16: int):
    """Rows that start at 16-byte boundaries (x itself, else a contiguous copy): tensor, pointer, strides of token and head."""
    p, (a, b, c) = x.data_ptr(), x.stride()
    if p & 15 or a % per16 or b % per16 or c != 1:
        a, b = _strides(x)
        if p & 15 or a % per16 or b % per16 or c != 1:
            x = x.contiguous() if not x.is_contiguous() else x.clone()
            p, (a, b) = x.data_ptr(), _strides(x)
    return x, p, a, b


def kvt_block_store(k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, kv_lens: torch.Tensor, k8: torch.Tensor,
                    v8: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, block_table: torch.Tensor,
                    seqs: Optional[torch.Tensor] = None) -> None:
    """Quantize rows k, v ([N, H, D] bf16 / fp16 / fp32) into the blocks of their positions: rows cu[j] .. cu[j + 1] are the
    last positions of request j's kv_lens[j] (both int32, as a plan gives them).

    A block's scale is the smallest power of two s with |x| <= 448 s (e4m3) or 127 s (int8) for the call's finite values,
    and never shrinks while the block fills: where it grows, the rows that the request held before are rounded to the new
    scale (exact for e4m3 codes, but for those that become subnormal).  Rows of a block that the request does not hold yet
    are left as they are, rows of k and v behind cu[n] are not read; N has to be cu[n] at least.  A block must be in the
    table of one request of the call only."""
    N, H, D = k.shape
    n = kv_lens.numel()
    nb, H8, B, D8 = _pool(k8, v8, ks, vs, block_table, n, seqs)
    assert v.shape == k.shape and (H, D) == (H8, D8), f"rows of {H} x {D} for blocks of {H8} x {D8}"
    assert k.dtype == v.dtype and k.dtype in _lib.DTYPE_CODE, k.dtype
    _i32("kv_lens", kv_lens, n)
    _i32("cu", cu, n + 1)
    if N == 0 or n == 0:
        return
    st = _stream(k, v, cu, kv_lens, k8, v8, ks, vs, block_table, seqs)
    per16 = 4 if k.dtype == torch.float32 else 8
    k, kp, kn, kh = _rows16(k, per16)
    v, vp, vn, vh = _rows16(v, per16)
    _lib.call("kvt_block_store", kp, vp, _lib.DTYPE_CODE[k.dtype], kn, kh, vn, vh, N, H, D, cu.data_ptr(),
              kv_lens.data_ptr(), n, _lib.ptr(seqs), block_table.data_ptr(), block_table.stride(0), *block_table.shape,
              CODE[k8.dtype], k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), nb, B, st)


def _grown(ws: dict, name: str, n: int, like: torch.Tensor, dtype=torch.float32, zero: bool = False) -> torch.Tensor:
    """A buffer of at least n entries on the device of `like`, kept in ws.  One that is outgrown stays there too (a captured
    graph may use it), so each is at least twice the last."""
    key = name, like.get_device()
    t = ws.get(key)
    if t is None or t.numel() < n:
        if t is not None:
            ws.setdefault("block_outgrown", []).append(t)
            n = max(n, 2 * t.numel())
        t = ws[key] = (torch.zeros if zero else torch.empty)(n, dtype=dtype, device=like.device)
    return t


def _parts(ws: dict, need: int, D: int, q: torch.Tensor, items: int):
    """Pointers of a split launch's partial buffers in ws: need rows of D values and of (maximum, sum), and the counters of
    `items` (0: none) whose parts the launch itself merges.  Those have to be zero, which every call leaves them; a capture
    does not make them, since its zeros would only be written by a replay."""
    o, ml = _grown(ws, "block_o", need * D, q), _grown(ws, "block_ml", need * 2, q)
    if items == 0:
        return o.data_ptr(), ml.data_ptr(), None
    c = ws.get(("block_counters", q.get_device()))
    if c is None or c.numel() < items:
        if torch.cuda.is_current_stream_capturing():
            return o.data_ptr(), ml.data_ptr(), None
        c = _grown(ws, "block_counters", items, q, _I32, True)
    return o.data_ptr(), ml.data_ptr(), c.data_ptr()


def _attn_args(q, out, H, D):
    assert q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float16), "queries are bf16 or fp16 [rows, Hq, D]"
    _, Hq, d = q.shape
    assert d == D, f"queries of {d} channels over blocks of {D}"
    if H == 0 or Hq == 0 or Hq % H or Hq // H > 16:
        raise ValueError(f"{Hq} q heads over {H} KV heads: a multiple, at most 16 each, is served")
    if out is None:
        out, so = torch.empty_like(q, memory_format=torch.contiguous_format), (Hq * D, D)
    else:
        assert out.shape == q.shape and out.dtype in _lib.DTYPE_CODE and out.stride(2) == 1
        so = _strides(out)
    return (*_rows16(q, 8), out, so, Hq)


def _splits(items: int, cap: int, blocks: int, least: int = 128) -> int:
    """Workgroups that share an item's positions: about `blocks` in all, none with fewer than `least` positions of the
    table's capacity."""
    return max(1, min(blocks // items, -(-cap // least)))


def kvt_block_decode(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor,
                     block_table: torch.Tensor, kv_lens: torch.Tensor, seqs: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     workspace: Optional[dict] = None, splits: Optional[int] = None) -> torch.Tensor:
    """Decode attention of one query token per request: q [n, Hq, D] (bf16 / fp16), request j over its kv_lens[j] positions.

    Returns out ([n, Hq, D], q's dtype unless a bf16 / fp16 / fp32 `out` is given); a request without positions gives
    NaN (0/0).  scale: > 0, default D ** -0.5.  The lengths are read on the device; `splits` follows from the number of
    requests and the block table's width unless given: workgroups that share the positions of a request and KV head, or
    minus the number of workgroups that share those of the whole call.  `workspace` (a dict) keeps the partial buffers across
    calls, and spares a launch where there are few parts: calls that share one must not overlap, a captured graph needs it
    as long as it is replayed, and one made before the capture is the faster one.  The results do not depend on it."""
    n = kv_lens.numel()
    nb, H, B, D = _pool(k8, v8, ks, vs, block_table, n, seqs)
    q, qp, qn, qh, out, so, Hq = _attn_args(q, out, H, D)
    if q.shape[0] != n:
        raise ValueError(f"{q.shape[0]} queries for {n} requests")
    _i32("kv_lens", kv_lens, n)
    if n == 0:
        return out
    st = _stream(q, k8, v8, ks, vs, block_table, kv_lens, seqs, out)
    cap = block_table.shape[1] * B
    if splits is not None:
        ns = int(splits)
    elif n >= _SHARE_REQUESTS and cap >= _SHARE_CAP:
        ns = -_DECODE_BLOCKS[D]
    else:
        ns = _splits(n * H, cap, 768 if n > 1 else _DECODE_BLOCKS[D])
    o = ml = counters = None
    if ns > 1 or ns < -1:
        ws = {} if workspace is None else workspace          # (held until the launch)
        o, ml, counters = _parts(ws, n * H * ns * 16 if ns > 1 else -2 * ns * 16, D, q,
                                 n * H if workspace is not None and ns <= _MERGE_SPLITS else 0)
    _lib.call("kvt_block_decode", qp, qn, qh, _lib.DTYPE_CODE[q.dtype], kv_lens.data_ptr(), n, H, Hq, D, CODE[k8.dtype],
              k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), nb, B, block_table.data_ptr(), block_table.stride(0),
              *block_table.shape, _lib.ptr(seqs), D ** -0.5 if scale is None else float(scale), ns, o, ml, counters,
              out.data_ptr(), _lib.DTYPE_CODE[out.dtype], *so, st)
    return out


def kvt_block_prefill(q: torch.Tensor, cu_q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, ks: torch.Tensor,
                      vs: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                      seqs: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None, workspace: Optional[dict] = None,
                      splits: Optional[int] = None) -> torch.Tensor:
    """Attention of chunks: q [total, Hq, D] (bf16 / fp16), request j owns rows cu_q[j] .. cu_q[j + 1] (int32 [n + 1]).

    causal: the chunk's queries are the last positions of request j (its keys are in the cache already) and each sees the
    positions up to its own: kv_lens[j] - chunk + i + 1 of them for query i.  causal=False: every query sees all
    kv_lens[j] positions -- cross attention to another sequence's states, of any length.  A query that sees nothing gives
    NaN (0/0).  Rows behind cu_q[n] (a padded step) are neither read nor written: they keep what a given `out` holds, and are
    uninitialized memory in one that is made here.  Other arguments as kvt_block_decode."""
    n = kv_lens.numel()
    nb, H, B, D = _pool(k8, v8, ks, vs, block_table, n, seqs)
    q, qp, qn, qh, out, so, Hq = _attn_args(q, out, H, D)
    _i32("kv_lens", kv_lens, n)
    _i32("cu_q", cu_q, n + 1)
    total = q.shape[0]
    if n == 0 or total == 0:
        return out
    st = _stream(q, cu_q, k8, v8, ks, vs, block_table, kv_lens, seqs, out)
    rows = _TILE_ROWS if total * (Hq // H) >= _TILE_MIN[D] * n or total * (Hq // H) // 16 + n > 65535 else 16
    items = total * (Hq // H) // rows + n
    if splits is not None:
        ns = int(splits)
    else:
        full = max(-(-total * (Hq // H) // rows), n) * H     # (items less the empty ones)
        cap = block_table.shape[1] * B
        if rows > 16:
            least = _TILE_LEAST if full * -(-cap // _TILE_LEAST) >= 128 else _TILE_LEAST // 2
            ns = _splits(full, cap, _TILE_BLOCKS[D] * (3 if n > 1 else 2) // 2, least)
        else:
            ns = _splits(full, cap, _DECODE_BLOCKS[D])
    o = ml = counters = None
    if ns > 1:
        ws = {} if workspace is None else workspace          # (held until the launch)
        o, ml, counters = _parts(ws, items * H * ns * rows, D, q,
                                 items * H if workspace is not None and rows == 16 and ns <= _MERGE_SPLITS else 0)
    _lib.call("kvt_block_prefill", qp, qn, qh, _lib.DTYPE_CODE[q.dtype], cu_q.data_ptr(), total, kv_lens.data_ptr(), n, H, Hq,
              D, CODE[k8.dtype], k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), nb, B, block_table.data_ptr(),
              block_table.stride(0), *block_table.shape, _lib.ptr(seqs), int(bool(causal)),
              D ** -0.5 if scale is None else float(scale), rows, ns, o, ml, counters, out.data_ptr(),
              _lib.DTYPE_CODE[out.dtype], *so, st)
    return out


class BlockKVCache:
    """Buffers of the 8-bit block cache for all layers of a model, and the step's calls over them.

    Per layer k8 / v8 [n_blocks, H, block, D] and ks / vs [n_blocks, H]; shared by the layers: block_table
    [max_seqs, max_blocks], seq_lens [max_seqs], the free list (a seeded permutation of the blocks) and its head.
    Lengths, blocks and the free list live on the device only; add_seq and release hand out table rows on the host."""

    def __init__(self, layers: int, H: int, D: int, n_blocks: int, max_seqs: int, max_blocks: int, device="cuda",
                 dtype: torch.dtype = torch.float8_e4m3fn, block: int = 64, seed: int = 0):
        if dtype not in CODE:
            raise ValueError(f"block codes are float8_e4m3fn or int8, not {dtype}")
        if block not in BLOCKS or D not in HEAD_DIMS:
            raise ValueError(f"blocks of {block} tokens x {D} channels: {BLOCKS} tokens and {HEAD_DIMS} channels are served")
        if n_blocks * block > 2 ** 31:
            raise ValueError(f"{n_blocks} blocks of {block} tokens: slots are int32")
        self.L, self.H, self.D, self.block, self.dtype = layers, H, D, block, dtype
        self.device = torch.device(device)
        z = dict(device=self.device)
        self.k8 = [torch.zeros(n_blocks, H, block, D, dtype=torch.int8, **z).view(dtype) for _ in range(layers)]
        self.v8 = [torch.zeros(n_blocks, H, block, D, dtype=torch.int8, **z).view(dtype) for _ in range(layers)]
        self.ks = [torch.zeros(n_blocks, H, dtype=torch.float32, **z) for _ in range(layers)]
        self.vs = [torch.zeros(n_blocks, H, dtype=torch.float32, **z) for _ in range(layers)]
        self.block_table = torch.full((max_seqs, max_blocks), -1, dtype=torch.int32, **z)
        self.seq_lens = torch.zeros(max_seqs, dtype=torch.int32, **z)
        g = torch.Generator().manual_seed(seed)
        self.free_list = torch.randperm(n_blocks, generator=g).to(torch.int32).to(self.device)
        self.free_head = torch.zeros(1, dtype=torch.int32, **z)
        self.status = torch.zeros(1, dtype=torch.int32, **z)
        self._rows: List[int] = list(range(max_seqs - 1, -1, -1))

    def add_seq(self) -> int:
        """A free table row for a new sequence."""
        if not self._rows:
            raise RuntimeError("no free sequence row")
        return self._rows.pop()

    def release(self, s: int) -> None:
        """Give a sequence's blocks back to the free list and its row back to add_seq (synchronizes the device)."""
        if s in self._rows or not 0 <= s < self.block_table.shape[0]:
            raise ValueError(f"row {s} holds no sequence")
        used = -(-int(self.seq_lens[s]) // self.block)
        blocks = self.block_table[s, :used]
        blocks = blocks[blocks >= 0]
        head = int(self.free_head) - blocks.numel()
        self.free_list[head:head + blocks.numel()] = blocks
        self.free_head.fill_(head)
        self.block_table[s].fill_(-1)
        self.seq_lens[s] = 0
        self._rows.append(s)

    def _vec(self, x: Union[torch.Tensor, Sequence[int]]) -> torch.Tensor:
        return x if isinstance(x, torch.Tensor) else torch.tensor(list(x), dtype=torch.int32).to(self.device)

    def plan(self, seqs, counts, n_tokens: Optional[int] = None, req_to_token: Optional[torch.Tensor] = None,
             commit: bool = True) -> BlockPlan:
        """kvt_block_plan over this cache.  seqs / counts: int32 device vectors or lists; n_tokens: a host bound of the
        counts' sum (needed with device counts; tokens and queries behind the sum are padding, which no call reads or
        writes)."""
        if n_tokens is None:
            if isinstance(counts, torch.Tensor):
                raise ValueError("plan: pass n_tokens (a host int >= the counts' sum) with counts on the device")
            n_tokens = sum(counts)
        return kvt_block_plan(self._vec(seqs), self._vec(counts), self.seq_lens, self.block_table, self.free_list,
                              self.free_head, n_tokens, self.block, self.status, req_to_token, commit)

    def check(self) -> None:
        """Raise RuntimeError if a plan could not be carried out in full since the last check (synchronizes the device)."""
        bits = int(self.status)
        if bits:
            self.status.zero_()
            names = [name for bit, name in ((POOL_SHORT, "block pool exhausted"), (ROW_FULL, "block table row full"),
                                            (TOKENS_OVER, "more tokens than n_tokens"),
                                            (BAD_ROW, "table row out of range or listed twice")) if bits & bit]
            raise RuntimeError("block plan: " + ", ".join(names))

    def append(self, layer: int, plan: BlockPlan, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write the plan's tokens (k, v: [n_tokens, H, D]) into layer `layer`."""
        kvt_block_store(k, v, plan.cu, plan.kv_lens, self.k8[layer], self.v8[layer], self.ks[layer], self.vs[layer],
                        self.block_table, plan.seqs)

    def decode(self, layer: int, plan: BlockPlan, q: torch.Tensor, **kw) -> torch.Tensor:
        """Attention of one query per request of the plan, over everything appended so far."""
        return kvt_block_decode(q, self.k8[layer], self.v8[layer], self.ks[layer], self.vs[layer], self.block_table,
                                plan.kv_lens, plan.seqs, **kw)

    def prefill(self, layer: int, plan: BlockPlan, q: torch.Tensor, **kw) -> torch.Tensor:
        """Attention of the plan's tokens (q: [n_tokens, Hq, D]).  Where n_tokens is more than the counts' sum, the rows
        behind that are not written: pass an `out` that holds what they should be, or do not read them."""
        return kvt_block_prefill(q, plan.cu, self.k8[layer], self.v8[layer], self.ks[layer], self.vs[layer],
                                 self.block_table, plan.kv_lens, plan.seqs, **kw)
