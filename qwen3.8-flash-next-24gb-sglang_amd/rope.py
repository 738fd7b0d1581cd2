"""Rotary positions of queries and keys, before they are written to a cache or attended: half and interleaved pairs, a
part of the head, frequencies scaled for long contexts.

    inv_freq, scale = rotary_frequencies(64, 1e6, method="yarn", factor=8, original=32768)
    q, k = kvt_rope(q, k, positions, inv_freq, scale)                                # a position per token
    q, k = kvt_rope(q, k, plan.kv_lens, inv_freq, scale, cu=plan.cu, seqs=plan.seqs, ahead=cache.evicted)   # a step's

The reference rotates in the serving framework it patches; it has no operator of its own for it.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .block_kv import _apart, _i32, _overlap, _stream, _strides

METHODS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(dim: int, base: float = 10000.0, method: Optional[str] = None, factor: float = 1.0,
                       original: Optional[int] = None, factors: Optional[Sequence[float]] = None,
                       beta_fast: float = 32.0, beta_slow: float = 1.0, attention: Optional[float] = None,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """fp64 [dim / 2] angles per position (radians), base^(-2 i / dim), and the factor of cosine and sine.

    method: "linear" divides every frequency by `factor`; "ntk" raises the base by factor^(dim / (dim - 2)), which leaves the
    highest frequency and divides the lowest by `factor`; "yarn" divides those whose period turns fewer than beta_slow
    times within `original` positions, leaves those that turn more than beta_fast times, with a ramp over the indexes
    between, and scales by 0.1 ln(factor) + 1.  factors: a divisor of each frequency instead.  attention: the factor of
    cosine and sine, where it is not the method's."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary part of {dim} channels: an even number is served")
    if method not in METHODS:
        raise ValueError(f"method {method!r}: one of {METHODS}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError(f"base {base} and factor {factor} have to be positive numbers")
    if factors is not None and (method is not None or len(factors) != dim // 2 or
                                not all(math.isfinite(f) and f > 0 for f in factors)):
        raise ValueError(f"factors: {dim // 2} divisors, positive numbers, and no method beside them")
    if method == "ntk":
        if dim < 4:
            raise ValueError("ntk: a rotary part of 4 channels at least")
        base = base * factor ** (dim / (dim - 2))
    inv = torch.tensor([base ** (-i / dim) for i in range(0, dim, 2)], dtype=torch.float64)
    scale = 1.0
    if factors is not None:
        inv = inv / torch.tensor(list(factors), dtype=torch.float64)
    elif method == "linear":
        inv = inv / factor
    elif method == "yarn":
        if original is None or original < 1 or base <= 1 or not 0 < beta_slow < beta_fast:
            raise ValueError("yarn: the original context, a base over 1 and beta_slow < beta_fast are needed")
        low, high = (dim * math.log(original / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (beta_fast, beta_slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    return inv.to(device), scale if attention is None else float(attention)


def _output(x: torch.Tensor, out: torch.Tensor, others: Sequence[Optional[torch.Tensor]]) -> None:
    """Refuses an output that overlaps x or another of the call's tensors, other than as x itself."""
    assert out.shape == x.shape and out.dtype == x.dtype and (out.numel() == 0 or out.stride(2) == 1), \
        "an output has its input's shape and type, and unit last stride"
    if out.numel() == 0:
        return
    _apart(out)
    in_place = out.data_ptr() == x.data_ptr() and _strides(out) == _strides(x)
    for y in others if in_place else (x, *others):
        if y is not None and _overlap(out, y):
            raise ValueError("an output overlaps an input: pass the input itself (in place), or other memory")


def _side(x: torch.Tensor, out: Optional[torch.Tensor]):
    """The output of x (a new tensor for None), and the pointers, strides and heads of both."""
    _, h, d = x.shape
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        so = (h * d, d)
    else:
        so = _strides(out)
    return out, (x.data_ptr(), *_strides(x), h, out.data_ptr(), *so)


def kvt_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
             scale: float = 1.0, interleaved: bool = False, cu: Optional[torch.Tensor] = None,
             seqs: Optional[torch.Tensor] = None, ahead: Optional[torch.Tensor] = None, inverse: bool = False,
             out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """Rotate the first 2 * len(inv_freq) channels of q [N, Hq, D] and k [N, H, D] (bf16 / fp16 / fp32; k may be None) to
    their positions; returns (out_q, out_k), new tensors unless given.  out_q=q or out_k=k rotates in place; outputs share no
    memory otherwise, with the inputs or each other (parts of one buffer are apart).

    Pairs are channels (i, i + rot / 2), or (2 i, 2 i + 1) with interleaved=True; cosines and sines are times `scale`.
    Positions: int32 or int64 [N], of any sign; angles are formed in 64 bits.  With cu (int32 [n + 1]) they are a step's, as
    a plan gives them: positions int32 [n] are the lengths with the step's tokens, of which rows cu[j] .. cu[j + 1] are the
    last, and `ahead` (int32, by seqs[j], default j) is added to them -- the entries that were evicted.  Rows behind cu[n] are
    neither read nor written.  inverse=True rotates back by the same angles: the transpose, so the gradient of an input is
    the inverse of the output's."""
    N, Hq, D = q.shape
    dtype = _lib.DTYPE_CODE.get(q.dtype)
    assert dtype is not None and (q.stride(2) == 1 or q.numel() == 0), "rows are [N, heads, D] in bf16, fp16 or fp32"
    if k is not None:
        n_k, Hk, d_k = k.shape
        assert k.dtype == q.dtype and (k.stride(2) == 1 or k.numel() == 0)
        assert n_k == N and d_k == D, f"keys of {tuple(k.shape)} beside queries of {tuple(q.shape)}"
    elif out_k is not None:
        raise ValueError("out_k without k")
    else:
        Hk = 0
    assert inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.is_contiguous(), "inv_freq is fp64 [rot / 2]"
    rot = 2 * inv_freq.numel()
    if not 2 <= rot <= D <= 256 or Hq < 1:
        raise ValueError(f"{rot} of {D} channels, {Hq} heads: up to 256 channels and a rotary part within them are served")
    n = n_rows = wide = 0
    if cu is None:
        wide = int(positions.dtype == torch.int64)
        assert (wide or positions.dtype == torch.int32) and positions.dim() == 1 and positions.is_contiguous()
        if positions.numel() < N:
            raise ValueError(f"{positions.numel()} positions for {N} tokens")
        if seqs is not None or ahead is not None:
            raise ValueError("seqs and ahead go with cu")
    else:
        n = positions.numel()
        _i32("positions", positions, n)
        _i32("cu", cu, n + 1)
        if seqs is not None:
            _i32("seqs", seqs, n)
        if ahead is not None:
            _i32("ahead", ahead, n if seqs is None else 0)
            n_rows = ahead.numel()
    if out_q is not None:
        _output(q, out_q, (k,))
    if out_k is not None:
        # (no pair is looked at twice)
        _output(k, out_k, (q, out_q) if out_q is not q else () if out_k is k else (q,))
    out_q, queries = _side(q, out_q)
    keys = (None, 0, 0, 0, None, 0, 0)
    if k is not None:
        out_k, side = _side(k, out_k)
        keys = side if Hk else keys
    if N == 0 or (cu is not None and n == 0):
        return out_q, out_k
    st = _stream(q, k, positions, inv_freq, cu, seqs, ahead, out_q, out_k)
    _lib.call("kvt_rope", *queries, *keys, dtype, N, D, rot, inv_freq.data_ptr(), positions.data_ptr(), wide, _lib.ptr(cu), n,
              _lib.ptr(seqs), _lib.ptr(ahead), n_rows, scale, bool(interleaved), bool(inverse), st)
    return out_q, out_k
