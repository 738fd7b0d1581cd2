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
from .block_kv import _stream, _strides

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
    if factors is not None and (method is not None or len(factors) != dim // 2):
        raise ValueError(f"factors: {dim // 2} divisors, and no method beside them")
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


def _span(x: torch.Tensor) -> Tuple[int, int]:
    first = x.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()


def _output(x: torch.Tensor, out: Optional[torch.Tensor], others: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """The output of x (a new tensor for None); one that overlaps x or another of the call's tensors, other than as x
    itself, is refused."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    assert out.shape == x.shape and out.dtype == x.dtype and out.stride(2) == 1, "an output has its input's shape and type"
    if out.numel() == 0:
        return out
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError("an output's elements have to be apart")
    if out.data_ptr() == x.data_ptr() and _strides(out) == _strides(x):
        return out                                          # in place
    a, b = _span(out)
    for y in (x, *others):
        if y is not None and y.numel() and y.get_device() == out.get_device():
            c, d = _span(y)
            if a < d and c < b:
                raise ValueError("an output overlaps an input: pass the input itself (in place), or other memory")
    return out


def kvt_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
             scale: float = 1.0, interleaved: bool = False, cu: Optional[torch.Tensor] = None,
             seqs: Optional[torch.Tensor] = None, ahead: Optional[torch.Tensor] = None, inverse: bool = False,
             out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """Rotate the first 2 * len(inv_freq) channels of q [N, Hq, D] and k [N, H, D] (bf16 / fp16 / fp32; k may be None) to
    their positions; returns (out_q, out_k), new tensors unless given.  out_q=q or out_k=k rotates in place.

    Pairs are channels (i, i + rot / 2), or (2 i, 2 i + 1) with interleaved=True; cosines and sines are times `scale`.
    Positions: int32 or int64 [N], of any sign; angles are formed in 64 bits.  With cu (int32 [n + 1]) they are a step's, as
    a plan gives them: positions int32 [n] are the lengths with the step's tokens, of which rows cu[j] .. cu[j + 1] are the
    last, and `ahead` (int32, by seqs[j], default j) is added to them -- the entries that were evicted.  Rows behind cu[n] are
    neither read nor written.  inverse=True rotates back by the same angles: the transpose, so the gradient of an input is
    the inverse of the output's."""
    assert q.dim() == 3 and q.dtype in _lib.DTYPE_CODE and (q.numel() == 0 or q.stride(2) == 1), "rows are [N, heads, D]"
    N, Hq, D = q.shape
    Hk = 0
    if k is not None:
        assert k.dim() == 3 and k.dtype == q.dtype and (k.numel() == 0 or k.stride(2) == 1)
        assert k.shape[0] == N and k.shape[2] == D, f"keys of {tuple(k.shape)} beside queries of {tuple(q.shape)}"
        Hk = k.shape[1]
    elif out_k is not None:
        raise ValueError("out_k without k")
    assert inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.is_contiguous(), "inv_freq is fp64 [rot / 2]"
    rot = 2 * inv_freq.numel()
    if not 2 <= rot <= D <= 256 or Hq < 1:
        raise ValueError(f"{rot} of {D} channels, {Hq} heads: up to 256 channels and a rotary part within them are served")
    n = n_rows = 0
    if cu is None:
        assert positions.dtype in (torch.int32, torch.int64) and positions.dim() == 1 and positions.is_contiguous()
        if positions.numel() < N:
            raise ValueError(f"{positions.numel()} positions for {N} tokens")
        if seqs is not None or ahead is not None:
            raise ValueError("seqs and ahead go with cu")
    else:
        assert cu.dtype == positions.dtype == torch.int32 and cu.dim() == positions.dim() == 1
        assert cu.is_contiguous() and positions.is_contiguous()
        n = positions.numel()
        if cu.numel() < n + 1:
            raise ValueError(f"cu has {cu.numel()} entries for {n} requests")
        if seqs is not None:
            assert seqs.dtype == torch.int32 and seqs.dim() == 1 and seqs.is_contiguous()
            if seqs.numel() < n:
                raise ValueError(f"seqs has {seqs.numel()} entries for {n} requests")
        if ahead is not None:
            assert ahead.dtype == torch.int32 and ahead.dim() == 1 and ahead.is_contiguous()
            n_rows = ahead.numel()
            if seqs is None and n_rows < n:
                raise ValueError(f"ahead has {n_rows} entries for {n} requests")
    q_out = _output(q, out_q, (k,))
    k_out = None if k is None else _output(k, out_k, (q, q_out))
    if N == 0 or (cu is not None and n == 0):
        return q_out, k_out
    st = _stream(q, k, positions, inv_freq, cu, seqs, ahead, q_out, k_out)
    keys = (None, 0, 0, 0, None, 0, 0) if Hk == 0 else (k.data_ptr(), *_strides(k), Hk, k_out.data_ptr(), *_strides(k_out))
    _lib.call("kvt_rope", q.data_ptr(), *_strides(q), Hq, q_out.data_ptr(), *_strides(q_out), *keys,
              _lib.DTYPE_CODE[q.dtype], N, D, rot, inv_freq.data_ptr(), positions.data_ptr(),
              int(positions.dtype == torch.int64), _lib.ptr(cu), n, _lib.ptr(seqs), _lib.ptr(ahead), n_rows, float(scale),
              int(bool(interleaved)), int(bool(inverse)), st)
    return q_out, k_out
