"""Plain 64-bit forms of the 8-bit block cache's operators (CPU, loops over requests), written from their definitions."""
import math

import torch

CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"fp8": 448.0, "int8": 127.0}


def values(codes: torch.Tensor) -> torch.Tensor:
    """float64 values of codes (e4m3 or int8)."""
    return codes.to(torch.float32).double()


def round_code(x: torch.Tensor, kv: str) -> torch.Tensor:
    """float64 -> the values that codes hold: nearest, ties to even, saturating; NaN -> NaN (e4m3) or 0 (int8)."""
    if kv == "int8":
        return torch.nan_to_num(x.round().clamp(-127, 127), nan=0.0)
    x = x.clamp(-448, 448)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.exp2(e) > x.abs().clamp(min=2.0 ** -6), e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= x.abs().clamp(min=2.0 ** -6), e + 1, e)
    step = torch.exp2(e - 3)
    return (x / step).round() * step


def scale_of(amax: float, kv: str) -> float:
    s = 2.0 ** -64
    while amax / s > QMAX[kv] and s < 2.0 ** 122:
        s *= 2
    return s


def plan(seqs, counts, seq_lens, table, free, head, n_tokens, B, rtt=None):
    """In place on table / rtt (lists of lists); (cu, slots, kv_lens, next head, status)."""
    cu, slots, kv, status, seen = [0], [], [], 0, set()
    for s, c in zip(seqs, counts):
        if not 0 <= s < len(table) or s in seen:
            status |= 8
            cu.append(cu[-1])
            kv.append(0)
            continue
        seen.add(s)
        if cu[-1] + max(c, 0) > n_tokens:
            status |= 4
        c = min(max(c, 0), n_tokens - cu[-1])
        for p in range(seq_lens[s], seq_lens[s] + c):
            lp = p // B
            if lp >= len(table[s]):
                status |= 2
                slots.append(-1)
                continue
            if p % B == 0:
                if head < len(free):
                    table[s][lp] = free[head]
                    head += 1
                else:
                    status |= 1
                    table[s][lp] = -1
            slot = table[s][lp] * B + p % B if table[s][lp] >= 0 else -1
            slots.append(slot)
            if rtt is not None and p < len(rtt[s]):
                rtt[s][p] = slot
        cu.append(cu[-1] + c)
        kv.append(seq_lens[s] + c)
    return cu, slots + [-1] * (n_tokens - len(slots)), kv, head, status


def store(x, cu, kv_lens, rows, table, codes, scale, kv):
    """One side of the write: x float64 [N, H, D]; codes float64 values [n_blocks, H, B, D] and scale float64
    [n_blocks, H], in place."""
    nb, H, B, D = codes.shape
    for r, row in enumerate(rows):
        n = cu[r + 1] - cu[r]
        old, p = kv_lens[r] - n, kv_lens[r] - n
        while p < kv_lens[r]:
            end = min(kv_lens[r], (p // B + 1) * B)
            b = table[row][p // B] if p // B < len(table[row]) else -1
            t = cu[r] + p - old
            if 0 <= b < nb:
                for h in range(H):
                    y = x[t:t + end - p, h]
                    fin = y[torch.isfinite(y)].abs()
                    s = scale_of(float(fin.max()) if fin.numel() else 0.0, kv)
                    if p % B:
                        was = float(scale[b, h])
                        if s > was:
                            codes[b, h, :p % B] = round_code(codes[b, h, :p % B] * (was / s), kv)
                        s = max(s, was)
                    scale[b, h] = s
                    codes[b, h, p % B:p % B + end - p] = round_code(y / s, kv)
            p = end


def attention(q, cu, kv_lens, rows, table, k, v, causal, scale):
    """q float64 [total, Hq, D]; k, v float64 values [n_blocks, H, B, D].  Returns (out, the weighted mean of |v|, the
    largest sum of |scale q k| of a row, the sum of |v|) float64; rows of no request stay 0."""
    nb, H, B, D = k.shape
    out, size, total = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(q.shape[:2], dtype=torch.float64)
    g = q.shape[1] // H
    for r, row in enumerate(rows):
        m = cu[r + 1] - cu[r]
        pos = [p for p in range(min(kv_lens[r], len(table[row]) * B)) if 0 <= table[row][p // B] < nb]
        at = torch.tensor(pos, dtype=torch.long)
        blk = torch.tensor([table[row][p // B] for p in pos], dtype=torch.long)
        for h in range(H):
            kk, vv = k[blk, h, at % B], v[blk, h, at % B]
            for j in range(g):
                qq = q[cu[r]:cu[r + 1], h * g + j]
                x = qq @ kk.t() * scale
                if causal:
                    last = kv_lens[r] - m + torch.arange(m)
                    x = x.masked_fill(at[None] > last[:, None], -math.inf)
                w = torch.softmax(x, -1) if pos else x
                out[cu[r]:cu[r + 1], h * g + j] = w @ vv if pos else math.nan
                size[cu[r]:cu[r + 1], h * g + j] = w @ vv.abs() if pos else math.nan
                total[cu[r]:cu[r + 1], h * g + j] = vv.abs().sum(0)
                if pos:
                    reach[cu[r]:cu[r + 1], h * g + j] = ((qq.abs() @ kk.abs().t()) * abs(scale)).amax(-1)
    return out, size, reach, total


def bound(out, size, reach, total, D, dtype):
    """How far a kernel's output may be from `out`: weights rounded to fp16 (half a step, 2^-11, on a weighted mean of
    |v|), scores summed in fp32 over D products (D 2^-24 of the sum of |q k|, twice in a quotient; with a little for the
    exponential), fp32 sums of the weights and of O (2^-20), and the output's own rounding.  Weights are held times 2^10
    (the largest of a row between 2^10 and 2^14) and times a V scale of at least 1/4 of the unit, so where they are fp16
    subnormals half a step, 2^-25, is at most 2^-25 / (2^10 / 4) = 2^-33 of the largest weight, which is at most their sum."""
    rel = 2.0 ** -11 + 2 * (D * 2.0 ** -24 * reach + 2.0 ** -20)
    return rel[..., None] * size + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -33 * total + 1e-30


def close(got, out, size, reach, total, D):
    dtype = got.dtype
    got = got.double().cpu()
    nan = torch.isnan(out)
    assert torch.equal(nan, torch.isnan(got)), "NaN pattern differs"
    tol = bound(out, size, reach, total, D, dtype)
    off = (got - out).abs()
    bad = (off > tol) & ~nan
    assert not bad.any(), (int(bad.sum()), float((off / tol)[bad].max()))
