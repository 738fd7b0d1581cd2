"""Plain 64-bit forms of the operators of a block cache within a budget, and of rotary positions (CPU, loops over
requests), written from their definitions."""
import math

import numpy as np
import torch

import block_testutil as ref


def rope(x, at, inv_freq, scale, interleaved, inverse=False):
    """x float64 [N, heads, D]; at: the N tokens' positions.  Returns (out, |a| + |b| of each element's pair times
    |scale|, |angle|); angles in extended precision."""
    out, size, turn = x.clone(), torch.zeros_like(x), torch.zeros_like(x)
    half = inv_freq.numel()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = np.array(at, dtype=np.longdouble) * np.longdouble(float(inv_freq[i])) * (-1 if inverse else 1)
        c = torch.tensor(np.cos(angle).astype(np.float64))[:, None] * scale
        s = torch.tensor(np.sin(angle).astype(np.float64))[:, None] * scale
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(scale)
        turn[..., a] = turn[..., b] = torch.tensor(np.abs(angle).astype(np.float64))[:, None]
    return out, size, turn


def rope_bound(out, size, turn, dtype):
    """Cosine and sine: the series is cut below 3e-9, its argument (at most pi / 4) and its five or six fp32 steps, whose
    later terms are small, round by at most 2^-22 together, the factor by 2^-24; the angle is off by three roundings of
    64 bits.  Two fp32 products and a sum: 2^-23.  All together below 2^-21 of |a| + |b|; then the output's rounding."""
    return (2.0 ** -21 + 3 * 2.0 ** -53 * turn) * size + torch.finfo(dtype).eps / 2 * out.abs() + torch.finfo(dtype).tiny * 2.0 ** -10


def weigh(q, cu, kv_lens, rows, table, k, prior, since, scale):
    """q float64 [total, Hq, D]; k float64 values [n_blocks, H, B, D] (times the scales); prior float64 [rows, H, width].
    Returns (out, a bound of each element's relative error but for the output's rounding)."""
    nb, H, B, D = k.shape
    out, rel = prior.clone(), torch.zeros_like(prior)
    g = q.shape[1] // H
    for r, row in enumerate(rows):
        if not 0 <= row < len(table):
            continue
        m = cu[r + 1] - cu[r]
        length = min(kv_lens[r], len(table[row]) * B)
        pos = [p for p in range(length) if 0 <= table[row][p // B] < nb]
        at = torch.tensor(pos, dtype=torch.long)
        blk = torch.tensor([table[row][p // B] for p in pos], dtype=torch.long)
        first = since[r] if since is not None else kv_lens[r] - m
        out[row, :, max(0, min(first, length)):length] = 0
        for h in range(H):
            kk = k[blk, h, at % B]
            reach = 0.0
            for j in range(g):
                qq = q[cu[r]:cu[r + 1], h * g + j]
                x = qq @ kk.t() * scale
                reach = max([reach] + (qq.abs() @ torch.nan_to_num(kk, 0, 0, 0).abs().t() * scale).flatten().tolist())
                last = kv_lens[r] - m + torch.arange(m)
                gone = at[None] > last[:, None]
                x = x.masked_fill(gone, -math.inf)
                w = torch.softmax(x, -1).masked_fill(gone, 0.0)
                out[row, h, at] += w.sum(0)
            # scores: D fp32 products and sums and their factor, of at most `reach` in all, twice in a quotient; sums of
            # `length` and of m * g terms; the exponential and the quotient
            rel[row, h, :length] = 2 * (D + 4) * 2.0 ** -24 * reach + (length + m * g) * 2.0 ** -24 + 2.0 ** -20
    return out, rel


def weigh_close(got, out, rel):
    got = got.double().cpu()
    nan = torch.isnan(out)
    assert torch.equal(nan, torch.isnan(got)), "NaN pattern differs"
    tol = (rel + 2.0 ** -24) * out.abs() + 1e-30
    off = (got - out).abs()
    bad = (off > tol) & ~nan
    assert not bad.any(), (int(bad.sum()), float((off / tol)[bad].max()))


def position(e, pos, held, evicted):
    return pos[e] if e < held else e + evicted


def keep(weights, length, budget, recent, sinks, pos=None, held=0, evicted=0):
    """src of one request and KV head; weights: a list."""
    if length <= budget:
        return [e if e < length else -1 for e in range(budget)]

    def order(e):
        at = position(e, pos, held, evicted) if pos is not None else e
        total = length + (evicted if pos is not None else 0)
        if e < sinks or at >= total - recent:
            return (0, 0.0, e)
        w = weights[e]
        return (2, 0.0, e) if w != w else (1, -w + 0.0, e)
    chosen = set(sorted(range(length), key=order)[:budget])
    comes = iter(sorted(e for e in chosen if e >= budget))
    return [e if e in chosen else next(comes) for e in range(budget)]


def evict(src, kv_lens, rows, table, codes, scales, kv, weights=None, pos=None, held=None, evicted=None):
    """In place: codes [float64 values [n_blocks, H, B, D]] and scales [float64 [n_blocks, H]] of both sides, weights
    and pos [rows, H, width]."""
    nb, H, B, _ = codes[0].shape
    for j, row in enumerate(rows):
        budget = len(src[j][0])
        if not 0 <= row < len(table) or kv_lens[j] <= budget:
            continue

        def block(e):
            b = table[row][e // B]
            return b if 0 <= b < nb else None
        for h in range(H):
            moves = [s if budget <= s < kv_lens[j] and block(s) is not None and block(e) is not None else e
                     for e, s in enumerate(src[j][h])]
            for lp in range(budget // B):
                es = list(range(lp * B, lp * B + B))
                if all(moves[e] == e for e in es):
                    continue
                to = block(lp * B)
                for c, z in zip(codes, scales):
                    x = torch.stack([c[block(moves[e]), h, moves[e] % B] for e in es])
                    s = torch.stack([z[block(moves[e]), h] for e in es])
                    if torch.isfinite(s).all():
                        y = x * s[:, None]
                        fin = y[torch.isfinite(y)].abs()
                        size = ref.scale_of(float(fin.max()) if fin.numel() else 0.0, kv)
                        x = ref.round_code(y / size, kv)
                    else:
                        size = math.nan
                    c[to, h], z[to, h] = x, size
            if weights is not None:
                was = weights[row, h].clone()
                for e, s in enumerate(moves):
                    weights[row, h, e] = was[s]
            if pos is not None:
                was = pos[row, h].tolist()
                for e, s in enumerate(moves):
                    pos[row, h, e] = position(s, was, int(held[row]), int(evicted[row]))


def trim(seqs, seq_lens, table, free, head, budget, B, held, evicted, n_free, commit=True):
    """In place on the lists; (kv_lens, next head, status)."""
    kv, freed, status, seen = [], [], 0, set()
    for s in seqs:
        if not 0 <= s < len(table) or s in seen:
            status |= 8
            kv.append(0)
            continue
        seen.add(s)
        n = max(seq_lens[s], 0)
        kv.append(min(n, budget))
        if n <= budget:
            continue
        for lp in range(budget // B, min(-(-n // B), len(table[s]))):
            if 0 <= table[s][lp] < n_free:
                freed.append(table[s][lp])
            if commit:
                table[s][lp] = -1
        if commit:
            seq_lens[s] = held[s] = budget
            evicted[s] += n - budget
    if len(freed) > head:
        status |= 16
    for i, b in enumerate(freed):
        if head - len(freed) + i >= 0:
            free[head - len(freed) + i] = b
    return kv, max(head - len(freed), 0), status
