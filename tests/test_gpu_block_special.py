"""8-bit block cache on the GPU: scales that are not finite.  A row is compared with the 64-bit form over what it sees; what it
does not see must not reach it."""
import math

import pytest
import torch

import block_testutil as ref
from test_gpu_block_kv import _pool, _tables, dev, i32, prefix

pytestmark = pytest.mark.gpu


def _sees(new, kv_lens, causal):
    """Positions that each query row sees."""
    return [max(min(L - n + i + 1 if causal else L, L), 0) for n, L in zip(new, kv_lens) for i in range(n)]


def _check(monkeypatch, kernel, kv, Hq, H, D, B, new, kv_lens, bad, causal=True, splits=None, seed=0, workspace=None):
    """kernel: "decode", or 16 / 128 for the chunk kernel of so many rows.  bad: {(request, block): (K scale, V scale)}, None for
    the one it has.  A row that sees a position of such a block is NaN, every other one as if the block's scales were 1."""
    from kvtier import block_kv
    if kernel != "decode":
        monkeypatch.setattr(block_kv, "_TILE_MIN", {D: 0 if kernel == 128 else 10 ** 9})
    causal = causal and kernel != "decode"
    g = torch.Generator().manual_seed(seed)
    table, nb = _tables(kv_lens, B, 2, seed)
    codes, sc = _pool(kv, nb, H, B, D, g)
    cu = prefix(new)
    q = torch.randn(cu[-1], Hq, D, generator=g).to(torch.bfloat16)
    dsc = [s.clone() for s in sc]
    for (r, lp), values in bad.items():
        for i in range(2):
            if values[i] is not None:
                dsc[i][table[r][lp], H - 1] = values[i]
                sc[i][table[r][lp], H - 1] = 1.0
    val = [ref.values(codes[i]) * sc[i].double()[..., None, None] for i in range(2)]
    want = list(ref.attention(q.double(), cu, kv_lens, range(len(new)), table, val[0], val[1], causal, D ** -0.5))
    t = 0
    for r, n in enumerate(new):
        for s in _sees([n], [kv_lens[r]], causal):
            if any(b == r and lp * B < s for b, lp in bad):
                want[0][t, (H - 1) * (Hq // H):] = math.nan
            t += 1
    args = [c.to(dev) for c in codes] + [s.to(dev) for s in dsc] + [i32(table), i32(kv_lens)]
    kw = dict(out=torch.zeros(q.shape, dtype=torch.float32, device=dev), splits=splits, workspace=workspace)
    if kernel == "decode":
        got = block_kv.kvt_block_decode(q.to(dev), *args, **kw)
    else:
        got = block_kv.kvt_block_prefill(q.to(dev), i32(cu), *args, causal=causal, **kw)
    ref.close(got, *want, D)


NAN, INF = math.nan, math.inf


@pytest.mark.parametrize("kernel", ["decode", 16, 128])
@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("Hq,H,D,B", [(4, 2, 64, 16), (8, 2, 128, 64), (16, 2, 256, 32)])
@pytest.mark.parametrize("scales", [(None, NAN), (NAN, None), (None, INF), (INF, None), (NAN, NAN)])
def test_scales_that_are_not_finite(kvt_pkg, monkeypatch, kernel, kv, Hq, H, D, B, scales):
    """In a request's only block, its first, one in the middle and its last: whatever the order, the rows that see it are NaN
    and no others are."""
    lens = [B - 3, 5 * B + 2, 5 * B + 2, 5 * B + 2, 3 * B]
    new = [1] * 5 if kernel == "decode" else [B - 3, 5 * B + 2, 70, 4 * B, 9]
    _check(monkeypatch, kernel, kv, Hq, H, D, B, new, lens, {(0, 0): scales, (1, 0): scales, (2, 2): scales, (3, 5): scales},
           seed=D + B)


@pytest.mark.parametrize("kernel,splits", [("decode", -9), ("decode", -40)] + [(k, s) for k in ("decode", 16, 128) for s in (2, 7, 30)])
@pytest.mark.parametrize("D", [64, 256])
def test_scales_that_are_not_finite_in_parts(kvt_pkg, monkeypatch, kernel, splits, D):
    """The same where the positions are split: a part without any finite score, merged in the launch and behind it."""
    lens = [2000, 700, 64]
    new = [1] * 3 if kernel == "decode" else [300, 40, 64]
    bad = {(0, lp): (NAN, NAN) for lp in range(26, 31)}
    for ws in (None, {}):
        _check(monkeypatch, kernel, "fp8", 8, 2, D, 64, new, lens, {**bad, (1, 0): (None, NAN)}, splits=splits, seed=5, workspace=ws)


@pytest.mark.parametrize("kernel", [16, 128])
def test_scales_that_are_not_finite_cross(kvt_pkg, monkeypatch, kernel):
    """Without the causal mask every query of the request sees the block."""
    _check(monkeypatch, kernel, "int8", 4, 4, 64, 32, [33, 40], [100, 77], {(1, 2): (None, NAN)}, causal=False, seed=2)
