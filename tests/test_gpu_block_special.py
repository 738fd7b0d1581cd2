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


@pytest.mark.parametrize("kernel,splits",
                         [("decode", -9), ("decode", -40)] + [(k, s) for k in ("decode", 16, 128) for s in (2, 7, 30)])
@pytest.mark.parametrize("D", [64, 256])
def test_scales_that_are_not_finite_in_parts(kvt_pkg, monkeypatch, kernel, splits, D):
    """The same where the positions are split: a part without any finite score, merged in the launch and behind it."""
    lens = [2000, 700, 64]
    new = [1] * 3 if kernel == "decode" else [300, 40, 64]
    bad = {(0, lp): (NAN, NAN) for lp in range(26, 31)}
    for ws in (None, {}):
        _check(monkeypatch, kernel, "fp8", 8, 2, D, 64, new, lens, {**bad, (1, 0): (None, NAN)}, splits=splits, seed=5,
               workspace=ws)


@pytest.mark.parametrize("kernel", [16, 128])
def test_scales_that_are_not_finite_cross(kvt_pkg, monkeypatch, kernel):
    """Without the causal mask every query of the request sees the block."""
    _check(monkeypatch, kernel, "int8", 4, 4, 64, 32, [33, 40], [100, 77], {(1, 2): (None, NAN)}, causal=False, seed=2)


@pytest.mark.parametrize("kernel", ["decode", 16, 128])
@pytest.mark.parametrize("Hq,H,D,B", [(2, 2, 64, 16), (8, 2, 128, 64), (16, 2, 256, 32)])
@pytest.mark.parametrize("splits", [None, 1, 3])
def test_nan_codes_reach_the_rows_that_see_them(kvt_pkg, monkeypatch, kernel, Hq, H, D, B, splits):
    """NaN codes of K and of V (e4m3) inside a causal chunk: a NaN in V makes its channel NaN for the queries from its position on,
    one in K every channel; earlier queries of the same tile are what they are without it."""
    from kvtier import block_kv
    if kernel != "decode":
        monkeypatch.setattr(block_kv, "_TILE_MIN", {D: 0 if kernel == 128 else 10 ** 9})
    lens = [70, 200, 333, 5, 40]
    new = [1] * 5 if kernel == "decode" else [70, 150, 9, 5, 1]
    g = torch.Generator().manual_seed(D)
    table, nb = _tables(lens, B, 2, D)
    codes, sc = _pool("fp8", nb, H, B, D, g)
    cu, causal = prefix(new), kernel != "decode"
    q = torch.randn(cu[-1], Hq, D, generator=g).to(torch.bfloat16)
    # (request, position, channel or None for K): in the first tile, at tile borders, near and at the end, twice in a channel
    spots = [(0, 0, 3), (0, 63, 5), (0, 64, 0), (0, 69, D - 1), (0, 20, 3), (0, 11, None), (1, 51, 7), (1, 100, 7), (1, 128, 8),
             (1, 199, 9), (1, 170, None), (2, 332, 1), (2, 326, 2), (2, 5, 4), (3, 4, 0), (4, 39, 60)]
    bits = [c.clone().view(torch.uint8) for c in codes]
    for j, (r, p, d) in enumerate(spots):
        at = (table[r][p // B], 0, p % B)
        codes[d is not None].view(torch.uint8)[at][d or 0] = 0
        bits[d is not None][at][d or 0] = 0x7F if j % 2 else 0xFF
    val = [ref.values(codes[i]) * sc[i].double()[..., None, None] for i in range(2)]
    want = list(ref.attention(q.double(), cu, lens, range(len(new)), table, val[0], val[1], causal, D ** -0.5))
    t = 0
    for r, n in enumerate(new):
        for s in _sees([n], [lens[r]], causal):
            for b, p, d in spots:
                if b == r and p < s:
                    want[0][t, :Hq // H, slice(None) if d is None else d] = math.nan
            t += 1
    args = [b.view(torch.float8_e4m3fn).to(dev) for b in bits] + [s.to(dev) for s in sc] + [i32(table), i32(lens)]
    if kernel == "decode":
        got = block_kv.kvt_block_decode(q.to(dev), *args, splits=splits)
    else:
        got = block_kv.kvt_block_prefill(q.to(dev), i32(cu), *args, splits=splits)
    # (a zero code for a NaN changes the other channels of rows that see it only through K, and those rows are NaN)
    ref.close(got, *want, D)


def test_a_nan_row_that_is_appended(kvt_pkg):
    """Through the cache: a token whose V is NaN leaves the queries before it, of its own prompt and of others, finite."""
    from kvtier import block_kv
    c = block_kv.BlockKVCache(1, 2, 128, n_blocks=20, max_seqs=2, max_blocks=10, block=32)
    rows = [c.add_seq(), c.add_seq()]
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(2, 150, 2, 128, device=dev, generator=g).to(torch.bfloat16)
    x[1, 80] = math.nan
    q = torch.randn(150, 8, 128, device=dev, generator=g).to(torch.bfloat16)
    plan = c.plan(rows, [100, 50])
    c.append(0, plan, x[0], x[1])
    bad = torch.isnan(c.prefill(0, plan, q)).flatten(1)
    assert not bad[:80].any() and bad[80:100].all() and not bad[100:].any()


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("n", [1, 30])
def test_a_scale_that_is_not_finite_stays(kvt_pkg, kv, n):
    """Rows appended to a block whose scale is NaN or infinite do not give the rows held there a finite scale; a block that the
    call opens takes no notice of what its scale was."""
    from kvtier import block_kv
    c = block_kv.BlockKVCache(1, 3, 64, n_blocks=4, max_seqs=1, max_blocks=4, block=16, dtype=ref.CODE[kv])
    s = c.add_seq()
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(2, 5 + n, 3, 64, device=dev, generator=g).to(torch.bfloat16)
    for t in (c.ks[0], c.vs[0]):
        t.fill_(math.nan)
    c.append(0, c.plan([s], [5]), x[0, :5], x[1, :5])
    first, later = int(c.block_table[s, 0]), [i for i in range(4) if i != int(c.block_table[s, 0])]
    for t in (c.ks[0], c.vs[0]):
        assert bool(torch.isfinite(t[first]).all()) and bool(torch.isnan(t[later]).all())
        t[first, 0], t[first, 1] = math.nan, math.inf
    plan = c.plan([s], [n])
    c.append(0, plan, x[0, 5:], x[1, 5:])
    for t in (c.ks[0], c.vs[0]):
        assert math.isnan(t[first, 0]) and math.isinf(t[first, 1]) and bool(torch.isfinite(t[first, 2]))
        for lp in range(1, -(-(5 + n) // 16)):
            assert bool(torch.isfinite(t[c.block_table[s, lp]]).all())
    q = torch.randn(n, 3, 64, device=dev, generator=g).to(torch.bfloat16)
    bad = torch.isnan(c.prefill(0, plan, q))
    assert bool(bad[:, :2].all()) and not bool(bad[:, 2].any())


@pytest.mark.parametrize("counts", [[5, 0, 33], [300, 1, 200]])
def test_a_padded_step(kvt_pkg, counts):
    """More rows than the counts' sum, NaN behind it: the cache and the queries' rows are those of the step without padding, a
    given out keeps its rows behind the sum, and one that is made there has the rows before it."""
    from kvtier import block_kv
    H, D, n = 2, 128, sum(counts)
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(2, n + 70, H, D, device=dev, generator=g).to(torch.bfloat16)
    q = torch.randn(n + 70, 8, D, device=dev, generator=g).to(torch.bfloat16)
    x[:, n:] = q[n:] = math.nan
    made = []
    for rows in (n, n + 70):
        c = block_kv.BlockKVCache(1, H, D, n_blocks=60, max_seqs=3, max_blocks=30, block=32, seed=4)
        seqs = i32([c.add_seq() for _ in counts])
        plan = c.plan(seqs, i32(counts), n_tokens=rows)
        c.append(0, plan, x[0, :rows], x[1, :rows])
        out = torch.full((rows, 8, D), 5.0, dtype=torch.bfloat16, device=dev)
        got = c.prefill(0, plan, q[:rows], out=out)
        assert got is out and bool((out[n:] == 5.0).all())
        val = [ref.values(x8[0].cpu()) * s[0].cpu().double()[..., None, None] for x8, s in ((c.k8, c.ks), (c.v8, c.vs))]
        want = ref.attention(q[:n].cpu().double(), prefix(counts), counts, seqs.tolist(), c.block_table.tolist(), *val,
                             True, D ** -0.5)
        for y in (out, c.prefill(0, plan, q[:rows])):
            ref.close(y[:n], *want, D)
        c.check()
        made.append(c)
    a, b = made
    for i, j in ((a.k8, b.k8), (a.v8, b.v8)):
        assert torch.equal(i[0].view(torch.int8), j[0].view(torch.int8))
    assert torch.equal(a.ks[0], b.ks[0]) and torch.equal(a.vs[0], b.vs[0]) and torch.equal(a.block_table, b.block_table)
