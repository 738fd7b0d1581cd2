"""A block cache within a budget on the GPU: accumulated attention weight, choice of entries, their move, blocks given back,
each against a plain 64-bit form (tests/evict_testutil.py), and all of them together as a serving program uses them."""
import math
import random

import pytest
import torch

import block_testutil as bref
import evict_testutil as ref

pytestmark = pytest.mark.gpu
dev = "cuda"
IO = {"bf16": torch.bfloat16, "f16": torch.float16}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prefix(x):
    out = [0]
    for y in x:
        out.append(out[-1] + y)
    return out


def pool(lens, max_blocks, n_rows, H, B, D, kv, seed, wide=1.0):
    """Codes, scales (powers of two) and tables of requests in rows of their own; (codes, scales, table, rows), on the CPU."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    blocks = [min(-(-x // B), max_blocks) for x in lens]
    nb = sum(blocks) + 2
    ids = list(range(nb))
    rng.shuffle(ids)
    rows = rng.sample(range(n_rows), len(lens))
    table = [[-1] * max_blocks for _ in range(n_rows)]
    for r, n in zip(rows, blocks):
        for lp in range(n):
            table[r][lp] = ids.pop()
    sides = []
    for gain in (wide, 1.0):
        x = torch.randn(nb, H, B, D, generator=g) * gain
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / bref.QMAX[kv])))
        sides.append((bref.round_code((x / s[..., None, None]).double(), kv).float().to(bref.CODE[kv]), s))
    return sides, table, rows


def values(side):
    return bref.values(side[0]) * side[1].double()[..., None, None]


# ------------------------------------------------------------------------------------------------------------ weigh
def run_weigh(case, fresh=False, apart=False, edit=None, ws=None, spare=0):
    from kvtier.block_evict import kvt_block_weigh
    lens, counts, hq, H, D, B, kv, io, seed = case
    one = counts is None
    m = [1] * len(lens) if one else counts
    max_blocks = max([-(-x // B) for x in lens] + [1]) + spare
    sides, table, rows = pool(lens, max_blocks, len(lens) + 2, H, B, D, kv, seed)
    g = torch.Generator().manual_seed(seed + 1)
    cu = prefix(m)
    q = torch.randn(cu[-1] + (0 if one else 3), hq, D, generator=g).to(IO[io])
    prior = torch.rand(len(table), H, max_blocks * B, generator=g)
    since = [0] * len(lens) if fresh else None
    if edit:
        sides, table, q = edit(sides, table, q, rows)
    (k8, ks) = sides[0]
    want, rel = ref.weigh(q.double(), cu, lens, rows, table, values((k8, ks)), prior.double(), since, D ** -0.5)
    w = prior.to(dev)
    out = torch.full_like(w, 9.0) if apart else None
    if apart:
        for r, n in zip(rows, lens):
            n = min(n, max_blocks * B)
            keep = torch.full_like(want[r], 9.0)
            keep[:, :n] = want[r][:, :n]
            want[r] = keep
        for r in set(range(len(table))) - set(rows):
            want[r] = 9.0
    got = kvt_block_weigh(q.to(dev), k8.to(dev), ks.to(dev), i32(table), i32(lens), w, None if one else i32(cu), i32(rows),
                          i32(since) if fresh else None, out=out, workspace=ws)
    assert got.data_ptr() == (out if apart else w).data_ptr()
    ref.weigh_close(got, want, rel)
    if apart:
        assert torch.equal(w.cpu(), prior)
    return got


WEIGH = [
    # lens, counts (None: one query each), hq, H, D, B, kv, io, seed
    ([1], None, 1, 1, 64, 16, "fp8", "bf16", 1),
    ([0, 1, 15, 16, 17, 64, 65], None, 12, 1, 128, 16, "int8", "f16", 2),
    ([777], None, 24, 2, 256, 64, "fp8", "bf16", 3),
    ([3000, 255, 256, 257, 5], None, 16, 2, 256, 32, "int8", "bf16", 4),
    ([2049, 1], None, 20, 20, 64, 32, "fp8", "f16", 5),
    ([1100, 300], None, 32, 2, 128, 64, "int8", "f16", 6),
    ([5], [5], 1, 1, 64, 16, "fp8", "bf16", 11),
    ([300, 0, 70, 1, 40], [7, 0, 70, 1, 2], 12, 1, 128, 64, "fp8", "bf16", 12),
    ([257], [257], 8, 8, 64, 16, "int8", "f16", 13),
    ([700, 100], [33, 100], 16, 2, 256, 32, "int8", "bf16", 14),
    ([2000], [61], 12, 1, 128, 64, "fp8", "f16", 15),
    ([520], [520], 24, 2, 256, 64, "fp8", "bf16", 16),
    ([400, 400, 400], [1, 1, 1], 32, 4, 64, 32, "fp8", "bf16", 17),
]


@pytest.mark.parametrize("case", WEIGH, ids=[str(c[-1]) for c in WEIGH])
def test_weigh(kvt_pkg, case):
    run_weigh(case)
    ws = {}
    a = run_weigh(case, fresh=True, apart=True, ws=ws, spare=3)
    b = run_weigh(case, fresh=True, apart=True, ws=ws, spare=3)
    assert torch.equal(a, b)


WIDE = [c for c in WEIGH if c[-1] in (2, 4, 12, 14, 15, 16, 17)] + [
    ([1500, 90, 2600], [1500, 90, 700], 16, 2, 128, 64, "fp8", "bf16", 18),
    ([3000, 7], [1200, 1], 8, 1, 64, 16, "int8", "f16", 19),
]


@pytest.mark.parametrize("case", WIDE, ids=[str(c[-1]) for c in WIDE])
def test_weigh_in_wide_tables(kvt_pkg, case):
    """Requests that fill little of their table, whose width is what the launch is sized by."""
    ws = {}
    run_weigh(case, ws=ws, spare=30000 // case[5])
    run_weigh(case, fresh=True, apart=True, ws=ws, spare=1000 // case[5])


@pytest.mark.parametrize("counts", [None, [40, 3, 20]])
@pytest.mark.parametrize("what", ["gone", "stale", "nan key", "scale", "nan query", "zero"])
def test_weigh_specials(kvt_pkg, counts, what):
    """Blocks that are not there; NaN codes behind a request's end, and in it; scales that are infinite, NaN and zero; a
    query of NaN."""
    lens = [150, 90, 64]

    def edit(sides, table, q, rows):
        (k8, ks), v = sides
        raw = k8.view(torch.int8).clone()
        if what == "gone":
            table[rows[0]][2] = -1
            table[rows[1]][0] = 10 ** 6
        if what == "stale":
            raw[table[rows[0]][-1 + -(-150 // 32)], :, 150 % 32:] = 0x7F
            raw[table[rows[1]][90 // 32], :, 90 % 32:] = 0x7F
        if what == "nan key":                      # (a late position of the chunk: earlier queries do not see it)
            raw[table[rows[0]][140 // 32], 1, 140 % 32, 5] = 0x7F
        if what == "scale":
            ks = ks.clone()
            ks[table[rows[0]][0], 0] = math.inf
            ks[table[rows[1]][2], 1] = math.nan
        if what == "zero":
            ks = ks.clone()
            ks[table[rows[0]][0], 0] = 0.0
        if what == "nan query":
            q = q.clone()
            q[1, 2, 7] = math.nan
        return [(raw.view(torch.float8_e4m3fn), ks), v], table, q
    run_weigh((lens, counts, 4, 2, 64, 32, "fp8", "bf16", 21), edit=edit)


def test_weigh_scale_and_strides(kvt_pkg):
    """A given scale, unaligned query rows, weights as a slice of a larger tensor, a table wider than its requests."""
    from kvtier.block_evict import kvt_block_weigh
    lens, H, B, D, hq = [200, 31], 2, 16, 64, 6
    sides, table, rows = pool(lens, 20, 4, H, B, D, "int8", 5)
    g = torch.Generator().manual_seed(6)
    buf = torch.randn(2, hq * D + 5, generator=g).to(torch.bfloat16)
    prior = torch.rand(4, 3, H, 20 * B + 7, generator=g)
    q = buf[:, 5:].unflatten(1, (hq, D))
    want, rel = ref.weigh(q.double(), [0, 1, 2], lens, rows, table, values(sides[0]), prior[:, 1].double(), [100, 40], 0.3)
    w = prior.to(dev)
    kvt_block_weigh(buf.to(dev)[:, 5:].unflatten(1, (hq, D)), sides[0][0].to(dev), sides[0][1].to(dev), i32(table), i32(lens),
                    w[:, 1], seqs=i32(rows), since=i32([100, 40]), scale=0.3)
    ref.weigh_close(w[:, 1], want, rel)
    assert torch.equal(w[:, 0].cpu(), prior[:, 0]) and torch.equal(w[:, 2].cpu(), prior[:, 2])


@pytest.mark.parametrize("counts", [None, True])
def test_weigh_many_ragged_requests(kvt_pkg, counts):
    """More requests than lanes, some without queries, some without entries."""
    rng = random.Random(3)
    lens = [rng.choice([0, 1, 5, 40, 130]) for _ in range(150)]
    m = None if counts is None else [rng.choice([0, 0, 1, 2, 9]) if n else 0 for n in lens]
    m = m if m is None else [min(a, b) for a, b in zip(m, lens)]
    run_weigh((lens, m, 4, 2, 64, 16, "int8", "bf16", 31))


def test_weigh_rows_and_lengths_out_of_range(kvt_pkg):
    """Table rows that are not there are left out; chunks longer than their request, and requests longer than their table."""
    from kvtier.block_evict import kvt_block_weigh
    H, B, D, hq = 2, 16, 64, 4
    sides, table, rows = pool([48, 30, 48], 3, 3, H, B, D, "fp8", 8)
    g = torch.Generator().manual_seed(6)
    prior = torch.rand(3, H, 48, generator=g)
    for lens, counts, seqs in (([3, 100, 20], [5, 2, 1], rows), ([40, 30, 20], [1, 1, 1], [rows[0], 7, -1]),
                               ([40, 30, 20], None, [rows[0], 3, -5])):
        cu = prefix(counts or [1, 1, 1])
        q = torch.randn(cu[-1], hq, D, generator=g).to(torch.bfloat16)
        want, rel = ref.weigh(q.double(), cu, lens, seqs, table, values(sides[0]), prior.double(), None, D ** -0.5)
        w = prior.to(dev)
        kvt_block_weigh(q.to(dev), sides[0][0].to(dev), sides[0][1].to(dev), i32(table), i32(lens), w,
                        i32(cu) if counts else None, i32(seqs))
        ref.weigh_close(w, want, rel)


def test_weigh_queries_before_the_first_request(kvt_pkg):
    """Queries before the first request's are nobody's; what a workspace holds from before does not matter."""
    from kvtier.block_evict import kvt_block_weigh
    H, B, D, hq, lens = 2, 16, 64, 8, [1300, 40]
    sides, table, rows = pool(lens, 90, 2, H, B, D, "fp8", 8)
    g = torch.Generator().manual_seed(9)
    prior, cu = torch.rand(2, H, 90 * B, generator=g), [37, 70, 75]
    q = torch.randn(80, hq, D, generator=g).to(torch.bfloat16)
    want, rel = ref.weigh(q.double(), cu, lens, rows, table, values(sides[0]), prior.double(), None, D ** -0.5)
    ws, outs = {}, []
    for _ in range(2):
        w = prior.to(dev)
        kvt_block_weigh(q.to(dev), sides[0][0].to(dev), sides[0][1].to(dev), i32(table), i32(lens), w, i32(cu), i32(rows),
                        workspace=ws)
        ref.weigh_close(w, want, rel)
        outs.append(w)
        for buffer in ws.values():
            buffer.fill_(1e9)
    assert torch.equal(*outs)


def test_weigh_of_no_queries(kvt_pkg):
    """An output of its own gets the weights as they are."""
    from kvtier.block_evict import kvt_block_weigh
    sides, table, rows = pool([48, 30], 3, 2, 1, 16, 64, "fp8", 8)
    w = torch.rand(2, 1, 48, device=dev)
    out = torch.zeros_like(w)
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=dev)
    kvt_block_weigh(q, sides[0][0].to(dev), sides[0][1].to(dev), i32(table), i32([48, 30]), w, i32([0, 0, 0]), i32(rows), out=out)
    assert torch.equal(out[rows[0]], w[rows[0]]) and torch.equal(out[rows[1], :, :30], w[rows[1], :, :30])
    assert not out[rows[1], :, 30:].any()


@pytest.mark.parametrize("counts", [None, [90, 2]])
@pytest.mark.parametrize("scale", [0.25, 40.0])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_weigh_scores_far_apart(kvt_pkg, counts, scale, order):
    """Scores that rise, or fall, by hundreds and by tens of thousands along the entries: maxima that lie far above the first tile's, and below."""
    from kvtier.block_evict import kvt_block_weigh
    lens, H, B, D, hq = [600, 300], 2, 64, 64, 4
    sides, table, rows = pool(lens, 10, 2, H, B, D, "int8", 5)
    k8, ks = sides[0]
    ks = ks.clone()
    for r, n in zip(rows, lens):
        blocks = table[r][:-(-n // B)]
        for i, b in enumerate(blocks if order == "rising" else reversed(blocks)):
            ks[b] *= 2.0 ** (i - 4)
    g = torch.Generator().manual_seed(6)
    cu = prefix(counts or [1, 1])
    q = torch.randn(cu[-1], hq, D, generator=g).to(torch.bfloat16)
    prior = torch.rand(2, H, 640, generator=g)
    want, rel = ref.weigh(q.double(), cu, lens, rows, table, values((k8, ks)), prior.double(), None, scale)
    w = prior.to(dev)
    kvt_block_weigh(q.to(dev), k8.to(dev), ks.to(dev), i32(table), i32(lens), w, None if counts is None else i32(cu), i32(rows),
                    scale=scale)
    got = w.double().cpu()
    assert torch.isfinite(got).all()
    # Large scores leave the weights few exact bits: `rel` is the bound of that while it is small, 1 + rel for e^rel.  And
    # every query's weights sum to one, but for what the scores of the two launches differ by, each of them off by half of
    # rel's first term, and the roundings of the sums: by rel in all.
    most = float(rel.max())
    if scale < 1:
        assert most < 0.05 and ((got - want).abs() <= (rel + 2.0 ** -24) * want.abs() + 1e-30).all()
    for i, r in enumerate(rows):
        new = (got[r] - torch.where(torch.arange(640) < lens[i] - (cu[i + 1] - cu[i]), prior[r].double(), 0.0))[:, :lens[i]]
        assert torch.allclose(new.sum(-1), torch.tensor(float((cu[i + 1] - cu[i]) * hq // H), dtype=torch.float64), rtol=most,
                              atol=0)


@pytest.mark.parametrize("at_once", [1, 2, 3, 100])
def test_weigh_requests_in_turns(kvt_pkg, monkeypatch, at_once):
    """Scores of a few requests at once: with rows and without, strides, given `since`; a workspace that an earlier call
    left larger changes nothing."""
    from kvtier import block_evict
    lens, hq, H, B, D = [700, 0, 65, 1500, 16, 333, 1], 12, 2, 32, 128
    n, mb = len(lens), 47
    monkeypatch.setattr(block_evict, "_SCORES", at_once * hq * mb * B)
    case = (lens, None, hq, H, D, B, "fp8", "bf16", 61)
    ws = {}
    outs = [run_weigh(case, fresh=True, apart=True, ws=w) for w in (ws, ws, {("weigh", 0): torch.empty(1 << 24, device=dev)}, None)]
    run_weigh(case, ws=ws)
    assert all(torch.equal(outs[0], x) for x in outs)
    sides, table, rows = pool(lens, mb, n, H, B, D, "int8", 62)
    table = [table[r] for r in rows]                       # (request j's row is j; one row more than requests)
    table.append([-1] * mb)
    g = torch.Generator().manual_seed(63)
    q = torch.randn(n, hq, D, generator=g).to(torch.float16)
    prior = torch.rand(n + 1, H, 2, mb * B, generator=g)
    since = [100, 0, 65, 7, 16, 332, 1]
    want, rel = ref.weigh(q.double(), list(range(n + 1)), lens, list(range(n)), table, values(sides[0]), prior[:, :, 1].double(),
                          since, D ** -0.5)
    w = prior.to(dev)
    block_evict.kvt_block_weigh(q.to(dev), sides[0][0].to(dev), sides[0][1].to(dev), i32(table), i32(lens), w[:, :, 1],
                                since=i32(since))
    ref.weigh_close(w[:, :, 1], want, rel)
    assert torch.equal(w[:, :, 0].cpu(), prior[:, :, 0])


LONG = [
    # lens, counts (None: one query each), hq, H, D, B, kv, io, seed
    ([9001, 5003, 1025], None, 8, 2, 64, 16, "fp8", "bf16", 71),
    ([8197, 300], None, 12, 1, 256, 64, "int8", "f16", 72),
    ([4099], None, 32, 2, 128, 32, "int8", "bf16", 73),
    ([2501, 777, 1300], [100, 3, 61], 8, 2, 64, 16, "fp8", "bf16", 74),
    ([2501, 1100], [101, 40], 12, 1, 256, 64, "int8", "bf16", 75),
    ([1800, 2100], [1800, 33], 4, 2, 128, 32, "int8", "f16", 76),
    ([2309], [2309], 2, 1, 256, 64, "fp8", "f16", 77),
    ([1300] * 3, [700, 0, 1300], 16, 1, 64, 64, "int8", "bf16", 78),
]


@pytest.mark.parametrize("case", LONG, ids=[str(c[-1]) for c in LONG])
def test_weigh_by_few_workgroups(kvt_pkg, monkeypatch, case):
    """As few workgroups as many requests over long tables leave each pair: one split over more than 4,096 positions (one
    query) or 1,024 (chunks), whose ids and scales are read again on the way, and workgroups of the sums that take
    1,024 positions, or 256 of a chunk, after others."""
    from kvtier import block_evict
    monkeypatch.setattr(block_evict, "_ROW_BLOCKS", 1)
    monkeypatch.setattr(block_evict, "_CHUNK_BLOCKS", 1)
    monkeypatch.setattr(block_evict, "_CHUNK_FIT", {64: 1, 128: 1, 256: 1})
    ws = {}
    a = run_weigh(case, fresh=True, apart=True, ws=ws)
    b = run_weigh(case, fresh=True, apart=True, ws=ws)
    assert torch.equal(a, b)
    run_weigh(case, spare=5)


@pytest.mark.parametrize("groups,splits", [(2, 1), (3, 2), (5, 7)])
def test_weigh_by_some_workgroups(kvt_pkg, groups, splits):
    """The same by the C entry's own numbers: several groups and splits, each of which takes more than one turn."""
    from kvtier import _lib
    H, hq, D, B = 2, 8, 64, 32
    for lens, counts, code, kv in (([9001, 2600], None, 0, "fp8"), ([3500, 1500], [150, 40], 1, "int8")):
        max_blocks = -(-max(lens) // B)
        sides, table, rows = pool(lens, max_blocks, 2, H, B, D, kv, 81)
        g = torch.Generator().manual_seed(82)
        cu = prefix(counts or [1, 1])
        q = torch.randn(cu[-1], hq, D, generator=g).to(torch.bfloat16)
        prior = torch.rand(2, H, max_blocks * B, generator=g)
        want, rel = ref.weigh(q.double(), cu, lens, rows, table, values(sides[0]), prior.double(), None, D ** -0.5)
        w, qd, k8, ks, t = prior.to(dev), q.to(dev), sides[0][0].to(dev), sides[0][1].to(dev), i32(table)
        floats = 2 * (hq * max_blocks * B + H * splits * 32) if counts is None else cu[-1] * hq * 2 * (splits + 1)
        work, n, c, r = torch.empty(floats, device=dev), i32(lens), i32(cu), i32(rows)
        _lib.call("kvt_block_weigh", qd.data_ptr(), hq * D, D, _lib.DTYPE_CODE[q.dtype], c.data_ptr() if counts else None,
                  cu[-1], n.data_ptr(), 2, H, hq, D, code, k8.data_ptr(), ks.data_ptr(), k8.shape[0], B, t.data_ptr(), max_blocks,
                  2, max_blocks, r.data_ptr(), D ** -0.5, None, w.data_ptr(), w.stride(0), w.stride(1), w.data_ptr(),
                  w.stride(0), w.stride(1), splits, 1, groups, 0, 1, work.data_ptr(), floats,
                  torch.cuda.current_stream().cuda_stream)
        ref.weigh_close(w, want, rel)


@pytest.mark.parametrize("counts", [None, [90, 2, 300], [1300, 2, 61]])
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("shape", ["1", "1/4", "16", "90 a tile", "91 a tile", "a jump", "waves"])
def test_weigh_of_exact_scores(kvt_pkg, monkeypatch, counts, few, shape):
    """Whole scores in powers of two, up to some 40,000 and exact in 32 bits, that rise along the entries for one q head, fall
    for the second, and neither for the others: every weight within what exponential, sums and quotient round."""
    from kvtier import block_evict
    if few:
        monkeypatch.setattr(block_evict, "_ROW_BLOCKS", 1)
        monkeypatch.setattr(block_evict, "_CHUNK_BLOCKS", 1)
        monkeypatch.setattr(block_evict, "_CHUNK_FIT", {64: 1})
    lens, H, B, D, hq = [2501, 70, 1400], 2, 32, 64, 8
    max_blocks = 80
    rise = {"1": lambda p: p, "1/4": lambda p: p // 4, "16": lambda p: 16 * p, "90 a tile": lambda p: p // 64 * 90,
            "91 a tile": lambda p: p // 64 * 91, "a jump": lambda p: 30_000 * (p > 1000), "waves": lambda p: abs(p % 700 - 350) * 3}[shape]
    sides, table, rows = pool(lens, max_blocks, 4, H, B, D, "fp8", 91)
    g = torch.Generator().manual_seed(92)
    # channels 0 .. 3: a position's rise in digits of 16, times 1, 16, 256, 4,096 by the query; 4 .. 11: noise.  Blocks of
    # scale 1 / 2 hold twice the value: all of it is exact in e4m3
    k8 = torch.zeros(len(sides[0][1]), H, B, D)
    ks = torch.exp2(-torch.randint(0, 2, sides[0][1].shape, generator=g).float())
    k8[..., 4:12] = torch.randint(-1, 2, (*k8.shape[:3], 8), generator=g).float()
    for r, n in zip(rows, lens):
        for p in range(n):
            v = rise(p)
            k8[table[r][p // B], :, p % B, :4] = torch.tensor([float(v >> 4 * i & 15) for i in range(4)])
    k8 = (k8 / ks[..., None, None]).to(torch.float8_e4m3fn)
    m = counts or [1, 1, 1]
    cu = prefix(m)
    q = torch.zeros(cu[-1], hq, D)
    q[..., 4:12] = torch.randint(-1, 2, (cu[-1], hq, 8), generator=g).float()
    for h in range(hq):
        q[:, h, :4] = torch.tensor([1.0, 16.0, 256.0, 4096.0]) * (1, -1, 0, 0)[h % 4]
    q = q.to(torch.bfloat16)
    prior = torch.rand(4, H, max_blocks * B, generator=g)
    # (the scale is ln 2: in fp32 its product with log2 e rounds to 1)
    assert float(torch.tensor(math.log(2), dtype=torch.float32) * torch.tensor(1 / math.log(2), dtype=torch.float32)) == 1.0
    want, _ = ref.weigh(q.double(), cu, lens, rows, table, values((k8, ks)), prior.double(), None, math.log(2))
    # exponential and quotient, and sums of up to `length` and of m * g terms; weights under 2^-99 are as good as none
    rel = torch.zeros_like(want)
    for r, n, c in zip(rows, lens, m):
        rel[r] = (n + c * hq // H) * 2.0 ** -24 + 2.0 ** -20
    w = prior.to(dev)
    block_evict.kvt_block_weigh(q.to(dev), k8.to(dev), ks.to(dev), i32(table), i32(lens), w, None if counts is None else i32(cu),
                                i32(rows), scale=math.log(2))
    ref.weigh_close(w, want, rel)


@pytest.mark.parametrize("D,few", [(64, True), (128, True), (256, True), (64, False)])
def test_weigh_long_columns(kvt_pkg, monkeypatch, D, few):
    """8,192 rows that all pay 1 / 37 to the same 37 entries (the others' weights are 2^-192): sums are formed by tiles of 64
    rows, and lose no more than that."""
    from kvtier import block_evict
    if few:
        monkeypatch.setattr(block_evict, "_CHUNK_BLOCKS", 1)
        monkeypatch.setattr(block_evict, "_CHUNK_FIT", {64: 1, 128: 1, 256: 1})
    m, hq, H, B, top = 2048, 4, 1, 64, 37
    n = m + top
    nb = -(-n // B)
    k8 = torch.zeros(nb, H, B, D)
    k8.view(nb * B, D)[top:, 0] = -192.0
    k8 = k8.to(torch.float8_e4m3fn)
    q = torch.zeros(m, hq, D, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    w = torch.full((1, H, nb * B), 9.0, device=dev)
    block_evict.kvt_block_weigh(q.to(dev), k8.to(dev), torch.ones(nb, H, device=dev), i32([list(range(nb))]), i32([n]), w, i32([0, m]),
                                since=i32([0]), scale=math.log(2))
    # Scores, exponentials and a row's sum, 37, are exact; one rounding of 1 / 37, 32 sums of a lane in a tile, one for each
    # of at most 128 tiles (splits are joined by fewer), one of a lane's two halves.
    got = w[0, 0, :n].double().cpu()
    assert ((got[:top] * top / (m * hq) - 1).abs() <= (1 + 32 + 128 + 1) * 2.0 ** -24).all(), float((got[:top] * top / (m * hq) - 1).abs().max())
    assert (got[top:] == 0).all() and (w[0, 0, n:] == 9).all()


def test_weigh_far_offsets(kvt_pkg):
    """Code offsets past 2^31 bytes and weight offsets past 2^31 entries."""
    from kvtier.block_evict import kvt_block_weigh
    H, B, D, hq = 8, 64, 256, 8
    nb = 16_500                                            # 2.16e9 bytes of codes
    k8 = torch.zeros(nb, H, B, D, dtype=torch.int8, device=dev)
    ks = torch.ones(nb, H, device=dev)
    max_blocks = 2 ** 22                                   # 2^28 entries a head
    table = torch.full((2, max_blocks), -1, dtype=torch.int32, device=dev)
    w = torch.empty(2, H, max_blocks * B, device=dev)      # 2^32 entries
    g = torch.Generator().manual_seed(3)
    ids = [16_499, 3, 16_450]
    codes = torch.randint(-127, 128, (3, H, B, D), generator=g, dtype=torch.int8)
    k8[ids] = codes.to(dev)
    ks[ids] = 2.0 ** -5
    table[1, :3] = i32(ids)
    prior = torch.rand(H, 192, generator=g)
    w[1, :, :192] = prior.to(dev)
    for m in (1, 3):
        q = torch.randn(m, hq, D, generator=g).to(torch.bfloat16)
        small = torch.zeros(3, H, B, D, dtype=torch.float64)
        small[:] = codes.double() * 2.0 ** -5
        want, rel = ref.weigh(q.double(), [0, m], [170], [0], [[0, 1, 2]], small, w[1:, :, :192].double().cpu(), None, D ** -0.5)
        kvt_block_weigh(q.to(dev), k8, ks, table, i32([170]), w, None if m == 1 else i32([0, m]), i32([1]))
        ref.weigh_close(w[1:, :, :192], want, rel)


# ------------------------------------------------------------------------------------------------------- keep and evict
def make_weights(n, kind, rng):
    if kind == "equal":
        return [1.0] * n
    if kind == "few":
        return [rng.choice([0.0, -0.0, 0.5, 1.0]) for _ in range(n)]
    if kind == "odd":
        return [rng.choice([math.nan, math.inf, -math.inf, -1.0, 0.0, 1e-45, 3.0, rng.random()]) for _ in range(n)]
    if kind == "rising":
        return [float(i) for i in range(n)]
    return [math.exp(rng.gauss(0, 3)) for _ in range(n)]


KEEP = [
    # lens, budget, recent, sinks, H
    ([5, 16, 17, 40], 16, 4, 2, 1),
    ([64, 65, 128, 1000], 64, 16, 4, 2),
    ([64, 65, 128, 1000], 64, 60, 4, 2),
    ([1, 0, 2], 1, 0, 0, 1),
    ([2047, 2049, 1025], 1024, 0, 0, 2),
    ([5000], 4096, 1000, 4, 3),
    ([40_000, 33_000], 16_384, 300, 4, 1),
    ([70_001, 32_769, 9000, 300], 301, 100, 4, 2),
    ([1_100_000], 5001, 0, 0, 1),
]


@pytest.mark.parametrize("kind", ["normal", "equal", "few", "odd", "rising"])
@pytest.mark.parametrize("lens,budget,recent,sinks,H", KEEP)
@pytest.mark.parametrize("moved", [False, True])
def test_keep(kvt_pkg, kind, lens, budget, recent, sinks, H, moved):
    from kvtier.block_evict import kvt_block_keep
    rng = random.Random(budget + H)
    n, width = len(lens), max(lens) + 13
    rows = rng.sample(range(n + 2), n)
    w = torch.zeros(n + 2, H, width)
    pos = torch.zeros(n + 2, H, width, dtype=torch.int32)
    held, evicted, want = [0] * (n + 2), [0] * (n + 2), []
    for j, r in enumerate(rows):
        if moved and lens[j]:
            held[r], evicted[r] = rng.randint(0, lens[j]), rng.randint(1, 500)
        per = []
        for h in range(H):
            x = make_weights(lens[j], kind, rng)
            w[r, h, :lens[j]] = torch.tensor(x)
            at = rng.sample(range(held[r] + evicted[r]), held[r])
            pos[r, h, :held[r]] = torch.tensor(at, dtype=torch.int32)
            per.append(ref.keep(w[r, h].tolist(), lens[j], budget, recent, sinks, pos[r, h].tolist() if moved else None,
                                held[r], evicted[r]))
        want.append(per)
    more = dict(pos=pos.to(dev), held=i32(held), evicted=i32(evicted)) if moved else {}
    ws = {}
    for _ in range(2):
        got = kvt_block_keep(w.to(dev), i32(lens), budget, i32(rows), recent, sinks, workspace=ws, **more)
        assert torch.equal(got.cpu(), torch.tensor(want, dtype=torch.int32).view(n, H, budget))


def test_keep_rows_and_strides(kvt_pkg):
    """Rows that are not there keep nothing; weights and pos as slices; more entries in kv_lens than the tensors have."""
    from kvtier.block_evict import kvt_block_keep
    w = torch.rand(3, 2, 4, 100, generator=torch.Generator().manual_seed(1))
    x = w.to(dev)[:, 1, :3]
    got = kvt_block_keep(x, i32([90, 50, 200, 60]), 32, i32([2, -1, 0, 7])).cpu()
    assert (got[1] == -1).all() and (got[3] == -1).all()
    for j, (r, n) in enumerate([(2, 90), (None, 0), (0, 100)]):
        for h in range(3):
            if r is not None:
                assert got[j, h].tolist() == ref.keep(w[r, 1, h].tolist(), n, 32, 0, 0)


def test_keep_of_many_pairs(kvt_pkg):
    """2^18 pairs of 16,130 entries each: 64 workgroups for each of them would be 2^32 threads.  Few are over the budget,
    one of them the last pair."""
    from kvtier.block_evict import kvt_block_keep
    n, budget, width = 1 << 18, 16_130, 32_800
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("57 GB of sources and workspace")
    g = torch.Generator().manual_seed(1)
    w = torch.randint(0, 5000, (1, 1, width), generator=g).float()
    lens = torch.full((n,), 7, dtype=torch.int32, device=dev)
    long = {0: 32_790, 70_000: 32_769, 131_072: 20_000, n - 1: 32_800}
    for j, x in long.items():
        lens[j] = x
    src = kvt_block_keep(w.to(dev), lens, budget, torch.zeros(n, dtype=torch.int32, device=dev), 100, 4)
    for j, x in long.items():
        assert src[j, 0].tolist() == ref.keep(w[0, 0].tolist(), x, budget, 100, 4)
    short = torch.full((budget,), -1, dtype=torch.int32, device=dev)
    short[:7] = torch.arange(7, device=dev)
    at = torch.arange(1, n - 1, 997, device=dev)
    assert (src[at[lens[at] == 7], 0] == short).all()


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("H,B,D", [(1, 16, 64), (2, 32, 128), (2, 64, 256), (3, 64, 64), (1, 16, 256), (2, 64, 128)])
@pytest.mark.parametrize("budget_blocks,share", [(1, 0.5), (4, 0.1), (5, 0.9)])
def test_evict(kvt_pkg, kv, H, B, D, budget_blocks, share):
    """Codes, scales, weights and positions to the bit; requests at and below the budget, and other blocks, untouched."""
    from kvtier.block_evict import kvt_block_evict
    budget = budget_blocks * B
    rng = random.Random(budget + D)
    lens = [budget + 1, budget, 3, budget + B, 3 * budget + 7, budget + 2 * B + 1]
    max_blocks = -(-max(lens) // B) + 1
    sides, table, rows = pool(lens, max_blocks, len(lens) + 1, H, B, D, kv, budget, wide=20.0)
    for (_, s) in sides:                                   # scales far apart, some smaller than the rows need
        s *= torch.exp2(torch.randint(-6, 7, s.shape, generator=torch.Generator().manual_seed(2)).float())
    n_rows, width = len(table), max_blocks * B + 5
    held = [rng.randint(0, budget) for _ in range(n_rows)]
    evicted = [rng.randint(0, 1000) for _ in range(n_rows)]
    pos = torch.tensor([rng.randint(0, 5000) for _ in range(n_rows * H * width)], dtype=torch.int32).view(n_rows, H, width)
    weights = torch.rand(n_rows, H, width, generator=torch.Generator().manual_seed(3))
    src = []
    for n in lens:
        per = []
        for _ in range(H):
            s = list(range(budget))
            free = sorted(rng.sample(range(budget), min(max(1, int(share * budget)), max(n - budget, 0))))
            for e, c in zip(free, sorted(rng.sample(range(budget, max(n, budget)), len(free)))):
                s[e] = c
            per.append(s)
        src.append(per)
    codes = [bref.values(c) for c, _ in sides]
    scales = [s.double() for _, s in sides]
    want_w, want_pos = weights.clone(), pos.clone()
    ref.evict(src, lens, rows, table, codes, scales, kv, want_w, want_pos, held, evicted)
    (k8, ks), (v8, vs) = [(c.clone().to(dev), s.to(dev)) for c, s in sides]
    w, p = weights.to(dev), pos.to(dev)
    args = (i32(src), i32(lens), k8, v8, ks, vs, i32(table), i32(rows), w, p, i32(held), i32(evicted))
    for _ in range(2):
        kvt_block_evict(*args)
        for got, want in ((k8, codes[0]), (v8, codes[1])):
            assert torch.equal(bref.values(got.cpu()), want)
        assert torch.equal(ks.cpu().double(), scales[0]) and torch.equal(vs.cpu().double(), scales[1])
        assert torch.equal(w.cpu(), want_w) and torch.equal(p.cpu(), want_pos)


def test_evict_specials(kvt_pkg):
    """NaN codes, blocks of zeros, scales that are not finite, sources that are none, blocks that are not there."""
    from kvtier.block_evict import kvt_block_evict
    B, H, D, budget = 16, 1, 64, 64
    lens = [120, 100]
    sides, table, rows = pool(lens, 8, 2, H, B, D, "fp8", 3)
    raw = [c.view(torch.int8).clone() for c, _ in sides]
    a, b = table[rows[0]], table[rows[1]]
    raw[0][a[5], 0, 3, 9] = 0x7F                    # a NaN that moves
    raw[1][a[0]] = 0
    raw[1][a[6]] = 0
    raw[1][a[3]] = 0                                # zeros to zeros: the smallest scale
    sides[0][1][a[7], 0] = math.inf                 # a moved row's scale
    sides[1][1][b[1], 0] = math.nan                 # a staying row's scale
    b[6] = -1
    src = [[list(range(budget))], [list(range(budget))]]
    src[0][0][5], src[0][0][20], src[0][0][21] = 5 * B + 3, 6 * B + 1, 7 * B + 2
    src[0][0][33], src[0][0][34], src[0][0][35] = 200, -7, 50     # behind the length, nothing, below the budget
    src[0][0][49] = 6 * B + 2
    for e in range(B):
        src[0][0][e] = 6 * B + e if e != 5 else 5 * B + 3
    src[0][0][36] = 120
    src[1][0][17], src[1][0][40] = 70, 6 * B        # (the second from a block that is not there)
    codes = [bref.values(c.view(torch.float8_e4m3fn)) for c in raw]
    scales = [s.double() for _, s in sides]
    ref.evict(src, lens, rows, table, codes, scales, "fp8")
    k8, v8 = (c.view(torch.float8_e4m3fn).to(dev) for c in raw)
    ks, vs = (s.to(dev) for _, s in sides)
    kvt_block_evict(i32(src), i32(lens), k8, v8, ks, vs, i32(table), i32(rows))
    for got, want in ((bref.values(k8.cpu()), codes[0]), (bref.values(v8.cpu()), codes[1]), (ks.cpu().double(), scales[0]),
                      (vs.cpu().double(), scales[1])):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, 1234.0), torch.nan_to_num(want, 1234.0))


def test_evict_alone(kvt_pkg):
    """Codes alone, without weights and positions; table rows that are not there; far blocks (offsets past 2^31 bytes)."""
    from kvtier.block_evict import kvt_block_evict
    H, B, D, nb = 8, 64, 256, 16_500
    k8, v8 = (torch.zeros(nb, H, B, D, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.ones(nb, H, device=dev) for _ in range(2))
    g = torch.Generator().manual_seed(3)
    ids = [16_499, 3, 16_450]
    small = [torch.randint(-127, 128, (3, H, B, D), generator=g, dtype=torch.int8) for _ in range(2)]
    scale = [torch.exp2(torch.randint(-3, 4, (3, H), generator=g).float()) for _ in range(2)]
    for x, z, c, s in ((k8, ks, small[0], scale[0]), (v8, vs, small[1], scale[1])):
        x[ids], z[ids] = c.to(dev), s.to(dev)
    src = [[list(range(B)) for _ in range(H)] for _ in range(3)]
    for h in range(H):
        src[1][h][5 + h], src[1][h][20] = 64 + h, 150
    codes, scales = [c.double() for c in small], [s.double() for s in scale]
    ref.evict(src, [170] * 3, [9, 0, -1], [[0, 1, 2]], codes, scales, "int8")
    kvt_block_evict(i32(src), i32([170] * 3), k8, v8, ks, vs, i32([ids]), i32([9, 0, -1]))
    for x, z, c, s in ((k8, ks, codes[0], scales[0]), (v8, vs, codes[1], scales[1])):
        assert torch.equal(x[ids].cpu().double(), c) and torch.equal(z[ids].cpu().double(), s)
    assert not k8[:3].any() and not v8[4:16_450].any() and (ks[4:16_450] == 1).all()


# ------------------------------------------------------------------------------------------------------------------ trim
@pytest.mark.parametrize("n,B,budget,longest", [(1, 64, 64, 65), (3, 16, 32, 300), (64, 64, 256, 400), (1024, 16, 16, 90), (5, 32, 64, 60),
                                                (7, 16, 32, 20_000), (200, 16, 48, 900), (2, 64, 64, 300_000)])
@pytest.mark.parametrize("commit", [True, False])
@pytest.mark.parametrize("bad", [False, True])
def test_trim(kvt_pkg, n, B, budget, longest, commit, bad):
    from kvtier.block_evict import kvt_block_trim
    rng = random.Random(n + B)
    n_rows, max_blocks = n + 4, -(-longest // B) + 1
    seqs = rng.sample(range(n_rows), n)
    lens = [0] * n_rows
    for s in range(n_rows):
        lens[s] = rng.choice([longest, budget, budget + 1, rng.randint(0, longest)])
    used = sum(-(-x // B) for x in lens)
    free = list(range(used + 9))
    rng.shuffle(free)
    table, head = [[-1] * max_blocks for _ in range(n_rows)], 0
    for s in range(n_rows):
        for lp in range(min(-(-lens[s] // B), max_blocks)):
            table[s][lp] = free[head]
            head += 1
    held, evicted = [0] * n_rows, [rng.randint(0, 50) for _ in range(n_rows)]
    if bad:
        seqs[0] = n_rows if n > 1 else -3
        if n > 2:
            seqs[2] = seqs[1]
        table[seqs[-1] if 0 <= seqs[-1] < n_rows else 0][max_blocks - 2] = -1
        head = min(head, 3)
    t = dict(seqs=i32(seqs), seq_lens=i32(lens), block_table=i32(table), free_list=i32(free), free_head=i32([head]),
             held=i32(held), evicted=i32(evicted), status=i32([0]))
    got = kvt_block_trim(budget=budget, block=B, commit=commit, **t)
    kv, nxt, status = ref.trim(seqs, lens, table, free, head, budget, B, held, evicted, len(free), commit)
    assert got.kv_lens.tolist() == kv and got.next_head.tolist() == [nxt] and t["status"].tolist() == [status]
    assert t["free_list"].tolist() == free and t["block_table"].tolist() == table
    assert t["seq_lens"].tolist() == lens and t["held"].tolist() == held and t["evicted"].tolist() == evicted
    assert t["free_head"].tolist() == [nxt if commit else head]


def test_trim_without_positions(kvt_pkg):
    from kvtier.block_evict import kvt_block_trim
    table, lens, free, head = i32([[3, 1, 0, 2]]), i32([100]), i32([3, 1, 0, 2, 4]), i32([4])
    got = kvt_block_trim(i32([0]), lens, table, free, head, 32, block=32)
    assert got.kv_lens.tolist() == [32] and head.tolist() == [1] and free.tolist() == [3, 1, 0, 2, 4]
    assert table.tolist() == [[3, -1, -1, -1]] and lens.tolist() == [32]
    got = kvt_block_trim(i32([]), lens, table, free, head, 32, block=32)
    assert got.kv_lens.numel() == 0 and got.next_head.tolist() == [1]


# -------------------------------------------------------------------------------------------------------------- together
def test_conversations_within_a_budget(kvt_pkg):
    """Prompts, steps, evictions: rotated keys are written, weighed and evicted; the cache's entries, positions and weights
    stay those of a plain record of the conversation, and decode attends to exactly the entries that are left."""
    from kvtier.block_kv import BlockKVCache
    from kvtier.rope import rotary_frequencies
    L, H, hq, D, B, budget, recent, sinks = 2, 2, 6, 64, 16, 64, 20, 3
    cache = BlockKVCache(L, H, D, 64, 4, 16, dev, block=B, evicting=True, seed=3)
    inv, scale = rotary_frequencies(32, 1e4)
    g = torch.Generator().manual_seed(9)
    a, b, c = cache.add_seq(), cache.add_seq(), cache.add_seq()
    cache.release(b)                                           # (rows out of order)
    seqs = [c, a]
    every = {s: torch.empty(L, 0, H, D, dtype=torch.float64) for s in seqs}     # rotated keys of all tokens
    # what each head holds: positions and weights, in the order of the cache's entries
    held = {s: [[[] for _ in range(H)] for _ in range(L)] for s in seqs}
    weight = {s: [[[] for _ in range(H)] for _ in range(L)] for s in seqs}
    most = torch.zeros(L, H, dtype=torch.float64)              # the largest scale of a head so far
    for step, counts in enumerate([[90, 33], [1, 1], [1, 50], [1, 1], [40, 1], [1, 1], [1, 1], [17, 1]]):
        total = sum(counts)
        q0 = torch.randn(total, hq, D, generator=g).to(torch.bfloat16)
        k0, v0 = (torch.randn(total, H, D, generator=g).to(torch.bfloat16) for _ in range(2))
        plan = cache.plan(seqs, counts)
        cu = prefix(counts)
        at = {s: list(range(every[s].shape[1], every[s].shape[1] + n)) for s, n in zip(seqs, counts)}
        new = {}
        for layer in range(L):
            q, k = cache.rotate(plan, q0.to(dev), (k0 * (layer + 1)).to(dev), inv, scale)
            out, size, turn = ref.rope((k0 * (layer + 1)).double(), [p for s in seqs for p in at[s]], inv.cpu(), scale, False)
            assert ((k.double().cpu() - out).abs() <= ref.rope_bound(out, size, turn, torch.bfloat16)).all()
            cache.append(layer, plan, k, v0.to(dev))
            new[layer] = k.double().cpu()
            if all(n == 1 for n in counts):
                o = cache.decode(layer, plan, q)
                cache.weigh_decode(layer, plan, q)
            else:
                o = cache.prefill(layer, plan, q)
                cache.weigh_prefill(layer, plan, q)
            table = cache.block_table.cpu().tolist()
            kk = bref.values(cache.k8[layer].cpu()) * cache.ks[layer].cpu().double()[..., None, None]
            vv = bref.values(cache.v8[layer].cpu()) * cache.vs[layer].cpu().double()[..., None, None]
            lens = plan.kv_lens.tolist()
            want, big, reach, tot = bref.attention(q.double().cpu(), cu, lens, seqs, table, kk, vv, True, D ** -0.5)
            bref.close(o, want, big, reach, tot, D)
            prior = torch.zeros(4, H, 256, dtype=torch.float64)
            for s in seqs:
                for h in range(H):
                    prior[s, h, :len(weight[s][layer][h])] = torch.tensor(weight[s][layer][h], dtype=torch.float64)
            want, rel = ref.weigh(q.double().cpu(), cu, lens, seqs, table, kk, prior, None, D ** -0.5)
            for i, s in enumerate(seqs):
                ref.weigh_close(cache.weights[layer, s, :, :lens[i]], want[s, :, :lens[i]], rel[s, :, :lens[i]])
                for h in range(H):
                    held[s][layer][h] += at[s]
                    weight[s][layer][h] = cache.weights[layer, s, h, :lens[i]].cpu().tolist()
                    # the cache's rows are the conversation's keys at those positions, within the codes' rounding
                    blocks = [table[s][e // B] for e in range(lens[i])]
                    rows = kk[torch.tensor(blocks), h, torch.arange(lens[i]) % B]
                    past = torch.cat((every[s][layer], new[layer][cu[i]:cu[i + 1]]))[:, h]
                    x = past[torch.tensor(held[s][layer][h])]
                    # half a step of e4m3; subnormals: half a step, 2^-10, of every scale that the row had on its way
                    # up by powers of two
                    most[layer, h] = max(most[layer, h], float(cache.ks[layer].cpu()[torch.tensor(blocks), h].max()))
                    assert ((rows - x).abs() <= x.abs() * 2.0 ** -4 + most[layer, h] * 2.0 ** -9).all()
        for i, s in enumerate(seqs):
            every[s] = torch.cat((every[s], torch.stack([new[layer][cu[i]:cu[i + 1]] for layer in range(L)])), 1)
        if step % 2 == 0 or step == 5:
            before = [int(x) for x in cache.seq_lens]
            cache.evict(seqs, budget, recent, sinks)
            cache.check()
            for s in seqs:
                n = before[s]
                for layer in range(L):
                    for h in range(H):
                        p, w = held[s][layer][h], weight[s][layer][h]
                        src = ref.keep(w, n, budget, recent, sinks, p, n, every[s].shape[1] - n)
                        if n > budget:
                            held[s][layer][h] = [p[e] for e in src]
                            weight[s][layer][h] = [w[e] for e in src]
                            got = cache.pos[layer, s, h, :budget].tolist()
                            assert got == held[s][layer][h]
                            assert cache.weights[layer, s, h, :budget].tolist() == weight[s][layer][h]
                m = min(n, budget)
                assert int(cache.seq_lens[s]) == m and int(cache.evicted[s]) == every[s].shape[1] - m
                assert [x >= 0 for x in cache.block_table[s].tolist()] == [lp < -(-m // B) for lp in range(16)]
            head = int(cache.free_head)
            used = [x for row in cache.block_table.tolist() for x in row if x >= 0]
            assert len(used) == head and sorted(used + cache.free_list[head:].tolist()) == list(range(64))
    for s in seqs:
        cache.release(s)
    assert int(cache.free_head) == 0 and not cache.evicted.any() and not cache.held.any()


def test_graph_of_a_step_with_eviction(kvt_pkg):
    """A decode step with rotation, write, attention, weighing and eviction in one graph, replayed with eager work between,
    against the same steps run eagerly on a cache of its own."""
    from kvtier.block_kv import BlockKVCache
    from kvtier.rope import rotary_frequencies
    L, H, hq, D, B, budget = 1, 2, 8, 64, 16, 48
    inv, scale = rotary_frequencies(64, 1e4)
    caches = [BlockKVCache(L, H, D, 32, 2, 8, dev, block=B, evicting=True) for _ in range(2)]
    g = torch.Generator().manual_seed(4)
    x = [torch.randn(100, n, D, generator=g).to(torch.bfloat16).to(dev) for n in (hq, H, H)]
    ones, wss = i32([1, 1]), ({}, {})
    rows = []
    for cache in caches:
        rows.append(i32([cache.add_seq(), cache.add_seq()]))
        plan = cache.plan(rows[-1], i32([50, 44]), 94)
        q, k = cache.rotate(plan, x[0][:94], x[1][:94], inv, scale)
        cache.append(0, plan, k, x[2][:94])
        cache.weigh_prefill(0, plan, q)
        cache.evict(rows[-1], budget, 8, 2)

    def step(i, q, k, v):
        c = caches[i]
        plan = c.plan(rows[i], ones, 2)
        q, k = c.rotate(plan, q, k, inv, scale)
        c.append(0, plan, k, v)
        out = c.decode(0, plan, q, workspace=wss[i])
        c.weigh_decode(0, plan, q, workspace=wss[i])
        c.evict(rows[i], budget, 8, 2)
        return out
    bufs = [t[:2].clone() for t in x]
    for i in range(2):
        step(i, *bufs)                                        # (workspaces; the two caches stay alike)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(0, *bufs)
    for r in range(20):
        for b, t in zip(bufs, x):
            b.copy_(t[2 * r + 3:2 * r + 5])
        graph.replay()
        torch.cuda.synchronize()
        want = step(1, *bufs)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("block_table", "seq_lens", "free_list", "free_head", "held", "evicted", "status"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
        n = caches[0].seq_lens.tolist()
        for s in range(2):
            assert torch.equal(caches[0].weights[0, s, :, :n[s]], caches[1].weights[0, s, :, :n[s]])
            assert torch.equal(caches[0].pos[0, s, :, :budget], caches[1].pos[0, s, :, :budget])
        assert torch.equal(caches[0].k8[0].view(torch.int8), caches[1].k8[0].view(torch.int8))
        assert torch.equal(caches[0].ks[0], caches[1].ks[0])
    caches[0].check()


def test_streams_of_their_own(kvt_pkg):
    """Two calls at once, on two streams, with a workspace each."""
    from kvtier.block_evict import kvt_block_keep, kvt_block_weigh
    lens, H, B, D, hq = [1500, 900], 2, 32, 128, 8
    sides, table, rows = pool(lens, 50, 2, H, B, D, "fp8", 3)
    g = torch.Generator().manual_seed(6)
    k8, ks = sides[0][0].to(dev), sides[0][1].to(dev)
    qs = [torch.randn(2, hq, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)]
    t, n, r = i32(table), i32(lens), i32(rows)
    streams, done = [torch.cuda.Stream() for _ in range(2)], []
    want = []
    for q in qs:
        w = torch.zeros(2, H, 1600, device=dev)
        kvt_block_weigh(q, k8, ks, t, n, w, seqs=r)
        want.append((w, kvt_block_keep(w, n, 256, r, 20, 4)))
    torch.cuda.synchronize()
    for _ in range(10):
        done = []
        for q, s in zip(qs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                w = torch.zeros(2, H, 1600, device=dev)
                kvt_block_weigh(q, k8, ks, t, n, w, seqs=r)
                done.append((w, kvt_block_keep(w, n, 256, r, 20, 4)))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(done, want):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_streams_with_a_workspace_each(kvt_pkg):
    """Calls of two streams at once that use their workspaces: chunks in splits, single queries, a choice of more than
    32,768 entries; over and over into the same buffers."""
    from kvtier.block_evict import kvt_block_keep, kvt_block_weigh
    lens, H, B, D, hq, width = [36_000, 900], 1, 64, 64, 8, 40_000
    sides, table, rows = pool(lens, width // B, 2, H, B, D, "fp8", 3)
    g = torch.Generator().manual_seed(6)
    k8, ks = sides[0][0].to(dev), sides[0][1].to(dev)
    t, n, r, cu = i32(table), i32(lens), i32(rows), i32([0, 30, 41])
    qs = [torch.randn(41, hq, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)]

    def calls(q, ws):
        w = torch.zeros(2, H, width, device=dev)
        kvt_block_weigh(q, k8, ks, t, n, w, cu, r, workspace=ws)
        kvt_block_weigh(q[:2], k8, ks, t, n, w, seqs=r, workspace=ws)
        return w, kvt_block_keep(w, n, 2048, r, 20, 4, workspace=ws)
    want = [calls(q, {}) for q in qs]
    torch.cuda.synchronize()
    assert not torch.equal(want[0][1], want[1][1])
    streams, wss = [torch.cuda.Stream() for _ in range(2)], [{}, {}]
    for _ in range(10):
        done = []
        for q, s, ws in zip(qs, streams, wss):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                done.append(calls(q, ws))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(done, want):
            assert torch.equal(a, c) and torch.equal(b, d)
    # (the caching allocator knows no other stream's use: the workspaces are each its own)
    assert all(k in ws for ws in wss for k in (("weigh", 0), ("keep", 0)))
