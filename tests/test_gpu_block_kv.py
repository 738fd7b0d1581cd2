"""8-bit block cache on the GPU: plan, quantizing write, decode and chunk attention against plain 64-bit forms
(tests/block_testutil.py), and the four together as a serving step uses them."""
import random

import pytest
import torch

import block_testutil as ref

pytestmark = pytest.mark.gpu
dev = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prefix(x):
    out = [0]
    for y in x:
        out.append(out[-1] + y)
    return out


# ------------------------------------------------------------------------------------------------------------- plan
def _plan_case(n, B, lens, counts, max_blocks, rows, pool, seed, rtt_cols=0):
    rng = random.Random(seed)
    free = list(range(pool))
    rng.shuffle(free)
    table = [[-1] * max_blocks for _ in range(rows)]
    seqs = rng.sample(range(rows), n)
    seq_lens = [0] * rows
    head = 0
    for s, L in zip(seqs, lens):
        seq_lens[s] = L
        for lp in range(-(-L // B)):
            table[s][lp] = free[head]
            head += 1
    rtt = [[7] * rtt_cols for _ in range(rows)] if rtt_cols else None
    return seqs, counts, seq_lens, table, free, head, rtt


def _run_plan(case, n_tokens, B, commit=True):
    from kvtier import block_kv
    seqs, counts, seq_lens, table, free, head, rtt = case
    d = dict(seqs=i32(seqs), counts=i32(counts), seq_lens=i32(seq_lens), block_table=i32(table), free_list=i32(free),
             free_head=i32([head]), status=i32([0]), req_to_token=None if rtt is None else i32(rtt))
    want_table, want_rtt = [list(r) for r in table], None if rtt is None else [list(r) for r in rtt]
    cu, slots, kv, nxt, status = ref.plan(seqs, counts, seq_lens, want_table, free, head, n_tokens, B, want_rtt)
    p = block_kv.kvt_block_plan(n_tokens=n_tokens, block=B, commit=commit, **d)
    assert p.cu.tolist() == cu and p.kv_lens.tolist() == kv and p.next_head.tolist() == [nxt]
    assert p.slots.tolist() == slots
    assert d["status"].tolist() == [status]
    assert d["block_table"].tolist() == want_table
    if rtt is not None:
        assert d["req_to_token"].tolist() == want_rtt
    after = list(seq_lens)
    if commit:
        for j, s in enumerate(seqs):
            if cu[j + 1] > cu[j]:
                after[s] = kv[j]
    assert d["seq_lens"].tolist() == after and d["free_head"].tolist() == [nxt if commit else head]
    return d, p


@pytest.mark.parametrize("n,B,longest,most,rtt", [(1, 64, 0, 1, 0), (1, 16, 63, 5, 80), (3, 32, 64, 1, 0), (64, 64, 700, 1, 0),
                                                  (65, 16, 200, 130, 333), (500, 64, 300, 40, 0), (1024, 16, 50, 9, 0)])
@pytest.mark.parametrize("commit", [True, False])
def test_plan(kvt_pkg, n, B, longest, most, rtt, commit):
    rng = random.Random(n + B)
    lens = [rng.randint(0, longest) for _ in range(n)]
    counts = [rng.randint(0, most) if most > 1 else 1 for _ in range(n)]
    case = _plan_case(n, B, lens, counts, (longest + most) // B + 2, n + 5, sum(-(-(a + b) // B) for a, b in zip(lens, counts)) + 2,
                      n, rtt)
    _run_plan(case, sum(counts) + 3, B, commit)


def test_plan_keeps_the_same_plan_until_committed(kvt_pkg):
    from kvtier import block_kv
    case = _plan_case(5, 16, [3, 16, 0, 47, 31], [20, 1, 5, 1, 40], 8, 9, 40, 1)
    d, p = _run_plan(case, 67, 16, commit=False)
    q = block_kv.kvt_block_plan(n_tokens=67, block=16, commit=True, **d)
    assert torch.equal(p.slots, q.slots) and torch.equal(p.kv_lens, q.kv_lens)
    assert d["free_head"].tolist() == q.next_head.tolist()


@pytest.mark.parametrize("short", ["pool", "row", "tokens"])
def test_plan_that_does_not_fit(kvt_pkg, short):
    lens, counts = [10, 64, 0, 100], [60, 9000 if short != "row" else 700, 33, 1]
    pool = 12 if short == "pool" else 300
    case = _plan_case(4, 64, lens, counts, 3 if short == "row" else 160, 6, pool, 2)
    _run_plan(case, sum(counts) - (40 if short == "tokens" else 0), 64)


def test_plan_rows_that_are_wrong_or_twice(kvt_pkg):
    """Rows out of range and rows listed again append nothing; more than 4,096 rows, so that stamps collide."""
    rows = 9000
    seqs = [5, -1, 4101, 5, 9000, 8197, 2 ** 30, 4101, 7]
    case = (seqs, [3, 4, 5, 6, 7, 8, 9, 10, 2], [0] * rows, [[-1] * 2 for _ in range(rows)], list(range(50)), 0, None)
    _run_plan(case, 60, 16)


def test_plan_of_nothing(kvt_pkg):
    _run_plan(_plan_case(3, 64, [5, 0, 64], [0, 0, 0], 2, 3, 4, 3), 0, 64)


@pytest.mark.parametrize("counts,n_tokens", [([100], 60), ([0, 100, 0], 60), ([0, 0, 7], 0), ([2 ** 31 - 1] * 3, 50),
                                             ([50, 0, 1], 50), ([30, -5, 20], 50)])
def test_plan_of_more_tokens_than_it_is_given(kvt_pkg, counts, n_tokens):
    """One request alone over n_tokens, none of the others with a token, no room at all; and counts that just fit."""
    n = len(counts)
    _run_plan(_plan_case(n, 16, [5, 0, 16][:n], counts, 30, 4, 40, 5), n_tokens, 16)


def test_plan_behind_a_full_row(kvt_pkg):
    """A row that an earlier step ran over is reported where tokens are appended to it, not where none are."""
    for counts, lens in (([0, 2], [70, 5]), ([1, 2], [70, 5]), ([0, 0], [64, 64])):
        case = _plan_case(2, 16, [min(n, 64) for n in lens], counts, 4, 3, 20, 6)
        for s, n in zip(case[0], lens):
            case[2][s] = n
        _run_plan(case, 4, 16)


def test_a_step_of_no_requests(kvt_pkg):
    """An idle step: an empty plan, and calls over it that do nothing."""
    from kvtier import block_kv
    c = block_kv.BlockKVCache(1, 2, 64, n_blocks=4, max_seqs=2, max_blocks=2, block=16)
    c.plan([c.add_seq()], [20])
    none = i32([])
    for n_tokens in (0, 3):
        before = [t.clone() for t in (c.block_table, c.seq_lens, c.free_head)]
        p = c.plan(none, none, n_tokens=n_tokens)
        assert p.cu.tolist() == [0] and p.slots.tolist() == [-1] * n_tokens and p.kv_lens.tolist() == [] and p.next_head.tolist() == [2]
        x = torch.randn(n_tokens, 2, 64, device=dev)
        c.append(0, p, x, x)
        assert c.decode(0, p, x[:0].half()).shape == (0, 2, 64)
        assert c.prefill(0, p, x.half()).shape == (n_tokens, 2, 64)
        assert all(torch.equal(a, b) for a, b in zip(before, (c.block_table, c.seq_lens, c.free_head)))
        c.check()
    p = c.plan([], [])
    assert p.cu.tolist() == [0] and p.slots.numel() == 0


# ------------------------------------------------------------------------------------------------------------ store
def _tables(kv_lens, B, extra, seed):
    rng = random.Random(seed)
    total = sum(-(-L // B) for L in kv_lens) + extra
    ids = list(range(total))
    rng.shuffle(ids)
    width = max(1, max(-(-L // B) for L in kv_lens)) + 1
    table = []
    for L in kv_lens:
        n = -(-L // B)
        table.append([ids.pop() for _ in range(n)] + [-1] * (width - n))
    return table, total


def _check_store(kv, dt, H, D, B, old, new, seed, x=None, table=None, mutate=None):
    from kvtier import block_kv
    kv_lens = [a + b for a, b in zip(old, new)]
    cu = prefix(new)
    tab, nb = _tables(kv_lens, B, 2, seed)
    table = table or tab
    g = torch.Generator().manual_seed(seed)
    raw = torch.randint(0, 256, (2, nb, H, B, D), dtype=torch.uint8, generator=g)
    if kv == "fp8":
        raw[(raw & 0x7F) == 0x7F] = 1                  # (no NaN among the codes held)
    else:
        raw[raw == 0x80] = 1
    codes = [raw[i].view(torch.int8).view(ref.CODE[kv]) for i in range(2)]
    scale = [2.0 ** torch.randint(-9, -5, (nb, H), generator=g).float() for _ in range(2)]
    if x is None:
        x = [(torch.randn(cu[-1], H, D, generator=g) * 2.0 ** torch.randint(-3, 4, (cu[-1], 1, 1), generator=g)).to(dt)
             for _ in range(2)]
    dx = [mutate(t.to(dev)) if mutate else t.to(dev) for t in x]
    dc, ds = [c.to(dev) for c in codes], [s.to(dev) for s in scale]
    block_kv.kvt_block_store(dx[0], dx[1], i32(cu), i32(kv_lens), dc[0], dc[1], ds[0], ds[1], i32(table))
    for i in range(2):
        want, ws = ref.values(codes[i]), scale[i].double()
        ref.store(x[i].double(), cu, kv_lens, range(len(old)), table, want, ws, kv)
        assert torch.equal(ds[i].cpu().double(), ws), "scales"
        got = ref.values(dc[i].cpu())
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), "codes"
        same = want == ref.values(codes[i])           # what is not written keeps its bytes
        rest = torch.ones_like(same)
        for r, row in enumerate(table):
            for lp in range(old[r] // B, -(-kv_lens[r] // B)):
                if lp < len(row) and 0 <= row[lp] < nb:
                    rest[row[lp], :, :min(B, kv_lens[r] - lp * B)] = False
        assert torch.equal(dc[i].cpu().view(torch.int8)[rest], codes[i].view(torch.int8)[rest])


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,D,B", [(2, 256, 64), (1, 256, 16), (3, 128, 32), (2, 128, 16), (5, 64, 64), (1, 64, 16)])
def test_store(kvt_pkg, kv, dt, H, D, B):
    _check_store(kv, dt, H, D, B, [0, 1, B - 1, B, 2 * B + 5, 7, 3], [1, 1, 1, 1, 3 * B + 2, B - 7, 0], seed=D + B + H)


@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_store_many_requests(kvt_pkg, kv):
    """More requests than one search round covers, tokens of one to many blocks."""
    rng = random.Random(5)
    old = [rng.randint(0, 90) for _ in range(300)]
    new = [rng.choice([0, 1, 1, 1, 2, 17, 64, 131]) for _ in range(300)]
    _check_store(kv, torch.bfloat16, 1, 64, 16, old, new, seed=9)


@pytest.mark.parametrize("kv,dt", [("fp8", torch.bfloat16), ("int8", torch.float16), ("fp8", torch.float32), ("int8", torch.bfloat16)])
@pytest.mark.parametrize("H,D,B", [(2, 256, 64), (5, 128, 16), (3, 64, 32)])
def test_store_few_rows_on_average(kvt_pkg, kv, dt, H, D, B):
    """Decode steps among which one request writes a prompt over several blocks, with values that are not finite."""
    old, new = [5, 0, 63, 64, 100, 17, 1, 31] * 12, [1, 0, 2, 1, 1, 1, 3, 1] * 12
    new[20] = 150
    x = torch.randn(2, sum(new), H, D, generator=torch.Generator().manual_seed(B)).to(dt)
    first = sum(new[:20])
    x[0, first + 3, 1, 5], x[1, first + 70, 0, 0], x[0, first + 149, H - 1, D - 1] = float("inf"), float("nan"), -float("inf")
    x[0, 0, 0, 0], x[1, -1, -1, -1] = float("nan"), float("inf")
    _check_store(kv, dt, H, D, B, old, new, seed=21, x=x)


@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_store_special_values(kvt_pkg, kv):
    """Infinities, NaN, zeros, the largest and the smallest values, ties: each in rows of its own block."""
    D, B = 64, 16
    rows = torch.zeros(7 * B, 1, D)
    g = torch.Generator().manual_seed(1)
    rows[0:B] = torch.randn(B, 1, D, generator=g)
    rows[3, 0, 5], rows[4, 0, 6], rows[5, 0, 7] = float("inf"), -float("inf"), float("nan")
    rows[2 * B:3 * B] = 3.3e38 * torch.rand(B, 1, D, generator=g)
    rows[3 * B:4 * B] = 1e-38 * torch.randn(B, 1, D, generator=g)
    rows[4 * B:5 * B] = (torch.randint(-64, 65, (B, 1, D), generator=g) + 0.5) * (1 if kv == "int8" else 4)
    rows[5 * B:6 * B] = float("nan")
    rows[6 * B:7 * B] = 127.0 if kv == "int8" else 448.0
    _check_store(kv, torch.float32, 1, D, B, [0], [7 * B], seed=3, x=[rows, -rows.flip(0)])


def test_store_growth_is_exact_for_e4m3(kvt_pkg):
    """Tokens one at a time, each twice the last: every growth of the scale is a power of two, so the codes of a block keep
    the values of a single write with the final scale, down to the subnormals."""
    from kvtier import block_kv
    D, B = 64, 16
    g = torch.Generator().manual_seed(4)
    x = torch.randn(B, 2, D, generator=g) * 2.0 ** torch.arange(B)[:, None, None]
    one = block_kv.BlockKVCache(1, 2, D, 1, 1, 1, block=B)
    all_ = block_kv.BlockKVCache(1, 2, D, 1, 1, 1, block=B)
    for c, steps in ((one, [1] * B), (all_, [B])):
        s, t = c.add_seq(), 0
        for n in steps:
            c.append(0, c.plan([s], [n]), x[t:t + n].to(dev), x[t:t + n].to(dev))
            t += n
        c.check()
    assert torch.equal(one.ks[0], all_.ks[0])
    a, b = ref.values(one.k8[0].cpu()), ref.values(all_.k8[0].cpu())
    normal = b.abs() >= 2.0 ** -6
    assert torch.equal(a[normal], b[normal])
    assert float((a - b).abs().max()) <= 2.0 ** -9


@pytest.mark.parametrize("how", ["heads", "tokens", "odd"])
def test_store_strided_rows(kvt_pkg, how):
    def mutate(t):
        n, h, d = t.shape
        if how == "heads":
            return torch.cat([t, t], 1)[:, :h]
        if how == "tokens":
            return torch.stack([t, t], 1).reshape(2 * n, h, d)[::2]
        big = torch.zeros(n, h, d + 3, dtype=t.dtype, device=t.device)
        big[..., 3:] = t
        return big[..., 3:]
    _check_store("fp8", torch.bfloat16, 2, 128, 32, [5, 0], [70, 33], seed=6, mutate=mutate)


def test_store_table_entries_that_are_no_block(kvt_pkg):
    """Positions whose entry is -1, beyond the pool, or past the table's columns are not written; the others are."""
    table = [[0, -1, 2], [99999, 3, -7]]
    _check_store("fp8", torch.bfloat16, 2, 64, 16, [4, 0], [60, 40], seed=7, table=table)


def test_store_lengths_that_do_not_fit(kvt_pkg):
    """kv_lens shorter than the call's rows, and prefix sums that run past the rows: nothing outside is touched."""
    from kvtier import block_kv
    c = block_kv.BlockKVCache(1, 1, 64, 4, 2, 2, block=16)
    c.block_table.copy_(i32([[0, 1], [2, 3]]))
    x = torch.randn(8, 1, 64, device=dev)
    block_kv.kvt_block_store(x, x, i32([0, 8, 8]), i32([3, 5]), c.k8[0], c.v8[0], c.ks[0], c.vs[0], c.block_table)
    block_kv.kvt_block_store(x, x, i32([0, 0, 2 ** 30]), i32([0, 4]), c.k8[0], c.v8[0], c.ks[0], c.vs[0], c.block_table)
    assert int(c.k8[0].view(torch.int8).abs().max()) == 0 and float(c.ks[0].max()) == 0


# -------------------------------------------------------------------------------------------------------- attention
def _pool(kv, nb, H, B, D, g, spread=2):
    """Codes (no NaN) and scales 2^-9 .. of a pool."""
    raw = torch.randint(0, 256, (2, nb, H, B, D), dtype=torch.uint8, generator=g)
    if kv == "fp8":
        raw = torch.where((raw & 0x78) > 0x50, raw & 0xD7, raw)     # |code| < 16: scores of a few units
        scale = 2.0 ** torch.randint(-4, -4 + spread, (2, nb, H), generator=g).float()
    else:
        raw[raw == 0x80] = 1
        scale = 2.0 ** torch.randint(-7, -7 + spread, (2, nb, H), generator=g).float()
    codes = [raw[i].view(torch.int8).view(ref.CODE[kv]) for i in range(2)]
    return codes, [scale[0].clone(), scale[1].clone()]


def _check_attn(kv, qt, Hq, H, D, B, new, kv_lens, causal=True, seed=0, decode=False, out_dtype=None, splits=None,
                change=None, q=None, scale=None, workspace=None):
    """change(codes, scales, table): alters the pool before both sides see it."""
    from kvtier import block_kv
    g = torch.Generator().manual_seed(seed)
    table, nb = _tables(kv_lens, B, 2, seed)
    codes, sc = _pool(kv, nb, H, B, D, g)
    if change:
        change(codes, sc, table)
    cu = prefix(new)
    tail = 0 if decode else 3                            # rows behind the last request
    if q is None:
        q = torch.randn(cu[-1] + tail, Hq, D, generator=g).to(qt)
    val = [ref.values(codes[i]) * sc[i].double()[..., None, None] for i in range(2)]
    f = D ** -0.5 if scale is None else scale
    want = ref.attention(q.double()[:cu[-1]], cu, kv_lens, range(len(new)), table, val[0], val[1], causal and not decode, f)
    dc, ds, tab, kl = [c.to(dev) for c in codes], [s.to(dev) for s in sc], i32(table), i32(kv_lens)
    out = torch.full(q.shape, 5.0, dtype=out_dtype or qt, device=dev)
    if decode:
        got = block_kv.kvt_block_decode(q.to(dev), dc[0], dc[1], ds[0], ds[1], tab, kl, scale=scale, out=out, splits=splits,
                                        workspace=workspace)
    else:
        got = block_kv.kvt_block_prefill(q.to(dev), i32(cu), dc[0], dc[1], ds[0], ds[1], tab, kl, causal=causal,
                                         scale=scale, out=out, splits=splits, workspace=workspace)
    assert got is out
    ref.close(got[:cu[-1]], *want, D)
    assert bool((got[cu[-1]:] == 5.0).all()), "rows behind the last request"
    return got


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("qt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,D,B", [(16, 2, 256, 64), (24, 2, 256, 16), (1, 1, 256, 32), (16, 1, 128, 64), (10, 2, 128, 16),
                                      (3, 3, 128, 32), (20, 4, 64, 16), (7, 1, 64, 64)])
def test_decode(kvt_pkg, kv, qt, Hq, H, D, B):
    _check_attn(kv, qt, Hq, H, D, B, [1] * len(LENS), LENS, decode=True, seed=Hq + D + B)


@pytest.mark.parametrize("splits", [1, 2, 3, 8, 40, -1, -2, -7, -64, -500])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_decode_splits_and_output_types(kvt_pkg, splits, out_dtype):
    _check_attn("fp8", torch.bfloat16, 16, 2, 128, 32, [1] * 4, [5000, 0, 129, 1000], decode=True, splits=splits,
                out_dtype=out_dtype, seed=splits)


@pytest.mark.parametrize("shares", [None, -1, -5, -300])
def test_decode_many_requests(kvt_pkg, shares):
    """More requests than a wavefront has lanes, empty ones among them: the equal shares' line is looked up in rounds."""
    rng = random.Random(17)
    lens = [rng.choice([0, 0, 1, 5, 33, 64, 200, rng.randint(1, 700)]) for _ in range(150)]
    _check_attn("fp8", torch.float16, 4, 2, 64, 16, [1] * 150, lens, decode=True, splits=shares, seed=18)


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("Hq,H,D,B", [(16, 2, 256, 64), (12, 1, 128, 16), (3, 3, 128, 64), (10, 2, 64, 32), (16, 1, 64, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill(kvt_pkg, kv, Hq, H, D, B, causal):
    """Ragged chunks: whole prompts, chunks behind a prefix, one token, none, more queries than positions (rows that see
    nothing), lengths around the tiles; few rows (the decode kernel), then enough for query tiles."""
    for new, kv_lens in (([65, 17, 1, 0, 40, 128, 5], [65, 200, 1, 50, 23, 131, 5]), ([513, 300, 0, 1, 257], [513, 700, 9, 77, 130])):
        _check_attn(kv, torch.bfloat16 if D != 64 else torch.float16, Hq, H, D, B, new, kv_lens, causal, seed=D + Hq)


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("Hq,H,D,B", [(16, 2, 256, 16), (5, 1, 256, 64), (8, 1, 128, 32), (20, 4, 64, 64)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", [16, 128])
def test_prefill_kernels(kvt_pkg, monkeypatch, kv, Hq, H, D, B, causal, rows):
    """Both kernels over the same chunks, whatever the rule would take."""
    from kvtier import block_kv
    monkeypatch.setattr(block_kv, "_TILE_MIN", {D: 0 if rows == 128 else 10 ** 9})
    new = [65, 17, 1, 0, 40, 128, 5]
    kv_lens = [65, 200, 1, 50, 23, 131, 5]
    _check_attn(kv, torch.bfloat16 if D != 64 else torch.float16, Hq, H, D, B, new, kv_lens, causal, seed=D + Hq)


@pytest.mark.parametrize("splits", [1, 2, 7])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_splits(kvt_pkg, splits, causal):
    _check_attn("int8", torch.float16, 8, 2, 128, 64, [33, 2, 300], [900, 700, 310], causal, seed=splits, splits=splits,
                out_dtype=torch.float32)


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_long(kvt_pkg, causal):
    """Enough rows for whole query tiles, a prefix, and an odd end."""
    _check_attn("fp8", torch.bfloat16, 16, 2, 256, 64, [513, 300], [1001, 300], causal, seed=11)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_attention_ignores_what_a_request_does_not_hold(kvt_pkg, decode, kv):
    """NaN codes (e4m3), the largest codes and huge scales behind the last position, and blocks that are not there."""
    lens = [37, 200, 100]

    def change(codes, sc, table):
        for c in codes:
            raw = c.view(torch.int8)
            for row, L in zip(table, lens):
                raw[row[L // 16], :, L % 16:] = 127       # (e4m3 0x7F: NaN)
        table[1][3], table[1][12], table[2][0] = -1, 10 ** 6, -2 ** 31
        for r, row in enumerate(table):
            row[-1] = (len(codes[0]) - 1)                 # an entry behind the length: another block, with NaN
        codes[0].view(torch.int8)[-1] = codes[1].view(torch.int8)[-1] = 127
        sc[0][-1] = sc[1][-1] = float("nan")
    new = [1, 1, 1] if decode else [37, 20, 3]
    _check_attn(kv, torch.bfloat16, 8, 2, 128, 16, new, lens, decode=decode, change=change, seed=3)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_scales_far_apart(kvt_pkg, decode):
    """V scales that differ by 2^60 from block to block (and blocks of zeros, and blocks that are not there between them),
    K scales by 2^6."""
    def change(codes, sc, table):
        n, H = sc[1].shape
        for row in table:
            row[3] = row[4] = row[9] = row[11] = -1
        e = torch.tensor([[-30, 30, 0, -64, 12][(i + h) % 5] for i in range(n) for h in range(H)]).view(n, H)
        sc[1].copy_(2.0 ** e.float())
        sc[0].mul_(2.0 ** ((torch.arange(n) % 4).float()[:, None] - 3))
        codes[1].view(torch.int8)[::7] = 0
    new = [1, 1] if decode else [70, 300]
    _check_attn("fp8", torch.bfloat16, 8, 2, 128, 16, new, [700, 333], decode=decode, change=change, seed=4,
                out_dtype=torch.float32)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_scales_at_the_ends(kvt_pkg, decode):
    """V scales from 2^-64 to 2^110 in one row: finite, and as exact as the largest ones ask."""
    def change(codes, sc, table):
        n, H = sc[1].shape
        e = torch.tensor([[-64, 110, -64, 0, 30][(i + h) % 5] for i in range(n) for h in range(H)]).view(n, H)
        sc[1].copy_(2.0 ** e.float())
    new = [1, 1] if decode else [70, 300]
    _check_attn("int8", torch.float16, 8, 2, 64, 16, new, [900, 333], decode=decode, change=change, seed=6,
                out_dtype=torch.float32)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("size", [1e-6, 40.0, 3e3])
def test_attention_query_sizes(kvt_pkg, decode, size):
    """Flat and one-hot softmax; bf16 queries far outside fp16's range times a small scale."""
    g = torch.Generator().manual_seed(2)
    new = [1, 1] if decode else [50, 40]
    n = sum(new) + (0 if decode else 3)
    q = (torch.randn(n, 8, 128, generator=g) * size * 1e6).to(torch.bfloat16)
    _check_attn("fp8", torch.bfloat16, 8, 2, 128, 32, new, [260, 90], decode=decode, seed=5, q=q, scale=128 ** -0.5 * 1e-6,
                out_dtype=torch.float32)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_offsets_past_32_bits(kvt_pkg, decode):
    """A pool of more than 4 GiB per side: the last blocks are read and written like the first."""
    from kvtier import block_kv
    H, B, D, nb = 2, 64, 256, 140_000                    # 4.6e9 bytes
    k8 = torch.zeros(nb, H, B, D, dtype=torch.int8, device=dev)
    v8 = torch.zeros(nb, H, B, D, dtype=torch.int8, device=dev)
    ks, vs = torch.zeros(nb, H, device=dev), torch.zeros(nb, H, device=dev)
    ids = [nb - 1, 0, nb - 2, 131_073]
    table, L = i32([ids]), 4 * B - 3
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(2, L, H, D, device=dev, generator=g).to(torch.bfloat16)
    block_kv.kvt_block_store(x[0], x[1], i32([0, L]), i32([L]), k8, v8, ks, vs, table)
    m = 1 if decode else 40
    q = torch.randn(m, 16, D, device=dev, generator=g).to(torch.bfloat16)
    at = torch.tensor(ids, device=dev)
    kc, vc = ((c[at].cpu().double() * s[at].cpu().double()[..., None, None]) for c, s in ((k8, ks), (v8, vs)))
    step = (x[0].abs().amax() / 127 * 2).item()          # a scale is below twice the largest value's share of a code
    back = kc.permute(0, 2, 1, 3).reshape(4 * B, H, D)[:L]
    assert float((back - x[0].double().cpu()).abs().max()) <= step / 2
    want = ref.attention(q.double().cpu(), [0, m], [L], [0], [[0, 1, 2, 3]], kc, vc, not decode, D ** -0.5)
    if decode:
        got = block_kv.kvt_block_decode(q, k8, v8, ks, vs, table, i32([L]))
    else:
        got = block_kv.kvt_block_prefill(q, i32([0, m]), k8, v8, ks, vs, table, i32([L]))
    ref.close(got, *want, D)


@pytest.mark.parametrize("kernel", ["decode", 16, 128])
@pytest.mark.parametrize("Hq,H,D,B,new,lens", [(12, 1, 128, 64, [61], [1758]), (16, 2, 256, 64, [70], [777]), (4, 4, 64, 16, [300], [300]),
                                               (8, 2, 128, 32, [33, 2, 300], [900, 700, 310]),
                                               (4, 2, 256, 16, [1] * 20, list(range(0, 1000, 50)))])
def test_attention_in_a_wide_table(kvt_pkg, monkeypatch, kernel, Hq, H, D, B, new, lens):
    """A table of 262,144 positions, as a cache for long contexts has it, over requests that fill little of it: 64 bits, with a
    kept workspace and without; and splits of one request's query tiles that hold 256 positions at least."""
    from kvtier import block_kv
    decode = kernel == "decode"
    monkeypatch.setattr(block_kv, "_TILE_MIN", {D: 0 if kernel == 128 else 10 ** 9})
    if decode:
        new = [1] * len(lens)
    g = torch.Generator().manual_seed(D)
    table, nb = _tables(lens, B, 2, D)
    codes, sc = _pool("fp8", nb, H, B, D, g)
    tab = torch.full((len(lens), 262_144 // B), -1, dtype=torch.int32)
    tab[:, :len(table[0])] = torch.tensor(table, dtype=torch.int32)
    cu = prefix(new)
    q = torch.randn(cu[-1], Hq, D, generator=g).to(torch.bfloat16)
    val = [ref.values(codes[i]) * sc[i].double()[..., None, None] for i in range(2)]
    want = ref.attention(q.double(), cu, lens, range(len(new)), table, val[0], val[1], not decode, D ** -0.5)
    args = [c.to(dev) for c in codes] + [s.to(dev) for s in sc] + [tab.to(dev), i32(lens)]

    def call(ws):
        out = torch.full(q.shape, 5.0, dtype=torch.float32, device=dev)
        if decode:
            return block_kv.kvt_block_decode(q.to(dev), *args, out=out, workspace=ws)
        return block_kv.kvt_block_prefill(q.to(dev), i32(cu), *args, out=out, workspace=ws)
    ws = {}
    for w in (None, ws, ws):
        ref.close(call(w), *want, D)
    if kernel == 128 and len(lens) == 1:
        ml = ws["block_ml", 0]
        ml.fill_(-7.0)
        call(ws)
        items = (cu[-1] * (Hq // H) // 128 + 1) * H
        used = (ml.view(items, -1, 128, 2) != -7.0).flatten(2).any(2).any(0).nonzero()
        assert 1 < used.numel() and int(used.max()) < -(-lens[0] // 256)


def test_attention_strided_queries_and_rows(kvt_pkg):
    """Queries as a slice of a fused projection (strided, and at an odd offset), table rows through seqs, a strided out."""
    from kvtier import block_kv
    g = torch.Generator().manual_seed(12)
    lens, B, H, D, Hq = [100, 50, 33], 32, 2, 64, 8
    table, nb = _tables(lens, B, 1, 12)
    codes, sc = _pool("fp8", nb, H, B, D, g)
    val = [ref.values(codes[i]) * sc[i].double()[..., None, None] for i in range(2)]
    seqs = [2, 0, 1]
    args = [codes[0].to(dev), codes[1].to(dev), sc[0].to(dev), sc[1].to(dev), i32(table)]
    for off in (0, 3):
        qkv = torch.randn(3, Hq + 5, D + off, generator=g).to(torch.bfloat16)
        q = qkv[:, 2:2 + Hq, off:]
        want = ref.attention(q.double(), [0, 1, 2, 3], [lens[s] for s in seqs], seqs, table, val[0], val[1], False, D ** -0.5)
        out = torch.zeros(3, Hq + 1, D, dtype=torch.float32, device=dev)
        got = block_kv.kvt_block_decode(qkv.to(dev)[:, 2:2 + Hq, off:], *args, i32([lens[s] for s in seqs]), seqs=i32(seqs),
                                        out=out[:, 1:])
        ref.close(got, *want, D)
        assert bool((out[:, 0] == 0).all())
    # rows that are no rows of the table see nothing
    got = block_kv.kvt_block_decode(q.to(dev), *args, i32([5, 5, 5]), seqs=i32([-1, 3, 0]))
    assert bool(torch.isnan(got[:2]).all()) and bool(torch.isfinite(got[2]).all())


@pytest.mark.parametrize("Hq,H,n", [(4, 2, 1), (1, 1, 3), (1, 1, 1)])
def test_one_row_or_head_of_an_odd_buffer(kvt_pkg, Hq, H, n):
    """Rows, queries and outputs whose dimensions of one entry have odd strides, on a 16-byte boundary and off it."""
    from kvtier import block_kv
    D, B = 64, 16
    g = torch.Generator().manual_seed(31)

    def odd(x, off):
        w = x.shape[1] * D
        buf = torch.zeros(x.shape[0] * (w + (8 if n > 1 else 5)) + off, dtype=x.dtype, device=dev)
        t = buf.as_strided(x.shape, (w + (8 if n > 1 else 5), D if x.shape[1] > 1 else 3, 1), off)
        return t.copy_(x)
    x = torch.randn(2, n, H, D, generator=g).to(torch.bfloat16)
    q = torch.randn(n, Hq, D, generator=g).to(torch.bfloat16)
    for off in (0, 1):
        c = block_kv.BlockKVCache(1, H, D, n_blocks=2, max_seqs=1, max_blocks=2, block=B)
        plan = c.plan([c.add_seq()], [n])
        c.append(0, plan, odd(x[0], off), odd(x[1], off))
        codes, sc = (c.k8[0], c.v8[0]), (c.ks[0], c.vs[0])
        val = [ref.values(codes[i].cpu()) * sc[i].cpu().double()[..., None, None] for i in range(2)]
        out = odd(torch.zeros(n, Hq, D), 0)
        got = c.prefill(0, plan, odd(q, off), out=out)
        assert got is out
        ref.close(got, *ref.attention(q.double(), [0, n], [n], [0], c.block_table.tolist(), val[0], val[1], True, D ** -0.5), D)
        if n == 1:
            assert torch.equal(c.decode(0, plan, odd(q, off), out=odd(torch.zeros(n, Hq, D), 0)), got)


# ----------------------------------------------------------------------------------------------------- the four together
def _step_reference(x, kv, B, H, D):
    """The cache that appending x (a list of [n, H, D] float64 per step, one sequence) leaves, as [1 + blocks] values."""
    n = sum(len(t) for t in x)
    nb = -(-n // B)
    codes, scale = torch.zeros(nb, H, B, D, dtype=torch.float64), torch.zeros(nb, H, dtype=torch.float64)
    L = 0
    for t in x:
        ref.store(t, [0, len(t)], [L + len(t)], [0], [list(range(nb))], codes, scale, kv)
        L += len(t)
    return codes * scale[..., None, None]


@pytest.mark.parametrize("kv,B,D", [("fp8", 64, 256), ("int8", 16, 128)])
def test_a_serving_run(kvt_pkg, kv, B, D):
    """Three sequences: prompts in ragged chunks, decode steps (one of them joins late), a release and a new sequence on its
    blocks; attention after every step against the reference's own cache."""
    from kvtier import block_kv
    H, Hq = 2, 8
    c = block_kv.BlockKVCache(2, H, D, n_blocks=60, max_seqs=3, max_blocks=400 // B, dtype=ref.CODE[kv], block=B, seed=3)
    g = torch.Generator().manual_seed(13)
    hist = {}
    a, b = c.add_seq(), c.add_seq()
    third = None
    steps = [[(a, 70), (b, 33)], [(b, 90), (a, 1)], [(a, 1), (b, 1)], "join", "release", [(a, 2), (b, 1)]]
    for step in steps:
        if step == "join":
            third = c.add_seq()
            step = [(third, 40), (a, 1), (b, 1)]
        elif step == "release":
            c.release(b)
            hist.pop(b)
            b = c.add_seq()
            step = [(b, 50), (third, 1)]
        seqs, counts = [s for s, _ in step], [n for _, n in step]
        plan = c.plan(seqs, counts)
        cu = prefix(counts)
        x = torch.randn(2, 2, cu[-1], H, D, generator=g).to(torch.bfloat16) * 3
        q = torch.randn(cu[-1], Hq, D, generator=g).to(torch.bfloat16)
        for j, s in enumerate(seqs):
            hist.setdefault(s, []).append(x[:, :, cu[j]:cu[j + 1]].double())
        for layer in range(2):
            c.append(layer, plan, x[layer, 0].to(dev), x[layer, 1].to(dev))
            got = c.prefill(layer, plan, q.to(dev))
            if all(n == 1 for n in counts):
                one = c.decode(layer, plan, q.to(dev))
            for j, s in enumerate(seqs):
                kv_ = [_step_reference([t[layer, i] for t in hist[s]], kv, B, H, D) for i in range(2)]
                L = sum(t.shape[2] for t in hist[s])
                want = ref.attention(q[cu[j]:cu[j + 1]].double(), [0, counts[j]], [L], [0], [list(range(len(kv_[0])))], kv_[0],
                                     kv_[1], True, D ** -0.5)
                ref.close(got[cu[j]:cu[j + 1]], *want, D)
                if all(n == 1 for n in counts):
                    ref.close(one[cu[j]:cu[j + 1]], *want, D)
    c.check()


def test_captured_decode_steps(kvt_pkg):
    """A decode step (plan, write, attention) captured once and replayed, with eager work between the replays, against the
    same steps made eagerly on a second cache; two graphs over one cache with workspaces of their own."""
    from kvtier import block_kv
    H, D, Hq, B, n = 2, 128, 16, 16, 3
    made = []
    for _ in range(2):
        c = block_kv.BlockKVCache(1, H, D, n_blocks=120, max_seqs=n, max_blocks=40, block=B, seed=1)
        for _ in range(n):
            c.add_seq()
        made.append(c)
    cap, eag = made
    g = torch.Generator(device=dev).manual_seed(14)
    lens = [5, 31, 200]
    x0 = torch.randn(2, sum(lens), H, D, device=dev, generator=g).to(torch.bfloat16)
    for c in made:
        c.append(0, c.plan([0, 1, 2], lens), x0[0], x0[1])
    seqs, ones = i32([0, 1, 2]), i32([1, 1, 1])
    k, v = torch.zeros(2, n, H, D, dtype=torch.bfloat16, device=dev).unbind(0)
    q = torch.zeros(n, Hq, D, dtype=torch.bfloat16, device=dev)

    def step(c, ws, out):
        plan = c.plan(seqs, ones, n_tokens=n)
        c.append(0, plan, k, v)
        return c.decode(0, plan, q, workspace=ws, out=out)

    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    before = {name: getattr(cap, name).clone() for name in ("block_table", "seq_lens", "free_head", "status")}
    keep = [t.clone() for t in (cap.k8[0].view(torch.int8), cap.v8[0].view(torch.int8), cap.ks[0], cap.vs[0])]
    spaces = [{}, {}]
    for ws, out in zip(spaces, outs):                    # (warm: the workspaces are allocated before the capture)
        step(cap, ws, out)
    torch.cuda.synchronize()
    for ws, out in zip(spaces, outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(cap, ws, out)
        graphs.append(gr)
    for name, t in before.items():
        getattr(cap, name).copy_(t)
    for t, u in zip((cap.k8[0].view(torch.int8), cap.v8[0].view(torch.int8), cap.ks[0], cap.vs[0]), keep):
        t.copy_(u)
    for i in range(40):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device=dev, generator=g).to(torch.bfloat16))
        graphs[i % 2].replay()
        want = step(eag, None, None)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want), i
    for t, u in zip((cap.k8[0], cap.v8[0]), (eag.k8[0], eag.v8[0])):
        assert torch.equal(t.view(torch.int8), u.view(torch.int8))
    assert torch.equal(cap.block_table, eag.block_table) and torch.equal(cap.seq_lens, eag.seq_lens)
    cap.check()


def test_on_another_stream(kvt_pkg):
    """Everything is enqueued on the current stream: a step on a side stream behind an event."""
    from kvtier import block_kv
    H, D = 2, 128
    c, e = (block_kv.BlockKVCache(1, H, D, n_blocks=40, max_seqs=1, max_blocks=20, block=64, seed=2) for _ in range(2))
    x = torch.randn(2, 700, H, D, device=dev).to(torch.bfloat16)
    q = torch.randn(700, 8, D, device=dev).to(torch.bfloat16)
    got = []
    for cache, st in ((c, torch.cuda.Stream()), (e, torch.cuda.current_stream())):
        s = cache.add_seq()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            plan = cache.plan([s], [700])
            cache.append(0, plan, x[0], x[1])
            got.append(cache.prefill(0, plan, q))
        torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    assert torch.equal(got[0], got[1])


def test_slots_serve_the_slot_pools(kvt_pkg):
    """A plan's slots and req_to_token are locations of the slot-indexed pools: rows written at them by
    quant_store_kv_int8 come back through the whole-prefix gather in order."""
    from kvtier import block_kv, sparse_attn
    H, D, B, nb = 2, 256, 64, 12
    g = torch.Generator(device=dev).manual_seed(15)
    seq_lens, table = i32([0, 0]), torch.full((2, 6), -1, dtype=torch.int32, device=dev)
    free, head = torch.randperm(nb).int().to(dev), i32([0])
    rtt = torch.zeros(2, 300, dtype=torch.int32, device=dev)
    counts = [130, 70]
    p = block_kv.kvt_block_plan(i32([1, 0]), i32(counts), seq_lens, table, free, head, 200, block=B, req_to_token=rtt)
    x = torch.randn(2, 200, H, D, device=dev, generator=g).to(torch.bfloat16)
    kb, vb = (torch.zeros(nb * B, H, D, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(nb * B, H, D // 64, dtype=torch.float16, device=dev) for _ in range(2))
    one = torch.ones(H, D, dtype=torch.float16, device=dev)
    sparse_attn.quant_store_kv_int8(x[0], x[1], p.slots, kb, vb, ks, vs, one, one)
    ok, ov = (torch.zeros(200, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    sparse_attn.qwen_sparse_prefix_gather_dequant_int8(kb, vb, ks, vs, one, one, rtt, p.seqs, p.kv_lens, p.cu, ok, ov, 2, 130)
    # a code is off by half a step of 1 / 127 of its group's largest value, the row by the rounding to bf16
    for got, want in ((ok, x[0]), (ov, x[1])):
        top = want.float().view(200, H, 4, 64).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 64).reshape(200, H, D)
        assert bool(((got.float() - want.float()).abs() <= top * (0.5 / 127 + 2.0 ** -8 + 2.0 ** -10)).all())


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("Hq,H,D,B,splits", [(1, 1, 64, 16, 2), (8, 2, 128, 32, 8), (32, 8, 128, 64, None), (32, 2, 256, 16, 16),
                                             (10, 2, 256, 64, None), (4, 4, 64, 64, 5)])
def test_merge_in_the_launch(kvt_pkg, kv, Hq, H, D, B, splits):
    """A kept workspace, over which few splits are merged inside the launch, used by decode steps and chunks of several sizes:
    64 bits, and the bits of a call without one; the counters are zero after every call."""
    ws = {}
    for lens, new in (([700], [3]), (LENS, [min(n, 4) for n in LENS]), ([2000, 0, 1, 900], [1, 0, 1, 2]), (LENS[3:5], [5, 1])):
        for decode in (True, False):
            got = [_check_attn(kv, torch.bfloat16, Hq, H, D, B, [1] * len(lens) if decode else new, lens, decode=decode, seed=19,
                               splits=splits, workspace=w, out_dtype=torch.float32) for w in (ws, ws, None)]
            for other in got[1:]:
                assert torch.equal(got[0].view(torch.int32), other.view(torch.int32))
            assert not ws["block_counters", 0].any()


@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("Hq,H,D,B,shares", [(4, 4, 64, 16, 7), (8, 1, 128, 64, 40), (32, 2, 128, 16, 33), (6, 2, 64, 32, 512),
                                             (16, 1, 64, 16, 128), (12, 2, 256, 64, 24)])
def test_merge_of_shares_in_the_launch(kvt_pkg, kv, Hq, H, D, B, shares):
    """The same over equal shares: pairs of two parts and of more than a wavefront's worth, several pairs of a workgroup, none."""
    ws = {}
    for lens in ([5000, 0, 3, 17], LENS * 2, [900, 1000, 1], [0, 0]):
        got = [_check_attn(kv, torch.bfloat16, Hq, H, D, B, [1] * len(lens), lens, decode=True, seed=20, splits=-shares, workspace=w,
                           out_dtype=torch.float32) for w in (ws, ws, None)]
        for other in got[1:]:
            assert torch.equal(got[0].view(torch.int32), other.view(torch.int32))
        assert not ws["block_counters", 0].any()


@pytest.mark.parametrize("warm", [True, False])
def test_workspace_of_a_captured_call_is_outgrown(kvt_pkg, warm):
    """A decode and a chunk captured over a workspace, made before the capture or inside it, which larger eager calls outgrow
    and use between the replays: every replay gives the eager bits."""
    from kvtier import block_kv
    H, D, Hq, B = 2, 128, 8, 32
    g = torch.Generator().manual_seed(23)
    lens = [900, 33, 1500, 1, 64, 700]
    table, nb = _tables(lens, B, 2, 23)
    codes, sc = _pool("fp8", nb, H, B, D, g)
    buf = (codes[0].to(dev), codes[1].to(dev), sc[0].to(dev), sc[1].to(dev))
    tab, kl = i32(table), i32(lens)
    q = torch.randn(6, Hq, D, generator=g).to(torch.bfloat16).to(dev)
    cq = torch.randn(6 * 5, Hq, D, generator=g).to(torch.bfloat16).to(dev)
    few = (tab[:2].contiguous(), kl[:2].contiguous())
    cu2, cu6 = i32([0, 5, 10]), i32([5 * i for i in range(7)])
    ws = {}

    def small(w, x, y):
        return (block_kv.kvt_block_decode(x[:2], *buf, *few, workspace=w),
                block_kv.kvt_block_prefill(y[:10], cu2, *buf, *few, workspace=w))

    def large(w):
        return (block_kv.kvt_block_decode(q, *buf, tab, kl, workspace=w),
                block_kv.kvt_block_prefill(cq, cu6, *buf, tab, kl, workspace=w))

    if warm:
        small(ws, q, cq)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = small(ws, q, cq)
    for i in range(4):
        q.normal_()
        cq.normal_()
        gr.replay()
        want = small(None, q, cq)
        torch.cuda.synchronize()
        # (the bits: queries of the request with fewer positions than queries see nothing and are NaN, which equals nothing)
        for a, b in (*zip(outs, want), *zip(large(ws), large(None))):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i
    assert ("block_outgrown" in ws) and not ws["block_counters", 0].any()


def test_calls_at_once_on_two_streams(kvt_pkg):
    """Steps over two caches at once, each on a stream and over a workspace of its own: the bits of the steps made alone."""
    from kvtier import block_kv
    H, D, Hq = 4, 128, 16
    streams = [torch.cuda.Stream() for _ in range(2)]
    g = torch.Generator(device=dev).manual_seed(25)
    x = torch.randn(2, 2, 900, H, D, device=dev, generator=g).to(torch.bfloat16)
    q = torch.randn(2, 900, Hq, D, device=dev, generator=g).to(torch.bfloat16)

    def run(i, c, ws, rows):
        out = []
        for n in ([600, 300], [2, 1], [1, 1], [1, 1], [40, 30]):
            plan = c.plan(rows, i32(n), n_tokens=sum(n))
            c.append(0, plan, x[i, 0, :sum(n)], x[i, 1, :sum(n)])
            out.append(c.prefill(0, plan, q[i, :sum(n)], workspace=ws))
            if n == [1, 1]:
                out.append(c.decode(0, plan, q[i, :2], workspace=ws))
        return out

    def made():
        c = block_kv.BlockKVCache(1, H, D, n_blocks=60, max_seqs=2, max_blocks=30, block=64, seed=3)
        return c, i32([c.add_seq(), c.add_seq()])

    alone = [run(i, *(lambda m: (m[0], {}, m[1]))(made())) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        pairs, got = [made() for _ in range(2)], [None, None]
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(i, pairs[i][0], {}, pairs[i][1])
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(got[i], alone[i]):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16))
