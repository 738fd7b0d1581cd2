"""Rotary positions on the GPU against a plain 64-bit form: layouts, parts of the head, types, strides, positions per
token and of a step, in place, inverse."""
import math
import random

import pytest
import torch

import evict_testutil as ref

pytestmark = pytest.mark.gpu
dev = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def close(got, x, at, inv, scale, inter, inverse=False):
    out, size, turn = ref.rope(x.double().cpu(), at, inv.cpu(), scale, inter, inverse)
    tol = ref.rope_bound(out, size, turn, got.dtype)
    off = (got.double().cpu() - out).abs()
    assert (off <= tol).all(), (int((off > tol).sum()), float((off / tol).max()))


def rows(n, heads, d, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads * d + pad, generator=g).to(dtype).to(dev)
    return x[:, pad:].unflatten(1, (heads, d))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,hq,h,d,rot", [(1, 24, 2, 256, 64), (7, 8, 8, 128, 128), (65, 20, 20, 64, 32), (3, 3, 1, 80, 20),
                                          (2, 1, 1, 2, 2), (5, 5, 3, 48, 18), (4, 2, 1, 256, 2), (4, 2, 1, 256, 256)])
def test_positions_per_token(kvt_pkg, inter, io, n, hq, h, d, rot):
    from kvtier.rope import kvt_rope, rotary_frequencies
    rng = random.Random(n * d + rot)
    at = [rng.choice([0, 1, -5, 262_143, 1_000_000, 2 ** 31 - 1, rng.randrange(10 ** 6)]) for _ in range(n)]
    inv, scale = rotary_frequencies(rot, 1e4 if n % 2 else 5e5)
    scale = scale if n % 3 else 1.25
    q, k = rows(n, hq, d, DT[io], 1), rows(n, h, d, DT[io], 2)
    for pos in (torch.tensor(at, dtype=torch.int32, device=dev), torch.tensor(at, device=dev)):
        a, b = kvt_rope(q, k, pos, inv, scale, interleaved=inter)
        close(a, q, at, inv, scale, inter)
        close(b, k, at, inv, scale, inter)
    a, b = kvt_rope(q, None, pos, inv, scale, interleaved=inter, inverse=True)
    assert b is None
    close(a, q, at, inv, scale, inter, True)


@pytest.mark.parametrize("io,pad", [("bf16", 8), ("bf16", 3), ("f32", 4), ("f16", 1)])
@pytest.mark.parametrize("inter", [False, True])
def test_strides_and_in_place(kvt_pkg, io, pad, inter):
    """q and k as views of one projection's output, aligned and not; in place, channels behind the part and the rest of
    the buffer stay bit for bit."""
    from kvtier.rope import kvt_rope, rotary_frequencies
    n, hq, h, d, rot = 33, 6, 2, 64, 32
    g = torch.Generator().manual_seed(5)
    buf = torch.randn(n, (hq + 2 * h) * d + pad, generator=g).to(DT[io]).to(dev)
    q, k = buf[:, pad:pad + hq * d].unflatten(1, (hq, d)), buf[:, pad + hq * d:pad + (hq + h) * d].unflatten(1, (h, d))
    at = list(range(1000, 1000 + n))
    pos = torch.tensor(at, dtype=torch.int32, device=dev)
    inv, scale = rotary_frequencies(rot, 1e4)
    a, b = kvt_rope(q, k, pos, inv, scale, interleaved=inter)
    close(a, q, at, inv, scale, inter)
    close(b, k, at, inv, scale, inter)
    was = buf.clone()
    kvt_rope(q, k, pos, inv, scale, interleaved=inter, out_q=q, out_k=k)
    assert torch.equal(q, a) and torch.equal(k, b)
    was[:, pad:pad + hq * d].unflatten(1, (hq, d))[..., :rot] = a[..., :rot]
    was[:, pad + hq * d:pad + (hq + h) * d].unflatten(1, (h, d))[..., :rot] = b[..., :rot]
    assert torch.equal(buf, was)
    # heads before tokens, and an output of its own strides
    qt = rows(hq, n, d, DT[io], 7).transpose(0, 1)
    out = torch.zeros(n, hq + 1, d, dtype=DT[io], device=dev)[:, 1:]
    got, _ = kvt_rope(qt, None, pos, inv, scale, interleaved=inter, out_q=out)
    assert got.data_ptr() == out.data_ptr()
    close(got, qt, at, inv, scale, inter)


@pytest.mark.parametrize("counts", [[1], [1, 1, 1, 1], [0, 5, 0, 130, 1], [300] + [1] * 70, [0, 0], [1] * 700])
def test_step_positions(kvt_pkg, counts):
    """Lengths, prefix sums, rows and evicted entries of a step; rows behind the last request stay as they are."""
    from kvtier.rope import kvt_rope, rotary_frequencies
    rng = random.Random(len(counts))
    n, N = len(counts), sum(counts) + 5
    cu = [sum(counts[:i]) for i in range(n + 1)]
    lens = [c + rng.randrange(200_000) for c in counts]
    seqs = rng.sample(range(n + 3), n)
    ahead = [rng.randrange(100_000) for _ in range(n + 3)]
    at = [lens[j] - c + i + ahead[seqs[j]] for j, c in enumerate(counts) for i in range(c)] + [0] * 5
    q, k = rows(N, 4, 64, torch.bfloat16, 3), rows(N, 1, 64, torch.bfloat16, 4)
    inv, scale = rotary_frequencies(64, 1e6, "yarn", 4.0, 8192)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    oq, ok = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    kvt_rope(q, k, i32(lens), inv, scale, cu=i32(cu), seqs=i32(seqs), ahead=i32(ahead), out_q=oq, out_k=ok)
    if sum(counts):
        close(oq[:-5], q[:-5], at[:-5], inv, scale, False)
        close(ok[:-5], k[:-5], at[:-5], inv, scale, False)
    assert (oq[-5:] == 7).all() and (ok[-5:] == 7).all()
    got, _ = kvt_rope(q, None, i32(lens), inv, scale, cu=i32(cu))
    if sum(counts):
        close(got[:-5], q[:-5], [a - ahead[s] for a, s in zip(at, [s for s, c in zip(seqs, counts) for _ in range(c)])],
              inv, scale, False)


def test_inverse_is_the_gradient(kvt_pkg):
    """sum(g * rope(x)) has the gradient inverse-rope(g): against differences of the 64-bit form, and against the
    operator's own transpose."""
    from kvtier.rope import kvt_rope, rotary_frequencies
    inv, scale = rotary_frequencies(16, 1e4, "yarn", 8.0, 4096)
    at = [3, 70_001]
    pos = torch.tensor(at, device=dev)
    x, g = rows(2, 2, 20, torch.float32, 1), rows(2, 2, 20, torch.float32, 2)
    for inter in (False, True):
        got = kvt_rope(g, None, pos, inv, scale, interleaved=inter, inverse=True)[0].double().cpu()
        x64, g64, step = x.double().cpu(), g.double().cpu(), 2.0 ** -12
        for i in range(2 * 2 * 20):
            d = torch.zeros(80, dtype=torch.float64)
            d[i] = step
            up, down = (float((g64 * ref.rope(x64 + s * d.view(2, 2, 20), at, inv.cpu(), scale, inter)[0]).sum()) for s in (1, -1))
            # a linear function: differences are exact but for 64-bit rounding; the operator within its bound
            assert abs((up - down) / (2 * step) - float(got.flatten()[i])) < 2.0 ** -20 * 4 * float(g64.abs().max())


def test_specials_empty_and_streams(kvt_pkg):
    from kvtier.rope import kvt_rope, rotary_frequencies
    inv, scale = rotary_frequencies(32, 1e4)
    q = rows(3, 2, 64, torch.bfloat16, 1).clone()
    q[1, 0, 3] = math.nan
    q[1, 1, 40] = math.inf                    # (behind the rotated part: copied)
    pos = torch.tensor([5, 6, 7], dtype=torch.int32, device=dev)
    got = kvt_rope(q, None, pos, inv, scale)[0]
    nan = torch.isnan(got)
    assert nan[1, 0, 3] and nan[1, 0, 19] and int(nan.sum()) == 2 and got[1, 1, 40] == math.inf
    for n in (0,):
        a, b = kvt_rope(q[:n], q[:n, :1], pos[:n], inv, scale)
        assert a.shape == (0, 2, 64) and b.shape == (0, 1, 64)
    a, b = kvt_rope(q, q[:, :0], pos, inv, scale)
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(got)) and b.shape == (3, 0, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kvt_rope(q, None, pos, inv, scale)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(torch.nan_to_num(other), torch.nan_to_num(got))


def test_graph(kvt_pkg):
    from kvtier.rope import kvt_rope, rotary_frequencies
    inv, scale = rotary_frequencies(64, 1e4)
    q, pos = rows(9, 4, 64, torch.bfloat16, 1), torch.arange(9, device=dev)
    out = torch.empty_like(q)
    kvt_rope(q, None, pos, inv, scale, out_q=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kvt_rope(q, None, pos, inv, scale, out_q=out)
    for i in range(4):
        pos.copy_(torch.arange(9, device=dev) * (i + 1))
        want = kvt_rope(q, None, pos, inv, scale)[0]
        out.fill_(0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_many_tokens(kvt_pkg):
    """Element offsets past 2^31."""
    from kvtier.rope import kvt_rope, rotary_frequencies
    n, hq, d = 131_100, 64, 256                               # 2.15e9 elements
    inv, scale = rotary_frequencies(64, 1e4)
    q = torch.empty(n, hq, d, dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    tail = torch.randn(40, hq, d, generator=g, device=dev).to(torch.bfloat16)
    q[-40:] = tail
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    kvt_rope(q, None, pos, inv, scale, out_q=q)
    close(q[-40:], tail, list(range(n - 40, n)), inv, scale, False)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
def test_outputs_in_one_buffer(kvt_pkg, io, inter):
    """Both outputs as column ranges of one buffer, as heads in turn, and one of them in place beside the other: the bits
    of separate outputs, and the rest of the buffer as it was."""
    from kvtier.rope import kvt_rope, rotary_frequencies
    n, hq, h, d, rot = 37, 4, 2, 64, 48
    inv, scale = rotary_frequencies(rot, 1e4)
    pos = torch.arange(500, 500 + n, device=dev)
    q, k = rows(n, hq, d, DT[io], 1), rows(n, h, d, DT[io], 2)
    a, b = kvt_rope(q, k, pos, inv, scale, interleaved=inter)
    close(a, q, list(range(500, 500 + n)), inv, scale, inter)
    buf = torch.full((n, hq + 2 * h, d), 3.0, dtype=DT[io], device=dev)
    kvt_rope(q, k, pos, inv, scale, interleaved=inter, out_q=buf[:, h:h + hq], out_k=buf[:, h + hq:])
    assert torch.equal(buf, torch.cat((torch.full_like(b, 3.0), a, b), 1))
    two = torch.full((n, h, 2, d), 3.0, dtype=DT[io], device=dev)
    kvt_rope(q[:, :h], k, pos, inv, scale, interleaved=inter, out_q=two[:, :, 0], out_k=two[:, :, 1])
    assert torch.equal(two, torch.stack((a[:, :h], b), 2))
    buf = torch.cat((q, k, k), 1)
    kvt_rope(buf[:, :hq], buf[:, hq:hq + h], pos, inv, scale, interleaved=inter, out_q=buf[:, :hq], out_k=buf[:, hq + h:])
    assert torch.equal(buf, torch.cat((a, k, b), 1))
