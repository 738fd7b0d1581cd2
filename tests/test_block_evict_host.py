"""Refusals of the operators of a block cache within a budget and of rotary positions, on the host: wrong shapes, types,
sizes and tensors off the GPU are errors before anything is launched; rotary frequencies against their formulas."""
import ctypes
import math
import random

import pytest
import torch


def _i(*x):
    return torch.tensor(x, dtype=torch.int32)


def _pool(nb=4, H=2, B=16, D=64, dtype=torch.float8_e4m3fn):
    return dict(k8=torch.zeros(nb, H, B, D, dtype=torch.int8).view(dtype), v8=torch.zeros(nb, H, B, D, dtype=torch.int8).view(dtype),
                ks=torch.zeros(nb, H), vs=torch.zeros(nb, H), block_table=torch.zeros(2, 3, dtype=torch.int32))


def _weigh(**over):
    from kvtier.block_evict import kvt_block_weigh
    p = _pool()
    a = dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), k8=p["k8"], ks=p["ks"], block_table=p["block_table"],
             kv_lens=_i(1, 1), weights=torch.zeros(2, 2, 48))
    return kvt_block_weigh(**{**a, **over})


def _keep(**over):
    from kvtier.block_evict import kvt_block_keep
    return kvt_block_keep(**{**dict(weights=torch.zeros(2, 2, 48), kv_lens=_i(40, 40), budget=16), **over})


def _evict(**over):
    from kvtier.block_evict import kvt_block_evict
    return kvt_block_evict(**{**dict(src=torch.zeros(2, 2, 16, dtype=torch.int32), kv_lens=_i(40, 40), **_pool()), **over})


def _trim(**over):
    from kvtier.block_evict import kvt_block_trim
    a = dict(seqs=_i(0), seq_lens=_i(40, 40), block_table=torch.zeros(2, 3, dtype=torch.int32), free_list=_i(0, 1),
             free_head=_i(1), budget=16, block=16)
    return kvt_block_trim(**{**a, **over})


def _rope(**over):
    from kvtier.rope import kvt_rope
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
             positions=torch.zeros(3, dtype=torch.int64), inv_freq=torch.ones(16, dtype=torch.float64))
    return kvt_rope(**{**a, **over})


@pytest.mark.parametrize("call", [_weigh, _keep, _evict, _trim, _rope])
def test_tensors_off_the_gpu_are_refused(kvt_pkg, call):
    with pytest.raises(AssertionError):
        call()


@pytest.mark.parametrize("over", [dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 4, 32, dtype=torch.bfloat16)),
                                  dict(weights=torch.zeros(2, 2, 48, dtype=torch.float64)), dict(weights=torch.zeros(2, 48, 2).transpose(1, 2)),
                                  dict(kv_lens=torch.zeros(2, dtype=torch.int64)), dict(since=torch.zeros(2)),
                                  dict(cu_q=torch.zeros(3, dtype=torch.int64)), dict(out=torch.zeros(2, 2, 48, dtype=torch.bfloat16)),
                                  dict(k8=torch.zeros(4, 2, 16, 64, dtype=torch.uint8))])
def test_weigh_contract(kvt_pkg, over):
    with pytest.raises(AssertionError):
        _weigh(**over)


@pytest.mark.parametrize("over", [dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 5, 64, dtype=torch.bfloat16)),
                                  dict(q=torch.zeros(2, 34, 64, dtype=torch.bfloat16)), dict(weights=torch.zeros(1, 2, 48)),
                                  dict(weights=torch.zeros(2, 2, 47)), dict(weights=torch.zeros(2, 1, 48)), dict(cu_q=_i(0, 1)),
                                  dict(since=_i(0)), dict(seqs=_i(0)), dict(out=torch.zeros(2, 2, 40)),
                                  dict(weights=torch.zeros(2, 1, 48).expand(2, 2, 48)), dict(out=torch.zeros(1, 2, 48).expand(2, 2, 48))])
def test_weigh_sizes(kvt_pkg, over):
    with pytest.raises(ValueError):
        _weigh(**over)


def test_weigh_refuses_an_output_that_overlaps(kvt_pkg):
    w = torch.zeros(3, 2, 48)
    for out in (w[1:], torch.as_strided(w, (2, 2, 47), (96, 48, 1))):
        with pytest.raises(ValueError):
            _weigh(weights=w[:2], out=out)
    with pytest.raises(AssertionError):            # (weights under another name are weights: on to the device's check)
        _weigh(weights=w[:2], out=w[:2])


def test_keep_refusals(kvt_pkg):
    pos, per_row = torch.zeros(2, 2, 48, dtype=torch.int32), _i(0, 0)
    for bad in (dict(weights=torch.zeros(2, 2, 48, dtype=torch.float16)), dict(kv_lens=torch.zeros(2)),
                dict(pos=pos.long(), held=per_row, evicted=per_row), dict(out=torch.zeros(2, 2, 16)),
                dict(out=torch.zeros(2, 2, 17, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            _keep(**bad)
    for bad in (dict(budget=0), dict(recent=-1), dict(recent=10, sinks=7), dict(pos=pos), dict(pos=pos, held=per_row),
                dict(pos=pos, held=per_row, evicted=_i(0)), dict(pos=pos[:1], held=per_row, evicted=per_row),
                dict(kv_lens=_i(1, 1, 1)), dict(seqs=_i(0)), dict(weights=torch.zeros(2, 2, 0))):
        with pytest.raises(ValueError):
            _keep(**bad)


def test_evict_refusals(kvt_pkg):
    pos, per_row = torch.zeros(2, 2, 48, dtype=torch.int32), _i(0, 0)
    for bad in (dict(src=torch.zeros(2, 2, 16, dtype=torch.int64)), dict(weights=torch.zeros(2, 2, 48, dtype=torch.float16)),
                dict(src=torch.zeros(2, 2, 32, dtype=torch.int32)[..., ::2]), dict(v8=torch.zeros(4, 2, 16, 64, dtype=torch.int8))):
        with pytest.raises(AssertionError):
            _evict(**bad)
    for bad in (dict(src=torch.zeros(2, 2, 24, dtype=torch.int32)), dict(src=torch.zeros(2, 2, 0, dtype=torch.int32)),
                dict(src=torch.zeros(1, 2, 16, dtype=torch.int32)), dict(weights=torch.zeros(2, 2, 40)), dict(pos=pos),
                dict(pos=pos, held=per_row), dict(pos=pos, held=_i(0), evicted=per_row), dict(seqs=_i(0)),
                dict(weights=torch.zeros(2, 1, 48).expand(2, 2, 48)),
                dict(pos=pos[:, :1].expand(2, 2, 48), held=per_row, evicted=per_row)):
        with pytest.raises(ValueError):
            _evict(**bad)


def test_trim_refusals(kvt_pkg):
    for bad in (dict(seqs=torch.zeros(1)), dict(free_head=torch.zeros(1, dtype=torch.int64)), dict(block_table=torch.zeros(2, 3))):
        with pytest.raises(AssertionError):
            _trim(**bad)
    for bad in (dict(budget=24), dict(budget=0), dict(block=48), dict(seq_lens=_i(1)), dict(held=_i(0, 0)),
                dict(held=_i(0, 0), evicted=_i(0)), dict(free_head=_i())):
        with pytest.raises(ValueError):
            _trim(**bad)


def test_rope_refusals(kvt_pkg):
    x = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    for bad in (dict(q=x.double()), dict(k=x.float()), dict(k=x[:2]), dict(inv_freq=torch.ones(16)),
                dict(positions=torch.zeros(3)), dict(cu=_i(0, 3), positions=torch.zeros(1, dtype=torch.int64)),
                dict(out_q=x.float()), dict(out_q=x[:2]), dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2))):
        with pytest.raises(AssertionError):
            _rope(**bad)
    two = torch.zeros(4, 4, 64, dtype=torch.bfloat16)
    for bad in (dict(positions=torch.zeros(2, dtype=torch.int64)), dict(inv_freq=torch.ones(33, dtype=torch.float64)),
                dict(inv_freq=torch.ones(0, dtype=torch.float64)), dict(seqs=_i(0)), dict(ahead=_i(0)),
                dict(cu=_i(0), positions=_i(1)), dict(cu=_i(0, 3), positions=_i(3), seqs=_i()),
                dict(cu=_i(0, 2, 3), positions=_i(3, 3), ahead=_i(0)), dict(k=None, out_k=x),
                dict(q=two[1:], out_q=two[:3]), dict(q=x, k=x[:, :2], out_q=x.clone(), out_k=x[:, 1:3]),
                dict(out_q=x[:1].expand(3, 4, 64)),
                dict(q=torch.zeros(3, 1, 320, dtype=torch.bfloat16), k=None)):
        with pytest.raises(ValueError):
            _rope(**bad)


def test_c_entries_refuse(kvt_pkg):
    """NULL pointers and sizes out of range come back as a status, without a launch."""
    lib = kvt_pkg._lib.lib()
    N = None

    def weigh(n=1, H=1, Hq=1, D=64, code=0, block=16, max_blocks=4, stride=4, rows=1, scale=1.0, splits=1, rs=1,
              groups=1, fit=0, most=0, floats=10 ** 6, q_type=0, cu=None, n_q=1, sq=64):
        return lib.kvt_block_weigh(N, sq, 64, q_type, cu, n_q, N, n, H, Hq, D, code, N, N, 4, block, N, stride, rows, max_blocks,
                                   N, scale, N, N, 0, 0, N, 0, 0, splits, rs, groups, fit, most, N, floats, N)
    for bad in (dict(n=0), dict(n=5000, rows=5000, n_q=5000), dict(Hq=17), dict(H=2, Hq=3), dict(D=96), dict(code=2), dict(block=48),
                dict(stride=3), dict(n=2), dict(scale=0.0), dict(scale=math.nan), dict(splits=0), dict(splits=2000), dict(rs=0),
                dict(groups=0), dict(fit=-1), dict(most=-1), dict(floats=10), dict(q_type=2), dict(sq=63), dict(n_q=0)):
        assert weigh(**bad) == -1, bad
    assert weigh(max_blocks=2 ** 28, stride=2 ** 28) == -3
    assert weigh(groups=1 << 24) == -3

    def keep(n=1, H=1, rows=1, cap=64, budget=16, recent=0, sinks=0, pos=None, held=None, ints=0, work=None):
        return lib.kvt_block_keep(N, 0, 0, N, n, H, rows, N, cap, budget, recent, sinks, pos, 0, 0, held, N, N, work, ints, N)
    for bad in (dict(n=0), dict(n=2), dict(cap=0), dict(budget=0), dict(recent=17), dict(sinks=-1), dict(pos=16), dict(held=16),
                dict(cap=40_000, ints=6227), dict(cap=40_000, work=8, ints=10 ** 6)):
        assert keep(**bad) == -1, bad
    assert keep(cap=2 ** 31) == -3 and keep(n=1 << 22, rows=1 << 22) == -3

    def evict(n=1, H=1, D=64, code=0, nb=4, block=16, stride=4, rows=1, mb=4, budget=16, pos=None, k8=None):
        return lib.kvt_block_evict(N, N, n, H, D, code, k8, N, N, N, nb, block, N, stride, rows, mb, N, budget, N, 0, 0, pos, 0, 0,
                                   N, N, N)
    for bad in (dict(n=0), dict(n=2), dict(D=32), dict(code=3), dict(nb=0), dict(block=8), dict(stride=2), dict(budget=8),
                dict(budget=24), dict(budget=80), dict(pos=16), dict(k8=8)):
        assert evict(**bad) == -1, bad
    assert evict(n=1 << 24, rows=1 << 24) == -3 and evict(mb=2 ** 27, stride=2 ** 27) == -3 and evict(nb=2 ** 28) == -3

    def trim(n=1, rows=1, stride=4, mb=4, n_free=4, block=16, budget=16, held=None, work=16):
        return lib.kvt_block_trim(n, N, N, rows, N, stride, mb, N, n_free, N, block, budget, held, N, N, N, N, 1, work, N)
    for bad in (dict(n=0), dict(n=1025), dict(rows=0), dict(stride=3), dict(n_free=-1), dict(block=12), dict(budget=15), dict(held=16),
                dict(work=None), dict(work=8)):
        assert trim(**bad) == -1, bad

    def rope(Hq=1, Hk=0, dtype=0, N_=1, D=64, rot=64, cu=None, n=0, wide=0, ahead=None, rows=0, on=64):
        return lib.kvt_rope(N, 64, 64, Hq, N, on, 64, N, 0, 0, Hk, N, 0, 0, dtype, N_, D, rot, N, N, wide, cu, n, N, ahead, rows, 1.0, 0,
                            0, N)
    for bad in (dict(Hq=0), dict(Hk=-1), dict(dtype=3), dict(D=258), dict(rot=66), dict(rot=7), dict(rot=0), dict(N_=-1),
                dict(cu=16), dict(cu=16, n=5000), dict(cu=16, n=1, wide=1), dict(cu=16, n=1, ahead=16), dict(ahead=16), dict(on=128)):
        assert rope(**bad) == -1, bad
    assert rope(N_=1 << 24) == -3 and rope(N_=0) == 0
    assert ctypes


def test_cache_without_evicting_refuses(kvt_pkg):
    from kvtier.block_kv import BlockKVCache
    c = BlockKVCache(1, 1, 64, 2, 1, 2, device="cpu")
    assert c.weights is None
    for call in (lambda: c.weigh_decode(0, None, None), lambda: c.weigh_prefill(0, None, None), lambda: c.evict([0], 64)):
        with pytest.raises(ValueError):
            call()
    c = BlockKVCache(2, 3, 64, 2, 1, 2, device="cpu", block=32, evicting=True)
    assert c.weights.shape == c.pos.shape == (2, 1, 3, 64)
    s = c.add_seq()
    c.evicted[s] = c.held[s] = 9
    c.release(s)
    assert int(c.evicted[s]) == int(c.held[s]) == 0
    c.status.fill_(16)
    with pytest.raises(RuntimeError, match="handed out"):
        c.check()


def test_rotary_frequencies(kvt_pkg):
    from kvtier.rope import rotary_frequencies
    plain, one = rotary_frequencies(64, 1e4, device="cpu")
    assert plain.dtype == torch.float64 and one == 1.0
    assert [abs(float(x) - 1e4 ** (-i / 32)) <= 1e-15 for i, x in enumerate(plain)] == [True] * 32
    assert torch.equal(rotary_frequencies(64, 1e4, "linear", 4.0, device="cpu")[0], plain / 4)
    ntk = rotary_frequencies(64, 1e4, "ntk", 4.0, device="cpu")[0]
    assert float(ntk[0]) == 1.0 and abs(float(ntk[-1] * 4 / plain[-1]) - 1) < 1e-12
    long, scale = rotary_frequencies(64, 1e4, "yarn", 4.0, 4096, device="cpu")
    assert abs(scale - (0.1 * math.log(4) + 1)) < 1e-15
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(long[turns > 40], plain[turns > 40])                   # fast ones stay, slow ones are divided
    assert torch.allclose(long[turns < 0.7], plain[turns < 0.7] / 4, rtol=1e-12)
    assert ((long <= plain) & (long >= plain / 4 * (1 - 1e-12))).all()
    own, s = rotary_frequencies(4, 100.0, factors=[1.0, 5.0], attention=1.5, device="cpu")
    assert own.tolist() == [1.0, 0.1 / 5.0] and s == 1.5
    for bad in (dict(dim=5), dict(dim=0), dict(method="other"), dict(factor=0.0), dict(base=-1.0), dict(factors=[1.0]),
                dict(factors=[1.0] * 4, method="linear"), dict(method="yarn"), dict(method="yarn", original=100, beta_fast=1.0),
                dict(dim=2, method="ntk")):
        with pytest.raises(ValueError):
            rotary_frequencies(**{**dict(dim=8, device="cpu"), **bad})


def test_overlaps_are_of_elements(kvt_pkg):
    """Views of one buffer against the elements that they hold: shared memory is always found, and column ranges, or heads,
    of one buffer are apart although their spans meet."""
    from kvtier.block_kv import _overlap
    rng = random.Random(1)
    where = torch.arange(4000, dtype=torch.int32)

    def both(x, y):
        return bool(set(x.flatten().tolist()) & set(y.flatten().tolist()))
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [rng.choice([1, 2, 3, 5]) for _ in range(3)]
            stride = [rng.choice([3, 8, 24, 40, 41, 64]), rng.choice([2, 4, 8, 13]), 1]
            views.append(torch.as_strided(where, shape, stride, rng.randrange(80)))
        assert _overlap(*views) or not both(*views)
    rows = where[:7 * 240].view(7, 240)
    parts = [rows[:, a:a + 8 * n].unflatten(1, (n, 8)) for a, n in ((0, 4), (32, 2), (48, 1), (56, 23), (40, 3))]
    groups = where[:7 * 240].view(7, 10, 24)
    parts += [groups[..., 0:8], groups[..., 8:16], groups[:, ::2, 16:24], groups[:, 1::2, 16:24]]
    for x in parts:
        for y in parts:
            assert _overlap(x, y) == both(x, y) or x.stride() != y.stride() and not both(x, y)
    for i, j in ((0, 1), (1, 2), (2, 3), (0, 4), (5, 6), (5, 7), (7, 8)):
        assert not _overlap(parts[i], parts[j]) and not _overlap(parts[j], parts[i]), (i, j)


def test_rope_outputs_and_the_other_tensors(kvt_pkg):
    """An output in place must be apart from the other tensors too; parts of one buffer are apart (and go on to the
    device's check)."""
    x = torch.zeros(3, 6, 64, dtype=torch.bfloat16)
    for bad in (dict(q=x, k=x[:, :2], out_q=x), dict(q=x, k=x, out_q=x), dict(q=x[:, 2:], k=x[:, 1:3], out_q=x[:, 2:]),
                dict(q=x[:, :4], k=x[:, 2:4], out_k=x[:, 2:4]), dict(q=x, k=x, out_q=x, out_k=x),
                dict(q=x[:, :2], k=x[:, 2:4], out_q=x[:, 2:4])):
        with pytest.raises(ValueError):
            _rope(**bad)
    q, k = x[:, :4], x[:, 4:]
    new = torch.zeros(3, 6, 64, dtype=torch.bfloat16)
    for good in (dict(out_q=new[:, :4], out_k=new[:, 4:]), dict(q=q, k=k, out_q=q, out_k=k), dict(q=q, k=k, out_q=q),
                 dict(q=q, k=k, out_q=new[:, 2:], out_k=new[:, :2]), dict(q=x[:, :2], k=x[:, 2:4], out_q=x[:, 4:])):
        with pytest.raises(AssertionError, match="device tensors"):
            _rope(**{**(dict(k=k, q=q) if "out_k" in good else {}), **good})


def test_weigh_output_beside_its_weights(kvt_pkg):
    """Sums and weights as parts of one buffer."""
    w = torch.zeros(2, 2, 2, 48)
    with pytest.raises(AssertionError, match="device tensors"):
        _weigh(weights=w[:, 0], out=w[:, 1])
    with pytest.raises(ValueError):
        _weigh(weights=w[:, 0], out=w[:, 0, :, 1:].as_strided((2, 2, 47), w[:, 0].stride(), 1))


def test_weigh_workspace_is_bounded(kvt_pkg, monkeypatch):
    """One query per request: the scores of as many requests as 2^30 floats hold, of one at least; what the call is given
    is what it asked for, whatever a workspace held before."""
    from kvtier import block_evict
    asked = []
    monkeypatch.setattr(block_evict, "_stream", lambda *x: 0)
    monkeypatch.setattr(block_evict._lib, "call", lambda name, *x: asked.append((name, x[-2])))
    monkeypatch.setattr(block_evict, "_grown", lambda ws, what, need, like, *x: asked.append(need) or torch.zeros(1))
    p = _pool(H=1)
    for n, hq, blocks, most in ((2, 16, 3, 2), (80, 16, 1 << 16, 64), (3, 16, 1 << 23, 1)):
        cap = 16 * blocks
        asked.clear()
        _weigh(q=torch.zeros(n, hq, 64, dtype=torch.bfloat16), k8=p["k8"], ks=p["ks"], kv_lens=torch.zeros(n, dtype=torch.int32),
               block_table=torch.empty(n, blocks, dtype=torch.int32), weights=torch.empty(n, 1, cap))
        assert most * hq * cap < asked[0] <= most * (hq * cap + 256 * 32), (n, asked)
        assert asked[1] == ("kvt_block_weigh", asked[0])


@pytest.mark.parametrize("bad", [0.0, -2.0, math.inf, math.nan])
def test_rotary_divisors_are_positive_numbers(kvt_pkg, bad):
    from kvtier.rope import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(8, factors=[1.0, 2.0, bad, 4.0], device="cpu")
