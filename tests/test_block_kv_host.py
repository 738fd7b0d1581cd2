"""Refusals of the 8-bit block cache's entry points, on the host: wrong shapes, types, sizes and tensors off the GPU are
errors before anything is launched, through the Python functions and through the C entries (NULL pointers, no GPU)."""
import ctypes

import pytest
import torch


def _pool(nb=4, H=2, B=16, D=64, dtype=torch.float8_e4m3fn):
    return dict(k8=torch.zeros(nb, H, B, D, dtype=torch.int8).view(dtype), v8=torch.zeros(nb, H, B, D, dtype=torch.int8).view(dtype),
                ks=torch.zeros(nb, H), vs=torch.zeros(nb, H), block_table=torch.zeros(2, 3, dtype=torch.int32))


def _i(*x):
    return torch.tensor(x, dtype=torch.int32)


def _decode(q=None, kv_lens=None, seqs=None, out=None, **over):
    from kvtier import block_kv
    p = {**_pool(), **over}
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16) if q is None else q
    return block_kv.kvt_block_decode(q, p["k8"], p["v8"], p["ks"], p["vs"], p["block_table"],
                                     _i(1, 1) if kv_lens is None else kv_lens, seqs=seqs, out=out)


def test_tensors_off_the_gpu_are_refused(kvt_pkg):
    from kvtier import block_kv
    p = _pool()
    with pytest.raises(AssertionError):
        _decode()
    with pytest.raises(AssertionError):
        block_kv.kvt_block_prefill(torch.zeros(2, 4, 64, dtype=torch.float16), _i(0, 1, 2), p["k8"], p["v8"], p["ks"],
                                   p["vs"], p["block_table"], _i(1, 1))
    with pytest.raises(AssertionError):
        x = torch.zeros(2, 2, 64)
        block_kv.kvt_block_store(x, x, _i(0, 1, 2), _i(1, 1), p["k8"], p["v8"], p["ks"], p["vs"], p["block_table"])
    with pytest.raises(AssertionError):
        block_kv.kvt_block_plan(_i(0), _i(1), _i(0, 0), p["block_table"], _i(0, 1), _i(0), 1)


@pytest.mark.parametrize("over", [dict(k8=torch.zeros(4, 2, 16, 64, dtype=torch.uint8)), dict(v8=torch.zeros(4, 2, 16, 64, dtype=torch.int8)),
                                  dict(ks=torch.zeros(4, 1)), dict(vs=torch.zeros(4, 2, dtype=torch.float16)),
                                  dict(block_table=torch.zeros(2, 3, dtype=torch.int64)),
                                  dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16)),
                                  dict(kv_lens=torch.zeros(2, dtype=torch.int64)),
                                  dict(seqs=torch.zeros(2, dtype=torch.int64)),
                                  dict(out=torch.zeros(2, 4, 64, dtype=torch.float64))])
def test_decode_contract(kvt_pkg, over):
    with pytest.raises(AssertionError):
        _decode(**over)


@pytest.mark.parametrize("over", [dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 5, 64, dtype=torch.bfloat16)),
                                  dict(q=torch.zeros(2, 34, 64, dtype=torch.bfloat16)), dict(seqs=torch.zeros(1, dtype=torch.int32)),
                                  dict(block_table=torch.zeros(1, 3, dtype=torch.int32)),
                                  dict(_pool(H=0)), dict(_pool(B=48)), dict(_pool(D=96), q=torch.zeros(2, 4, 96, dtype=torch.bfloat16))])
def test_decode_sizes(kvt_pkg, over):
    with pytest.raises(ValueError):
        _decode(**over)


def test_plan_contract(kvt_pkg):
    from kvtier import block_kv
    ok = dict(seqs=_i(0), counts=_i(1), seq_lens=_i(0, 0), block_table=torch.zeros(2, 3, dtype=torch.int32),
              free_list=_i(0, 1), free_head=_i(0), n_tokens=1)
    for bad in (dict(seqs=torch.zeros(1, dtype=torch.int64)), dict(free_head=torch.zeros(1)),
                dict(block_table=torch.zeros(2, 3)), dict(req_to_token=torch.zeros(2, 9, dtype=torch.int64))):
        with pytest.raises(AssertionError):
            block_kv.kvt_block_plan(**{**ok, **bad})
    for bad in (dict(counts=_i()), dict(seq_lens=_i(0)), dict(req_to_token=torch.zeros(1, 9, dtype=torch.int32))):
        with pytest.raises(ValueError):
            block_kv.kvt_block_plan(**{**ok, **bad})


def test_cache_refusals(kvt_pkg):
    from kvtier.block_kv import BlockKVCache
    for bad in (dict(dtype=torch.uint8), dict(block=48), dict(D=96), dict(n_blocks=2 ** 28)):
        with pytest.raises(ValueError):
            BlockKVCache(**{**dict(layers=0, H=1, D=64, n_blocks=2, max_seqs=1, max_blocks=2, device="cpu"), **bad})
    c = BlockKVCache(1, 1, 64, 2, 1, 2, device="cpu")
    s = c.add_seq()
    with pytest.raises(RuntimeError):
        c.add_seq()
    with pytest.raises(ValueError):
        c.release(s + 1)
    with pytest.raises(ValueError):
        c.plan(_i(0), _i(1))                     # device counts need a host bound
    c.release(s)
    with pytest.raises(ValueError):
        c.release(s)
    assert c.add_seq() == s
    c.status.fill_(3)
    with pytest.raises(RuntimeError, match="pool exhausted, block table row full"):
        c.check()
    c.check()


def test_release_gives_blocks_back(kvt_pkg):
    from kvtier.block_kv import BlockKVCache
    c = BlockKVCache(1, 1, 64, 6, 2, 3, device="cpu", block=16)
    s = c.add_seq()
    ids = c.free_list[:3].tolist()
    c.block_table[s] = torch.tensor([ids[0], ids[1], -1], dtype=torch.int32)   # (the third found no block)
    c.seq_lens[s], c.free_head[0] = 40, 3
    c.release(s)
    assert int(c.free_head) == 1 and c.free_list[1:3].tolist() == ids[:2]
    assert c.block_table[s].tolist() == [-1] * 3 and int(c.seq_lens[s]) == 0


def test_c_entries_refuse_sizes(kvt_pkg):
    """EINVAL / ERANGE come before any pointer is looked at or anything is launched."""
    L = kvt_pkg._lib.lib()
    N = None

    def plan(n=1, rows=1, stride=4, max_blocks=4, n_free=4, block=64, n_tokens=1, rtt=N, rtt_stride=0, rtt_cols=0):
        return L.kvt_block_plan(n, N, N, N, rows, N, stride, max_blocks, N, n_free, N, block, n_tokens, N, N, N, N, N, rtt,
                                rtt_stride, rtt_cols, 0, N)
    for bad in (dict(n=0), dict(n=1025), dict(rows=0), dict(max_blocks=0), dict(stride=3), dict(n_free=-1), dict(block=48),
                dict(n_tokens=-1), dict(rtt=64, rtt_stride=4, rtt_cols=5)):
        assert plan(**bad) == -1, bad
    assert plan(n_tokens=2 ** 30 + 1) == -3 and plan(n_free=2 ** 26) == -3

    def store(dtype=0, s=64, n_tokens=1, H=1, D=64, n=1, n_rows=1, stride=4, max_blocks=4, code=0, n_blocks=1, block=64, k=N):
        return L.kvt_block_store(k, N, dtype, s, s, s, s, n_tokens, H, D, N, N, n, N, N, stride, n_rows, max_blocks, code, N,
                                 N, N, N, n_blocks, block, N)
    for bad in (dict(dtype=3), dict(s=60), dict(dtype=2, s=62), dict(n_tokens=-1), dict(H=0), dict(D=96), dict(n=0),
                dict(n=4097, n_rows=4097), dict(n=2), dict(stride=3), dict(max_blocks=0), dict(code=2), dict(n_blocks=0),
                dict(block=8), dict(k=8)):
        assert store(**bad) == -1, bad
    assert store(H=65536) == -3 and store(n_tokens=2 ** 30, H=16, block=16) == -3
    assert store(n_tokens=0) == 0                # nothing to do, nothing launched

    def attn(fn, n=1, H=1, Hq=1, D=64, code=0, n_blocks=1, block=64, stride=4, n_rows=1, max_blocks=4, splits=1, s=64, qt=0,
             ot=0, q=N, n_q=1, cu=64, item_rows=16, scale=1.0, part=N, so=None, out=N):
        head = (q, s, s, qt) + ((cu, n_q) if fn == "kvt_block_prefill" else ())
        mid = (0,) if fn == "kvt_block_prefill" else ()
        rows = (item_rows,) if fn == "kvt_block_prefill" else ()
        return getattr(L, fn)(*head, N, n, H, Hq, D, code, N, N, N, N, n_blocks, block, N, stride, n_rows, max_blocks, N, *mid,
                              scale, *rows, splits, part, part, N, out, ot, s if so is None else so, s if so is None else so, N)
    for fn in ("kvt_block_decode", "kvt_block_prefill"):
        for bad in (dict(n=0), dict(n=4097, n_rows=4097), dict(n=2), dict(H=0), dict(Hq=0), dict(H=2, Hq=3), dict(Hq=17),
                    dict(D=32), dict(code=2), dict(n_blocks=0), dict(block=128), dict(stride=3), dict(n_rows=0),
                    dict(max_blocks=0), dict(splits=0), dict(splits=2), dict(s=60), dict(qt=2), dict(ot=3), dict(q=8),
                    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(out=8), dict(so=60), dict(ot=2, so=62)):
            assert attn(fn, **bad) == -1, (fn, bad)
        assert attn(fn, max_blocks=2 ** 26, stride=2 ** 26) == -3
    assert attn("kvt_block_prefill", n_q=-1) == -1 and attn("kvt_block_prefill", cu=N) == -1
    assert attn("kvt_block_prefill", item_rows=32) == -1 and attn("kvt_block_prefill", n_q=2 ** 20, Hq=1) == -3
    assert attn("kvt_block_decode", splits=1025) == -3 and attn("kvt_block_decode", splits=-65536) == -1
    assert attn("kvt_block_decode", splits=-65536, part=64) == -3 and attn("kvt_block_prefill", splits=-2) == -1
    assert attn("kvt_block_decode", splits=-2 ** 31, part=64) == -3 and attn("kvt_block_decode", splits=-65536, H=2 ** 16, Hq=2 ** 16) == -3
    assert attn("kvt_block_prefill", n_q=2 ** 30, H=2 ** 4, Hq=2 ** 4, item_rows=128) == -3      # (2^32 threads)
    assert attn("kvt_block_prefill", n_q=0) == 0


def test_attention_refuses_tables_whose_positions_run_past_32_bits(kvt_pkg):
    """The kernels' 32-bit positions run up to 4,096 ahead of a request's last one: tables within 8,192 of 2^31 are ERANGE."""
    L = kvt_pkg._lib.lib()
    for block in (16, 32, 64):
        for positions in (2 ** 31 - block, 2 ** 31 - 8192 + block):
            m = positions // block
            tail = (1.0, 1, None, None, None, None, 0, 64, 64, None)
            pool = (0, None, None, None, None, 1, block, None, m, 1, m, None)
            assert L.kvt_block_decode(None, 64, 64, 0, None, 1, 1, 1, 64, *pool, *tail) == -3, (block, positions)
            for rows in (16, 128):
                assert L.kvt_block_prefill(None, 64, 64, 0, 64, 1, None, 1, 1, 1, 64, *pool, 1, 1.0, rows, *tail[1:]) == -3


def test_block_kernels_hold_no_instructions_in_asm(kvt_pkg):
    """The compiler puts no wait before asm that reads a matrix product's result, so the kernels' asm is empty (a register is
    pinned) or a wait."""
    import os
    import re
    src = os.path.join(os.path.dirname(kvt_pkg._lib.__file__), "csrc")
    for name in sorted(f for f in os.listdir(src) if f.startswith("block_")):
        with open(os.path.join(src, name)) as f:
            for text in re.findall(r"\basm\b(?:\s+volatile)?\s*\(\s*((?:\"[^\"]*\"\s*)+)", f.read()):
                assert re.fullmatch(r'"(s_waitcnt vmcnt\(0\))?"\s*', text), (name, text)


@pytest.mark.parametrize("shape,strides", [((1, 2, 64), (133, 64, 1)), ((3, 1, 64), (64, 1, 1)), ((1, 1, 64), (7, 5, 1)),
                                           ((3, 1, 64), (72, 3, 1))])
def test_strides_of_single_entries_do_not_matter(kvt_pkg, shape, strides):
    """One token, or one head, out of an odd-pitched buffer is taken as it is; off a 16-byte boundary it is copied once, and the
    copy's strides are ones that the entry points take."""
    from kvtier import block_kv
    buf = torch.arange(1024, dtype=torch.float32)
    for dtype, per16 in ((torch.float16, 8), (torch.float32, 4)):
        b = buf.to(dtype)
        base = -b.data_ptr() % 16 // b.element_size()
        for off in (0, 1):
            x = b.as_strided(shape, strides, base + off)
            y, p, sn, sh = block_kv._rows16(x, per16)
            assert p == y.data_ptr() and p % 16 == 0 and sn % per16 == 0 and sh % per16 == 0
            assert (y is x) == (off == 0)
            at = y.as_strided(shape, (sn, sh, 1)) if off == 0 else y
            assert torch.equal(at, x)
