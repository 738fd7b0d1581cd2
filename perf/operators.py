"""Performance cases of the 8-bit block cache: keys and values held in 8 bits (e4m3 or int8) in blocks of B tokens, with
one power-of-two scale per block, KV head and side.

Four operators, as a serving step calls them:

  plan    block tables and slot maps on the device from the requests' lengths and the step's token counts
  store   quantizing write of the step's K/V rows into their blocks, growing a block's scale where it has to
  decode  attention of one query token per request over its blocks
  chunk   attention of a chunk of query tokens per request, causal, or over another sequence's states (cross attention)

Layouts: k8 / v8 [n_blocks, H, B, D] codes, ks / vs fp32 [n_blocks, H] scales, block_table int32 [rows, max_blocks],
cu int32 [n + 1] prefix sums of token counts, kv_lens int32 [n] lengths with the step's tokens counted.

`run` computes an operator from elementary torch operations where `own` is false and calls the framework's operator
where it is true; `exact` restates it in 64 bits.  K is N(0, 1) with one channel in 32 eight times larger (the outlier
channels of real keys), V is N(0, 1), queries are N(0, 1): scores spread over several units.  Lengths and counts follow
from the case alone (log-uniform, the longest as stated), values, table rows and block ids from the seed.
"""
import math
import random

import torch

own = False

QMAX = {"fp8": 448.0, "int8": 127.0}
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
IO = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MIN_EXP, MAX_EXP = -64, 122
#: (query heads, KV heads, head size) of the attention cases that are drawn
HEADS = [(16, 2, 256), (24, 2, 256), (12, 1, 128), (64, 8, 128), (8, 8, 128), (20, 20, 64), (32, 4, 64)]


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 conversations: one token each, some of which open a block
        dict(name="plan_decode", op="plan", batch=64, len=16384, new=1, block=64, rtt=False),
        # prompt ingestion of many requests at once, blocks of 16, with the slot table of the slot-indexed readers
        dict(name="plan_prompts", op="plan", batch=512, len=4096, new=2500, block=16, rtt=True),
        # the write of a decode step: one token per request into a block that holds some already
        dict(name="store_decode", op="store", batch=32, len=4000, new=1, h=2, d=256, block=64, kv="fp8", io="bf16"),
        # the write of a prompt chunk: some 8,000 tokens over a few requests, each going on inside a block
        dict(name="store_prompt", op="store", batch=4, len=1500, new=3600, h=2, d=256, block=64, kv="fp8", io="bf16"),
        # many short prompts of a model with more, smaller heads, int8 codes, fp16 rows, blocks of 16
        dict(name="store_int8", op="store", batch=48, len=900, new=1400, h=8, d=128, block=16, kv="int8", io="f16"),
        # one short conversation: latency and launches count
        dict(name="decode_short", op="decode", batch=1, len=777, hq=24, h=2, d=256, block=64, kv="fp8", io="bf16"),
        # a mixed batch of medium contexts, the served model's heads
        dict(name="decode_ragged", op="decode", batch=32, len=16384, hq=24, h=2, d=256, block=64, kv="fp8", io="bf16"),
        # the longest conversation, alone
        dict(name="decode_262k", op="decode", batch=1, len=262144, hq=16, h=2, d=256, block=64, kv="fp8", io="bf16"),
        # a full serving batch of a model with 8 KV heads, int8 codes, blocks of 16
        dict(name="decode_int8", op="decode", batch=64, len=8191, hq=64, h=8, d=128, block=16, kv="int8", io="f16"),
        # a short chunk behind a long prefix, on a rank that holds one KV head: few rows, long axis
        dict(name="chunk_prefix", op="chunk", batch=1, len=60000, new=61, hq=12, h=1, d=128, block=64, kv="fp8",
             io="bf16", causal=True),
        # a whole prompt of 10,001 tokens
        dict(name="chunk_prompt", op="chunk", batch=1, len=10001, new=10001, hq=16, h=2, d=256, block=64, kv="fp8",
             io="bf16", causal=True),
        # decoder rows over an encoder's cached states, of other lengths: cross attention
        dict(name="chunk_cross", op="chunk", batch=8, len=1500, new=448, hq=20, h=20, d=64, block=32, kv="int8",
             io="f16", causal=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["plan", "store", "decode", "decode", "chunk", "chunk"])
    block = rng.choice([16, 32, 64])
    kv = rng.choice(["fp8", "int8"])
    if op == "plan":
        batch = _log_int(rng, 1, 700)
        return dict(op=op, batch=batch, len=_log_int(rng, 1, 8000), new=_log_int(rng, 1, min(4000, 500_000 // batch)),
                    block=block, rtt=rng.random() < 0.5)
    if op == "store":
        _, h, d = rng.choice(HEADS)
        batch = _log_int(rng, 1, 64)
        return dict(op=op, batch=batch, len=_log_int(rng, 1, 4000), new=_log_int(rng, 1, max(1, 12_000 // batch)),
                    h=h, d=d, block=block, kv=kv, io=rng.choice(["bf16", "bf16", "f16", "f32"]))
    hq, h, d = rng.choice(HEADS)
    io = rng.choice(["bf16", "f16"])
    if op == "decode":
        batch = _log_int(rng, 1, 64)
        return dict(op=op, batch=batch, len=_log_int(rng, 1, min(262_144, 130_000_000 // (batch * h * d))), hq=hq, h=h,
                    d=d, block=block, kv=kv, io=io)
    batch = _log_int(rng, 1, 8)
    pairs = 150_000_000_000 // (batch * hq * d)                      # (query, position) pairs of a request at most
    new = _log_int(rng, 2, min(5000, math.isqrt(pairs) // 2))
    return dict(op=op, batch=batch, len=new + _log_int(rng, 1, min(60_000, pairs // new - new)), new=new, hq=hq, h=h, d=d,
                block=block, kv=kv, io=io, causal=rng.random() < 0.75)


def _lengths(case):
    """(tokens held before the step, tokens of the step) of each request, from the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, op = case["batch"], case["op"]
    if op == "decode":
        return [0] * n, [case["len"]] + [_log_int(rng, max(1, case["len"] // 16), case["len"]) for _ in range(n - 1)]
    if op == "chunk":
        new = [case["new"]] + [_log_int(rng, max(1, case["new"] // 8), case["new"]) for _ in range(n - 1)]
        if not case["causal"]:   # lengths of the other sequence: nothing to do with the queries'
            return [0] * n, new
        return [case["len"] - new[0]] + [rng.randint(0, case["len"] - m) for m in new[1:]], new
    old = [rng.randint(0, case["len"]) for _ in range(n)]
    if case["new"] == 1:
        return old, [1] * n
    return old, [case["new"]] + [_log_int(rng, max(1, case["new"] // 8), case["new"]) for _ in range(n - 1)]


def _kv_lengths(case):
    old, new = _lengths(case)
    if case["op"] == "chunk" and not case["causal"]:
        rng = random.Random(case["len"])
        return [case["len"]] + [_log_int(rng, max(1, case["len"] // 8), case["len"]) for _ in old[1:]]
    return [a + b for a, b in zip(old, new)]


# ------------------------------------------------------------------------------------------------------------ inputs
def _prefix(values):
    out = [0]
    for x in values:
        out.append(out[-1] + x)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case, held, planned, gen):
    """Block ids in a random order: a table with the blocks of `held` tokens per row, and the order itself."""
    b = case["block"]
    blocks = [-(-x // b) for x in held]
    total = sum(-(-x // b) for x in planned) + 3
    order = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(held), max(1, max(-(-x // b) for x in planned))), -1, dtype=torch.int32, device="cuda")
    cu = _prefix(blocks)
    for r, n in enumerate(blocks):
        table[r, :n] = order[cu[r]:cu[r + 1]]
    return table, order, cu[-1]


def _pow2(amax, qmax):
    """The smallest power of two s with amax / s <= qmax, as fp32, within 2^MIN_EXP .. 2^MAX_EXP."""
    m, e = torch.frexp(amax)
    top, bits = math.frexp(qmax)
    e = (e - bits + (m > top)).clamp(MIN_EXP, MAX_EXP)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return ((e.int() + 127) << 23).view(torch.float32)


def _codes(x, kv):
    """fp32 values within the codes' range -> codes, rounded to nearest even."""
    return x.to(torch.float8_e4m3fn) if kv == "fp8" else x.round().to(torch.int8)


def _keys(shape, h, d, gen):
    gain = torch.ones(h, d, device="cuda")
    gain[:, torch.randperm(d, generator=gen, device="cuda")[:max(1, d // 32)]] = 8.0
    return torch.randn(shape, generator=gen, device="cuda"), gain


def _pool(case, n_blocks, gen):
    """Codes and scales of a pool whose every block is full."""
    h, b, d = case["h"], case["block"], case["d"]
    k, gain = _keys((n_blocks, h, b, d), h, d, gen)
    out = []
    for x in (k * gain[:, None], torch.randn((n_blocks, h, b, d), generator=gen, device="cuda")):
        s = _pow2(x.abs().amax((2, 3)), QMAX[case["kv"]])
        out.append((_codes(x / s[..., None, None], case["kv"]), s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    old, new = _lengths(case)
    n = len(old)
    s = dict(case=dict(case))
    if case["op"] == "plan":
        table, order, used = _table(case, old, [a + b for a, b in zip(old, new)], gen)
        rows = torch.randperm(n, generator=gen, device="cuda")
        spread = torch.full_like(table, -1)
        spread[rows] = table
        lens = torch.zeros(n, dtype=torch.int32, device="cuda")
        lens[rows] = _i32(old)
        s.update(seqs=rows.int(), counts=_i32(new), seq_lens=lens, block_table=spread, free_list=order,
                 free_head=_i32([used]), n_tokens=sum(new), status=_i32([0]),
                 req_to_token=torch.zeros(n, spread.shape[1] * case["block"], dtype=torch.int32, device="cuda")
                 if case["rtt"] else None)
        return s
    kv_lens = _kv_lengths(case)
    table, _, used = _table(case, kv_lens, kv_lens, gen)
    k8, v8, ks, vs = _pool(case, used + 3, gen)
    s.update(k8=k8, v8=v8, ks=ks, vs=vs, block_table=table, kv_lens=_i32(kv_lens))
    if case["op"] == "store":
        k, gain = _keys((sum(new), case["h"], case["d"]), case["h"], case["d"], gen)
        level = 2.0 ** (torch.rand(sum(new), 1, 1, generator=gen, device="cuda") - 0.5)   # rows differ in size
        s.update(k=(k * gain * level).to(IO[case["io"]]),
                 v=(torch.randn(k.shape, generator=gen, device="cuda") * level).to(IO[case["io"]]),
                 cu=_i32(_prefix(new)))
        return s
    rows = n if case["op"] == "decode" else sum(new)
    s.update(q=torch.randn(rows, case["hq"], case["d"], generator=gen, device="cuda").to(IO[case["io"]]), workspace={})
    if case["op"] == "chunk":
        s.update(cu_q=_i32(_prefix(new)), max_q=max(new), max_len=max(kv_lens))
    else:
        s.update(max_len=max(kv_lens))
    return s


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return _run_own(s)
    return {"plan": _plan, "store": _store, "decode": _decode, "chunk": _chunk}[s["case"]["op"]](s)


def _run_own(s):
    from kvtier import block_kv

    op = s["case"]["op"]
    if op == "plan":
        p = block_kv.kvt_block_plan(s["seqs"], s["counts"], s["seq_lens"], s["block_table"], s["free_list"], s["free_head"],
                                    s["n_tokens"], block=s["case"]["block"], status=s["status"],
                                    req_to_token=s["req_to_token"], commit=False)
        out = dict(cu=p.cu, slots=p.slots, kv_lens=p.kv_lens, next_head=p.next_head, block_table=s["block_table"],
                   status=s["status"])
        return out if s["req_to_token"] is None else dict(out, req_to_token=s["req_to_token"])
    if op == "store":
        block_kv.kvt_block_store(s["k"], s["v"], s["cu"], s["kv_lens"], s["k8"], s["v8"], s["ks"], s["vs"],
                                 s["block_table"])
        return dict(k8=s["k8"], v8=s["v8"], ks=s["ks"], vs=s["vs"])
    if op == "decode":
        return block_kv.kvt_block_decode(s["q"], s["k8"], s["v8"], s["ks"], s["vs"], s["block_table"], s["kv_lens"],
                                         workspace=s["workspace"])
    return block_kv.kvt_block_prefill(s["q"], s["cu_q"], s["k8"], s["v8"], s["ks"], s["vs"], s["block_table"],
                                      s["kv_lens"], causal=s["case"]["causal"], workspace=s["workspace"])


def _plan(s):
    b = s["case"]["block"]
    seqs, table = s["seqs"].long(), s["block_table"]
    counts, old = s["counts"].long(), s["seq_lens"][seqs].long()
    cu = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    kv_lens = old + counts
    first, last = (old + b - 1) // b, (kv_lens + b - 1) // b       # the blocks that a request opens
    taken = (last - first).cumsum(0) - (last - first)
    head = s["free_head"].long()
    lp = torch.arange(table.shape[1], device="cuda")[None]
    opens = (lp >= first[:, None]) & (lp < last[:, None])
    at = (head + taken[:, None] + lp - first[:, None]).clamp(0, s["free_list"].numel() - 1)
    rows = torch.where(opens, s["free_list"][at], table[seqs])
    table[seqs] = rows
    t = torch.arange(s["n_tokens"], device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True)
    pos = old[r] + t - cu[r]
    slots = (rows[r, pos // b] * b + pos % b).int()
    out = dict(cu=cu.int(), slots=slots, kv_lens=kv_lens.int(), next_head=(head + (last - first).sum()).int(),
               block_table=table, status=s["status"])
    if s["req_to_token"] is not None:
        s["req_to_token"][seqs[r], pos] = slots
        out["req_to_token"] = s["req_to_token"]
    return out


def _store(s):
    b, kv = s["case"]["block"], s["case"]["kv"]
    cu, kv_lens, table = s["cu"].long(), s["kv_lens"].long(), s["block_table"].long()
    old = kv_lens - (cu[1:] - cu[:-1])
    t = torch.arange(s["k"].shape[0], device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True)
    pos = old[r] + t - cu[r]
    block, row = table[r, pos // b], pos % b
    part = table[torch.arange(old.numel(), device="cuda"), old // b]     # the block a request goes on in, if it is open
    held = torch.arange(b, device="cuda")[None] < (old % b)[:, None]     # and the rows it holds
    for x, codes, scale in ((s["k"], s["k8"], s["ks"]), (s["v"], s["v8"], s["vs"])):
        x = x.float()
        amax = torch.zeros_like(scale).index_reduce_(0, block, x.abs().amax(-1), "amax")
        need = _pow2(amax, QMAX[kv])
        before = torch.zeros_like(scale)
        before[part] = torch.where(held.any(1)[:, None], scale[part], before[part])
        after = torch.maximum(need, before)
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
        touched[block] = True
        raw = codes.view(torch.int8)                                     # (moved as bytes)
        was = raw[part]
        grown = _codes(was.view(CODE[kv]).float() * (before[part] / after[part])[..., None, None], kv).view(torch.int8)
        raw[part] = torch.where(held[:, None, :, None], grown, was)
        scale.copy_(torch.where(touched[:, None], after, scale))
        raw[block, :, row] = _codes(x / after[block][..., None], kv).view(torch.int8)
    return dict(k8=s["k8"], v8=s["v8"], ks=s["ks"], vs=s["vs"])


def _gathered(s):
    """fp32 K, V [n, H, positions, D] of every request, padded to the longest."""
    b = s["case"]["block"]
    table = s["block_table"][:, :-(-s["max_len"] // b)].long().clamp(min=0)
    out = []
    for codes, scale in ((s["k8"], s["ks"]), (s["v8"], s["vs"])):
        x = codes.view(torch.int8)[table].view(codes.dtype).float()       # [n, blocks, H, B, D]
        x = x * scale[table][..., None, None]
        out.append(x.transpose(1, 2).flatten(2, 3))
    return out


def _softmax_v(q, k, v, visible):
    """softmax(q k^T) v for q [n, H, rows, D]; row i of request n sees the first visible[n, i] positions."""
    x = torch.matmul(q, k.transpose(2, 3).contiguous())
    gone = torch.arange(k.shape[2], device="cuda")[None, None] >= visible[..., None]
    x.masked_fill_(gone[:, None], float("-inf"))
    p = (x - x.amax(-1, keepdim=True)).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _decode(s):
    q, h, d = s["q"], s["case"]["h"], s["case"]["d"]
    k, v = _gathered(s)
    g = q.shape[1] // h
    x = q.float().view(-1, h, g, d) * d ** -0.5
    o = _softmax_v(x, k, v, s["kv_lens"][:, None].expand(-1, g))
    return o.reshape(q.shape).to(q.dtype)


def _chunk(s):
    q, h, d, cu = s["q"], s["case"]["h"], s["case"]["d"], s["cu_q"].long()
    k, v = _gathered(s)
    n, g, m = cu.numel() - 1, q.shape[1] // h, s["max_q"]
    j = torch.arange(m, device="cuda")[None]
    at = (cu[:-1, None] + j).clamp(max=q.shape[0] - 1)
    x = (q[at].float() * d ** -0.5).view(n, m, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * m, d)
    visible = s["kv_lens"][:, None].expand(n, m)
    if s["case"]["causal"]:
        visible = visible - (cu[1:] - cu[:-1])[:, None] + j + 1
    visible = visible.clamp(min=1)                                        # padding rows: anything but nothing
    o = _softmax_v(x, k, v, visible.repeat(1, g))
    o = o.view(n, h, g, m, d).permute(0, 3, 1, 2, 4).reshape(n, m, h * g, d)
    t = torch.arange(q.shape[0], device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True)
    return o[r, t - cu[r]].to(q.dtype)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    old, new = _lengths(case)
    b = case["block"]
    if case["op"] == "plan":
        blocks = sum(-(-(x + y) // b) - -(-x // b) for x, y in zip(old, new))
        per_token = 8 if case["rtt"] else 4
        return {"bytes": sum(new) * per_token + blocks * 8 + len(old) * 20, "flops": 0}
    h, d = case["h"], case["d"]
    kv = _kv_lengths(case)
    if case["op"] == "store":
        blocks = sum(-(-(x + y) // b) - x // b for x, y in zip(old, new))
        return {"bytes": 2 * sum(new) * h * d * (IO[case["io"]].itemsize + 1) + blocks * (8 * h + 4), "flops": 0}
    blocks = sum(-(-x // b) for x in kv)
    read = 2 * sum(kv) * h * d + blocks * (8 * h + 4)
    hq, pairs = case["hq"], sum(kv)
    rows = len(kv)
    if case["op"] == "chunk":
        rows = sum(new)
        pairs = sum(x * y for x, y in zip(kv, new))
        if case["causal"]:
            pairs -= sum(y * (y - 1) // 2 for y in new)
    return {"bytes": read + 4 * rows * hq * d, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------------- exact
def _round_e4m3(x):
    """float64 -> the nearest e4m3 value (ties to even), |x| <= 448."""
    e = torch.frexp(x.abs())[1].clamp(min=-5).double() - 4      # spacing 2^(exponent - 3), subnormals 2^-9
    step = torch.exp2(e)
    return torch.round(x / step) * step


def _exact_scale(amax, kv):
    if amax == 0:
        return 2.0 ** MIN_EXP
    e = math.ceil(math.log2(amax / QMAX[kv]))
    while amax / 2.0 ** e > QMAX[kv]:
        e += 1
    while amax / 2.0 ** (e - 1) <= QMAX[kv]:
        e -= 1
    return 2.0 ** min(max(e, MIN_EXP), MAX_EXP)


def _exact_store(case, s):
    b, kv = case["block"], case["kv"]
    old, new = _lengths(case)
    table, cu = s["block_table"].tolist(), _prefix(new)
    out = {}
    for name, x, codes, scale in (("k", s["k"], s["k8"], s["ks"]), ("v", s["v"], s["v8"], s["vs"])):
        x, codes, scale = x.double(), codes.double(), scale.double()
        top = x.abs().amax(-1).cpu()
        for r, (first, count) in enumerate(zip(old, new)):
            p = first
            while p < first + count:
                end = min(first + count, (p // b + 1) * b)
                block, held, t0, t1 = table[r][p // b], p % b, cu[r] + p - first, cu[r] + end - first
                size = [_exact_scale(a, kv) for a in top[t0:t1].amax(0).tolist()]
                if held:
                    before = scale[block].tolist()
                    size = [max(a, c) for a, c in zip(size, before)]
                    y = codes[block, :, :held] * (scale[block] / torch.tensor(size, device="cuda").double())[:, None, None]
                    codes[block, :, :held] = _round_e4m3(y) if kv == "fp8" else y.round()
                scale[block] = torch.tensor(size, dtype=torch.float64, device="cuda")
                y = x[t0:t1].transpose(0, 1) / scale[block][:, None, None]
                codes[block, :, held:held + end - p] = _round_e4m3(y) if kv == "fp8" else y.round()
                p = end
        out[name + "8"], out[name + "s"] = (codes if kv == "fp8" else None), scale
    return dict(k8=out["k8"], v8=out["v8"], ks=out["ks"], vs=out["vs"])


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(case, s)
    b, g = case["block"], case["hq"] // case["h"]
    _, new = _lengths(case)
    if case["op"] == "decode":
        new = [1] * len(new)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    cu = _prefix(new)
    for r, (length, m) in enumerate(zip(_kv_lengths(case), new)):
        blocks = s["block_table"][r, :-(-length // b)].long()
        for h in range(case["h"]):
            k, v = ((c.view(torch.int8)[blocks, h].view(c.dtype).double() * z[blocks, h].double()[:, None, None]).flatten(0, 1)[:length]
                    for c, z in ((s["k8"], s["ks"]), (s["v8"], s["vs"])))
            for j in range(g):
                x = s["q"][cu[r]:cu[r + 1], h * g + j].double() @ k.t().contiguous() / math.sqrt(case["d"])
                if case["op"] == "chunk" and case["causal"]:
                    last = length - m + torch.arange(m, device="cuda")
                    x.masked_fill_(torch.arange(length, device="cuda")[None] > last[:, None], float("-inf"))
                out[cu[r]:cu[r + 1], h * g + j] = torch.softmax(x, -1) @ v
    return out
