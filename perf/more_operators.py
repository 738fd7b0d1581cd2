"""Performance cases of a long conversation kept within a budget of the 8-bit block cache: keys and queries rotated to their
positions, attention weight accumulated per cache entry, the lightest entries evicted, their blocks given back.

Five operators, as a serving step calls them:

  rope    rotary positions on a step's queries and keys: half and interleaved layouts, part of the head, scaled frequencies
  weigh   softmax weights of the step's queries (one per request, or a causal chunk), summed over queries and the q heads
          of a KV head, added to the weight of each entry
  keep    which entries stay: the heaviest, with the first `sinks` and the last `recent` positions always among them
  evict   the entries that stay move into the places of those that go; a block that changes gets its scale anew
  trim    lengths are cut to the budget, blocks behind it return to the free list

Layouts: k8 / v8 [n_blocks, H, B, D] codes (e4m3 or int8), ks / vs fp32 [n_blocks, H] power-of-two scales, block_table int32
[rows, max_blocks], kv_lens int32 [n], weights fp32 and pos int32 [rows, H, max_blocks * B]; cu int32 [n + 1] prefix sums of
token counts.  Entry e of a head that was never moved (e >= held) sits at position e + evicted of its conversation, another
one at pos[e].  `src` int32 [n, H, budget]: the entry that goes to place e (itself where it stays, -1 where there is none);
entries from behind the budget, in order, fill the places that become free, in order.

`run` computes an operator from elementary torch operations where `own` is false and calls the framework's operator
where it is true; `exact` restates it in 64 bits.  Queries are N(0, 1), K is N(0, 1) with one channel in 32 eight times
larger (the outlier channels of real keys), V is N(0, 1); accumulated weights are log-normal (a few entries hold most),
with some equal ones and zeros among them.  Lengths and counts follow from the case alone, values, table rows and block
ids from the seed.
"""
import math
import random

import torch

own = False

QMAX = {"fp8": 448.0, "int8": 127.0}
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
IO = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MIN_EXP, MAX_EXP = -64, 122
SINKS = 4
#: (query heads, KV heads, head size) of the drawn cases
HEADS = [(16, 2, 256), (24, 2, 256), (12, 1, 128), (64, 8, 128), (8, 8, 128), (20, 20, 64), (32, 4, 64)]


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 long conversations, a quarter of the head rotated: latency counts
        dict(name="rope_decode", op="rope", batch=64, new=1, hq=24, h=2, d=256, rot=64, io="bf16", inter=False, scaled=False,
             fused=False, far=262144),
        # prompt chunks of a model that interleaves the pairs and stretches its context, q and k in one projection's output
        dict(name="rope_prompt", op="rope", batch=3, new=4001, hq=64, h=8, d=128, rot=128, io="f16", inter=True, scaled=True,
             fused=True, far=131072),
        # the heavy-hitter sums of a mixed decode batch
        dict(name="weigh_decode", op="weigh", batch=32, len=16384, new=1, hq=24, h=2, d=256, block=64, kv="fp8", io="bf16",
             fresh=False),
        # a full serving batch with 8 KV heads, int8 codes, blocks of 16
        dict(name="weigh_int8", op="weigh", batch=64, len=8191, new=1, hq=64, h=8, d=128, block=16, kv="int8", io="f16",
             fresh=False),
        # a long prompt weighed by its last 61 queries only, before it is cut down
        dict(name="weigh_window", op="weigh", batch=1, len=60000, new=61, hq=12, h=1, d=128, block=64, kv="fp8", io="bf16",
             fresh=True),
        # a whole prompt of 10,001 tokens weighed by all of its queries
        dict(name="weigh_prompt", op="weigh", batch=1, len=10001, new=10001, hq=16, h=2, d=256, block=64, kv="fp8",
             io="bf16", fresh=False),
        # a serving batch that has grown one block over its budget
        dict(name="keep_steady", op="keep", batch=64, len=4160, budget=4096, recent=256, h=8, block=64),
        # the longest prompt, cut to a sixteenth
        dict(name="keep_prompt", op="keep", batch=1, len=262144, budget=16384, recent=1000, h=2, block=64),
        # the same batch's entries moved: a row or two of most blocks
        dict(name="evict_steady", op="evict", batch=64, len=4160, budget=4096, h=8, d=128, block=64, kv="fp8"),
        # prompts of some 30,000 tokens cut to 8,192: most places change
        dict(name="evict_prompt", op="evict", batch=4, len=30011, budget=8192, h=2, d=256, block=32, kv="int8"),
        # a block of each of 64 conversations given back
        dict(name="trim_steady", op="trim", batch=64, len=4160, budget=4096, block=64),
        # long prompts' tails given back, blocks of 16
        dict(name="trim_prompts", op="trim", batch=200, len=12000, budget=2048, block=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["rope", "weigh", "weigh", "keep", "evict", "evict", "trim"])
    block = rng.choice([16, 32, 64])
    hq, h, d = rng.choice(HEADS)
    batch = _log_int(rng, 1, 64)
    if op == "rope":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 80_000_000 // (batch * (hq + h) * d)))
        return dict(op=op, batch=batch, new=new, hq=hq, h=h, d=d, rot=rng.choice([d, d, d // 2, d // 4, 20]),
                    io=rng.choice(["bf16", "bf16", "f16", "f32"]), inter=rng.random() < 0.5, scaled=rng.random() < 0.5,
                    fused=rng.random() < 0.5, far=_log_int(rng, 8000, 1_000_000))
    if op == "weigh":
        kv, io = rng.choice(["fp8", "int8"]), rng.choice(["bf16", "f16"])
        if rng.random() < 0.5:
            return dict(op=op, batch=batch, len=_log_int(rng, 1, min(262_144, 130_000_000 // (batch * h * d))), new=1, hq=hq,
                        h=h, d=d, block=block, kv=kv, io=io, fresh=rng.random() < 0.3)
        batch = _log_int(rng, 1, 8)
        pairs = min(200_000_000_000 // (batch * hq * d), 1_400_000_000 // (batch * hq))   # (query, position) of a request
        new = _log_int(rng, 2, min(5000, math.isqrt(pairs) // 2))
        return dict(op=op, batch=batch, len=new + _log_int(rng, 1, min(60_000, pairs // new - new)), new=new, hq=hq, h=h, d=d,
                    block=block, kv=kv, io=io, fresh=rng.random() < 0.5)
    if op == "trim":
        batch = _log_int(rng, 1, 500)
    most = 262_144 if op == "keep" else 60_000 if op == "trim" else 120_000_000 // (batch * h * d)
    most = min(most, 2_400_000 // batch)
    length = _log_int(rng, 2 * block, max(2 * block, most))
    budget = min(length // block, _log_int(rng, 1, length // block)) * block
    out = dict(op=op, batch=batch, len=length, budget=budget, block=block)
    if op == "keep":
        out.update(recent=rng.randint(0, max(0, budget - SINKS) // 2), h=h)
    if op == "evict":
        out.update(h=h, d=d, kv=rng.choice(["fp8", "int8"]))
    return out


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _counts(case, rng):
    return [case["new"]] + [_log_int(rng, max(1, case["new"] // 8), case["new"]) for _ in range(case["batch"] - 1)]


def _lengths(case):
    """(entries of each request, queries of each request) from the case alone."""
    rng = _rng(case)
    top, n = case["len"], case["batch"]
    if case["op"] == "weigh":
        new = _counts(case, rng)
        if case["new"] == 1:
            return [top] + [_log_int(rng, max(1, top // 16), top) for _ in range(n - 1)], new
        return [top] + [rng.randint(m, top) for m in new[1:]], new
    # most requests are over their budget, some are not there yet
    low = max(1, case["budget"] - (top - case["budget"]) // 4)
    return [top] + [rng.randint(low, top) for _ in range(n - 1)], None


# ------------------------------------------------------------------------------------------------------------ inputs
def _prefix(values):
    out = [0]
    for x in values:
        out.append(out[-1] + x)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


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


def _table(case, lens, gen):
    """Block ids in a random order: a table with the blocks of each row's entries, the order, and the blocks in use."""
    b = case["block"]
    blocks = [-(-x // b) for x in lens]
    total = sum(blocks) + 3
    order = torch.randperm(total, generator=gen, device="cuda").int()
    lp = torch.arange(max(blocks), device="cuda")[None]
    cu, each = _i32(_prefix(blocks)).long(), _i32(blocks).long()[:, None]
    table = torch.where(lp < each, order[(cu[:-1, None] + lp).clamp(max=total - 1)], torch.full_like(order[:1], -1))
    return table, order, sum(blocks)


def _side(case, n_blocks, gain, gen):
    """Codes and scales of one side of a pool whose every block is full."""
    x = torch.randn((n_blocks, case["h"], case["block"], case["d"]), generator=gen, device="cuda")
    if gain is not None:
        x *= gain[:, None]
    s = _pow2(x.abs().amax((2, 3)), QMAX[case["kv"]])
    return _codes(x / s[..., None, None], case["kv"]), s


def _outliers(case, gen):
    gain = torch.ones(case["h"], case["d"], device="cuda")
    gain[:, torch.randperm(case["d"], generator=gen, device="cuda")[:max(1, case["d"] // 32)]] = 8.0
    return gain


def _weights(shape, gen):
    """Accumulated weights: log-normal; one in 16 rounded to a power of two (equal ones), one in 64 zero."""
    w = torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda"))
    u = torch.rand(shape, generator=gen, device="cuda")
    w = torch.where(u < 1 / 16, torch.exp2(torch.log2(w).round()), w)
    return torch.where(u > 63 / 64, torch.zeros_like(w), w)


def _moved(case, lens, rows, gen):
    """held, evicted (int32 [rows]) and pos int32 [rows, H, width] of conversations that were cut before: the entries held
    then sit at positions of their own, in no order."""
    b, h, n = case["block"], case["h"], len(lens)
    width = -(-max(lens) // b) * b
    held = (_i32(lens) * torch.rand(n, generator=gen, device="cuda")).int()
    evicted = torch.randint(1, 200_000, (n,), generator=gen, device="cuda").int() * (held > 0)
    pos = (torch.rand((n, h, width), generator=gen, device="cuda") * (held + evicted)[:, None, None]).int()
    out = torch.zeros_like(held), torch.zeros_like(evicted), torch.zeros_like(pos)
    for a, x in zip(out, (held, evicted, pos)):
        a[rows] = x
    return out


def _frequencies(case):
    """fp64 [rot / 2] angles per position and the factor of cosine and sine.  scaled: frequencies of periods beyond the
    original context divided by 8, those that turn often there left, a ramp between (YaRN)."""
    rot, base, orig, factor = case["rot"], 1e6 if case["scaled"] else 1e4, 16384, 8.0
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if not case["scaled"]:
        return inv.cuda(), 1.0
    at = [rot * math.log(orig / (beta * 2 * math.pi)) / (2 * math.log(base)) for beta in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return (inv / factor * ramp + inv * (1 - ramp)).cuda(), 0.1 * math.log(factor) + 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=dict(case))
    if case["op"] == "rope":
        rng = _rng(case)
        new = _counts(case, rng)
        n, hq, h, d = sum(new), case["hq"], case["h"], case["d"]
        cols = (hq + 2 * h) * d if case["fused"] else (hq + h) * d
        x = torch.randn(n, cols, generator=gen, device="cuda").to(IO[case["io"]])
        q, k = x[:, :hq * d].unflatten(1, (hq, d)), x[:, hq * d:(hq + h) * d].unflatten(1, (h, d))
        if not case["fused"]:
            q, k = q.contiguous(), k.contiguous()
        lens = [m + rng.randint(0, case["far"]) for m in new]    # entries with the step's own
        inv, scale = _frequencies(case)
        rows = torch.randperm(len(new), generator=gen, device="cuda")
        s.update(q=q, k=k, inv_freq=inv, scale=scale, cu=_i32(_prefix(new)), kv_lens=_i32(lens), seqs=rows.int(),
                 ahead=torch.randint(0, case["far"], (len(new),), generator=gen, device="cuda").int(), n_tokens=n)
        return s
    lens, new = _lengths(case)
    n = len(lens)
    table, order, used = _table(case, lens, gen)
    s.update(block_table=table, kv_lens=_i32(lens))
    width = table.shape[1] * case["block"]
    if case["op"] == "trim":
        # rows in another order than the requests'
        rows = torch.randperm(n, generator=gen, device="cuda")
        spread, seq_lens = torch.full_like(table, -1), torch.zeros_like(s["kv_lens"])
        spread[rows], seq_lens[rows] = table, s["kv_lens"]
        s.update(seqs=rows.int(), block_table=spread, seq_lens=seq_lens, free_list=order, free_head=_i32([used]),
                 status=_i32([0]))
        return s
    if case["op"] == "weigh":
        s["k8"], s["ks"] = _side(case, used + 3, _outliers(case, gen), gen)
        s.update(q=torch.randn(sum(new), case["hq"], case["d"], generator=gen, device="cuda").to(IO[case["io"]]),
                 weights=_weights((n, case["h"], width), gen), workspace={}, cu_q=_i32(_prefix(new)), max_q=max(new),
                 since=torch.zeros_like(s["kv_lens"]) if case["fresh"] else s["kv_lens"] - _i32(new))
        s["out"] = torch.zeros_like(s["weights"])
        return s
    rows = torch.arange(n, device="cuda")
    s["weights"] = _weights((n, case["h"], width), gen)
    s["held"], s["evicted"], s["pos"] = _moved(case, lens, rows, gen)
    if case["op"] == "keep":
        s["workspace"] = {}
        return s
    s["src"] = _select(s["weights"], s["kv_lens"], case["budget"], 0, s["pos"], s["held"], s["evicted"])
    s["k8"], s["ks"] = _side(case, used + 3, _outliers(case, gen), gen)
    s["v8"], s["vs"] = _side(case, used + 3, None, gen)
    return s


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return _run_own(s)
    return {"rope": _rope, "weigh": _weigh, "keep": _keep, "evict": _evict, "trim": _trim}[s["case"]["op"]](s)


def _run_own(s):
    from kvtier import block_evict, rope

    c = s["case"]
    if c["op"] == "rope":
        q, k = rope.kvt_rope(s["q"], s["k"], s["kv_lens"], s["inv_freq"], scale=s["scale"], interleaved=c["inter"],
                             cu=s["cu"], seqs=s["seqs"], ahead=s["ahead"])
        return dict(q=q, k=k)
    if c["op"] == "weigh":
        return block_evict.kvt_block_weigh(s["q"], s["k8"], s["ks"], s["block_table"], s["kv_lens"], s["weights"],
                                           cu_q=None if c["new"] == 1 else s["cu_q"], since=s["since"], out=s["out"],
                                           workspace=s["workspace"])
    if c["op"] == "keep":
        return block_evict.kvt_block_keep(s["weights"], s["kv_lens"], c["budget"], recent=c["recent"], sinks=SINKS,
                                          pos=s["pos"], held=s["held"], evicted=s["evicted"], workspace=s["workspace"])
    if c["op"] == "evict":
        block_evict.kvt_block_evict(s["src"], s["kv_lens"], s["k8"], s["v8"], s["ks"], s["vs"], s["block_table"],
                                    weights=s["weights"], pos=s["pos"], held=s["held"], evicted=s["evicted"])
        return dict(k8=s["k8"], v8=s["v8"], ks=s["ks"], vs=s["vs"], weights=s["weights"], pos=s["pos"])
    t = block_evict.kvt_block_trim(s["seqs"], s["seq_lens"], s["block_table"], s["free_list"], s["free_head"], c["budget"],
                                   block=c["block"], status=s["status"], commit=False)
    return dict(kv_lens=t.kv_lens, next_head=t.next_head, free_list=s["free_list"], status=s["status"])


def _rope(s):
    c, cu = s["case"], s["cu"].long()
    t = torch.arange(s["n_tokens"], device="cuda")
    r = torch.searchsorted(cu[1:], t, right=True)
    at = s["kv_lens"].long()[r] - cu[r + 1] + t + s["ahead"].long()[s["seqs"].long()[r]]
    angle = at.double()[:, None] * s["inv_freq"][None]
    cos, sin = ((f(angle) * s["scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        a, b = _pairs(x[..., :c["rot"]], c["inter"])
        y = (a * cos - b * sin, b * cos + a * sin)
        y = torch.stack(y, -1).flatten(-2) if c["inter"] else torch.cat(y, -1)
        out[name] = torch.cat((y, x[..., c["rot"]:]), -1).to(s[name].dtype)
    return out


def _pairs(x, inter):
    return (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, -1)


def _weigh(s):
    c, cu = s["case"], s["cu_q"].long()
    q, h, d = s["q"], c["h"], c["d"]
    n, g, m = cu.numel() - 1, q.shape[1] // h, s["max_q"]
    table = s["block_table"].long().clamp(min=0)
    k = s["k8"].view(torch.int8)[table].view(s["k8"].dtype).float() * s["ks"][table][..., None, None]
    k = k.transpose(1, 2).flatten(2, 3)                                     # [n, H, positions, D]
    j = torch.arange(m, device="cuda")[None]
    x = q[(cu[:-1, None] + j).clamp(max=q.shape[0] - 1)].float() * d ** -0.5
    x = x.view(n, m, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * m, d)
    x = torch.matmul(x, k.transpose(2, 3).contiguous())                     # [n, H, (q head, query), positions]
    kv_lens, count = s["kv_lens"].long(), cu[1:] - cu[:-1]
    e = torch.arange(k.shape[2], device="cuda")
    sees = (kv_lens - count)[:, None] + j + 1                               # [n, m]
    sees = torch.where(j < count[:, None], sees, torch.zeros_like(sees)).repeat(1, g)
    gone = e[None, None] >= sees.clamp(min=1)[..., None]                    # (a row of no query sees one entry)
    x.masked_fill_(gone[:, None], float("-inf"))
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).mul_((sees > 0)[:, None, :, None])
    total = p.sum(2) + torch.where(e < s["since"][:, None], 1.0, 0.0)[:, None] * s["weights"]
    s["out"].copy_(torch.where((e < kv_lens[:, None])[:, None], total, s["out"]))
    return s["out"]


def _select(weights, kv_lens, budget, recent, pos, held, evicted):
    """src [n, H, budget] of requests in the order of the table's rows."""
    e = torch.arange(weights.shape[2], device="cuda")
    lens, held, evicted = (x.long()[:, None, None] for x in (kv_lens, held, evicted))
    at = torch.where(e < held, pos.long(), e + evicted)
    always = (e < SINKS) | (at >= lens + evicted - recent)
    key = torch.where(always, torch.full_like(weights, float("inf")), weights)
    key = torch.where(e < lens, key, torch.full_like(key, float("-inf")))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    stays = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order, True) & (e < lens)
    free, comes = ~stays[..., :budget], stays[..., budget:]
    behind = torch.sort(comes.to(torch.int8), dim=-1, descending=True, stable=True).indices + budget
    rank = free.long().cumsum(-1) - 1
    pad = torch.zeros_like(free, dtype=torch.long)
    behind = torch.cat((behind, pad), -1)
    src = torch.where(free, torch.gather(behind, -1, rank.clamp(min=0)), e[:budget].expand_as(pad))
    here = torch.where(e[:budget] < lens, e[:budget].expand_as(pad), torch.full_like(pad, -1))
    return torch.where(lens > budget, src, here).int()


def _keep(s):
    c = s["case"]
    return _select(s["weights"], s["kv_lens"], c["budget"], c["recent"], s["pos"], s["held"], s["evicted"])


def _evict(s):
    c = s["case"]
    b, h, kv, budget = c["block"], c["h"], c["kv"], c["budget"]
    over = s["kv_lens"] > budget
    e = torch.arange(budget, device="cuda")
    src = torch.where(over[:, None, None], s["src"].long(), e)              # [n, H, budget]
    at = torch.where(e < s["held"][:, None, None], s["pos"][..., :budget], e + s["evicted"][:, None, None])
    rest = torch.where(src < s["held"][:, None, None], torch.gather(s["pos"], 2, src), src + s["evicted"][:, None, None])
    at = torch.where(src == e, at, rest).int()
    table = s["block_table"].long().clamp(min=0)
    n, hh = torch.arange(c["batch"], device="cuda")[:, None, None], torch.arange(h, device="cuda")[None, :, None]
    from_block, from_row = table[n, src // b], src % b
    changes = (src != e).view(c["batch"], h, -1, b).any(-1)                 # [n, H, blocks]
    to = table[:, :budget // b][:, None].expand_as(changes)[changes]
    heads = hh.expand_as(changes)[changes]
    pick = changes.repeat_interleave(b, 2)
    for codes, scale in ((s["k8"], s["ks"]), (s["v8"], s["vs"])):
        raw = codes.view(torch.int8)
        hp = hh.expand_as(src)[pick]
        x = raw[from_block[pick], hp, from_row[pick]].view(codes.dtype).float() * scale[from_block[pick], hp][:, None]
        x = x.view(-1, b, c["d"])
        size = _pow2(x.abs().amax((1, 2)), QMAX[kv])
        raw[to, heads] = _codes(x / size[:, None, None], kv).view(torch.int8)
        scale[to, heads] = size
    s["weights"][..., :budget] = torch.gather(s["weights"], 2, src)
    s["pos"][..., :budget] = torch.where(over[:, None, None], at, s["pos"][..., :budget])
    return dict(k8=s["k8"], v8=s["v8"], ks=s["ks"], vs=s["vs"], weights=s["weights"], pos=s["pos"])


def _trim(s):
    c = s["case"]
    b, seqs, table = c["block"], s["seqs"].long(), s["block_table"]
    lens = s["seq_lens"].long()[seqs]
    lp = torch.arange(table.shape[1], device="cuda")[None]
    last = torch.where(lens > c["budget"], (lens + b - 1) // b, torch.zeros_like(lens))
    goes = (lp >= c["budget"] // b) & (lp < last[:, None])
    freed = table[seqs][goes]                                               # by request, then by block
    head = s["free_head"] - freed.numel()
    at = torch.arange(freed.numel(), device="cuda") + head
    s["free_list"][at] = freed
    return dict(kv_lens=lens.clamp(max=c["budget"]).int(), next_head=head.int(), free_list=s["free_list"],
                status=s["status"])


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    b = case.get("block")
    if case["op"] == "rope":
        n = sum(_counts(case, _rng(case)))
        size = n * (case["hq"] + case["h"]) * case["d"] * IO[case["io"]].itemsize
        return {"bytes": 2 * size + 12 * case["batch"], "flops": 3 * n * (case["hq"] + case["h"]) * case["rot"]}
    lens, new = _lengths(case)
    budget, total = case.get("budget"), sum(lens)
    if case["op"] == "trim":
        freed = sum(-(-x // b) - budget // b for x in lens if x > budget)
        return {"bytes": 8 * freed + 12 * len(lens), "flops": 0}
    h = case["h"]
    if case["op"] == "weigh":
        blocks = sum(-(-x // b) for x in lens)
        older = 0 if case["fresh"] else total - sum(new)
        pairs = sum(x * y - y * (y - 1) // 2 for x, y in zip(lens, new))
        read = total * h * case["d"] + blocks * 4 * (h + 1) + 2 * sum(new) * case["hq"] * case["d"]
        return {"bytes": read + 4 * h * (total + older), "flops": 2 * case["d"] * case["hq"] * pairs}
    cut = [x for x in lens if x > budget]
    if case["op"] == "keep":
        return {"bytes": 4 * h * (sum(cut) + budget * len(lens)), "flops": 0}
    # entries that move, if all are as likely to stay, and the blocks that get any: their rows are read, for the scale,
    # and the moved ones written
    moved = [budget * (x - budget) / x for x in cut]
    nb = budget // b
    changed = [nb * (1 - (1 - 1 / nb) ** m) if nb > 1 else 1.0 for m in moved]
    rows = sum(changed) * b + sum(moved)
    per_head = 2 * case["d"] * rows + 12 * len(cut) * budget + 8 * sum(moved) + 16 * sum(changed)
    return {"bytes": int(h * per_head) + 1, "flops": 0}


# ------------------------------------------------------------------------------------------------------------- exact
def _round_e4m3(x):
    """float64 -> the nearest e4m3 value (ties to even), |x| <= 448."""
    e = torch.frexp(x.abs())[1].clamp(min=-5).double() - 4      # spacing 2^(exponent - 3), subnormals 2^-9
    step = torch.exp2(e)
    return torch.round(x / step) * step


def _exact_scale(amax, kv):
    """float64 [..] -> the smallest power of two that holds amax in the codes' range."""
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -100) / QMAX[kv]))
    e = torch.where(amax > QMAX[kv] * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= QMAX[kv] * torch.exp2(e - 1), e - 1, e)
    return torch.exp2(e.clamp(MIN_EXP, MAX_EXP))


def _exact_rope(case, s):
    cu, new = s["cu"].tolist(), _counts(case, _rng(case))
    out = {name: s[name].double() for name in ("q", "k")}
    rot = case["rot"]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["inter"] else (slice(0, rot // 2), slice(rot // 2, rot))
    for r, m in enumerate(new):
        start = int(s["kv_lens"][r]) - m + int(s["ahead"][int(s["seqs"][r])])
        turn = torch.polar(torch.full((m, rot // 2), float(s["scale"]), dtype=torch.float64, device="cuda"),
                           torch.arange(start, start + m, device="cuda").double()[:, None] * s["inv_freq"])[:, None]
        for x in out.values():
            part = x[cu[r]:cu[r + 1]]
            z = torch.complex(part[..., first], part[..., second]) * turn
            part[..., first], part[..., second] = z.real, z.imag
    return out


def _exact_weigh(case, s):
    lens, new = _lengths(case)
    b, g, cu = case["block"], case["hq"] // case["h"], _prefix(new)
    out = s["out"].double()
    for r, (length, m) in enumerate(zip(lens, new)):
        blocks = s["block_table"][r, :-(-length // b)].long()
        since = int(s["since"][r])
        for h in range(case["h"]):
            k = s["k8"].view(torch.int8)[blocks, h].view(s["k8"].dtype).double()
            k = (k * s["ks"][blocks, h].double()[:, None, None]).flatten(0, 1)[:length].t().contiguous()
            out[r, h, :since] = s["weights"][r, h, :since].double()
            for j in range(g):
                x = s["q"][cu[r]:cu[r + 1], h * g + j].double() @ k / math.sqrt(case["d"])
                if m > 1:
                    last = length - m + torch.arange(m, device="cuda")
                    x.masked_fill_(torch.arange(length, device="cuda")[None] > last[:, None], float("-inf"))
                out[r, h, :length] += torch.softmax(x, -1).sum(0)
    return out


def _exact_evict(case, s):
    lens, _ = _lengths(case)
    b, kv, nb = case["block"], case["kv"], case["budget"] // case["block"]
    out = {}
    here = torch.arange(case["budget"], device="cuda").view(nb, b)
    for name, scales in (("k8", "ks"), ("v8", "vs")):
        codes, scale = s[name].to(torch.float32), s[scales].double()
        if kv == "fp8":
            out[name] = codes.double()
        for r, length in enumerate(lens):
            if length <= case["budget"]:
                continue
            table = s["block_table"][r].long()
            for h in range(case["h"]):
                src = s["src"][r, h].long().view(nb, b)
                moved = (src != here).any(1)
                from_block = table[src[moved] // b]
                x = codes[from_block, h, src[moved] % b].double() * s[scales][from_block, h].double()[..., None]
                size = _exact_scale(x.abs().amax((1, 2)), kv)
                scale[table[:nb][moved], h] = size
                if kv == "fp8":
                    out[name][table[:nb][moved], h] = _round_e4m3(x / size[:, None, None])
        out[scales] = scale
    weights = s["weights"].double()
    for r, length in enumerate(lens):
        if length > case["budget"]:
            weights[r, :, :case["budget"]] = torch.gather(s["weights"][r].double(), 1, s["src"][r].long())
    return dict(k8=out.get("k8"), v8=out.get("v8"), ks=out["ks"], vs=out["vs"], weights=weights, pos=None)


def exact(case, seed):
    if case["op"] in ("keep", "trim"):
        return None
    return {"rope": _exact_rope, "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](case, prepare(case, seed))
