"""Operators for long texts that are measured: a paged cache held in 4 bits (rows written and read back, attention over it), and attention that reads
only those blocks of the cache that a score of their bounds selects for each query row.

``own`` False: the plain form, elementary tensor operations in fp32; True: the calls of ``NativeOps``.

Fields of a case:
  op        store | attend | sparse
  hq, hkv, dim   query heads, key heads, head dim
  store     tokens: rows that are written (``skip``: every so many of them has no slot, 0: none)
  attend, sparse   seqs: sequences of the step; ctx_lo, ctx_hi: tokens they have in the cache before it, spread evenly between; rows: new tokens per sequence
  attend    window, first: a row sees the last ``window`` tokens up to itself and the first ``first`` ones (window 0: all before it)
  sparse    kv: bf16 | e4m3 | int4, what the cache holds; count: blocks that a row reads, ``lead`` at the text's start and ``tail`` at its end among them
  sinks     whether each head has a logit of its own in the sum; cap: soft-cap of the scores (0: none)
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

BLOCK = 16


def _attend(name, seqs, ctx_lo, ctx_hi, rows, hq, hkv, dim, window=0, first=0, sinks=False, cap=0.0):
    return dict(name=name, op="attend", seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, rows=rows, hq=hq, hkv=hkv, dim=dim, window=window, first=first, sinks=sinks,
                cap=cap)


def _sparse(name, seqs, ctx_lo, ctx_hi, rows, hq, hkv, dim, kv, count, lead=1, tail=2, sinks=False, cap=0.0):
    return dict(name=name, op="sparse", seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, rows=rows, hq=hq, hkv=hkv, dim=dim, kv=kv, count=count, lead=lead, tail=tail,
                sinks=sinks, cap=cap)


def listed():
    return [
        # the row of one user's new token, and a full prefill step of the 8B preset's heads
        dict(name="store_1", op="store", tokens=1, hkv=8, dim=128, skip=0),
        dict(name="store_8192", op="store", tokens=8192, hkv=8, dim=128, skip=0),
        # one user, one token, a short text: latency
        _attend("attend_1", 1, 900, 900, 1, 32, 8, 128),
        # a full batch of long conversations, the heads of the 8B preset
        _attend("attend_64", 64, 4000, 32000, 1, 32, 8, 128),
        # heads of 64 with a logit of their own, a window and first tokens that end inside pages
        _attend("attend_48_window", 48, 900, 9001, 1, 64, 8, 64, 1000, 130, sinks=True),
        # chunks of two long prompts
        _attend("attend_prompt_2x2048", 2, 2500, 6143, 2048, 32, 8, 128),
        # chunks of odd lengths under a window
        _attend("attend_prompt_3x777", 3, 1, 3001, 777, 64, 8, 64, 512, 16),
        # one user behind a long text
        _sparse("sparse_1", 1, 30000, 30000, 1, 32, 8, 128, "bf16", 64),
        # a full batch of long conversations that read 2048 tokens each
        _sparse("sparse_64", 64, 4000, 32000, 1, 32, 8, 128, "bf16", 128),
        # the same over caches of 8 and of 4 bits, ragged, some texts shorter than what is read
        _sparse("sparse_24_fp8", 24, 100, 9000, 1, 64, 8, 64, "e4m3", 48, sinks=True),
        _sparse("sparse_40_int4", 40, 1000, 20000, 1, 40, 8, 128, "int4", 96),
        # chunks of two prompts, each row with blocks of its own
        _sparse("sparse_prompt_2x301", 2, 3000, 6001, 301, 32, 8, 128, "bf16", 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds that neither form can do without, roughly: the fp32 products of the plain form weigh most."""
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 5e13


def _held(case):
    """Values that the plain form holds at a time: scores, and gathered keys."""
    if case["op"] == "store":
        return 0
    reach = case["ctx_hi"] + case["rows"]
    if case["op"] == "attend":
        cols = min(reach, case["window"] + case["rows"] + case["first"]) if case["window"] else reach
        return max(case["seqs"] * case["hq"] * case["rows"] * cols, case["seqs"] * case["hkv"] * cols * case["dim"])
    rows = case["seqs"] * case["rows"]
    return max(rows * case["hkv"] * case["count"] * BLOCK * case["dim"], rows * case["hkv"] * reach // BLOCK)


def draw(rng):
    top, most = {}, {}
    for c in listed():
        top[c["op"]] = max(top.get(c["op"], 0.0), _cost(c))
        most[c["op"]] = max(most.get(c["op"], 0), _held(c))
    while True:
        op = rng.choice(["store", "attend", "attend", "attend", "sparse", "sparse", "sparse"])
        hkv, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128])
        if op == "store":
            c = dict(op=op, tokens=_log(rng, 1, 8192), hkv=hkv, dim=dim, skip=rng.choice([0, 0, 2, 5]))
        else:
            hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
            ctx = _log(rng, 1 if op == "attend" else 64, 32000)
            common = dict(seqs=_log(rng, 1, 64), ctx_lo=rng.randint(max(1, ctx // 8), ctx), ctx_hi=ctx, hq=hq, hkv=hkv, dim=dim, sinks=rng.random() < 0.3,
                          cap=rng.choice([0.0, 0.0, 0.0, 30.0]))
            if op == "attend":
                window = rng.choice([0, _log(rng, 32, 4096)])
                c = dict(op=op, rows=rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)]), window=window, first=_log(rng, 1, 256) if window else 0, **common)
            else:
                c = dict(op=op, rows=rng.choice([1, 1, 1, _log(rng, 2, 300)]), kv=rng.choice(["bf16", "e4m3", "int4"]), count=_log(rng, 4, 160),
                         lead=rng.randint(0, 2), tail=rng.randint(1, 2), **common)
        if _cost(c) <= top[op] and _held(c) <= most[op]:
            return c


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _row_bytes(case):
    kv = case.get("kv", "int4")
    return {"bf16": 2 * case["dim"], "e4m3": case["dim"], "int4": case["dim"] // 2 + 4}[kv]


# ------------------------------------------------------------------ the 4-bit rows
def _bits(x):
    return x.view(torch.int32)


def _down(x):
    """fp32 rounded down to what bf16 holds."""
    b = _bits(x)
    cut = b & -65536
    return torch.where((cut != b) & (b < 0), cut + 65536, cut).view(torch.float32)


def _up(x):
    """fp32 >= 0 rounded up to what bf16 holds."""
    return ((_bits(x) + 65535) & -65536).view(torch.float32)


def _encode(x):
    """[..., dim] -> uint8 [..., dim / 2 + 4]: codes (even dims in the low half of a byte), step and lowest value as bf16."""
    x = x.float()
    fine = torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(fine, x, torch.zeros_like(x))
    low = _down(x.amin(-1, keepdim=True))
    step = _up(torch.div(x.amax(-1, keepdim=True) - low, torch.full_like(low, 15)))       # (a number as divisor would become a factor)
    code = torch.where(step > 0, torch.round((x - low) / step).clamp(0, 15), torch.zeros_like(x)).to(torch.uint8)
    step = torch.where(fine, step, torch.full_like(step, math.nan))
    tail = torch.cat([step, low], -1).to(torch.bfloat16).view(torch.uint8)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, tail], -1)


def _decode(rows):
    """uint8 [..., dim / 2 + 4] -> fp32 [..., dim]"""
    half = rows.shape[-1] - 4
    par = rows[..., half:].contiguous().view(torch.bfloat16).float()
    code = torch.stack([rows[..., :half] & 15, rows[..., :half] >> 4], -1).flatten(-2)
    return code.float() * par[..., :1] + par[..., 1:]


def _values(rows, kv):
    return _decode(rows) if kv == "int4" else rows.view(torch.float8_e4m3fn).float() if kv == "e4m3" else rows.float()


# ------------------------------------------------------------------ bounds of blocks
def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _unit(top):
    """The smallest e with top <= 127 x 2^e."""
    e = torch.frexp(top)[1] - 7
    return torch.where(top > 127 * _pow2(e), e + 1, e)


def _code_bounds(k):
    """fp32 [..., block, dim] -> int8 [..., 2 dim + 16]: upper and lower bounds of every channel over the block in units of 2^e, then e."""
    hi, lo = k.amax(-2), k.amin(-2)
    top = torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True)
    e = torch.where(top > 0, _unit(top).clamp(min=-120), torch.full_like(top, -120, dtype=torch.int32))
    unit = _pow2(-e)
    rest = torch.zeros(*e.shape[:-1], 16, dtype=torch.int8, device=k.device)
    rest[..., :1] = e.to(torch.int8)
    return torch.cat([torch.ceil(hi * unit).to(torch.int8), torch.floor(lo * unit).to(torch.int8), rest], -1)


def _pool(g, blocks, case, leaning):
    """A pool of keys or values. ``leaning``: the keys of a block have a direction in common, as those of neighbouring tokens do."""
    kv, hkv, dim = case.get("kv", "int4"), case["hkv"], case["dim"]
    if kv == "int4" and not leaning:                         # codes of 4 bits as they come, steps and lowest values of rows of about unit size
        codes = torch.randint(0, 256, (blocks, hkv, BLOCK, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
        step = 0.2 + 0.1 * torch.rand(blocks, hkv, BLOCK, 1, generator=g, device="cuda")
        low = -step * (7 + torch.rand(blocks, hkv, BLOCK, 1, generator=g, device="cuda"))
        return torch.cat([codes, torch.cat([step, low], -1).to(torch.bfloat16).view(torch.uint8)], -1)
    out = torch.empty(blocks, hkv, BLOCK, _row_bytes(case) // (2 if kv == "bf16" else 1), device="cuda", dtype=torch.bfloat16 if kv == "bf16" else torch.uint8)
    for b in range(0, blocks, 4096):
        n = min(4096, blocks - b)
        x = torch.randn(n, hkv, BLOCK, dim, generator=g, device="cuda", dtype=torch.bfloat16)
        if leaning:
            x = x + torch.randn(n, hkv, 1, dim, generator=g, device="cuda", dtype=torch.bfloat16)
        out[b:b + n] = _encode(x) if kv == "int4" else x.to(torch.float8_e4m3fn).view(torch.uint8) if kv == "e4m3" else x
    return out


def _tables(g, lens, blocks):
    """Pages of each sequence at random places of the pool; block 0 behind the last one."""
    need = [-(-n // BLOCK) for n in lens]
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    cols = torch.arange(max(need), device="cuda")
    t = order[(starts[:, None] + cols).clamp(max=blocks - 1)]
    return torch.where(cols < torch.tensor(need, device="cuda")[:, None], t, torch.zeros_like(t)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    s = SimpleNamespace(case=case, op=case["op"])
    hkv, dim = case["hkv"], case["dim"]
    if case["op"] == "store":
        T = case["tokens"]
        blocks = -(-T // BLOCK) + 3
        s.k = 2 * torch.randn(T, hkv * dim, generator=g, device="cuda", dtype=torch.bfloat16)
        s.v = torch.randn(T, hkv * dim, generator=g, device="cuda", dtype=torch.bfloat16)
        s.slots = torch.randperm(blocks * BLOCK, generator=g, device="cuda")[:T].to(torch.int32)
        if case["skip"]:
            s.slots[case["skip"] - 1::case["skip"]] = -1
        s.live = torch.nonzero(s.slots >= 0)[:, 0]
        s.kc = torch.zeros(blocks, hkv, BLOCK, dim // 2 + 4, dtype=torch.uint8, device="cuda")
        s.vc = torch.zeros_like(s.kc)
        return s
    ctx, n = _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"]), case["rows"]
    B, T, lens = len(ctx), len(ctx) * n, [c + n for c in ctx]
    blocks = sum(-(-x // BLOCK) for x in lens) + 3
    s.tables = _tables(g, lens, blocks)
    s.kc, s.vc = _pool(g, blocks, case, case["op"] == "sparse"), _pool(g, blocks, case, False)
    s.q = 1.5 * torch.randn(T, case["hq"] * dim, generator=g, device="cuda", dtype=torch.bfloat16)
    s.sinks = torch.randn(case["hq"], generator=g, device="cuda") if case["sinks"] else None
    s.scale = dim ** -0.5
    s.starts, s.lens, s.ctx = i32([n * i for i in range(B + 1)]), i32(lens), i32(ctx)
    s.row_seq = torch.arange(B, dtype=torch.int32, device="cuda").repeat_interleave(n)
    s.local = torch.arange(n, dtype=torch.int32, device="cuda").repeat(B)
    s.positions = s.ctx[s.row_seq.long()] + s.local
    s.max_len = max(lens)
    s.meta = SimpleNamespace(q_starts=s.starts, seq_lens=s.lens, num_seqs=B, num_tokens=T, max_q_len=n, min_q_len=n, max_kv_len=s.max_len)
    if case["op"] == "sparse":
        s.slots = s.tables[s.row_seq.long(), (s.positions // BLOCK).long()] * BLOCK + s.positions % BLOCK
        s.full = (s.slots[s.slots % BLOCK == BLOCK - 1] // BLOCK).long()             # blocks that the step's rows complete
        s.bounds = torch.empty(blocks, hkv, 2 * dim + 16, dtype=torch.int8, device="cuda")
        for b in range(0, blocks, 4096):
            s.bounds[b:b + 4096] = _code_bounds(_values(s.kc[b:b + 4096], case["kv"]))
        s.bounds[s.full] = 0                                                         # whose bounds the step has to find
        if case["kv"] == "e4m3":
            s.kc, s.vc = s.kc.view(torch.float8_e4m3fn), s.vc.view(torch.float8_e4m3fn)
    return s


_ops = {}


def _native():
    from fllm_b200.ops.native import NativeOps
    dev = torch.device("cuda", torch.cuda.current_device())
    if dev not in _ops:
        _ops[dev] = NativeOps(dev)
    return _ops[dev]


def run(state):
    s, c = state, state.case
    if own:
        ops = _native()
        if s.op == "store":
            ops.kv4_write(s.k, s.v, s.slots, s.kc, s.vc)
            return ops.kv4_read(s.kc, s.slots), ops.kv4_read(s.vc, s.slots)
        if s.op == "attend":
            return ops.attention(s.q, s.kc, s.vc, s.tables, s.row_seq, s.positions, c["hq"], c["hkv"], c["dim"], s.scale, c["window"], s.sinks, c["cap"],
                                 meta=s.meta, first=c["first"])
        ops.kv_bounds(s.kc, s.bounds, s.slots)
        picks = ops.select_blocks(s.q, s.bounds, s.tables, c["hq"], c["hkv"], c["dim"], BLOCK, c["count"], s.meta, lead=c["lead"], tail=c["tail"])
        out = ops.attention_blocks(s.q, s.kc, s.vc, s.tables, picks, c["hq"], c["hkv"], c["dim"], s.scale, s.meta, s.sinks, c["cap"])
        return out, picks, s.bounds
    if s.op == "store":
        return _plain_store(s)
    if s.op == "attend":
        return _plain_attend(s)
    return _plain_sparse(s)


def _plain_store(s):
    hkv, dim = s.case["hkv"], s.case["dim"]
    at, out = s.slots[s.live].long(), []
    for x, cache in ((s.k, s.kc), (s.v, s.vc)):
        cache[at // BLOCK, :, at % BLOCK] = _encode(x[s.live].view(-1, hkv, dim))
        back = torch.zeros(x.shape, device="cuda")
        back[s.live] = _decode(cache[at // BLOCK, :, at % BLOCK]).flatten(1)
        out.append(back)
    return tuple(out)


def _weights(score, seen, sinks):
    """Softmax over the last axis of what is seen; a row that sees nothing has weights of 0."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return p / total.clamp(min=1e-30)


def _plain_attend(s):
    c = s.case
    hq, hkv, D, W, F, R = c["hq"], c["hkv"], c["dim"], c["window"], c["first"], c["rows"]
    # columns: the first tokens, then those from where the first row's window begins
    lo = (s.ctx + 1 - W).clamp(min=0) if W else torch.zeros_like(s.ctx)
    F = min(F, s.max_len) if W else 0
    span = min(s.max_len, W + R) if W else s.max_len
    col = torch.arange(F + span, device="cuda")
    tok = torch.where(col < F, col, lo[:, None] + col - F)                                           # [B, C]
    there = (tok < s.lens[:, None]) & ((col < F) | (tok >= F))
    at = tok.clamp(max=s.max_len - 1)
    page = torch.gather(s.tables, 1, (at // BLOCK).long()).long()
    K = _decode(s.kc[page, :, at % BLOCK])
    q = s.q.float().view(-1, R, hkv, hq // hkv, D)
    score = torch.einsum("brhgd,bchd->bhgrc", q, K) * s.scale
    del K
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    pos = s.ctx[:, None] + torch.arange(R, device="cuda")                                            # [B, R]
    seen = (tok[:, None] <= pos[:, :, None]) & there[:, None]
    if W:
        seen &= (tok[:, None] > pos[:, :, None] - W) | (tok[:, None] < F)
    V = _decode(s.vc[page, :, at % BLOCK])
    p = _weights(score, seen[:, None, None], None if s.sinks is None else s.sinks.view(1, hkv, hq // hkv, 1, 1))
    return torch.einsum("bhgrc,bchd->brhgd", p, V).reshape(-1, hq * D).to(s.q.dtype)


def _plain_sparse(s):
    c = s.case
    hq, hkv, D, count, lead, tail = c["hq"], c["hkv"], c["dim"], c["count"], c["lead"], c["tail"]
    T, G = s.q.shape[0], hq // hkv
    raw = lambda t: t.view(torch.uint8) if c["kv"] == "e4m3" else t
    kc, vc = raw(s.kc), raw(s.vc)
    s.bounds[s.full] = _code_bounds(_values(kc[s.full], c["kv"]))
    # scores of blocks: whole numbers below 2^24 times a power of two, so these products and sums are what they are in any order
    q = s.q.float().view(T, hkv, G, D)
    u = torch.cat([q.clamp(min=0).sum(2), (-q).clamp(min=0).sum(2)], -1)                             # [T, hkv, 2 D]
    top = u.amax(-1, keepdim=True)
    u = torch.round(u * _pow2(-_unit(top))) * torch.cat([torch.ones(D, device="cuda"), -torch.ones(D, device="cuda")])
    b = s.bounds[s.tables.long()]                                                                    # [B, blocks, hkv, 2 D + 16]
    code = b[..., :2 * D].float()
    score = torch.einsum("brhd,bnhd->brhn", u.view(-1, c["rows"], hkv, 2 * D), code)
    score = (score * _pow2(b[..., 2 * D]).transpose(1, 2)[:, None]).flatten(0, 1)        # [T, hkv, blocks]
    n = (s.positions // BLOCK + 1)[:, None, None]
    i = torch.arange(score.shape[-1], device="cuda")
    score = torch.where(i >= n, torch.full_like(score, -math.inf), torch.where((i < lead) | (i >= n - tail), torch.full_like(score, math.inf), score))
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :count]
    best = torch.cat([best, torch.full((T, hkv, max(0, count - best.shape[-1])), 1 << 30, device="cuda")], -1)
    best = torch.where(best < n, best, torch.full_like(best, 1 << 30)).sort(-1)[0]
    picks = torch.where(best < (1 << 30), best, torch.full_like(best, -1))
    # attention over their tokens
    tok = (picks.clamp(min=0)[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten(-2)   # [T, hkv, C]
    seen = (tok <= s.positions[:, None, None]) & (picks >= 0).repeat_interleave(BLOCK, -1)
    page = torch.gather(s.tables.long()[s.row_seq.long()][:, None].expand(-1, hkv, -1), 2, (tok // BLOCK).clamp(max=s.tables.shape[1] - 1))
    head = torch.arange(hkv, device="cuda")[:, None]
    score = torch.einsum("thgd,thcd->thgc", q, _values(kc[page, head, tok % BLOCK], c["kv"])) * s.scale
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    V = _values(vc[page, head, tok % BLOCK], c["kv"])
    p = _weights(score, seen[:, :, None], None if s.sinks is None else s.sinks.view(1, hkv, G, 1))
    return torch.einsum("thgc,thcd->thgd", p, V).reshape(T, hq * D).to(s.q.dtype), picks.to(torch.int32), s.bounds


def work(case):
    hkv, D = case["hkv"], case["dim"]
    if case["op"] == "store":             # the rows of keys and values, their slots, the rows in 4 bits, and what these stand for
        live = case["tokens"] - (case["tokens"] // case["skip"] if case["skip"] else 0)
        return {"bytes": 2 * live * hkv * (2 * D + D // 2 + 4) + 4 * case["tokens"] + 8 * case["tokens"] * hkv * D, "flops": 8 * live * hkv * D}
    ctx, n = _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"]), case["rows"]
    T, row = len(ctx) * n, 2 * _row_bytes(case) * hkv
    io = 4 * T * case["hq"] * D
    if case["op"] == "attend":
        W, F = case["window"], case["first"]
        keys = pairs = pages = 0
        for c in ctx:
            lo = max(0, c + 1 - W) if W else 0
            keys += c + n - lo + min(F, lo)
            pages += -(-(c + n) // BLOCK)
            for i in range(n):
                beg = max(0, c + i + 1 - W) if W else 0
                pairs += c + i + 1 - beg + min(F, beg)
        return {"bytes": keys * row + io + 4 * pages, "flops": 4 * pairs * case["hq"] * D}
    read = scored = pairs = fresh = 0
    for c in ctx:
        have = -(-(c + n) // BLOCK)
        read += min(have, case["count"] * n) if n > 1 else min(have, case["count"])      # blocks of a sequence, each once at least
        scored += have if have > case["count"] else 0
        fresh += (c + n) // BLOCK - c // BLOCK
        for i in range(n):
            pairs += min(c + i + 1, case["count"] * BLOCK)
    # picks are written, and read by the attention; each bound and each block that is looked at is read once; keys of new blocks are read for their bounds
    blocks = sum(-(-(c + n) // BLOCK) for c in ctx)
    bounds = (scored + fresh) * hkv * (2 * D + 16)
    return {"bytes": read * BLOCK * row + bounds + fresh * BLOCK * row // 2 + io + 4 * T * hkv * case["count"] + 4 * blocks,
            "flops": 4 * pairs * case["hq"] * D + (4 * n * scored * hkv * D)}


def exact(case, seed):
    """Sequence by sequence in fp64, from the definitions."""
    if case["op"] == "store":
        return _exact_store(case, seed)
    s = prepare(case, seed)
    hq, hkv, D, n, G = case["hq"], case["hkv"], case["dim"], case["rows"], case["hq"] // case["hkv"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for b, c in enumerate(_spread(case["ctx_lo"], case["ctx_hi"], case["seqs"])):
        pages = s.tables[b, :-(-(c + n) // BLOCK)].long()
        keys, values = (_exact_rows(t[pages], case).transpose(0, 1).flatten(1, 2) for t in (s.kc, s.vc))     # [hkv, tokens, D]
        j = torch.arange(keys.shape[1], device="cuda")
        me = c + torch.arange(n, device="cuda")
        seen = j[None] <= me[:, None]
        if case["op"] == "attend" and case["window"]:
            seen = seen & ((me[:, None] - j[None] < case["window"]) | (j[None] < case["first"]))
        for h in range(hkv):
            q = s.q[b * n:(b + 1) * n, h * G * D:(h + 1) * G * D].to(torch.float64).view(n, G, D)
            look = seen if case["op"] == "attend" else seen & _exact_choice(q, keys[h], me, case)
            x = torch.einsum("rgd,cd->rgc", q, keys[h]) * s.scale
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            x = torch.where(look[:, None], x, torch.full_like(x, -math.inf))
            if s.sinks is not None:
                x = torch.cat([x, s.sinks[h * G:(h + 1) * G].to(torch.float64).view(1, G, 1).expand(n, G, 1)], 2)
            p = torch.softmax(x, 2)[..., :keys.shape[1]]
            out[b * n:(b + 1) * n, h * G * D:(h + 1) * G * D] = torch.einsum("rgc,cd->rgd", p, values[h]).flatten(1)
    return out if case["op"] == "attend" else (out, None, None)


def _exact_rows(t, case):
    kv, D = case.get("kv", "int4"), case["dim"]
    if kv != "int4":
        return t.to(torch.float64)
    word = t.to(torch.int64)
    d = torch.arange(D, device="cuda")
    code = word[..., d // 2] >> (4 * (d % 2)) & 15
    step, low = ((word[..., D // 2 + i:D // 2 + i + 1] | word[..., D // 2 + i + 1:D // 2 + i + 2] << 8).to(torch.int16).view(torch.bfloat16).to(torch.float64)
                 for i in (0, 2))
    return (low + step * code).float().to(torch.float64)


def _exact_choice(q, keys, me, case):
    """Tokens [rows, tokens] of the blocks that each row reads."""
    n, tokens = q.shape[0], keys.shape[0]
    blocks = tokens // BLOCK
    k = keys.view(blocks, BLOCK, -1)
    hi, lo = k.amax(1), k.amin(1)
    unit = torch.maximum(hi.abs(), lo.abs()).amax(1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(unit / 127)))
    hi, lo = torch.ceil(hi / unit), torch.floor(lo / unit)
    plus, minus = q.clamp(min=0).sum(1), (-q).clamp(min=0).sum(1)
    one = torch.exp2(torch.ceil(torch.log2(torch.maximum(plus, minus).amax(1, keepdim=True) / 127)))
    score = (torch.round(plus / one) @ hi.T - torch.round(minus / one) @ lo.T) * unit.T
    keep = torch.zeros(n, blocks, dtype=torch.bool, device="cuda")
    for r in range(n):
        last = int(me[r]) // BLOCK + 1
        keep[r, :last] = True
        if last <= case["count"]:
            continue
        between = score[r, case["lead"]:last - case["tail"]]
        order = torch.argsort(between, descending=True, stable=True)[case["count"] - case["lead"] - case["tail"]:]
        keep[r, case["lead"] + order] = False
    return keep.repeat_interleave(BLOCK, 1)


def _exact_store(case, seed):
    s = prepare(case, seed)
    out = []
    for rows in (s.k, s.v):
        x = rows.to(torch.float64).view(-1, case["hkv"], case["dim"])
        low = _eight_bits(x.amin(-1, keepdim=True), torch.floor)
        step = _eight_bits(torch.div(x.amax(-1, keepdim=True) - low, torch.full_like(low, 15)), torch.ceil)
        value = low + step * torch.round((x - low) / step).clamp(0, 15)
        out.append(torch.where((s.slots >= 0)[:, None], value.flatten(1), torch.zeros_like(value.flatten(1))))
    return tuple(out)


def _eight_bits(x, way):
    """x on the grid of 8 significant bits, rounded the way that is given."""
    unit = torch.exp2((torch.frexp(x)[1] - 8).to(torch.float64))
    return way(x / unit) * unit
