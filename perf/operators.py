"""Operators over the paged key / value cache that are measured: attention under a sliding window with a few first tokens that stay
visible, attention for trees of drafted tokens, copies of blocks (forks) and the move of accepted tree rows to their places.

``own`` False: the plain form, elementary tensor operations in fp32 on the pages that are visible; True: the calls of ``NativeOps``.

Fields of a case:
  op        window | tree | copy | compact
  seqs      sequences of the step; ctx_lo, ctx_hi: tokens they have in the cache before it, spread evenly between
  rows      window: new tokens per sequence (1: decode). tree, compact: nodes_lo, nodes_hi drafted nodes per sequence, the root among them
  hq, hkv, dim   query heads, key heads, head dim (hq is not used by copy and compact); layers: of the pool that is copied in
  window, first  a row sees the last ``window`` tokens up to itself and the first ``first`` ones (window 0: all before it)
  kv        bf16 | e4m3, what the cache holds
  sinks     whether each head has a logit of its own in the sum; cap: soft-cap of the scores (0: none)
  pairs     copy: blocks that are copied
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

BLOCK = 16
DEPTH = 6            # levels of a draft tree below its root, at most


def _attn(name, op, seqs, ctx_lo, ctx_hi, hq, hkv, dim, window=0, first=0, kv="bf16", sinks=False, cap=0.0, **more):
    return dict(name=name, op=op, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, hq=hq, hkv=hkv, dim=dim, window=window, first=first, kv=kv, sinks=sinks,
                cap=cap, **more)


def listed():
    return [
        # one user, one token: what a step costs that reads next to nothing
        _attn("window_decode_1", "window", 1, 700, 700, 32, 8, 128, 256, 4, rows=1),
        # a full batch of long conversations, the heads of the 8B preset
        _attn("window_decode_64", "window", 64, 4000, 32000, 32, 8, 128, 4096, 4, rows=1),
        # heads of 64 with a logit of their own, an 8-bit cache, a window and first tokens that end inside pages and tiles
        _attn("window_decode_48_fp8", "window", 48, 900, 9001, 64, 8, 64, 1000, 130, kv="e4m3", sinks=True, rows=1),
        # chunks of two long prompts
        _attn("window_prompt_2x2048", "window", 2, 2500, 6143, 32, 8, 128, 1024, 64, rows=2048),
        # chunks of odd lengths over an 8-bit cache
        _attn("window_prompt_3x777_fp8", "window", 3, 1, 3001, 64, 8, 64, 512, 16, kv="e4m3", rows=777),
        # one user's draft tree
        _attn("tree_1", "tree", 1, 900, 900, 32, 8, 128, nodes_lo=12, nodes_hi=12),
        # trees of 64 nodes behind contexts of many lengths
        _attn("tree_16x64", "tree", 16, 1000, 12000, 32, 8, 128, nodes_lo=64, nodes_hi=64),
        # ragged trees, some of more than 64 nodes, five heads to a key head, window and first tokens, an 8-bit cache
        _attn("tree_40_fp8", "tree", 40, 100, 8000, 40, 8, 128, 2048, 4, kv="e4m3", nodes_lo=8, nodes_hi=100),
        # one sequence that writes into a shared last block, and a beam's worth of them; pools of 36 and of 24 layers
        dict(name="fork_1", op="copy", layers=36, hkv=8, dim=128, kv="bf16", pairs=1),
        dict(name="fork_160", op="copy", layers=36, hkv=8, dim=128, kv="bf16", pairs=160),
        # accepted rows of a few small trees (8-bit cache), and of a full batch of large ones
        dict(name="compact_3_fp8", op="compact", layers=24, hkv=8, dim=64, kv="e4m3", seqs=3, nodes_lo=9, nodes_hi=30),
        dict(name="compact_64", op="compact", layers=36, hkv=8, dim=128, kv="bf16", seqs=64, nodes_lo=20, nodes_hi=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds that neither form can do without, roughly: the fp32 products of the plain form weigh most."""
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 5e13


def _scores(case):
    """Scores that the plain form holds at a time: rows by columns of the longest sequence."""
    rows = case["rows"] if case["op"] == "window" else case["nodes_hi"]
    cols = min(case["ctx_hi"] + rows, case["window"] + rows + case["first"]) if case["window"] else case["ctx_hi"] + rows
    return case["seqs"] * case["hq"] * rows * cols


def draw(rng):
    top = {c["op"]: 0.0 for c in listed()}
    for c in listed():
        top[c["op"]] = max(top[c["op"]], _cost(c))
    while True:
        op = rng.choice(["window", "window", "window", "tree", "tree", "tree", "copy", "compact"])
        kv = rng.choice(["bf16", "bf16", "e4m3"])
        hkv, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128])
        if op == "copy":
            c = dict(op=op, layers=rng.randint(1, 36), hkv=hkv, dim=dim, kv=kv, pairs=_log(rng, 1, 160))
        elif op == "compact":
            lo = _log(rng, 1, 60)
            c = dict(op=op, layers=rng.randint(1, 36), hkv=hkv, dim=dim, kv=kv, seqs=_log(rng, 1, 64), nodes_lo=lo, nodes_hi=rng.randint(lo, 100))
        else:
            hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
            windowed = op == "window" or rng.random() < 0.4
            window = _log(rng, 32, 4096) if op == "window" else _log(rng, 128, 4096) if windowed else 0
            first = _log(rng, 1, 256) if windowed else 0
            ctx = _log(rng, 1, 16000)
            c = _attn("", op, _log(rng, 1, 64), rng.randint(max(1, ctx // 8), ctx), ctx, hq, hkv, dim, window, first, kv, rng.random() < 0.3,
                      rng.choice([0.0, 0.0, 0.0, 30.0]))
            del c["name"]
            if op == "window":
                c["rows"] = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
            else:
                c["nodes_lo"] = _log(rng, 1, 64)
                c["nodes_hi"] = rng.randint(c["nodes_lo"], 160)
        if _cost(c) <= top[op] and (op in ("copy", "compact") or _scores(c) <= 420_000_000):
            return c


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _tree(rng, nodes):
    """Parents of a draft tree of ``nodes`` nodes (node 0 the root, the token that was emitted last): nodes in the order of their depth, the
    likelier ones with more children."""
    parents, depth = [-1], [0]
    width = max(2, (nodes - 1 + DEPTH - 1) // DEPTH)
    level = [0]
    while len(parents) < nodes:
        nxt = []
        for _ in range(min(width, nodes - len(parents))):
            p = level[min(len(level) - 1, int(rng.expovariate(1.0)))]
            nxt.append(len(parents))
            parents.append(p)
            depth.append(depth[p] + 1)
        parents[nxt[0]:] = sorted(parents[nxt[0]:])
        level = nxt if len(nxt) == width else level
    return parents


def _bits(parents):
    m = []
    for i, p in enumerate(parents):
        m.append((1 << i) | (m[p] if p >= 0 else 0))
    return m


def _lens(case):
    """Per sequence: tokens in the cache before the step, new rows, and (trees) parents."""
    if case["op"] == "window":
        ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"])
        return ctx, [case["rows"]] * case["seqs"], None
    n = _spread(case["nodes_lo"], case["nodes_hi"], case["seqs"])
    rng = random.Random(case["seqs"] * 1000 + case["nodes_hi"])
    rng.shuffle(n)
    trees = [_tree(rng, k) for k in n]
    if case["op"] == "compact":
        return [rng.randint(1, 40) for _ in n], n, trees
    return _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"]), n, trees


def _normal(g, shape, kv):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    return x.to(torch.float8_e4m3fn) if kv == "e4m3" else x


def _tables(g, lens, blocks):
    """Pages of each sequence at random places of the pool; block 0 behind the last one."""
    need = [-(-n // BLOCK) for n in lens]
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    cols = torch.arange(max(need), device="cuda")
    t = order[(starts[:, None] + cols).clamp(max=blocks - 1)]
    return torch.where(cols < torch.tensor(need, device="cuda")[:, None], t, torch.zeros_like(t)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    s = SimpleNamespace(case=case, op=case["op"])
    if case["op"] == "copy":
        blocks = 2 * case["pairs"] + 8
        s.store = _normal(g, (case["layers"], 2, blocks, case["hkv"], BLOCK, case["dim"]), case["kv"])
        s.pairs = torch.randperm(blocks, generator=g, device="cuda")[:2 * case["pairs"]].view(-1, 2).to(torch.int32).contiguous()
        return s
    ctx, rows, trees = _lens(case)
    lens = [c + n for c, n in zip(ctx, rows)]
    blocks = sum(-(-n // BLOCK) for n in lens) + 3
    s.tables = _tables(g, lens, blocks)
    if case["op"] == "compact":
        # accepted paths: the first child of the root, then nodes behind the last place that is written (a path's rows never overwrite
        # what the same move would read again, so the call can be made again on the same state)
        rng = random.Random(seed)
        paths = []
        for parents in trees:
            path = [0]
            if len(parents) > 1:
                path.append(1)
            limit = rng.randint(1, DEPTH)
            while len(path) < limit:
                nxt = [i for i in range(DEPTH + 1, len(parents)) if parents[i] == path[-1] or (len(path) == 2 and i > path[-1])]
                if not nxt:
                    break
                path.append(rng.choice(nxt))
            paths.append(path[:limit])
        s.store = _normal(g, (case["layers"], 2, blocks, case["hkv"], BLOCK, case["dim"]), case["kv"])
        s.base = i32(ctx)
        s.path = i32([p + [0] * (DEPTH + 1 - len(p)) for p in paths])
        s.counts = i32([len(p) for p in paths])
        return s
    T, B = sum(rows), len(rows)
    shape = (blocks, case["hkv"], BLOCK, case["dim"])
    s.k, s.v = _normal(g, shape, case["kv"]), _normal(g, shape, case["kv"])
    s.q = 1.5 * torch.randn(T, case["hq"] * case["dim"], generator=g, device="cuda", dtype=torch.bfloat16)
    s.sinks = torch.randn(case["hq"], generator=g, device="cuda") if case["sinks"] else None
    s.scale = case["dim"] ** -0.5
    starts = [sum(rows[:i]) for i in range(B)] + [T]
    s.starts, s.lens, s.ctx = i32(starts), i32(lens), i32(ctx)
    s.row_seq = torch.repeat_interleave(torch.arange(B, dtype=torch.int32, device="cuda"), i32(rows).long())
    s.local = torch.arange(T, dtype=torch.int32, device="cuda") - s.starts[s.row_seq.long()]       # row of its sequence
    s.max_rows, s.min_rows, s.max_len = max(rows), min(rows), max(lens)
    s.meta = SimpleNamespace(q_starts=s.starts, seq_lens=s.lens, num_seqs=B, num_tokens=T, max_q_len=s.max_rows, min_q_len=s.min_rows,
                             max_kv_len=s.max_len)
    if case["op"] == "window":
        s.positions = s.ctx[s.row_seq.long()] + s.local
        return s
    words = -(-s.max_rows // 64)
    flat = []
    for t in trees:
        for m in _bits(t):
            parts = [(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
            flat.append([x - (1 << 64) if x >> 63 else x for x in parts])
    s.masks = torch.tensor(flat, dtype=torch.int64, device="cuda")
    s.base = s.ctx[s.row_seq.long()].contiguous()
    s.positions = s.lens[s.row_seq.long()] - 1
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
        if s.op == "copy":
            ops.kv_copy_blocks([s.store.flatten(0, 1)], s.pairs)
            return _bytes(s.store)
        if s.op == "compact":
            ops.kv_compact([s.store.flatten(0, 1)], s.tables, s.base, s.path, s.counts)
            return _bytes(s.store)
        if s.op == "window":
            return ops.attention(s.q, s.k, s.v, s.tables, s.row_seq, s.positions, c["hq"], c["hkv"], c["dim"], s.scale, c["window"], s.sinks,
                                 c["cap"], meta=s.meta, first=c["first"])
        return ops.attention_tree(s.q, s.k, s.v, s.tables, s.row_seq, s.positions, s.masks, s.base, c["hq"], c["hkv"], c["dim"], s.scale,
                                  c["window"], s.sinks, c["cap"], first=c["first"], meta=s.meta)
    if s.op == "copy":
        flat = _bytes(s.store)
        flat[:, :, s.pairs[:, 1].long()] = flat[:, :, s.pairs[:, 0].long()]
        return flat
    if s.op == "compact":
        return _plain_compact(s)
    return _plain_attention(s)


def _bytes(store):
    """The pool as whole numbers: copies are equal bit by bit."""
    return store.view(torch.uint8 if store.element_size() == 1 else torch.int16)


def _plain_compact(s):
    flat = _bytes(s.store)
    n = s.path.shape[1]
    step = torch.arange(n, device="cuda")
    live = step < s.counts[:, None]
    src, dst = s.base[:, None] + s.path, s.base[:, None] + step
    page = lambda at: torch.gather(s.tables, 1, (at // BLOCK).clamp(max=s.tables.shape[1] - 1).long())[live].long()
    rows = flat[:, :, page(src), :, (src % BLOCK)[live].long()]
    flat[:, :, page(dst), :, (dst % BLOCK)[live].long()] = rows
    return flat


def _plain_attention(s):
    c = s.case
    hq, hkv, D, W, F = c["hq"], c["hkv"], c["dim"], c["window"], c["first"]
    B, R = s.lens.shape[0], s.max_rows
    # columns: the first tokens, then those from where the first row's window begins
    lo = (s.ctx + 1 - W).clamp(min=0) if W else torch.zeros_like(s.ctx)
    F = min(F, s.max_len) if W else 0
    span = min(s.max_len, W + R) if W else s.max_len
    col = torch.arange(F + span, device="cuda")
    tok = torch.where(col < F, col, lo[:, None] + col - F)                                           # [B, C]
    there = (tok < s.lens[:, None]) & ((col < F) | (tok >= F))
    at = tok.clamp(max=s.max_len - 1)
    page = torch.gather(s.tables, 1, (at // BLOCK).long()).long()
    K = s.k.view(torch.uint8)[page, :, at % BLOCK].view(s.k.dtype).float() if c["kv"] == "e4m3" else s.k[page, :, at % BLOCK].float()
    V = s.v.view(torch.uint8)[page, :, at % BLOCK].view(s.v.dtype).float() if c["kv"] == "e4m3" else s.v[page, :, at % BLOCK].float()
    q = torch.zeros(B, R, hq * D, device="cuda")
    seq, loc = s.row_seq.long(), s.local.long()
    q[seq, loc] = s.q.float()
    q = q.view(B, R, hkv, hq // hkv, D)
    score = torch.einsum("brhgd,bchd->bhgrc", q, K) * s.scale
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    row = torch.arange(R, device="cuda")
    if c["op"] == "window":
        pos = s.ctx[:, None] + row                                                                   # [B, R]
        seen = tok[:, None] <= pos[:, :, None]
        seen &= (tok[:, None] > pos[:, :, None] - W) | (tok[:, None] < F)
    else:
        words = torch.zeros(B, R, s.masks.shape[1], dtype=torch.int64, device="cuda")
        words[seq, loc] = s.masks
        node = (tok - s.ctx[:, None])                                                                # [B, C], negative: context
        inside = node.clamp(0, s.masks.shape[1] * 64 - 1)
        word = torch.gather(words, 2, (inside // 64).long()[:, None].expand(B, R, inside.shape[1]))
        anc = ((word >> (inside % 64)[:, None]) & 1).bool() & (node >= 0)[:, None]                   # ancestors and the node itself
        seen = anc | (node < 0)[:, None]
        if W:
            every = torch.arange(R, device="cuda")
            own_bits = (torch.gather(words, 2, (every // 64)[None, None].expand(B, R, R)) >> (every % 64)) & 1   # [B, row, node]
            depth = own_bits.sum(2) - 1                                                              # [B, R]
            place = s.ctx[:, None] + torch.gather(depth, 1, node.clamp(0, R - 1).long())             # of a node's token in its path
            place = torch.where(node < 0, tok, place)
            pos = s.ctx[:, None] + depth
            seen &= (place[:, None] > pos[:, :, None] - W) | (place[:, None] < F)
    seen = seen & there[:, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s.sinks is not None:
        extra = s.sinks.view(1, hkv, hq // hkv, 1, 1)
        top = torch.maximum(top, extra)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(extra - top)
    o = torch.einsum("bhgrc,bchd->brhgd", p / total.clamp(min=1e-30), V)
    return o.reshape(B, R, hq * D)[seq, loc].to(s.q.dtype)


def work(case):
    elem = 1 if case["kv"] == "e4m3" else 2
    if case["op"] == "copy":
        block = case["layers"] * 2 * case["hkv"] * BLOCK * case["dim"] * elem
        return {"bytes": 2 * case["pairs"] * block + 8 * case["pairs"], "flops": 0}
    ctx, rows, _ = _lens(case)
    if case["op"] == "compact":           # three rows or so per sequence move
        row = case["layers"] * 2 * case["hkv"] * case["dim"] * elem
        return {"bytes": sum(2 * row * max(0, min(n, 4) - 2) + 40 for n in rows), "flops": 0}
    W, F = case["window"], case["first"]
    keys = pairs = 0
    for c, n in zip(ctx, rows):
        if case["op"] == "window":
            lo = max(0, c + 1 - W)
            keys += c + n - lo + min(F, lo)
            for i in ([0] if n == 1 else range(n)):
                beg = max(0, c + i + 1 - W)
                pairs += c + i + 1 - beg + min(F, beg)
        else:
            lo = max(0, c + 1 - W) if W else 0
            keys += c + n - lo + min(F, lo)
            pairs += n * (c - lo + min(F, lo) + min(n, DEPTH))
    D, T = case["dim"], sum(rows)
    return {"bytes": keys * case["hkv"] * D * 2 * elem + 4 * T * case["hq"] * D + 4 * sum(-(-n // BLOCK) for n in [c + r for c, r in zip(ctx, rows)]),
            "flops": 4 * pairs * case["hq"] * D}


def exact(case, seed):
    """Sequence by sequence and head by head in fp64: what each row sees is written down from the definition, token by token."""
    if case["op"] in ("copy", "compact"):
        return None
    s = prepare(case, seed)
    ctx, rows, trees = _lens(case)
    hq, hkv, D, W, F = case["hq"], case["hkv"], case["dim"], case["window"], case["first"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    k, v, t0 = s.k.to(torch.float64), s.v.to(torch.float64), 0
    for b, (c, n) in enumerate(zip(ctx, rows)):
        pages = s.tables[b, :-(-(c + n) // BLOCK)].long()
        kb = k[pages].transpose(0, 1).reshape(hkv, -1, D)[:, :c + n]
        vb = v[pages].transpose(0, 1).reshape(hkv, -1, D)[:, :c + n]
        j = torch.arange(c + n, device="cuda")
        if trees is None:
            where, me = j, j[c:]                                    # place of a token in the text, and of each row
            seen = j[None] <= me[:, None]
        else:
            depth, path = [], []
            for i, p in enumerate(trees[b]):
                depth.append(0 if p < 0 else depth[p] + 1)
                path.append([i] if p < 0 else path[p] + [i])
            where = torch.cat([j[:c], c + torch.tensor(depth, device="cuda")])
            me = where[c:]
            seen = torch.zeros(n, c + n, dtype=torch.bool)
            seen[:, :c] = True
            for i, line in enumerate(path):
                seen[i, [c + x for x in line]] = True
            seen = seen.cuda()
        if W:
            seen = seen & ((me[:, None] - where[None] < W) | (where[None] < F))
        for h in range(hq):
            x = (s.q[t0:t0 + n, h * D:(h + 1) * D].to(torch.float64) @ kb[h // (hq // hkv)].T) * s.scale
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            if s.sinks is not None:
                x = torch.cat([x, s.sinks[h].to(torch.float64).expand(n, 1)], 1)
            p = torch.softmax(x, 1)[:, :c + n]
            out[t0:t0 + n, h * D:(h + 1) * D] = p @ vb[h // (hq // hkv)]
        t0 += n
    return out
