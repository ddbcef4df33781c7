"""fp64 statement of attention under a window with first tokens and of draft trees, token by token, and how far the kernels may be from it.

The bound of an output: its weights w_j are rounded to bf16 for the product with the values (relative 2^-8, f16: 2^-11), the output once more (2^-8 of
it); a score is off by at most (D + 4) 2^-24 sum_d |q_d k_d| scale from its fp32 sum and by 2^-22 |s| from its factor, its exponent and a soft-cap (twice
that of its magnitude), e^x and the sums over n keys add (n + 64) 2^-24. An error e of all scores moves an output by at most 2 e A,
A = sum_j w_j |v_j|. So |o' - o| <= (2^-8 + 2 e_s) A + 2^-8 |o| + tiny, second-order terms covered by a factor of 1.1. Beside an e4m3
cache queries may lose 2^-17 of the row's largest magnitude in their small values, which moves a score by 2^-17 max|q| sum_d |k_d| scale; weights are f16
there, and 2 x 2^-17 max|q| sum|k| scale <= 2^-8 - 2^-11 up to max|q| sum|k| scale = 223 (here: at most 6.75 x 256 x 0.8 / 16 = 87), so the bound is the
same.
"""
import math
from types import SimpleNamespace

import torch


def tree_paths(parents):
    path, depth = [], []
    for i, p in enumerate(parents):
        path.append([i] if p < 0 else path[p] + [i])
        depth.append(0 if p < 0 else depth[p] + 1)
    return path, depth


def masks_of(parents, words):
    rows = []
    for line in tree_paths(parents)[0]:
        m = sum(1 << i for i in line)
        parts = [(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
        rows.append([x - (1 << 64) if x >> 63 else x for x in parts])
    return rows


def seen_rows(ctx, n, window, first, parents=None):
    """[n, ctx + n] truth values: what every row of a sequence sees."""
    j = torch.arange(ctx + n)
    if parents is None:
        where, me = j, j[ctx:]
        seen = j[None] <= me[:, None]
    else:
        path, depth = tree_paths(parents)
        where = torch.cat([j[:ctx], ctx + torch.tensor(depth, dtype=torch.long)])
        me = where[ctx:]
        seen = torch.zeros(n, ctx + n, dtype=torch.bool)
        seen[:, :ctx] = True
        for i, line in enumerate(path):
            seen[i, [ctx + x for x in line]] = True
    if window:
        seen = seen & ((me[:, None] - where[None] < window) | (where[None] < first))
    return seen


def attend(q, k, v, seen, scale, sinks=None, cap=0.0):
    """q [n, hq, D], k, v [N, hkv, D], seen [n, N] -> (outputs, bounds) [n, hq, D] in fp64."""
    q, k, v = q.double(), k.double(), v.double()
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    k = torch.where(seen.any(0).to(k.device)[:, None, None], k, torch.zeros_like(k))          # what nobody sees may be anything
    v = torch.where(seen.any(0).to(k.device)[:, None, None], v, torch.zeros_like(v))
    s = torch.einsum("nhd,mhd->nhm", q, k) * scale
    size = torch.einsum("nhd,mhd->nhm", q.abs(), k.abs()) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    vis = seen.to(s.device)[:, None]
    s = s.masked_fill(~vis, -math.inf)
    top = s.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks.double().to(s.device)[None, :, None])
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks.double().to(s.device)[None, :, None] - top)
    w = w / total.clamp(min=1e-300)
    o = torch.einsum("nhm,mhd->nhd", w, v)
    D, N = q.shape[2], k.shape[0]
    off = (size.masked_fill(~vis, 0).amax(-1) * ((D + 4) * 2.0 ** -24 + 2.0 ** -21) + (N + 64) * 2.0 ** -24)[..., None]
    A = torch.einsum("nhm,mhd->nhd", w, v.abs())
    return o, 1.1 * ((2.0 ** -8 + 2 * off) * A + 2.0 ** -8 * o.abs()) + 1e-30


def setup(rows, ctx, hq, hkv, D, kv="bf16", block=16, words=0, trees=None, seed=0, device="cuda", spare=4, fill=0.0, q_scale=1.5, pool_blocks=0, q_pitch=0):
    """Caches with the sequences' pages at random places, queries, the step batch; `fill`: what every other place of the pools holds."""
    g = torch.Generator(device=device).manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, rows)]
    need = [-(-n // block) for n in lens]
    blocks = pool_blocks or sum(need) + spare
    order = (torch.randperm(sum(need) + spare, generator=g, device=device) + (blocks - sum(need) - spare)).int()
    tables = torch.full((len(rows), max(max(need), 1)), -1, dtype=torch.int32, device=device)
    pools, flat = [], []
    for _ in range(2):
        pools.append(torch.full((blocks, hkv, block, D), fill, dtype=torch.bfloat16, device=device))
        flat.append([])
    at = 0
    for s, n in enumerate(lens):
        pages = order[at:at + need[s]]
        at += need[s]
        tables[s, :need[s]] = pages
        tok = torch.arange(n, device=device)
        for pool, mine in zip(pools, flat):
            x = torch.randn(n, hkv, D, generator=g, device=device).bfloat16()
            if kv == "e4m3":
                x = x.to(torch.float8_e4m3fn).bfloat16()
            if n:
                pool[pages.long()[tok // block], :, tok % block] = x
            mine.append(x)
    if kv == "e4m3":
        pools = [p.to(torch.float8_e4m3fn) for p in pools]
    T = sum(rows)
    q = torch.randn(T, q_pitch or hq * D, generator=g, device=device)[:, :hq * D]
    q = (q * q_scale).bfloat16() if not q_pitch else (torch.randn(T, q_pitch, generator=g, device=device) * q_scale).bfloat16()[:, q_pitch - hq * D:]
    starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=device)
    seq = [s for s, n in enumerate(rows) for _ in range(n)]
    meta = SimpleNamespace(q_starts=i32(starts), seq_lens=i32(lens), num_seqs=len(rows), num_tokens=T, max_q_len=max(rows), min_q_len=min(rows),
                           max_kv_len=max(lens))
    out = SimpleNamespace(q=q, k=pools[0], v=pools[1], keys=flat[0], values=flat[1], tables=tables, meta=meta, row_seq=i32(seq), rows=rows, ctx=ctx, starts=starts,
                          lens=lens, trees=trees, hq=hq, hkv=hkv, D=D, base=i32([ctx[s] for s in seq]),
                          positions=i32([(ctx[s] + i if trees is None else lens[s] - 1) for s, n in enumerate(rows) for i in range(n)]))
    if trees is not None:
        out.masks = torch.tensor([m for t in trees for m in masks_of(t, words)], dtype=torch.int64, device=device)
    return out


def want(c, scale, window, first, sinks=None, cap=0.0):
    os, bs = [], []
    for s, n in enumerate(c.rows):
        if not n:
            continue
        q = c.q[c.starts[s]:c.starts[s] + n].reshape(n, c.hq, c.D)
        o, b = attend(q, c.keys[s], c.values[s], seen_rows(c.ctx[s], n, window, first, None if c.trees is None else c.trees[s]), scale, sinks, cap)
        os.append(o.reshape(n, -1))
        bs.append(b.reshape(n, -1))
    return torch.cat(os), torch.cat(bs)


def check(y, o, bound):
    y = y.double()
    assert torch.equal(torch.isnan(y), torch.isnan(o)), "NaN in other places"
    fine = torch.isfinite(o)
    assert torch.equal(y[~fine & ~torch.isnan(o)], o[~fine & ~torch.isnan(o)])
    over = ((y - o).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"{over.max().item()} over the bound, {(over > 0).sum().item()} of {over.numel()} values"


def grow(nodes, seed, fan=3):
    import random
    r = random.Random(seed)
    return [-1] + [max(0, i - r.randint(1, fan)) for i in range(1, nodes)] if nodes else []
