"""Attention under a window with first tokens that stay visible, draft trees over the cache, and moves inside the pools, on the kernels
against fp64."""
import math
from types import SimpleNamespace

import pytest
import torch

import span_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fllm_b200.ops.native import NativeOps
    return NativeOps(torch.device("cuda:0"))


def _window(ops, c, window, first, sinks=None, cap=0.0):
    return ops.attention(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.hq, c.hkv, c.D, c.D ** -0.5, window, sinks, cap, meta=c.meta, first=first)


def _tree(ops, c, window=0, first=0, sinks=None, cap=0.0):
    return ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks, c.base, c.hq, c.hkv, c.D, c.D ** -0.5, window, sinks, cap,
                              first=first, meta=c.meta)


def _sinks(hq):
    return torch.linspace(-3, 3, hq, device="cuda")


HEADS = [(8, 2, 128), (16, 2, 64), (4, 4, 64), (5, 1, 128), (14, 2, 128), (32, 2, 64), (8, 4, 256)]


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("window,first,sink,cap", [(33, 4, False, 0.0), (128, 70, True, 0.0), (1, 1, False, 0.0), (250, 16, False, 20.0)])
def test_window_rows(ops, hq, hkv, D, kv, window, first, sink, cap):
    """Decode and short rows of sequences of many lengths, one of no row and ones shorter than the window or the first tokens."""
    rows, ctx = [1, 2, 1, 0, 7, 1, 3], [0, 5, 300, 10, 129, 1777, 15]
    c = so.setup(rows, ctx, hq, hkv, D, kv, seed=hq + D, fill=float("nan"))
    s = _sinks(hq) if sink else None
    y = _window(ops, c, window, first, s, cap)
    so.check(y, *so.want(c, D ** -0.5, window, first, s, cap))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("window,first", [(64, 5), (500, 130), (17, 200)])
def test_window_prompts(ops, hq, hkv, D, kv, window, first):
    """Chunks of prompts beside decode rows, chunks from the first token on, tiles that end inside pages."""
    rows, ctx = [130, 1, 257, 64], [0, 900, 411, 1]
    c = so.setup(rows, ctx, hq, hkv, D, kv, seed=hq * D, fill=float("nan"))
    y = _window(ops, c, window, first)
    so.check(y, *so.want(c, D ** -0.5, window, first))
    assert ops.check_status() == 0


def test_window_long_prompt_with_sinks_and_cap(ops):
    c = so.setup([700], [1300], 8, 2, 128, seed=3)
    s = _sinks(8)
    so.check(_window(ops, c, 600, 40, s, 15.0), *so.want(c, 128 ** -0.5, 600, 40, s, 15.0))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("window,first,sink", [(0, 0, False), (40, 3, True), (4, 2, False)])
def test_tree(ops, hq, hkv, D, kv, window, first, sink):
    """Trees of 1 to 200 nodes behind contexts of none to many tokens; windows that cut context and ancestors."""
    nodes, ctx = [1, 13, 64, 3, 200, 65], [50, 0, 333, 1, 129, 1030]
    c = so.setup(nodes, ctx, hq, hkv, D, kv, words=4, trees=[so.grow(n, n) for n in nodes], seed=D, fill=float("nan"))
    s = _sinks(hq) if sink else None
    y = _tree(ops, c, window, first, s)
    so.check(y, *so.want(c, D ** -0.5, window, first, s))
    assert ops.check_status() == 0


@pytest.mark.parametrize("words", [1, 2, 3, 4])
def test_tree_words_and_chains(ops, words):
    """A chain is a plain causal chunk; masks of one to four words."""
    n = 64 * words - 1
    chain = list(range(-1, n - 1))
    c = so.setup([n, 2], [77, 500], 8, 2, 128, words=words, trees=[chain, [-1, 0]], seed=words)
    if words == 1:
        c.masks = c.masks.view(-1)
    y = _tree(ops, c)
    so.check(y, *so.want(c, 128 ** -0.5, 0, 0))
    plain = SimpleNamespace(**{**vars(c), "trees": None})
    so.check(y, *so.want(plain, 128 ** -0.5, 0, 0))


def test_tree_equals_the_kernel_without_a_step_batch(ops):
    c = so.setup([30, 64], [100, 611], 8, 2, 128, words=1, trees=[so.grow(30, 1), so.grow(64, 2)], seed=11)
    o, bound = so.want(c, 128 ** -0.5, 0, 0)
    y = ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks.view(-1), c.base, 8, 2, 128, 128 ** -0.5)
    so.check(y, o, bound)
    so.check(_tree(ops, c), o, bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq", [2, 32])
def test_rows_that_see_nothing(ops, D, hq):
    """A mask of no bits behind an empty context: 0, with and without sinks; its neighbours are not disturbed."""
    c = so.setup([20], [0], hq, 2, D, words=1, trees=[so.grow(20, 5)], seed=2)
    c.masks[3] = 0
    c.masks[11] = 0
    for s in (None, _sinks(hq)):
        o, bound = so.want(c, D ** -0.5, 0, 0, s)
        y = _tree(ops, c, sinks=s)
        keep = [i for i in range(20) if i not in (3, 11)]
        so.check(y[keep], o[keep], bound[keep])
        assert (y[[3, 11]] == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", [(2, 2, 128), (8, 2, 128), (40, 2, 64), (4, 2, 256)])
def test_infinities_and_nan_of_other_branches(ops, hq, hkv, D, kv):
    """Keys and values of a node that only some rows see: the others are as if they were not there, the ones that see them get what the
    formula gives."""
    nodes = 40
    par = [-1] + [max(0, i - 4) for i in range(1, nodes)]          # a root with four chains, one odd value in each
    c = so.setup([nodes], [133], hq, hkv, D, kv, words=1, trees=[par], seed=5)
    bad = {9: float("nan"), 22: float("inf"), 31: -float("inf")}
    if kv == "e4m3":
        bad = {9: float("nan"), 22: float("nan")}
    for node, x in bad.items():
        tok = 133 + node
        blk, off = int(c.tables[0, tok // 16]), tok % 16
        c.v[blk, :, off, 5] = x
        c.values[0][tok, :, 5] = x
    blk, off = int(c.tables[0, (133 + 16) // 16]), (133 + 16) % 16
    c.k[blk, :, off, 3] = float("nan")
    c.keys[0][133 + 16, :, 3] = float("nan")
    seen = so.seen_rows(133, nodes, 0, 0, par)
    y = _tree(ops, c).view(nodes, hq, D)
    clean = [i for i in range(nodes) if not seen[i, [133 + n for n in list(bad) + [16]]].any()]
    assert 0 < len(clean) < nodes
    vals = torch.nan_to_num(c.values[0].float(), 0, 0, 0)
    keys = torch.nan_to_num(c.keys[0].float(), 0, 0, 0)
    o, bound = so.attend(c.q.view(nodes, hq, D), keys, vals, seen, D ** -0.5)
    so.check(y[clean], o[clean], bound[clean])
    for node, x in bad.items():
        rows = [i for i in range(nodes) if seen[i, 133 + node] and not seen[i, 133 + 16] and not any(seen[i, 133 + n] for n in bad if n != node)]
        assert rows
        for i in rows:
            assert (torch.isnan(y[i, :, 5]) if math.isnan(x) else y[i, :, 5] == x).all()
            rest = [d for d in range(D) if d != 5]
            so.check(y[i][:, rest], o[i][:, rest], bound[i][:, rest])
    hit = [i for i in range(nodes) if seen[i, 133 + 16]]
    assert torch.isnan(y[hit]).all()


@pytest.mark.parametrize("hq,rows", [(2, 1), (8, 100)])
def test_stale_values_behind_and_before_what_is_seen(ops, hq, rows):
    """NaN in the rest of the last page, in pages that the window has passed and in tokens of its first page in front of it."""
    ctx, window, first = 700, 90, 20
    c = so.setup([rows], [ctx], hq, 2, 128, seed=8, fill=float("nan"))
    o, bound = so.want(c, 128 ** -0.5, window, first)
    for tok in range(first, ctx + 1 - window):
        blk, off = int(c.tables[0, tok // 16]), tok % 16
        c.v[blk, :, off] = float("nan")
        c.k[blk, :, off] = float("inf")
    for page in range(2, (ctx + 1 - window) // 16):
        c.tables[0, page] = -1                        # freed
    y = _window(ops, c, window, first)
    so.check(y, o, bound)
    assert ops.check_status() == 0


def test_strided_queries_and_larger_blocks(ops):
    c = so.setup([3, 150], [100, 200], 8, 2, 64, block=48, seed=4, q_pitch=8 * 64 + 264)
    assert c.q.stride(0) == 8 * 64 + 264
    y = _window(ops, c, 77, 9)
    so.check(y, *so.want(c, 0.125, 77, 9))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [1, 70])
def test_pools_of_more_than_32_bits(ops, kv, rows):
    """Pages behind 2^32 bytes and 2^31 values of a pool."""
    blocks = (1 << 31) // (8 * 16 * 128) + 500
    c = so.setup([rows], [300], 16, 8, 128, kv, seed=6, pool_blocks=blocks)
    assert int(c.tables.min()) * 8 * 16 * 128 > 1 << 31
    y = _window(ops, c, 200, 30)
    so.check(y, *so.want(c, 128 ** -0.5, 200, 30))
    pools = [c.k[None], c.v[None]]
    a = int(c.tables[0, 0])
    ops.kv_copy_blocks(pools, [(a, 1), (a, blocks - 1)])
    for t in (c.k, c.v):
        assert torch.equal(t[1].view(torch.uint8), t[a].view(torch.uint8)) and torch.equal(t[blocks - 1].view(torch.uint8), t[a].view(torch.uint8))
    assert ops.check_status() == 0


@pytest.mark.parametrize("rows", [1, 90])
def test_pages_that_are_not_there(ops, rows):
    """Entries of the block table that name no block are not followed; the status word says so."""
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    c = so.setup([rows], [300], 8, 2, 128, seed=9)
    good = c.tables.clone()
    for entry in (-1, c.k.shape[0], 1 << 30):
        c.tables.copy_(good)
        c.tables[0, 18] = entry
        _window(mine, c, 200, 4)
        assert mine.check_status() == 3
    c.tables.copy_(good)
    c.meta.seq_lens += 1 << 20                         # longer than its table
    _window(mine, c, 100, 4)
    assert mine.check_status() == 3


def test_streams_graphs_and_many_calls(ops):
    """On another stream, captured and replayed with other lengths and contents, two graphs replayed in turn, call after call."""
    c = so.setup([1, 40, 3], [600, 100, 2000], 8, 2, 128, seed=12)
    t = so.setup([30, 7], [500, 1500], 8, 2, 128, words=1, trees=[so.grow(30, 1), so.grow(7, 2)], seed=13)
    w1, w2 = so.want(c, 128 ** -0.5, 300, 4), so.want(t, 128 ** -0.5, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = _window(ops, c, 300, 4)
    side.synchronize()
    so.check(y, *w1)
    graphs, outs = [], []
    for f in (lambda: _window(ops, c, 300, 4), lambda: _tree(ops, t)):
        f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    so.check(outs[0], *w1)
    so.check(outs[1], *w2)
    # the same graph on shorter sequences: the lengths are read on the device
    short = so.setup([1, 40, 3], [77, 0, 1999], 8, 2, 128, seed=14)
    c.q.copy_(short.q)
    c.tables.fill_(-1)
    c.tables[:, :short.tables.shape[1]].copy_(short.tables)
    c.meta.seq_lens.copy_(short.meta.seq_lens)
    n = short.k.shape[0]
    c.k[:n].copy_(short.k)
    c.v[:n].copy_(short.v)
    graphs[0].replay()
    torch.cuda.synchronize()
    so.check(outs[0], *so.want(short, 128 ** -0.5, 300, 4))
    assert ops.check_status() == 0


def test_same_call_same_bits(ops):
    c = so.setup([33, 1, 256], [5000, 9000, 300], 16, 2, 128, seed=15)
    first = _window(ops, c, 1000, 64)
    for _ in range(5):
        assert torch.equal(_window(ops, c, 1000, 64), first)


def test_refusals(ops):
    c = so.setup([2], [40], 4, 2, 64, words=1, trees=[[-1, 0]], seed=1)
    call = lambda **kw: ops.attention(**{**dict(q=c.q, k_cache=c.k, v_cache=c.v, block_tables=c.tables, row_seq=c.row_seq, positions=c.positions, hq=4,
                                                hkv=2, head_dim=64, scale=0.125, window=16, first=4, meta=c.meta), **kw})
    bad = [dict(meta=None), dict(first=-1), dict(window=-3), dict(bidirectional=True), dict(q=c.q.float()), dict(q=c.q[:, 1:]), dict(scale=0.0),
           dict(scale=float("nan")), dict(softcap=-1.0), dict(hkv=3), dict(head_dim=96), dict(k_cache=c.k[..., :32]), dict(v_cache=c.v.float()),
           dict(k_cache=c.k.transpose(1, 2)), dict(block_tables=c.tables.long()), dict(sinks=torch.zeros(3, device="cuda")), dict(sinks=torch.zeros(4)),
           dict(q=c.q.cpu())]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    tree = lambda **kw: ops.attention_tree(**{**dict(q=c.q, k_cache=c.k, v_cache=c.v, block_tables=c.tables, row_seq=c.row_seq, positions=c.positions,
                                                     tree_mask=c.masks, tree_base=c.base, hq=4, hkv=2, head_dim=64, scale=0.125, meta=c.meta), **kw})
    tree()
    for kw in [dict(tree_mask=c.masks.int()), dict(tree_mask=c.masks[:1]), dict(tree_mask=c.masks.expand(2, 5).contiguous()), dict(tree_base=c.base.long()),
               dict(meta=None, first=2, tree_mask=c.masks.view(-1)), dict(window=-1)]:
        with pytest.raises((ValueError, RuntimeError)):
            tree(**kw)
    pool = torch.zeros(3, 6, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    for args in [([], [(0, 1)]), ([pool], [(0, 6)]), ([pool], [(-1, 2)]), ([pool], i32([0, 1])), ([pool], i32([[0, 1]]).long()), ([pool[0]], [(0, 1)]),
                 ([pool.transpose(2, 3)], i32([[0, 1]])), ([pool, pool[:, :5]], i32([[0, 1]])), ([pool.cpu()], i32([[0, 1]]))]:
        with pytest.raises((ValueError, RuntimeError, IndexError)):
            ops.kv_copy_blocks(*args)
    ok = (i32([[0, 1]]), i32([3]), i32([[0, 2]]), i32([2]))
    ops.kv_compact([pool], *ok)
    for k, x in [(0, i32([0, 1])), (0, i32([[0, 1]]).long()), (1, i32([])), (2, i32([0, 2])), (3, torch.tensor([2], dtype=torch.int32))]:
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv_compact([pool], *[x if k == j else a for j, a in enumerate(ok)])
    assert ops.check_status() == 0


# ------------------------------------------------------------------------------------------ moves
def _pools(kind, blocks, bs=16):
    g = torch.Generator(device="cuda").manual_seed(blocks)
    bits = lambda *s: torch.randint(0, 256, s, generator=g, device="cuda", dtype=torch.uint8)
    as_type = lambda x, t: x.view(t)
    if kind == "kv":
        return [as_type(bits(6, blocks, 3, bs, 256), torch.bfloat16)]
    if kind == "e4m3":
        return [as_type(bits(4, blocks, 2, bs, 64), torch.float8_e4m3fn)]
    if kind == "planes":                     # every second plane of a larger tensor
        return [as_type(bits(5, 2, blocks, 2, bs, 128), torch.bfloat16)[:, 1]]
    if kind == "rows":                       # a latent row, heads with a factor each, value rows of another width
        return [as_type(bits(1, blocks, 1, bs, 1152), torch.bfloat16), as_type(bits(1, blocks, 4, bs, 4), torch.float32), as_type(bits(1, blocks, 4, bs, 192), torch.bfloat16)]
    if kind == "odd":                        # rows of 6 bytes
        return [as_type(bits(2, blocks, 3, bs, 6), torch.bfloat16)]
    return [as_type(bits(1, blocks, 1, bs, 16), torch.bfloat16) for _ in range(100)]


def _same(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


KINDS = ["kv", "e4m3", "planes", "rows", "odd", "many"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [16, 5])
def test_copies_of_blocks(ops, kind, bs):
    from fllm_b200.ops.reference import RefOps
    pools = _pools(kind, 23, bs)
    ref = [t.clone() for t in pools]
    pairs = [(0, 22), (5, 6), (7, 8), (7, 9), (11, 11)]
    RefOps().kv_copy_blocks(ref, pairs)
    ops.kv_copy_blocks(pools, torch.tensor(pairs, dtype=torch.int32, device="cuda"))
    assert _same(pools, ref)
    chain = [(1, 2), (2, 3), (4, 2), (3, 1), (1, 4), (1, 5)]          # a list means one after the other
    RefOps().kv_copy_blocks(ref, chain)
    ops.kv_copy_blocks(pools, chain)
    assert _same(pools, ref)
    ops.kv_copy_blocks(pools, [])
    ops.kv_copy_blocks(pools, torch.zeros(0, 2, dtype=torch.int32, device="cuda"))
    assert _same(pools, ref) and ops.check_status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [16, 5])
def test_accepted_rows(ops, kind, bs):
    """Paths whose sources and destinations overlap, longer than a batch and than a thread block's list, of no node and of one."""
    from fllm_b200.ops.reference import RefOps
    pools = _pools(kind, 120, bs)
    ref = [t.clone() for t in pools]
    paths = [[0, 1, 2], [0, 2, 3, 7, 8, 9, 10, 11, 12, 13, 14, 40], [], [1], list(range(3, 93)), [5, 6, 7]]
    counts = [3, 12, 0, 1, 90, 2]
    depth = 95
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    per = -(-140 // bs)
    tables = torch.full((6, per), -1, dtype=torch.int32)
    order = torch.randperm(120, generator=torch.Generator().manual_seed(3)).int()
    used = [-(-n // bs) for n in (20, 60, 1, 9, 130, 16)]
    for s, n in enumerate(used):
        tables[s, :n] = order[sum(used[:s]):sum(used[:s]) + n]
    args = (tables.cuda(), i32([3, 17, 0, 5, 30, 8]), i32([p + [-7] * (depth - len(p)) for p in paths]), i32(counts))
    RefOps().kv_compact(ref, *args)
    ops.kv_compact(pools, *args)
    assert _same(pools, ref) and ops.check_status() == 0


def test_moves_that_name_no_block(ops):
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    pools = _pools("kv", 20)
    ref = [t.clone() for t in pools]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    mine.kv_copy_blocks(pools, i32([[0, 20], [-1, 3], [1 << 30, 2]]))
    assert mine.check_status() == 3 and _same(pools, ref)
    for base, path in [(0, [0, 70]), (40, [0, 5]), (-9, [0, 2]), (4, [3, 0])]:
        mine.kv_compact(pools, i32([[1, -1, 30]]), i32([base]), i32([path]), i32([2]))
        assert mine.check_status() == 3
        if path != [3, 0]:
            assert _same(pools, ref)


def test_moves_in_graphs_and_on_other_streams(ops):
    from fllm_b200.ops.reference import RefOps
    pools = _pools("kv", 30)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    pairs, path, counts = i32([[0, 1], [2, 3]]), i32([[0, 2, 5]]), i32([3])
    tables, base = i32([[7, 8, 9]]), i32([14])
    side = torch.cuda.Stream()
    ref = [t.clone() for t in pools]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.kv_copy_blocks(pools, pairs)
        ops.kv_compact(pools, tables, base, path, counts)
    side.synchronize()
    RefOps().kv_copy_blocks(ref, pairs)
    RefOps().kv_compact(ref, tables, base, path, counts)
    assert _same(pools, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_copy_blocks(pools, pairs)
        ops.kv_compact(pools, tables, base, path, counts)
    pairs.copy_(i32([[4, 5], [6, 10]]))
    path.copy_(i32([[0, 1, 4]]))
    g.replay()
    torch.cuda.synchronize()
    RefOps().kv_copy_blocks(ref, pairs)
    RefOps().kv_compact(ref, tables, base, path, counts)
    assert _same(pools, ref) and ops.check_status() == 0


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("window,first", [(0, 0), (50, 4)])
def test_tree_step_and_the_plain_step_after_it(ops, window, first):
    """A forked sequence (its shared last block copied) runs a tree step; the accepted path's rows move to their places; a plain step on the
    compacted cache sees exactly what a step after the accepted tokens alone would see."""
    from fllm_b200.models.decoder import KVCache
    from fllm_b200.runtime.speculative import DraftTree
    hq, hkv, D, ctx = 8, 2, 128, 133
    tree = DraftTree([5, 6, 7, 8, 9, 10, 11], [-1, 0, 0, 1, 2, 2, 5])
    kv = KVCache(3, 40, hkv, 16, D, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    text = torch.randn(3, 2, ctx, hkv, D, generator=g, device="cuda").bfloat16()
    node = torch.randn(3, 2, len(tree), hkv, D, generator=g, device="cuda").bfloat16()
    table = list(range(10, 20))
    for j in range(ctx):
        kv.store[:, :, table[j // 16], :, j % 16] = text[:, :, j]
    kv.copy_blocks([(table[8], 30)], ops)              # the block that is written next was shared
    table[8] = 30
    for i in range(len(tree)):
        kv.store[:, :, table[(ctx + i) // 16], :, (ctx + i) % 16] = node[:, :, i]
    assert torch.equal(kv.store[:, :, 18, :, 5], torch.zeros_like(kv.store[:, :, 18, :, 5]))           # the parent's copy has none of it
    M = len(tree)
    q = torch.randn(M, hq * D, generator=g, device="cuda").bfloat16()
    meta = SimpleNamespace(q_starts=i32([0, M]), seq_lens=i32([ctx + M]), num_seqs=1, num_tokens=M, max_q_len=M, min_q_len=M, max_kv_len=ctx + M)
    masks = torch.tensor(tree.masks_i64(), device="cuda")
    for layer in range(3):
        y = ops.attention_tree(q, kv.k(layer), kv.v(layer), i32([table]), i32([0] * M), i32([ctx + M - 1] * M), masks, i32([ctx] * M), hq, hkv, D,
                               D ** -0.5, window, first=first, meta=meta)
        o, b = so.attend(q.view(M, hq, D), torch.cat([text[layer, 0], node[layer, 0]]), torch.cat([text[layer, 1], node[layer, 1]]),
                         so.seen_rows(ctx, M, window, first, tree.parents), D ** -0.5)
        so.check(y.view(M, hq, D), o, b)
    path, bonus = tree.verify_greedy(5, [7, 0, 10, 0, 0, 11, 3])
    assert path == [0, 2, 5, 6] and bonus == 3
    kv.compact(i32([table]), i32([ctx]), i32([path]), i32([len(path)]), ops)
    n = ctx + len(path)
    q1 = torch.randn(1, hq * D, generator=g, device="cuda").bfloat16()
    meta = SimpleNamespace(q_starts=i32([0, 1]), seq_lens=i32([n]), num_seqs=1, num_tokens=1, max_q_len=1, min_q_len=1, max_kv_len=n)
    for layer in range(3):
        y = ops.attention(q1, kv.k(layer), kv.v(layer), i32([table]), i32([0]), i32([n - 1]), hq, hkv, D, D ** -0.5, window, meta=meta, first=first)
        k, v = (torch.cat([text[layer, i], node[layer, i][path]]) for i in (0, 1))
        o, b = so.attend(q1.view(1, hq, D), k, v, so.seen_rows(n - 1, 1, window, first), D ** -0.5)
        so.check(y.view(1, hq, D), o, b)
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("n", [1, 40])
def test_first_nodes_that_lie_far_behind(ops, kv, hq, n):
    """Two deep branches of a tree in a text that begins with it: the second one's upper nodes are among the first tokens, but stored behind the first one."""
    par = [-1] + list(range(0, 50)) + [0] + list(range(51, 150))
    c = so.setup([151] * n, [0, 3, 1, 9] * (n // 4) if n > 1 else [0], hq, 2, 128, kv, words=3, trees=[par] * n, seed=77)
    for window, first in ((4, 4), (20, 7)):
        so.check(_tree(ops, c, window, first), *so.want(c, 128 ** -0.5, window, first))
    assert ops.check_status() == 0


# ------------------------------------------------------------------------------------------ up to eight packed rows
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", [(8, 1, 64), (6, 2, 128), (4, 4, 256), (7, 1, 128), (2, 2, 64), (16, 2, 256)])
@pytest.mark.parametrize("n,longest", [(1, 900), (5, 1500), (90, 700), (1, 16000)])
def test_decode_rows(ops, hq, hkv, D, kv, n, longest):
    """One row a sequence, some of no row, from one to many splits; places that a row does not see hold NaN."""
    rows, ctx = [1 if i % 4 != 2 else 0 for i in range(n)], [(i * 397) % longest if i else longest for i in range(n)]
    c = so.setup(rows, ctx, hq, hkv, D, kv, seed=n + D, fill=float("nan"))
    for window, first, s, cap in ((50, 3, None, 0.0), (longest // 2, 100, _sinks(hq), 0.0), (1, 1, None, 20.0), (0, 0, None, 0.0) if n == 1 else (33, 40, None, 0.0)):
        window = window or 1 << 20
        so.check(_window(ops, c, window, max(first, 1), s, cap), *so.want(c, D ** -0.5, window, max(first, 1), s, cap))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("G,D", [(1, 128), (2, 64), (4, 256), (2, 128)])
def test_trees_of_few_rows(ops, G, D, kv):
    """Trees of up to 8 / G nodes: infinities and NaN of a node's values reach the nodes below it and no others; masks of no bits."""
    nodes = 8 // G
    par = [-1] + [0] * (nodes - 1)
    for n, ctx in ((1, 37), (3, 700), (70, 90)):
        c = so.setup([nodes] * n, [ctx + i for i in range(n)], 2 * G, 2, D, kv, words=1, trees=[par] * n, seed=n, fill=float("nan"))
        so.check(_tree(ops, c, 60, 5), *so.want(c, D ** -0.5, 60, 5))
        o, bound = so.want(c, D ** -0.5, 0, 0)
        so.check(_tree(ops, c), o, bound)
        tok = c.ctx[n - 1] + 1                          # the last sequence's second node: its own row alone sees it
        for at, x in ((7, float("nan")), (D - 2, float("inf") if kv == "bf16" else float("nan"))):
            c.v[int(c.tables[n - 1, tok // 16]), :, tok % 16, at] = x
        y = _tree(ops, c)
        mine = (n - 1) * nodes + 1
        keep = torch.arange(n * nodes, device="cuda") != mine
        so.check(y[keep], o[keep], bound[keep])
        got = y[mine].view(2 * G, D).float()
        assert torch.isnan(got[:, 7]).all() and (torch.isnan(got[:, D - 2]) if kv == "e4m3" else got[:, D - 2] == float("inf")).all()
        rest = [d for d in range(D) if d not in (7, D - 2)]
        so.check(y[mine].view(2 * G, D)[:, rest], o[mine].view(2 * G, D)[:, rest], bound[mine].view(2 * G, D)[:, rest])
        c.masks.zero_()
        c.base.zero_()
        assert (_tree(ops, c) == 0).all()
    assert ops.check_status() == 0


# ------------------------------------------------------------------------------------------ the tensor-memory kernel
# (few rows in all go to the kernel for few rows: what follows is large enough for the other one)
def _trees(n, nodes, hq, hkv, D, kv="bf16", ctx=700, seed=0, fill=0.0, words=1):
    par = [-1] + [max(0, i - 4) for i in range(1, nodes)]              # a root with four chains
    return so.setup([nodes] * n, [ctx + 17 * i for i in range(n)], hq, hkv, D, kv, words=words, trees=[par] * n, seed=seed, fill=fill), par


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (40, 2, 64), (6, 2, 64)])
@pytest.mark.parametrize("n", [2, 30])
def test_infinities_and_nan_of_other_branches_in_many_rows(ops, hq, hkv, D, kv, n):
    """One and two row tiles, whole and cut items: NaN and infinities in one sequence's nodes reach only the rows that see them."""
    nodes, ctx = 60, 2500
    c, par = _trees(n, nodes, hq, hkv, D, kv, ctx, seed=21, fill=float("nan"))
    o, bound = so.want(c, D ** -0.5, 0, 0)
    where = n - 1
    bad = {9: float("nan"), 22: float("inf") if kv == "bf16" else float("nan")}
    for node, x in bad.items():
        tok = c.ctx[where] + node
        c.v[int(c.tables[where, tok // 16]), :, tok % 16, 5] = x
    tok = c.ctx[where] + 31
    c.k[int(c.tables[where, tok // 16]), :, tok % 16, 3] = float("nan")
    y = _tree(ops, c)
    first = where * nodes
    so.check(y[:first], o[:first], bound[:first])
    seen = so.seen_rows(c.ctx[where], nodes, 0, 0, par)
    mine = y[first:].view(nodes, hq, D)
    o, bound = o[first:].view(nodes, hq, D), bound[first:].view(nodes, hq, D)
    hit = {m: [i for i in range(nodes) if seen[i, c.ctx[where] + m]] for m in (9, 22, 31)}
    clean = [i for i in range(nodes) if not any(i in h for h in hit.values())]
    assert clean and all(hit.values())
    so.check(mine[clean], o[clean], bound[clean])
    rest = [d for d in range(D) if d != 5]
    for m, x in bad.items():
        got = mine[hit[m]][:, :, 5].float()
        assert (torch.isnan(got) if math.isnan(x) else got == x).all()
        so.check(mine[hit[m]][:, :, rest], o[hit[m]][:, :, rest], bound[hit[m]][:, :, rest])
    assert torch.isnan(mine[hit[31]]).all()
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,D", [(8, 128), (32, 64)])
def test_stale_values_around_prompts(ops, hq, D, kv):
    """NaN in pages that the window has passed, in tokens in front of it and behind the last one; freed pages; several row tiles."""
    rows, ctx, window, first = [600, 333], [900, 1501], 190, 20
    c = so.setup(rows, ctx, hq, 2, D, kv, seed=8, fill=float("nan"))
    o, bound = so.want(c, D ** -0.5, window, first)
    for s in range(2):
        for tok in range(first, ctx[s] + 1 - window):
            blk, off = int(c.tables[s, tok // 16]), tok % 16
            c.v[blk, :, off] = float("nan")
            c.k[blk, :, off] = float("nan")
        for page in range(2, (ctx[s] + 1 - window) // 16):
            c.tables[s, page] = -1
    so.check(_window(ops, c, window, first), o, bound)
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_rows_that_see_nothing_among_many(ops, kv):
    c, _ = _trees(40, 30, 8, 2, 128, kv, ctx=200, seed=3)
    c.base.zero_()                                      # no context: what the masks name is all there is
    c.masks.zero_()
    c.masks[::3] = 7
    y = _tree(ops, c)
    empty = torch.ones(len(y), dtype=torch.bool, device="cuda")
    empty[::3] = False
    assert (y[empty] == 0).all() and torch.isfinite(y).all()
    for i in (0, 3, 597, 1197):
        s = i // 30
        o, b = so.attend(c.q[i:i + 1].view(1, 8, 128), c.keys[s][:3], c.values[s][:3], torch.ones(1, 3, dtype=torch.bool), 128 ** -0.5)
        so.check(y[i].view(1, 8, 128), o, b)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prompts_in_pools_of_more_than_32_bits(ops, kv):
    blocks = (1 << 31) // (8 * 16 * 128) + 500
    c = so.setup([500], [300], 32, 8, 128, kv, seed=6, pool_blocks=blocks)
    assert int(c.tables.min()) * 8 * 16 * 128 > 1 << 31
    so.check(_window(ops, c, 200, 30), *so.want(c, 128 ** -0.5, 200, 30))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prompt_pages_that_are_not_there(ops, kv):
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    c = so.setup([700], [300], 16, 2, 128, kv, seed=9)
    good = c.tables.clone()
    for entry in (-1, c.k.shape[0], 1 << 30):
        c.tables.copy_(good)
        c.tables[0, 40] = entry
        _window(mine, c, 200, 4)
        assert mine.check_status() == 3
    c.tables.copy_(good)
    _window(mine, c, 200, 4)
    assert mine.check_status() == 0
    c.meta.seq_lens += 1 << 20
    _window(mine, c, 100, 4)
    assert mine.check_status() == 3


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("sink", [False, True])
def test_long_sequences_beside_short_ones(ops, kv, sink):
    """Trees of which some are cut into pieces and some are not, decode rows of one long sequence, and both in one call."""
    s = _sinks(8) if sink else None
    nodes, ctx = [40, 33, 5, 64, 2, 4, 1], [9000, 50, 700, 300, 0, 3000, 20]
    c = so.setup(nodes, ctx, 8, 1, 128, kv, words=1, trees=[so.grow(n, n) for n in nodes], seed=31, fill=float("nan"))
    so.check(_tree(ops, c, sinks=s), *so.want(c, 128 ** -0.5, 0, 0, s))
    one = so.setup([1], [20000], 8, 1, 128, kv, seed=32)
    so.check(_window(ops, one, 19000, 100, s), *so.want(one, 128 ** -0.5, 19000, 100, s))
    both = so.setup([1, 1, 900], [15000, 7, 500], 8, 1, 128, kv, seed=33)
    so.check(_window(ops, both, 12000, 64, s), *so.want(both, 128 ** -0.5, 12000, 64, s))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,hq,hkv", [([704, 640], 16, 2), ([2400], 8, 1), ([1500, 20, 1400], 8, 2)])
def test_last_rounds_of_prompts(ops, kv, rows, hq, hkv):
    """Whole tiles that two blocks share, tiles of what is left of rows, sequences that end where others go on; first tokens in the window's tiles."""
    c = so.setup(rows, [400 + 77 * i for i in range(len(rows))], hq, hkv, 64, kv, seed=61, fill=float("nan"))
    for window, first in ((130, 3), (65, 40), (500, 1)):
        so.check(_window(ops, c, window, first), *so.want(c, 0.125, window, first))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (16, 2, 64), (8, 4, 256)])
@pytest.mark.parametrize("n,at", [(10, [9]), (150, [0, 131]), (400, [128, 255, 399])])
def test_a_few_prompts_among_many_rows(ops, hq, hkv, D, kv, n, at):
    """Prompts at the ends of the ranges in which blocks look their sequence up, beside decode rows and sequences of no row."""
    rows, ctx = [(1, 1, 0, 3, 1)[i % 5] for i in range(n)], [37 * i % 300 for i in range(n)]
    for k, i in enumerate(at):
        rows[i] = 700 - 121 * k
    c = so.setup(rows, ctx, hq, hkv, D, kv, seed=n + D, fill=float("nan"))
    so.check(_window(ops, c, 100, 5), *so.want(c, D ** -0.5, 100, 5))
    assert ops.check_status() == 0
    nodes = [min(r, 100) for r in rows]
    t = so.setup(nodes, ctx, hq, hkv, D, kv, words=2, trees=[so.grow(m, m) for m in nodes], seed=n, fill=float("nan"))
    so.check(_tree(ops, t), *so.want(t, D ** -0.5, 0, 0))
    assert ops.check_status() == 0


def test_lengths_that_a_ragged_batch_does_not_announce():
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    n, at = 300, 140
    rows = [1] * n
    rows[at] = 900
    for D in (128, 256):
        c = so.setup(rows, [50] * n, 8, 2, D, seed=5)
        o, bound = so.want(c, D ** -0.5, 60, 5)
        good = c.meta.q_starts.clone()
        for s, delta in ((299, 5), (at, -3), (0, -1)):
            c.meta.q_starts.copy_(good)
            c.meta.q_starts[s + (s == 299)] += delta
            y = _window(mine, c, 60, 5)
            assert mine.check_status() == 3, (D, s)
        c.meta.q_starts.copy_(good)
        c.meta.max_q_len = 899
        y = _window(mine, c, 60, 5)
        assert mine.check_status() == 3
        so.check(y[:at], o[:at], bound[:at])
        so.check(y[at + 900:], o[at + 900:], bound[at + 900:])


def test_prompts_in_graphs_and_on_streams(ops):
    """Two captured graphs of the tensor-memory kernel replayed in turn and on two streams at once, then on other lengths."""
    c = so.setup([500, 40, 3], [600, 1100, 2000], 16, 2, 128, seed=12)
    t, _ = _trees(24, 50, 16, 2, 128, ctx=500, seed=13)
    w1, w2 = so.want(c, 128 ** -0.5, 300, 4), so.want(t, 128 ** -0.5, 0, 0)
    graphs, outs = [], []
    for f in (lambda: _window(ops, c, 300, 4), lambda: _tree(ops, t)):
        f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    so.check(outs[0], *w1)
    so.check(outs[1], *w2)
    short = so.setup([500, 40, 3], [0, 77, 1999], 16, 2, 128, seed=14)
    c.q.copy_(short.q)
    c.tables.fill_(-1)
    c.tables[:, :short.tables.shape[1]].copy_(short.tables)
    c.meta.seq_lens.copy_(short.meta.seq_lens)
    c.k[:short.k.shape[0]].copy_(short.k)
    c.v[:short.k.shape[0]].copy_(short.v)
    graphs[0].replay()
    torch.cuda.synchronize()
    so.check(outs[0], *so.want(short, 128 ** -0.5, 300, 4))
    assert ops.check_status() == 0


def test_large_magnitudes_beside_an_8_bit_cache(ops):
    """Queries of very different magnitudes from row to row, up to 2^120 and down to 2^-130 with a scale that makes up for it, zero rows, and rows with
    an infinity or a NaN, which are NaN and disturb no other."""
    for rows, ctx in ([3, 1], [200, 90]), ([500, 333], [300, 700]):
        c = so.setup(rows, ctx, 16, 2, 128, "e4m3", seed=41)
        T = sum(rows)
        c.q[::5] = 0
        for up, scale in ((2.0 ** 118, 2.0 ** -118), (2.0 ** -118, 2.0 ** 118)):
            q = (c.q.float() * up).bfloat16()
            d = SimpleNamespace(**{**vars(c), "q": q})
            call = lambda x: ops.attention(x, c.k, c.v, c.tables, c.row_seq, c.positions, 16, 2, 128, 128 ** -0.5 * scale, 150, meta=c.meta, first=9)
            o, bound = so.want(d, 128 ** -0.5 * scale, 150, 9)
            so.check(call(q), o, bound)
            q2 = q.clone()
            q2[T - 1, 3] = float("inf")
            q2[1, 200] = float("nan")
            y = call(q2)
            assert torch.isnan(y[T - 1, :128]).all() and torch.isnan(y[1, 128:256]).all()
            keep = torch.ones(T, dtype=torch.bool, device="cuda")
            keep[[1, T - 1]] = False
            so.check(y[keep], o[keep], bound[keep])
    assert ops.check_status() == 0


@pytest.mark.parametrize("rows,ctx", [([3, 1], [200, 90]), ([300, 290], [300, 700])])
def test_lengths_that_the_batch_does_not_announce(rows, ctx):
    """More rows in a sequence than the batch says, rows behind the query's, a length that no table reaches: reported. Fewer rows than it says: right."""
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    c = so.setup(rows, ctx, 16, 2, 128, seed=51, fill=float("nan"))
    o, bound = so.want(c, 128 ** -0.5, 150, 9)
    c.meta.max_q_len -= 1
    c.meta.min_q_len = min(c.meta.min_q_len, c.meta.max_q_len)
    y = _window(mine, c, 150, 9)
    assert mine.check_status() == 3
    so.check(y[rows[0]:], o[rows[0]:], bound[rows[0]:])
    c.meta.max_q_len += 1
    c.meta.min_q_len = c.meta.max_q_len
    so.check(_window(mine, c, 150, 9), o, bound)
    assert mine.check_status() == 0
    good = c.meta.q_starts.clone()
    for bad in ([-1, rows[0], sum(rows)], [0, sum(rows), rows[0]], [0, rows[0], sum(rows) + 1]):
        c.meta.q_starts.copy_(torch.tensor(bad))
        c.meta.max_q_len = sum(rows) + 1
        _window(mine, c, 150, 9)
        assert mine.check_status() == 3, bad
    c.meta.q_starts.copy_(good)
    c.meta.seq_lens[1] = 2 ** 31 - 1
    y = _window(mine, c, 150, 9)
    assert mine.check_status() == 3
    so.check(y[:rows[0]], o[:rows[0]], bound[:rows[0]])


def test_compaction_beyond_every_table():
    from fllm_b200.ops.native import NativeOps
    mine = NativeOps(torch.device("cuda:0"), 1 << 20)
    pool = torch.randn(2, 4, 2, 16, 64, device="cuda").bfloat16()
    before = pool.clone()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    for base, node in ((2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 8, 20), (-5, 9), (0, 64)):
        mine.kv_compact([pool], i32([[0, 1, 2, 3]]), i32([base]), i32([[node]]), i32([1]))
        assert mine.check_status() == 3 and torch.equal(pool, before)
    mine.kv_compact([pool], i32([[0, 1, 2, 3]]), i32([1]), i32([[5, 5, 7]]), i32([3]))         # the same node twice: copied twice
    assert mine.check_status() == 0
    for to, node in ((1, 6), (2, 6), (3, 8)):
        assert torch.equal(pool[:, 0, :, to], before[:, 0, :, node])


def test_served_model_keeps_its_first_tokens():
    """An engine whose windows leave the first tokens visible: prompts in chunks, decode steps from captured graphs, the blocks between freed; the
    tokens are those of an engine that frees nothing, and the logits follow the PyTorch operators."""
    from fllm_b200.config import EngineConfig, preset
    from fllm_b200.models.decoder import Decoder, KVCache, StepBatch
    from fllm_b200.ops.reference import RefOps
    from fllm_b200.runtime import LLMEngine, SamplingParams
    cfg = preset("qwen3-tiny")
    cfg.sliding_window, cfg.window_first = 40, 20
    prompt = [(7 * i) % 50 + 1 for i in range(150)]
    outs = []
    for free in (True, False):
        eng = LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=96, max_model_len=256, max_num_batched_tokens=64), device="cuda:0")
        if not free:
            eng.scheduler.window = 0
        outs.append(eng.generate([prompt, prompt[:30]], SamplingParams(max_tokens=12)))
    assert outs[0] == outs[1]
    n = len(prompt)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    b = StepBatch(i32(prompt), i32(list(range(n))), i32(list(range(n))), i32([0] * n), i32([list(range(16))]), i32([n - 1]), num_seqs=1, num_tokens=n,
                  max_kv_len=n, max_q_len=n, min_q_len=n, seq_lens=i32([n]), q_starts=i32([0, n]))
    logits = []
    for o in (eng.ops, RefOps()):
        kv = KVCache(cfg.num_layers, 20, cfg.num_kv_heads, 16, cfg.head_dim, "cuda")
        logits.append(Decoder(cfg, eng.weights, kv, o, eng.spec).forward(b).float())
    assert (logits[0] - logits[1]).abs().max() <= 0.05 * logits[1].abs().max()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,nodes,ctx", [(2, 2, [3], [200]), (2, 1, [3, 5], [900, 40]), (2, 2, [2], [9500]), (16, 2, [64], [6000]), (32, 8, [33] * 40, [800] * 40)])
def test_rows_that_see_nothing_have_no_sink_either(ops, hq, hkv, nodes, ctx, kv):
    """A row that sees nothing is 0 whatever its head's sink is; a sink of -inf, or of a magnitude that log2 e takes to -inf, is none for the others.
    Few rows whole, in a cluster and over a merge; many rows in pieces and whole."""
    c = so.setup(nodes, ctx, hq, hkv, 64, kv, words=1, trees=[so.grow(n, n) for n in nodes], seed=hq, fill=float("nan"))
    blind = [c.starts[s] + n - 1 for s, n in enumerate(nodes)]
    c.masks[blind] = 0
    c.base[blind] = 0
    keep = [i for i in range(sum(nodes)) if i not in blind]
    low = torch.finfo(torch.float32).min
    for values in ([-math.inf, low], [low, -math.inf, 1.0, -2.0], [-1e38, math.inf], [math.nan, -math.inf]):
        s = torch.tensor((values * hq)[:hq], device="cuda")
        o, bound = so.want(c, 64 ** -0.5, 0, 0, s)
        y = _tree(ops, c, sinks=s)
        so.check(y[keep], o[keep], bound[keep])
        assert (y[blind] == 0).all()
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,ctx", [([1], [9000]), ([2, 1], [16000, 8800]), ([1], [40])])
def test_batches_that_announce_more_rows_than_there_are(ops, rows, ctx, kv):
    """Every sequence is said to have more rows than the batch has, so that both kernels' rows are spoken for: answered all the same. A batch that is said
    to have none is answered or reported."""
    c = so.setup(rows, ctx, 32, 8, 64, kv, seed=sum(ctx))
    o, bound = so.want(c, 0.125, 20000, 4)
    for most, least in ((20, 20), (5000, 300), (17, 5)):
        c.meta.max_q_len, c.meta.min_q_len = most, least
        torch.full((sum(rows), 32 * 64), math.nan, dtype=torch.bfloat16, device="cuda")        # (what an output would otherwise begin as)
        so.check(_window(ops, c, 20000, 4), o, bound)
        assert ops.check_status() == 0
    c.meta.max_q_len = c.meta.min_q_len = 0
    y = _window(ops, c, 20000, 4)
    if max(rows) == 1:
        so.check(y, o, bound)
        assert ops.check_status() == 0
    else:
        assert ops.check_status() != 0
    ops.status.zero_()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,rows,ctx", [(2, [1], [70]), (8, [2], [500]), (2, [1], [9500]), (32, [40], [6000]), (32, [64] * 40, [700] * 40)])
def test_nan_of_values_with_weights_below_every_number(ops, hq, rows, ctx, kv):
    """A NaN that a row sees shows wherever its page is summed, though e^x of its score is 0 beside the others': in another warp, split or piece."""
    c = so.setup(rows, ctx, hq, 2, 64, kv, seed=hq)
    c.q.fill_(4.0)
    for s, n in enumerate(ctx):
        for at, n_at in ((n // 3, 3), (2, 5)):           # (token, dim)
            tok = torch.arange(c.lens[s], device="cuda")
            c.keys[s].fill_(4.0)
            c.keys[s][:n // 2] = -4.0
            c.values[s][at, :, n_at] = math.nan
        page = c.tables[s, tok // 16].long()
        c.k[page, :, tok % 16] = c.keys[s].to(c.k.dtype)
        c.v[page, :, tok % 16] = c.values[s].to(c.v.dtype)
    window = max(c.lens)                                 # everything is seen, the first tokens by `first` at the latest
    y = _window(ops, c, window, 16).view(-1, hq, 64)
    nan = torch.zeros_like(y, dtype=torch.bool)
    nan[..., 3] = nan[..., 5] = True
    assert torch.equal(torch.isnan(y), nan)
    assert ops.check_status() == 0


def test_a_list_of_copies_does_not_wait_for_the_stream(ops):
    """The copies of a host list are queued behind what the stream has to do, however often; their source is read when they run."""
    pool = torch.zeros(4, 64, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    pool[:, 0] = 1
    ops.kv_copy_blocks([pool], [(0, 1)])
    a = torch.randn(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    b = a
    for _ in range(6):                                 # some 100 ms in fp32
        b = a @ a
    pool[:, 2] = b[0, 0].bfloat16()
    for i in range(40):
        ops.kv_copy_blocks([pool], [(2, 3 + i), (3 + i, 60)])
    done = torch.cuda.Event()
    done.record()
    assert not done.query(), "the call waited for the stream"
    torch.cuda.synchronize()
    assert all(torch.equal(pool[:, i], pool[:, 2]) for i in list(range(3, 43)) + [60])
    assert ops.check_status() == 0


@pytest.mark.parametrize("kind,n", [("kv", 1), ("kv", 96), ("rows", 97), ("odd", 200), ("many", 250)])
def test_lists_of_many_copies(ops, kind, n):
    """More pairs than a launch holds, chains among them, and the same list from a captured graph."""
    from fllm_b200.ops.reference import RefOps
    pools = _pools(kind, 2 * n + 3)
    pairs = [(2 * i, 2 * i + 1) for i in range(n)] + [(1, 2 * n), (2 * n, 2 * n + 2)]
    for graph in (False, True):
        ref = [t.clone() for t in pools]
        RefOps().kv_copy_blocks(ref, pairs)
        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                ops.kv_copy_blocks(pools, list(pairs))
            g.replay()
        else:
            ops.kv_copy_blocks(pools, pairs)
        torch.cuda.synchronize()
        assert _same(pools, ref)
        for t in pools:                                # other sources for the graph
            t[:, 0:2 * n:2] = t[:, 1:2 * n:2].flip(1)
    assert ops.check_status() == 0


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [[1, 1], [40, 3]])
def test_windows_below_zero_are_none(ops, rows, kv):
    """Without first tokens, and for trees without a step batch, a negative window is no window."""
    c = so.setup(rows, [300, 77], 8, 2, 128, kv, seed=3)
    for meta in (c.meta, None):
        call = lambda window: ops.attention(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, 8, 2, 128, 128 ** -0.5, window, meta=meta)
        assert torch.equal(call(-1), call(0))
    t = so.setup(rows, [300, 77], 8, 2, 128, words=1, trees=[so.grow(n, n) for n in rows], seed=4)
    tree = lambda window: ops.attention_tree(t.q, t.k, t.v, t.tables, t.row_seq, t.positions, t.masks.view(-1), t.base, 8, 2, 128, 128 ** -0.5, window)
    assert torch.equal(tree(-7), tree(0))
    assert ops.check_status() == 0
