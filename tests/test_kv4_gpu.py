"""A cache held in 4 bits on the kernels: rows written (with and without a rotation) and read, attention over it, against the encoding's statement and fp64."""
import math

import pytest
import torch

import kv4_oracle as ko
import span_oracle as so
from fllm_b200.ops.kv4 import kv4_decode, kv4_encode, kv4_width
from fllm_b200.ops.reference import RefOps

pytestmark = pytest.mark.gpu
HEADS = [(8, 2, 128), (16, 2, 64), (4, 4, 64), (5, 1, 128), (14, 2, 128), (32, 2, 64), (8, 4, 256), (24, 2, 256)]


@pytest.fixture(scope="module")
def ops():
    from fllm_b200.ops.native import NativeOps
    return NativeOps(torch.device("cuda:0"))


def _caches(blocks, hkv, block, D):
    g = torch.Generator(device="cuda").manual_seed(7)
    return [torch.randint(0, 256, (blocks, hkv, block, kv4_width(D)), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]


def _odd_rows(n, width, D, seed):
    """Normal rows, and at their start heads that are alike, tiny, huge, of one large value, of a zero range, not finite, of a range that fp32 does not hold."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, width, generator=g, device="cuda").bfloat16()
    kinds = [lambda r: r.fill_(3.25), lambda r: r.mul_(1e-38), lambda r: r.mul_(1e37), lambda r: r[3:4].fill_(1000.0), lambda r: r.fill_(0.0),
             lambda r: r[D - 1:].fill_(float("nan")), lambda r: r[:1].fill_(float("inf")), lambda r: r[5:6].fill_(-float("inf")),
             lambda r: (r[:1].fill_(3e38), r[1:2].fill_(-3e38)), lambda r: r.add_(100.0), lambda r: r.copy_(torch.arange(D, device="cuda") % 16), lambda r: r.fill_(-0.0)]
    for i, f in enumerate(kinds):
        if i < n:
            f(x[i, :D])
    return x


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hkv,block,n", [(1, 16, 1), (3, 16, 37), (8, 32, 300), (2, 5, 64)])
def test_write_and_read(ops, D, hkv, block, n):
    """Every byte is the one of the encoding's statement; places without a slot stay; reading gives what the bytes stand for, bit for bit."""
    blocks = n // block + 3
    k, v = _odd_rows(n, hkv * D, D, 1), _odd_rows(n, hkv * D, D, 2).flip(0).contiguous()
    wide = torch.randn(n, hkv * D + 24, device="cuda").bfloat16()
    wide[:, 8:8 + hkv * D] = v
    slots = torch.randperm(blocks * block, device="cuda")[:n].int()
    slots[2::5] = -1
    kc, vc = _caches(blocks, hkv, block, D)
    want = [c.clone() for c in (kc, vc)]
    RefOps().kv4_write(k, v, slots, *want)
    ops.kv4_write(k, wide[:, 8:8 + hkv * D], slots, kc, vc)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    for c in (kc, vc):
        assert torch.equal(ops.kv4_read(c, slots).view(torch.int32), RefOps().kv4_read(c, slots).view(torch.int32)) or \
            torch.equal(torch.nan_to_num(ops.kv4_read(c, slots), nan=7.5), torch.nan_to_num(RefOps().kv4_read(c, slots), nan=7.5))
    assert ops.check_status() == 0


def test_error_of_the_encoding(ops):
    """Half a step at most for every value of a finite row (and what fp32 rounds in z + s c), the ends of the range within it."""
    x = _odd_rows(500, 128, 128, 3)
    x = x[torch.isfinite(x.float()).all(1) & torch.isfinite(x.float().amax(1) - x.float().amin(1))]
    kc, vc = _caches(40, 1, 16, 128)
    slots = torch.arange(len(x), dtype=torch.int32, device="cuda")
    ops.kv4_write(x, x, slots, kc, vc)
    rows = kc.transpose(1, 2).reshape(-1, 68)[:len(x)]
    step = rows[:, 64:66].contiguous().view(torch.bfloat16).double()
    y = ops.kv4_read(kc, slots).double()
    assert ((y - x.double()).abs() <= step / 2 * (1 + 2.0 ** -22) + x.double().abs().amax(1, keepdim=True) * 2.0 ** -23).all()
    assert (step <= (x.double().amax(1, keepdim=True) - x.double().amin(1, keepdim=True)) / 15 * (1 + 2.0 ** -7) + 1e-40).all()


def test_slots_behind_the_pool_are_reported(ops):
    kc, vc = _caches(2, 2, 16, 64)
    k = torch.randn(3, 128, device="cuda").bfloat16()
    before = kc.clone()
    ops.kv4_write(k, k, torch.tensor([32, -5, 1 << 30], dtype=torch.int32, device="cuda"), kc, vc)
    assert ops.check_status() != 0 and torch.equal(kc, before)
    assert (ops.kv4_read(kc, torch.tensor([40], dtype=torch.int32, device="cuda")) == 0).all()
    assert ops.check_status() != 0


def test_no_rows(ops):
    kc, vc = _caches(2, 2, 16, 64)
    k = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.kv4_write(k, k, none, kc, vc)
    assert ops.kv4_read(kc, none).shape == (0, 128)


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("hq,hkv,D,rot,style,norm", [(8, 2, 128, 128, 0, True), (4, 4, 64, 64, 0, False), (8, 4, 256, 256, 0, True), (6, 3, 128, 64, 1, False),
                                                     (4, 1, 64, 32, 0, True), (4, 2, 128, 128, 1, True)])
def test_rotation_and_write(ops, T, hq, hkv, D, rot, style, norm):
    """The rotated rows of a bf16 cache, encoded: the same bytes, and the same queries."""
    g = torch.Generator(device="cuda").manual_seed(T + D)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device="cuda").bfloat16()
    w = [torch.rand(D, generator=g, device="cuda").bfloat16() + 0.5 for _ in range(2)] if norm else [None, None]
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda").float() / rot)
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda").int()
    blocks = T // 16 + 2
    slots = torch.randperm(blocks * 16, device="cuda")[:T].int()
    slots[1::7] = -1
    plain = [torch.zeros(blocks, hkv, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kc, vc = _caches(blocks, hkv, 16, D)
    before = [kc.clone(), vc.clone()]
    a = ops.rope_kv_write(qkv.clone(), pos, slots, inv, *w, *plain, hq, hkv, D, rot, style, 1e-6)
    b = ops.rope_kv_write(qkv.clone(), pos, slots, inv, *w, kc, vc, hq, hkv, D, rot, style, 1e-6)
    assert torch.equal(a, b)
    at = slots[slots >= 0].long()
    for x, c, old in zip(plain, (kc, vc), before):
        want = old.clone()
        want[at // 16, :, at % 16] = kv4_encode(x[at // 16, :, at % 16])
        assert torch.equal(c, want)


@pytest.mark.parametrize("D,splits", [(64, 2), (128, 3), (128, 8), (256, 7)])
def test_rotation_and_write_of_partial_sums(ops, D, splits):
    hq, hkv, T = 4, 2, 5
    width = (hq + 2 * hkv) * D
    ws = torch.randn((64 << 10) // 4 + splits * T * width, device="cuda")
    bias = torch.randn(width, device="cuda").bfloat16()
    inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
    pos, slots = torch.arange(T, device="cuda").int() * 11, torch.tensor([3, 19, -1, 0, 30], dtype=torch.int32, device="cuda")
    plain = [torch.zeros(2, hkv, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    four = _caches(2, hkv, 16, D)
    qs = []
    for caches in (plain, four):
        q = torch.empty(T, hq * D, device="cuda", dtype=torch.bfloat16)
        ops.k.rope_kv_write_splitk(ws, splits, bias, q, pos, slots, inv, None, None, *caches, hq, hkv, D, D, 0, 1e-6, 1.0)
        qs.append(q)
    assert torch.equal(*qs)
    at = slots[slots >= 0].long()
    for x, c in zip(plain, four):
        assert torch.equal(c[at // 16, :, at % 16], kv4_encode(x[at // 16, :, at % 16]))


# ------------------------------------------------------------------ attention
def _attend(ops, c, window=0, first=0, sinks=None, cap=0.0):
    return ops.attention(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.hq, c.hkv, c.D, c.D ** -0.5, window, sinks, cap, meta=c.meta, first=first)


def _sinks(hq):
    return torch.linspace(-3, 3, hq, device="cuda")


@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("window,first,sink,cap", [(0, 0, False, 0.0), (33, 4, False, 0.0), (128, 70, True, 0.0), (1, 1, False, 0.0), (250, 16, False, 20.0), (0, 0, True, 30.0)])
def test_rows(ops, hq, hkv, D, window, first, sink, cap):
    """Decode and short rows of sequences of many lengths, one of no row and ones shorter than the window or the first tokens."""
    rows, ctx = [1, 2, 1, 0, 7, 1, 3], [0, 5, 300, 10, 129, 1777, 15]
    c = ko.setup(rows, ctx, hq, hkv, D, seed=hq + D, fill=float("nan"))
    s = _sinks(hq) if sink else None
    so.check(_attend(ops, c, window, first, s, cap), *ko.want(c, D ** -0.5, window, first, s, cap))
    assert ops.check_status() == 0


@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("window,first", [(0, 0), (64, 5), (500, 130), (17, 200)])
def test_prompts(ops, hq, hkv, D, window, first):
    """Chunks of prompts beside decode rows, chunks from the first token on, tiles that end inside pages."""
    rows, ctx = [130, 1, 257, 64], [0, 900, 411, 1]
    c = ko.setup(rows, ctx, hq, hkv, D, seed=hq * D, fill=float("nan"))
    so.check(_attend(ops, c, window, first), *ko.want(c, D ** -0.5, window, first))
    assert ops.check_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_long_prompt_with_sinks_and_cap(ops, D):
    c = ko.setup([700, 300], [1300, 2], 8, 2, D, seed=3, fill=float("nan"))
    s = _sinks(8)
    so.check(_attend(ops, c, 600, 40, s, 15.0), *ko.want(c, D ** -0.5, 600, 40, s, 15.0))
    so.check(_attend(ops, c, 0, 0, s), *ko.want(c, D ** -0.5, 0, 0, s))
    assert ops.check_status() == 0


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (16, 2, 64), (8, 4, 256), (32, 2, 64)])
@pytest.mark.parametrize("window,first,sink", [(0, 0, False), (40, 3, True)])
def test_trees(ops, hq, hkv, D, window, first, sink):
    nodes, ctx = [1, 13, 64, 3, 200, 65], [50, 0, 333, 1, 129, 1030]
    c = ko.setup(nodes, ctx, hq, hkv, D, words=4, trees=[so.grow(n, n) for n in nodes], seed=D, fill=float("nan"))
    s = _sinks(hq) if sink else None
    y = ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks, c.base, hq, hkv, D, D ** -0.5, window, s, 0.0, first=first, meta=c.meta)
    so.check(y, *ko.want(c, D ** -0.5, window, first, s))
    assert ops.check_status() == 0


@pytest.mark.parametrize("block", [32, 64, 48])
def test_larger_blocks(ops, block):
    c = ko.setup([1, 40, 3], [700, 77, 31], 8, 2, 128, block=block, seed=block, fill=float("nan"))
    so.check(_attend(ops, c), *ko.want(c, 128 ** -0.5, 0, 0))
    assert ops.check_status() == 0


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (40, 4, 64)])
def test_many_splits_and_long_texts(ops, hq, hkv, D):
    """One sequence behind 20,000 tokens (parts through memory), two of 6000 (parts of a cluster)."""
    for rows, ctx in ([1], [20000]), ([2, 1], [6000, 5999]):
        c = ko.setup(rows, ctx, hq, hkv, D, seed=5)
        so.check(_attend(ops, c), *ko.want(c, D ** -0.5, 0, 0))
    assert ops.check_status() == 0


@pytest.mark.parametrize("T", [1, 80])
def test_values_that_are_not_finite(ops, T):
    """A token with a NaN among its keys (a row that reads as NaN) is NaN in the rows that see it and nowhere else; so with its values."""
    for which in ("k", "v"):
        c = ko.setup([T, 1], [100, 300], 8, 2, 128, seed=9)
        tok = 99 if T == 1 else 140                       # rows from 140 - 100 on see it
        blk, off = int(c.tables[0, tok // 16]), tok % 16
        pool, flat = (c.k, c.keys) if which == "k" else (c.v, c.values)
        row = torch.zeros(2, 128, device="cuda")
        row[:, 7] = float("nan")
        pool[blk, :, off] = kv4_encode(row)
        y = _attend(ops, c)
        flat[0][tok] = 0.0
        o, bound = ko.want(c, 128 ** -0.5, 0, 0)
        sees = torch.zeros(T + 1, dtype=torch.bool, device="cuda")
        sees[max(0, tok - 100) if T > 1 else 0:T] = True
        assert torch.isnan(y[sees]).all()
        so.check(y[~sees], o[~sees], bound[~sees])


@pytest.mark.parametrize("hq,nodes", [(2, 60), (2, 14), (8, 200), (32, 200)])
def test_a_branch_of_values_that_are_not_finite(ops, hq, nodes):
    """Two chains in turn behind one root: every value of the first is NaN, and the rows of the second are as if it were not there, whatever lanes hold of it."""
    par = [-1] + [max(0, i - 2) for i in range(1, nodes)]
    c = ko.setup([nodes], [201], hq, 2, 128, words=4, trees=[par], seed=3)
    row = torch.full((2, 128), float("nan"), device="cuda")
    for node in range(1, nodes, 2):                       # at even places of the text
        tok = 201 + node
        c.v[int(c.tables[0, tok // 16]), :, tok % 16] = kv4_encode(row)
        c.values[0][tok] = 0.0
    y = ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks, c.base, hq, 2, 128, 128 ** -0.5, meta=c.meta)
    o, bound = ko.want(c, 128 ** -0.5, 0, 0)
    second = torch.arange(nodes, device="cuda") % 2 == 0
    assert torch.isnan(y[~second]).all()
    so.check(y[second], o[second], bound[second])
    assert ops.check_status() == 0


@pytest.mark.parametrize("k_scale,v_scale", [(1e-20, 1.0), (1.0, 1e-30), (1.0, 1e30), (50.0, 1e4), (1.0, 1e37)])
def test_magnitudes(ops, k_scale, v_scale):
    """Steps of any size: of a cache's tokens alike."""
    c = so.setup([1, 20], [400, 33], 8, 2, 128, seed=4, q_scale=min(1.5, 1.5 / k_scale))
    c.k, c.v = kv4_encode(c.k.float() * k_scale), kv4_encode(c.v.float() * v_scale)
    c.keys = [kv4_decode(kv4_encode(k.float() * k_scale)) for k in c.keys]
    c.values = [kv4_decode(kv4_encode(v.float() * v_scale)) for v in c.values]
    o, bound = so.want(c, 128 ** -0.5, 0, 0)
    so.check(_attend(ops, c), o, bound + 2.0 ** -11 * 8 * 0.6 * v_scale)


def test_steps_of_different_sizes(ops):
    """Small values of heavy tokens beside large ones of light tokens, and large ones that come last: each keeps its part."""
    D, n = 128, 400
    c = so.setup([1], [n - 1], 8, 2, D, seed=6)
    size = torch.where(torch.arange(n, device="cuda") % 50 == 49, 300.0, 0.01)[:, None, None]
    size[-1] = 1000.0
    vals = (c.values[0].float() * size).bfloat16()
    tok = torch.arange(n, device="cuda")
    c.v[c.tables[0].long()[tok // 16], :, tok % 16] = vals
    c.k, c.v = kv4_encode(c.k), kv4_encode(c.v)
    c.keys, c.values = [kv4_decode(kv4_encode(c.keys[0]))], [kv4_decode(kv4_encode(vals))]
    o, bound = so.want(c, D ** -0.5, 0, 0)
    step = (vals.float().amax(-1) - vals.float().amin(-1)) / 15                # [n, hkv]
    w = torch.softmax(torch.einsum("hd,nhd->hn", c.q[0].view(8, D).double(), c.keys[0].double().repeat_interleave(4, 1)) * D ** -0.5, -1)
    extra = (w * step.double().repeat_interleave(4, 1).T).sum(-1) * 2.0 ** -11 * 8 * 1.1
    so.check(_attend(ops, c), o, bound + extra[:, None].expand(8, D).reshape(1, -1))


def test_far_pages(ops):
    """Pages behind 4 GB of a pool."""
    c = ko.setup([1, 3], [300, 200], 8, 8, 128, seed=8)
    blocks = 560_000                                       # x 8704 bytes
    for name in "kv":
        pool = torch.zeros(blocks, 8, 16, 68, dtype=torch.uint8, device="cuda")
        small = getattr(c, name)
        pool[-small.shape[0]:] = small
        setattr(c, name, pool)
    c.tables = torch.where(c.tables >= 0, c.tables + blocks - small.shape[0], c.tables)
    so.check(_attend(ops, c), *ko.want(c, 128 ** -0.5, 0, 0))
    slots = torch.tensor([(blocks - 1) * 16 + 3], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 8 * 128, device="cuda").bfloat16()
    ops.kv4_write(x, x, slots, c.k, c.v)
    assert torch.equal(ops.kv4_read(c.k, slots), kv4_decode(kv4_encode(x.view(1, 8, 128))).flatten(1))
    assert ops.check_status() == 0


def test_pages_that_are_not_there(ops):
    """Table entries that name no block, lengths behind the table: reported, the other sequences are answered."""
    c = ko.setup([1, 1], [200, 200], 8, 2, 128, seed=1)
    c.tables[0, 3] = 1 << 20
    y = _attend(ops, c)
    assert ops.check_status() != 0
    o, bound = ko.want(c, 128 ** -0.5, 0, 0)
    so.check(y[1:], o[1:], bound[1:])


def test_a_captured_step_reads_new_lengths(ops):
    """Rows written and read in a graph, replayed for the next tokens; another stream than the default one."""
    hq, hkv, D, B = 8, 2, 128, 3
    c = ko.setup([1] * B, [40, 100, 7], hq, hkv, D, seed=2, spare=40)
    c.tables = torch.nn.functional.pad(c.tables, (0, 4), value=0)
    free = sorted(set(range(c.k.shape[0])) - set(c.tables[c.tables >= 0].tolist()))
    c.tables[c.tables < 0] = 0
    for s in range(B):
        for p in range(-(-c.lens[s] // 16), c.tables.shape[1]):
            c.tables[s, p] = free.pop()
    c.meta.max_kv_len = 200
    k, v = (torch.randn(B, hkv * D, device="cuda").bfloat16() for _ in range(2))
    lens = c.meta.seq_lens

    def step():
        at = lens - 1
        slots = c.tables.gather(1, (at // 16).long()[:, None])[:, 0] * 16 + at % 16
        ops.kv4_write(k, v, slots.int(), c.k, c.v)
        return _attend(ops, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for turn in range(20):
        k.normal_()
        v.normal_()
        if turn:
            lens += 1
        graph.replay()
        for s in range(B):
            new = [kv4_decode(kv4_encode(x[s].view(1, hkv, D))) for x in (k, v)]
            c.keys[s], c.values[s] = (torch.cat([old[:c.lens[s] - 1 + turn], n]) for old, n in zip((c.keys[s], c.values[s]), new))
    c.ctx = [len(x) - 1 for x in c.keys]
    so.check(y, *ko.want(c, D ** -0.5, 0, 0))
    assert ops.check_status() == 0


def test_refusals(ops):
    c = ko.setup([1], [20], 8, 2, 128)
    args = (c.tables, c.row_seq, c.positions, 8, 2, 128, 1.0)
    with pytest.raises(ValueError, match="step batch"):
        ops.attention(c.q, c.k, c.v, *args)
    with pytest.raises(ValueError, match="causal"):
        ops.attention(c.q, c.k, c.v, *args, meta=c.meta, bidirectional=True)
    with pytest.raises(ValueError, match="step batch"):
        ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, torch.ones(1, dtype=torch.int64, device="cuda"), c.positions, 8, 2, 128, 1.0)
    with pytest.raises(RuntimeError, match="v_cache"):
        ops.attention(c.q, c.k, c.v[:-1], *args, meta=c.meta)
    x = torch.randn(1, 256, device="cuda").bfloat16()
    slots = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.kv4_write(x.float(), x, slots, c.k, c.v), lambda: ops.kv4_write(x[:, :128], x, slots, c.k, c.v),
                lambda: ops.kv4_write(x, x, slots.long(), c.k, c.v), lambda: ops.kv4_write(x, x, slots, c.k, c.v[:, :1]),
                lambda: ops.kv4_write(x, x, slots[:0], c.k, c.v), lambda: ops.kv4_read(c.k[..., :66], slots), lambda: ops.kv4_read(c.k[:, :, ::2], slots),
                lambda: ops.kv4_write(torch.randn(2, 260, device="cuda").bfloat16()[:, :256], x.expand(2, -1), slots, c.k, c.v)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        kv4_width(96)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hq", [2, 8, 32])
def test_queries_of_the_largest_size_beside_keys_of_zero(ops, D, hq):
    """Few rows: scores are 0 where the keys are, whatever the queries' size."""
    c = ko.setup([1, 3], [200, 33], hq, 2, D, seed=D)
    c.q = (c.q.float() * 2.0 ** 122).bfloat16()
    c.k.zero_()
    c.keys = [torch.zeros_like(k) for k in c.keys]
    o, bound = so.want(c, D ** -0.5, 0, 0)
    so.check(_attend(ops, c), o, bound + ko.slack(c))
    assert ops.check_status() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [3, 400])
def test_codes_beside_ties(ops, D, T):
    """Values at the middle between two codes, and one bf16 number next to it: rows written with a rotation by nothing, and without one, are the statement's."""
    g = torch.Generator(device="cuda").manual_seed(D + T)
    hq, hkv = 4, 2
    n = T * hkv
    size = torch.exp2(torch.randint(-120, 110, (n, 1), generator=g, device="cuda").float())
    lo = (size * torch.randn(n, 1, generator=g, device="cuda")).bfloat16().float()
    hi = (lo + size * (0.01 + torch.rand(n, 1, generator=g, device="cuda"))).bfloat16().float()
    ends = torch.cat([lo, hi, lo.expand(n, D - 2)], 1)
    step = kv4_encode(ends)[:, D // 2:D // 2 + 2].contiguous().view(torch.bfloat16).float()
    x = (lo + step * (torch.randint(0, 15, (n, D), generator=g, device="cuda") + 0.5)).bfloat16()
    x = (x.view(torch.int16) + torch.randint(-1, 2, (n, D), generator=g, device="cuda").to(torch.int16)).view(torch.bfloat16)
    x = torch.minimum(torch.maximum(torch.nan_to_num(x.float()), lo), hi)
    x[:, :2] = ends[:, :2]
    x = x.bfloat16()
    rows = kv4_encode(x).view(T, hkv, -1)
    blocks = T // 16 + 2
    slots = torch.randperm(blocks * 16, generator=g, device="cuda")[:T].int()
    flat = x.view(T, hkv * D)
    inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
    for how in ("rows", "rotated"):
        kc, vc = _caches(blocks, hkv, 16, D)
        if how == "rows":
            ops.kv4_write(flat, flat, slots, kc, vc)
        else:
            qkv = torch.cat([torch.zeros(T, hq * D, device="cuda").bfloat16(), flat, flat], 1)
            ops.rope_kv_write(qkv, torch.zeros(T, dtype=torch.int32, device="cuda"), slots, inv, None, None, kc, vc, hq, hkv, D, D, 0, 1e-6)
        at = slots.long()
        assert torch.equal(kc[at // 16, :, at % 16], rows) and torch.equal(vc[at // 16, :, at % 16], rows), how
