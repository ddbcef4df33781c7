"""Prompts and trees over a cache held in 4 bits on the tensor-memory kernel, where tokens of a tile, or tiles of a text, are of different sizes.

Rows of the cache are written code by code: step 2^a, lowest value -8 x 2^a, so a code stands for (c - 8) 2^a and every power of two times it is an f16 number. What
the kernel widens is then exact as long as a token keeps a unit of its own, and the bound of span_oracle holds as it stands (weights f16, 2^-11 of each). Beside it:
a weight below 2^-14 in the kernel's units is within 2^-25 of what it was, or gone. The largest of a row's weights is at least 2^6 there, so is their sum, and values are
below 2^-6 in a unit whose largest value so far is at least 2^-9: such a token is off by 2^-25 2^-6 / (2^6 2^-9) U = 2^-28 U at most, U the largest value that rows of its CTA
(at most 256 packed ones) see, and by no more than what it adds itself."""
import pytest
import torch

import span_oracle as so
from fllm_b200.ops.kv4 import kv4_decode

pytestmark = pytest.mark.gpu
SHAPES = [(400, 500), (24, 6100)]          # two row tiles and one, the second in pieces of the walk
HQ, HKV = 8, 2


@pytest.fixture(scope="module")
def ops():
    from fllm_b200.ops.native import NativeOps
    return NativeOps(torch.device("cuda:0"))


def _rows(g, n, D, exp, low=None):
    """[n, HKV, D / 2 + 4]: random codes of step 2^exp, or (low) rows whose values are all low."""
    codes = torch.randint(0, 256, (n, HKV, D // 2), generator=g, device="cuda", dtype=torch.uint8)
    step = torch.exp2(torch.as_tensor(exp, device="cuda", dtype=torch.float32)).expand(n).clone()
    z = -8 * step
    if low is not None:
        alike = torch.isfinite(low)
        step, z = torch.where(alike, 0.0, step), torch.where(alike, low, z)
    tail = torch.stack([step, z], -1)[:, None].expand(n, HKV, 2).to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([codes, tail], -1)


def _case(rows, ctx, D, k, v, q=None, hq=HQ, trees=None, span=None):
    """A sequence whose tokens' rows are k and v."""
    c = so.setup([rows], [ctx], hq, HKV, D, seed=rows + D, words=4 if trees else 0, trees=trees and [trees])
    tok = torch.arange(rows + ctx, device="cuda")
    for name, x in (("k", k), ("v", v)):
        pool = torch.zeros(*getattr(c, name).shape[:3], D // 2 + 4, dtype=torch.uint8, device="cuda")
        pool[c.tables[0].long()[tok // 16], :, tok % 16] = x
        setattr(c, name, pool)
    c.keys, c.values = [kv4_decode(k)], [kv4_decode(v)]
    if q is not None:
        c.q = q.bfloat16().view(rows, hq * D)
    tiles = -(-rows * (hq // HKV) // 16) * HKV * -(-(span or rows + ctx) // 16)
    assert tiles > 28 * torch.cuda.get_device_properties(0).multi_processor_count, "too little for the tensor-memory kernel"
    return c


def _want(c, ignored=None, sinks=None, cap=0.0, window=0, first=0):
    """(outputs, bounds); `ignored`: tokens whose weights are nothing beside the others (below e^-30 2^20 of them)."""
    n, N, D, scale = c.rows[0], c.lens[0], c.D, c.D ** -0.5
    q, k, v = c.q.view(n, c.hq, D), c.keys[0], c.values[0]
    seen = so.seen_rows(c.ctx[0], n, window, first, c.trees[0] if c.trees else None).cuda()
    size = v.double().abs().amax((1, 2))
    last = (c.ctx[0] + torch.arange(n, device="cuda") + 256).clamp(max=N - 1) if c.trees is None else torch.full((n,), N - 1, device="cuda")
    most = size.cummax(0)[0][last]
    if ignored is not None:
        seen[:, ignored] = False
    o, bound = so.attend(q, k, v, seen, scale, sinks, cap)
    s = torch.einsum("nhd,mhd->nhm", q.double(), k.double().repeat_interleave(c.hq // HKV, 1)) * scale
    s = cap * torch.tanh(s / cap) if cap else s
    w = torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), -1)
    extra = torch.minimum(w * size, most[:, None, None] * 2.0 ** -28).sum(-1)
    return o.reshape(n, -1), (bound + extra[..., None] + 1e-7).reshape(n, -1)


def _attend(ops, c, sinks=None, cap=0.0, window=0, first=0):
    if c.trees:
        return ops.attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks, c.base, c.hq, HKV, c.D, c.D ** -0.5, window, sinks, cap, meta=c.meta, first=first)
    return ops.attention(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.hq, HKV, c.D, c.D ** -0.5, window, sinks, cap, meta=c.meta, first=first)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,ctx", SHAPES)
@pytest.mark.parametrize("kind", ["zero queries", "small queries", "large keys"])
@pytest.mark.parametrize("sink", [False, True])
def test_scores_of_zero(ops, D, rows, ctx, kind, sink):
    """Queries of zero, and small ones, beside a tile of keys that are zero; queries that are zero where a tile's keys are very large: finite, as the formula is."""
    g = torch.Generator(device="cuda").manual_seed(D + rows)
    n = rows + ctx
    at = (ctx + rows // 2) // 128 * 128
    k, v = _rows(g, n, D, -2), _rows(g, n, D, -2)
    q = 1.5 * torch.randn(rows, HQ, D, generator=g, device="cuda")
    if kind == "large keys":
        k = torch.zeros_like(k)
        k[at:at + 128, :, 0] = 0xF0                       # dim 1: code 15
        k[at:at + 128, :, D // 2:] = torch.tensor([2.0 ** 122, 0.0], device="cuda").bfloat16().view(torch.uint8)
        q *= 2.0 ** 20
        q[:, :, 1] = 0.0
    else:
        k[at:at + 128] = 0
        if kind == "zero queries":
            q[::3] = 0.0
        else:
            q *= 2.0 ** -40
    c = _case(rows, ctx, D, k, v, q)
    s = torch.linspace(-3, 3, HQ, device="cuda") if sink else None
    so.check(_attend(ops, c, s), *_want(c, sinks=s))
    assert ops.check_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,ctx", SHAPES)
@pytest.mark.parametrize("kind,cap", [("values", 0.0), ("keys", 0.0), ("both", 0.0), ("both", 30.0), ("first", 0.0), ("growing", 0.0), ("shrinking", 0.0), ("ratio", 0.0)])
def test_tokens_of_different_sizes(ops, D, rows, ctx, kind, cap):
    """A few very large tokens without weight, before and behind other rows' ends; values that grow or shrink from tile to tile; sizes that change from token to
    token: every token keeps its bits."""
    g = torch.Generator(device="cuda").manual_seed(D + rows)
    n = rows + ctx
    tok = torch.arange(n, device="cuda")
    q = 1.5 * torch.randn(rows, HQ, D, generator=g, device="cuda") + 1.0
    k_exp, v_exp = torch.full((n,), -1.0, device="cuda"), torch.full((n,), -2.0, device="cuda")
    large = (tok == 3) if kind == "first" else (tok % 150 == 77) | (tok == ctx + rows // 2)
    ignored = None
    low = torch.full((n,), float("nan"), device="cuda")
    if kind in ("values", "keys", "both", "first"):
        ignored = large
        low[large] = -2.0 ** 17 if kind in ("keys", "both") else -8.0
        if kind != "keys":
            v_exp[large] = 12.0
    elif kind == "ratio":
        k_exp -= torch.randint(0, 10, (n,), generator=g, device="cuda") * 2
        v_exp -= torch.randint(0, 12, (n,), generator=g, device="cuda") * 2
    else:
        v_exp += (tok // 128 if kind == "growing" else -(tok // 128)) * (3.0 if n < 2000 else 0.5) // 1
    c = _case(rows, ctx, D, _rows(g, n, D, k_exp, low), _rows(g, n, D, v_exp), q)
    so.check(_attend(ops, c, cap=cap), *_want(c, ignored, cap=cap))
    assert ops.check_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,first", [(300, 20), (200, 130), (77, 1)])
def test_windows_with_first_tokens_of_other_sizes(ops, D, window, first):
    """First tokens and tokens of the window that are much larger, or much smaller, than the others of their tile."""
    g = torch.Generator(device="cuda").manual_seed(D + window)
    rows, ctx = 1500, 611
    n = rows + ctx
    tok = torch.arange(n, device="cuda")
    large = (tok == 0) | (tok % 190 == 100)
    low = torch.where(large, -2.0 ** 15, float("nan"))
    k = _rows(g, n, D, torch.where(tok % 7 == 3, -9.0, -1.0), low)
    v = _rows(g, n, D, torch.where(large, 12.0, torch.where(tok % 5 == 1, -13.0, -2.0)))
    q = 1.5 * torch.randn(rows, 64, D, generator=g, device="cuda") + 1.0
    c = _case(rows, ctx, D, k, v, q, 64, span=min(rows + ctx, window + first + rows))
    so.check(_attend(ops, c, window=window, first=first), *_want(c, large, window=window, first=first))
    assert ops.check_status() == 0


def test_a_tree_with_large_nodes(ops):
    """Nodes of large values that their descendants do not weigh, beside branches that do not see them."""
    g = torch.Generator(device="cuda").manual_seed(5)
    nodes, ctx, D, hq = 200, 313, 128, 32
    n = nodes + ctx
    large = torch.zeros(n, dtype=torch.bool, device="cuda")
    large[[40, ctx + 20, ctx + 77]] = True
    low = torch.where(large, -2.0 ** 17, float("nan"))
    q = 1.5 * torch.randn(nodes, hq, D, generator=g, device="cuda") + 1.0
    c = _case(nodes, ctx, D, _rows(g, n, D, -1, low), _rows(g, n, D, torch.where(large, 12.0, -2.0)), q, hq, so.grow(nodes, 3))
    so.check(_attend(ops, c), *_want(c, large))
    assert ops.check_status() == 0


@pytest.mark.parametrize("rows,ctx", SHAPES)
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("sizes", [False, True])
def test_a_row_that_is_not_finite(ops, rows, ctx, which, sizes):
    """NaN in the rows that see it and nowhere else, with other tokens of the tile of other sizes or not."""
    D = 128
    g = torch.Generator(device="cuda").manual_seed(rows)
    n, bad = rows + ctx, ctx + rows // 3
    exp = -2.0 - (torch.randint(0, 6, (n,), generator=g, device="cuda") * 4 if sizes else torch.zeros(n, device="cuda"))
    k, v = _rows(g, n, D, exp), _rows(g, n, D, exp)
    c = _case(rows, ctx, D, k, v)
    row = (k if which == "k" else v)[bad:bad + 1].clone()
    row[..., D // 2:D // 2 + 2] = torch.tensor([float("nan")], device="cuda").bfloat16().view(torch.uint8)
    getattr(c, which)[int(c.tables[0, bad // 16]), :, bad % 16] = row[0]
    y = _attend(ops, c)
    sees = torch.arange(rows, device="cuda") >= bad - ctx
    assert torch.isnan(y[sees]).all()
    o, bound = _want(c)
    so.check(y[~sees], o[~sees], bound[~sees])
