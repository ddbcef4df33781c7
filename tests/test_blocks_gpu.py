"""Bounds of blocks, the choice of blocks from their scores, and attention that reads only them, on the kernels: bounds and choices equal the statement's,
attention is compared with fp64."""
from types import SimpleNamespace

import pytest
import torch

import kv4_oracle as ko
import span_oracle as so
from fllm_b200.ops.blocks import bounds_width, code_bounds
from fllm_b200.ops.kv4 import cache_values
from fllm_b200.ops.reference import RefOps

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "e4m3", "int4"]


@pytest.fixture(scope="module")
def ops():
    from fllm_b200.ops.native import NativeOps
    return NativeOps(torch.device("cuda:0"))


def _setup(kind, *args, **more):
    return ko.setup(*args, **more) if kind == "int4" else so.setup(*args, kv=kind, **more)


def _bounds(c):
    return code_bounds(cache_values(c.k, c.D)).contiguous()


def _cpu(meta):
    return SimpleNamespace(**{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in vars(meta).items()})


def _choices(c, bounds, block, count, lead, tail):
    return RefOps().select_blocks(c.q.cpu(), bounds.cpu(), c.tables.cpu(), c.hq, c.hkv, c.D, block, count, _cpu(c.meta), lead, tail)


def _choose(ops, c, bounds, block, count, lead=1, tail=2):
    return ops.select_blocks(c.q, bounds, c.tables, c.hq, c.hkv, c.D, block, count, c.meta, lead=lead, tail=tail)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 48])
def test_bounds(ops, kind, D, block):
    """Blocks whose last place a slot names; the others stay. Tiny, huge, equal, zero and not finite keys."""
    g = torch.Generator(device="cuda").manual_seed(D)
    k = torch.randn(30, 3, block, D, generator=g, device="cuda")
    k *= torch.exp2(torch.randint(-30, 30, (30, 3, 1, 1), generator=g, device="cuda").float()) if kind != "e4m3" else 1
    k[0, 0], k[1, 0, 2, 3], k[2, 1, 0, 0], k[3, 2] = 0.0, float("nan"), float("inf") if kind != "e4m3" else 0.5, 2.0
    k[4, 0], k[5, 1] = 127.0, -127.0
    if kind != "e4m3":
        k[6, 0] *= 1e-38
        k[7, 0, 0, 0] = 3e38
    from fllm_b200.ops.kv4 import kv4_encode
    cache = {"bf16": lambda: k.bfloat16(), "e4m3": lambda: k.to(torch.float8_e4m3fn), "int4": lambda: kv4_encode(k)}[kind]()
    want = code_bounds(cache_values(cache, D))
    bounds = torch.full((30, 3, bounds_width(D)), 77, dtype=torch.int8, device="cuda")
    done = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 20, 29], device="cuda")
    slots = torch.cat([done * block + block - 1, torch.tensor([-1, 12 * block, 13 * block + block - 2, -block - 1], device="cuda")]).int()
    ops.kv_bounds(cache, bounds, slots[torch.randperm(len(slots), device="cuda")])
    assert torch.equal(bounds[done], want[done])
    rest = [i for i in range(30) if i not in done.tolist()]
    assert (bounds[rest] == 77).all() and ops.check_status() == 0
    # what they say: no key is outside
    v, e = cache_values(cache, D).double(), want[..., 2 * D].double()
    fine = (e < 127)[..., None, None].expand_as(v) & torch.isfinite(v)
    unit = torch.exp2(e)[..., None, None]
    assert (v <= want[..., :D].double()[:, :, None] * unit)[fine].all() and (v >= want[..., D:2 * D].double()[:, :, None] * unit)[fine].all()
    ops.kv_bounds(cache, bounds, torch.tensor([30 * block + block - 1], dtype=torch.int32, device="cuda"))
    assert ops.check_status() != 0


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (4, 4, 64), (10, 1, 128), (8, 4, 256), (40, 2, 64)])
@pytest.mark.parametrize("count,lead,tail", [(3, 1, 2), (8, 0, 1), (20, 2, 3), (100, 1, 1), (400, 1, 2)])
def test_choices_of_decode_rows(ops, hq, hkv, D, count, lead, tail):
    """Texts shorter and longer than what is read, empty ones, ones that end at a block's end, rows of no token."""
    c = so.setup([1, 1, 0, 2, 1, 1, 5], [0, 5000, 100, 30, 1599, 1600, 777], hq, hkv, D, seed=count)
    b = _bounds(c)
    c.tables[c.tables < 0] = 0
    assert torch.equal(_choose(ops, c, b, 16, count, lead, tail).cpu(), _choices(c, b, 16, count, lead, tail))
    assert ops.check_status() == 0


@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (6, 1, 64), (4, 2, 256)])
def test_choices_of_prompt_rows(ops, hq, hkv, D):
    """Tiles of many rows, those of a chunk from the first token on, beside decode rows (looked up), larger blocks."""
    for block, rows, ctx in (16, [70, 1, 9], [0, 900, 400]), (32, [129, 1, 1, 1, 1, 1, 1, 1], [600, 3, 90, 10, 10, 10, 10, 2000]):
        c = so.setup(rows, ctx, hq, hkv, D, block=block, seed=D)
        b = _bounds(c)
        c.tables[c.tables < 0] = 0
        assert torch.equal(_choose(ops, c, b, block, 7).cpu(), _choices(c, b, block, 7, 1, 2))
    assert ops.check_status() == 0


def test_rows_that_take_turns_in_the_scores_memory(ops):
    """Room for 64 rows at a time: the choices are the same, tiles that lie in two turns among them."""
    c = so.setup([150, 1, 41], [700, 900, 30], 8, 2, 128, seed=6)
    b = _bounds(c)
    c.tables[c.tables < 0] = 0
    m = c.meta
    few, n = ops.k.select_blocks(c.q, b, c.tables, m.q_starts, m.seq_lens, m.num_seqs, m.max_q_len, m.max_kv_len, 8, 2, 128, 16, 7, 1, 2, ops.status, 1)
    assert n == 6 and torch.equal(few, _choose(ops, c, b, 16, 7)) and torch.equal(few.cpu(), _choices(c, b, 16, 7, 1, 2))
    assert ops.check_status() == 0


def test_equal_scores_go_to_the_lower_block(ops):
    """Blocks with the same keys, queries of zeros: every score is met many times."""
    c = so.setup([1, 3], [3000, 1000], 8, 2, 128, seed=1)
    b = _bounds(c)
    b[:] = b[torch.arange(len(b), device="cuda") % 3]
    c.tables[c.tables < 0] = 0
    assert torch.equal(_choose(ops, c, b, 16, 50).cpu(), _choices(c, b, 16, 50, 1, 2))
    c.q.zero_()
    y = _choose(ops, c, b, 16, 50)
    assert (y[0] == torch.tensor(list(range(48)) + [186, 187], device="cuda")).all()


def test_values_that_are_not_finite(ops):
    """Blocks with a NaN come first; infinite queries count as 0, queries of any magnitude choose alike."""
    c = so.setup([1], [4000], 8, 2, 128, seed=2)
    tok = 16 * 77 + 3
    c.k[int(c.tables[0, 77]), 1, 3, 5] = float("nan")
    b = _bounds(c)
    y = _choose(ops, c, b, 16, 10)
    assert 77 in y[0, 1].tolist() and torch.equal(y.cpu(), _choices(c, b, 16, 10, 1, 2))
    base = y
    for f in (2.0 ** 100, 2.0 ** -100):
        d = SimpleNamespace(**{**vars(c), "q": (c.q.float() * f).bfloat16()})
        assert torch.equal(_choose(ops, d, b, 16, 10), base)
    c.q[0, 3], c.q[0, 300] = float("inf"), float("nan")
    assert torch.equal(_choose(ops, c, b, 16, 10).cpu(), _choices(c, b, 16, 10, 1, 2))
    c.q.fill_(3e38)
    assert torch.equal(_choose(ops, c, b, 16, 10).cpu(), _choices(c, b, 16, 10, 1, 2))


def test_choice_of_a_very_long_text(ops):
    """30,000 blocks, most of them the same ones (the table names them again and again)."""
    c = so.setup([1], [1000], 4, 1, 64, seed=3)
    b = _bounds(c)
    n = 30_000
    g = torch.Generator(device="cuda").manual_seed(1)
    c.tables = torch.randint(0, len(b), (1, n), generator=g, device="cuda").int()
    c.meta.seq_lens[0] = n * 16 - 5
    c.meta.max_kv_len = n * 16
    assert torch.equal(_choose(ops, c, b, 16, 500).cpu(), _choices(c, b, 16, 500, 1, 2))
    assert ops.check_status() == 0


def test_texts_longer_than_said_are_cut_and_reported(ops):
    c = so.setup([1, 1], [1000, 100], 4, 1, 64, seed=4)
    b = _bounds(c)
    c.tables[c.tables < 0] = 0
    c.meta.max_kv_len = 500
    y = _choose(ops, c, b, 16, 6)
    assert ops.check_status() != 0 and y.max() < 32
    c.meta.max_kv_len = 1001
    c.tables[0, 20] = 1 << 20                              # a block that is not there is never the best
    y = _choose(ops, c, b, 16, 6)
    assert ops.check_status() != 0 and 20 not in y[0].tolist()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (16, 2, 64), (12, 1, 128), (40, 2, 64), (8, 4, 256), (9, 1, 256)])
@pytest.mark.parametrize("sink,cap", [(False, 0.0), (True, 20.0)])
def test_attention(ops, kind, hq, hkv, D, sink, cap):
    """What is chosen is read and nothing else (what is not holds NaN), up to the row's own token."""
    rows, ctx = [1, 3, 0, 1, 1], [0, 700, 50, 2500, 47]
    c = _setup(kind, rows, ctx, hq, hkv, D, seed=D + hq, fill=float("nan"))
    c.tables[c.tables < 0] = 0
    b = _bounds(c)
    picks = _choose(ops, c, b, 16, 9)
    s = torch.linspace(-2, 2, hq, device="cuda") if sink else None
    read = {int(c.tables[int(c.row_seq[r]), i]) for r in range(len(picks)) for i in picks[r].flatten().tolist() if i >= 0}
    for p in (c.k, c.v):
        raw = p.view(torch.uint8) if p.element_size() == 1 else p
        for i in set(range(len(raw))) - read:
            raw[i] = 0xFF if p.element_size() == 1 else float("nan")
    y = ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, hq, hkv, D, D ** -0.5, c.meta, s, cap)
    so.check(y, *ko.want_blocks(c, picks, D ** -0.5, s, cap))
    assert ops.check_status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_lists_of_the_callers_own(ops, kind):
    """Lists of no block (0), of one, with larger blocks and many splits; a name behind the text is reported and ends the list."""
    c = _setup(kind, [1, 2], [4000, 3000], 8, 2, 128, block=32, seed=3)
    picks = torch.full((3, 2, 90), -1, dtype=torch.int32, device="cuda")
    picks[0, 0, :1] = 0
    picks[1, 0, :90] = torch.arange(3, 93, device="cuda")
    picks[1, 1, :3] = torch.tensor([0, 50, 93], device="cuda")
    picks[2, 1, :2] = torch.tensor([7, 93], device="cuda")
    s = torch.zeros(8, device="cuda")
    for sinks in (None, s):
        y = ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, 8, 2, 128, 128 ** -0.5, c.meta, sinks)
        so.check(y, *ko.want_blocks(c, picks, 128 ** -0.5, sinks))
        assert (y[0, 4 * 128:] == 0).all()
    assert ops.check_status() == 0
    picks[0, 0, 1] = 126
    ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, 8, 2, 128, 128 ** -0.5, c.meta)
    assert ops.check_status() != 0


def test_all_blocks_are_plain_attention(ops):
    for kind in KINDS:
        c = _setup(kind, [1, 4], [900, 60], 8, 2, 128, seed=5)
        c.tables[c.tables < 0] = 0
        picks = _choose(ops, c, _bounds(c), 16, 64)
        y = ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, 8, 2, 128, 128 ** -0.5, c.meta)
        so.check(y, *(ko if kind == "int4" else so).want(c, 128 ** -0.5, 0, 0))


@pytest.mark.parametrize("kind", KINDS)
def test_steps_in_a_graph(ops, kind):
    """Rows written, bounds of blocks that they complete, choice and attention as a decode step runs them, captured once and replayed over the ends of blocks;
    two graphs do not share scores."""
    hq, hkv, D, B, count = 8, 2, 64, 2, 5
    c = _setup(kind, [1] * B, [300, 150], hq, hkv, D, seed=2, spare=40)
    free = sorted(set(range(c.k.shape[0])) - set(c.tables[c.tables >= 0].tolist()))
    c.tables = torch.nn.functional.pad(c.tables, (0, 6), value=-1)
    for s in range(B):
        for p in range(c.tables.shape[1]):
            if c.tables[s, p] < 0:
                c.tables[s, p] = free.pop()
    bounds = _bounds(c)
    c.meta.max_kv_len = c.tables.shape[1] * 16
    lens, k, v = c.meta.seq_lens, torch.zeros(B, hkv * D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, hkv * D, device="cuda", dtype=torch.bfloat16)

    def step():
        at = lens - 1
        slots = (c.tables.gather(1, (at // 16).long()[:, None])[:, 0] * 16 + at % 16).int()
        if kind == "int4":
            ops.kv4_write(k, v, slots, c.k, c.v)
        else:
            for x, p in ((k, c.k), (v, c.v)):
                raw = p.view(torch.uint8) if kind == "e4m3" else p
                new = x.view(B, hkv, D).to(p.dtype)
                raw[slots.long() // 16, :, slots.long() % 16] = new.view(torch.uint8) if kind == "e4m3" else new
        ops.kv_bounds(c.k, bounds, slots)
        picks = _choose(ops, c, bounds, 16, count)
        return picks, ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, hq, hkv, D, D ** -0.5, c.meta)
    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for turn in range(40):
        k.normal_()
        v.normal_()
        lens += 1
        for graph, out in graphs:
            graph.replay()
    for graph, (picks, y) in graphs:
        assert torch.equal(picks.cpu(), _choices(c, bounds, 16, count, 1, 2))
    n = lens.tolist()
    tok = [torch.arange(x, device="cuda") for x in n]
    raw = lambda p: cache_values(p, D)
    c.keys = [raw(c.k)[c.tables[s].long()[t // 16], :, t % 16] for s, t in enumerate(tok)]
    c.values = [raw(c.v)[c.tables[s].long()[t // 16], :, t % 16] for s, t in enumerate(tok)]
    c.lens, c.positions = n, lens - 1
    for _, (picks, y) in graphs:
        so.check(y, *ko.want_blocks(c, picks, D ** -0.5))
    full = [int(c.tables[s, i]) for s in range(B) for i in range(n[s] // 16)]
    assert torch.equal(bounds[full], _bounds(c)[full]) and ops.check_status() == 0


def test_refusals(ops):
    c = so.setup([1], [200], 8, 2, 128)
    b = _bounds(c)
    picks = torch.zeros(1, 2, 4, dtype=torch.int32, device="cuda")
    for count, lead, tail in (2, 1, 2), (5, -1, 1), (5, 1, 0):
        with pytest.raises(ValueError, match="room"):
            _choose(ops, c, b, 16, count, lead, tail)
    with pytest.raises(ValueError, match="step batch"):
        ops.select_blocks(c.q, b, c.tables, 8, 2, 128, 16, 5, None)
    with pytest.raises(ValueError, match="step batch"):
        ops.attention_blocks(c.q, c.k, c.v, c.tables, picks, 8, 2, 128, 1.0, None)
    for bad in (lambda: ops.select_blocks(c.q, b[..., :-16], c.tables, 8, 2, 128, 16, 5, c.meta), lambda: ops.select_blocks(c.q.float(), b, c.tables, 8, 2, 128, 16, 5, c.meta),
                lambda: ops.select_blocks(c.q, b, c.tables, 8, 4, 128, 16, 5, c.meta), lambda: ops.kv_bounds(c.k, b[:-1], picks.flatten()),
                lambda: ops.kv_bounds(c.k, b, picks.flatten().long()), lambda: ops.kv_bounds(c.k[..., :64], b, picks.flatten()),
                lambda: ops.attention_blocks(c.q, c.k, c.v, c.tables, picks.long(), 8, 2, 128, 1.0, c.meta),
                lambda: ops.attention_blocks(c.q, c.k, c.v, c.tables, picks[:, :1], 8, 2, 128, 1.0, c.meta)):
        with pytest.raises(RuntimeError):
            bad()
