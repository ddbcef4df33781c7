"""Windows with first tokens, draft trees under them, moves of blocks and rows, and the bookkeeping that goes with them, on the PyTorch operators."""
from types import SimpleNamespace

import pytest
import torch

import span_oracle as so
from fllm_b200.ops.reference import RefOps
from fllm_b200.ops.span import ordered_copies


@pytest.mark.parametrize("window,first", [(5, 2), (16, 30), (1, 0), (100, 3)])
def test_reference_window(window, first):
    c = so.setup([1, 4, 20], [30, 7, 0], 4, 2, 64, seed=1, device="cpu", fill=0.0)
    y = RefOps().attention(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, 4, 2, 64, 0.125, window, meta=c.meta, first=first)
    so.check(y, *so.want(c, 0.125, window, first))


@pytest.mark.parametrize("window,first", [(0, 0), (6, 3), (2, 1)])
def test_reference_tree(window, first):
    c = so.setup([9, 70], [20, 0], 4, 2, 64, words=2, trees=[so.grow(9, 1), so.grow(70, 2)], seed=2, device="cpu")
    y = RefOps().attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks, c.base, 4, 2, 64, 0.125, window, first=first, meta=c.meta)
    so.check(y, *so.want(c, 0.125, window, first))


def test_arguments():
    ops, c = RefOps(), so.setup([1], [3], 2, 2, 64, device="cpu", words=1, trees=[[-1]])
    args = (c.q, c.k, c.v, c.tables, c.row_seq, c.positions)
    for kw in (dict(window=4, first=-1), dict(window=-1), dict(window=4, first=1, bidirectional=True)):
        with pytest.raises(ValueError):
            ops.attention(*args, 2, 2, 64, 0.125, **kw)
    with pytest.raises(ValueError):
        ops.attention_tree(*args, c.masks.view(-1), c.base, 2, 2, 64, 0.125, window=4, first=1)


def test_copies_keep_their_order():
    assert ordered_copies([(0, 1), (0, 2), (3, 3)], 9) == [[(0, 1), (0, 2)]]
    assert ordered_copies([(0, 1), (1, 2)], 9) == [[(0, 1)], [(1, 2)]]
    assert ordered_copies([(0, 1), (4, 0), (5, 1)], 9) == [[(0, 1)], [(4, 0), (5, 1)]]
    for pair in ((0, 9), (-1, 2), (9, 0)):
        with pytest.raises(ValueError):
            ordered_copies([pair], 9)
    store = torch.arange(2 * 9 * 4).float().view(2, 9, 1, 2, 2)
    want = store.clone()
    pairs = [(0, 1), (1, 2), (5, 1), (2, 0)]
    for s, d in pairs:
        want[:, d] = want[:, s]
    RefOps().kv_copy_blocks([store], pairs)
    assert torch.equal(store, want)


def test_accepted_rows_move_in_their_order():
    store = torch.arange(10 * 4).float().view(1, 10, 1, 4, 1)
    text = torch.arange(40).float()
    RefOps().kv_compact([store], torch.tensor([list(range(10))]), torch.tensor([6]), torch.tensor([[0, 2, 3, 9]]), torch.tensor([4]))
    want = text.clone()
    want[6:10] = text[[6, 8, 9, 15]]
    assert torch.equal(store.view(-1), want)
    with pytest.raises(ValueError):
        RefOps().kv_compact([store], torch.tensor([[0]]), torch.tensor([0]), torch.tensor([[1, 0]]), torch.tensor([2]))


def test_caches_name_their_pools():
    from fllm_b200.models.decoder import KVCache
    from fllm_b200.models.row_cache import RowCache, RowSpec
    ops = RefOps()
    kv = KVCache(2, 6, 3, 4, 8, "cpu", torch.float32)
    kv.store.normal_()
    want = kv.store.clone()
    want[:, :, 5] = want[:, :, 1]
    kv.copy_blocks([(1, 5)], ops)
    assert torch.equal(kv.store, want)
    rc = RowCache([RowSpec(16), RowSpec(8, 2), RowSpec(8, 2, 4, 3)], 6, 4, "cpu", torch.float32)
    for t in rc.rows + [f for f in rc.factors + rc.value_rows if f is not None]:
        t.normal_()
    all_of = lambda: [t.clone() for t in rc.rows + [f for f in rc.factors + rc.value_rows if f is not None]]
    before = all_of()
    rc.copy_blocks([(2, 0)], ops)
    for a, b in zip(before, all_of()):
        a[0] = a[2]
        assert torch.equal(a, b)
    before = all_of()
    rc.compact(torch.tensor([[3, 4]]), torch.tensor([1]), torch.tensor([[0, 4]]), torch.tensor([2]), ops)
    for a, b in zip(before, all_of()):
        if a.dim() == 3 and a.shape[1] == 4:
            a[3, 2] = a[4, 1]
        else:
            a[3, :, 2] = a[4, :, 1]
        assert torch.equal(a, b)


def test_first_blocks_are_not_pruned():
    from fllm_b200.runtime.block_manager import BlockManager
    bm = BlockManager(40, 4, False)
    bm.allocate(1, list(range(90)))
    assert bm.ensure_capacity(1, 90)
    sb = bm.seqs[1]
    sb.num_tokens = 90
    before = list(sb.table)
    free = len(bm.free)
    freed = bm.prune_window(1, 20, 6)
    assert [i for i, b in enumerate(sb.table) if b < 0] == list(range(2, 17)) and freed == 15 and len(bm.free) == free + 15
    assert sb.table[:2] == before[:2] and sb.table[17:] == before[17:]
    assert bm.prune_window(1, 20, 6) == 0


def _engine(first):
    from fllm_b200.config import EngineConfig, preset
    from fllm_b200.runtime import LLMEngine
    cfg = preset("qwen3-tiny")
    cfg.sliding_window, cfg.window_first = 24, first
    return LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=64, max_model_len=256), device="cpu")


def test_engine_keeps_the_first_tokens():
    """A served model whose windows leave the first tokens visible: the blocks of the text between are freed, the tokens are those of the whole text
    under the same mask."""
    from fllm_b200.runtime import SamplingParams
    prompt = [(7 * i) % 50 + 1 for i in range(90)]
    outs = {}
    for first in (0, 20):
        eng = _engine(first)
        outs[first] = eng.generate([prompt], SamplingParams(max_tokens=8))
        stepped = eng.generate([prompt[:40]], SamplingParams(max_tokens=8))
        whole = _engine(first)
        whole.scheduler.window = 0                      # nothing is freed
        assert whole.generate([prompt], SamplingParams(max_tokens=8)) == outs[first]
        assert whole.generate([prompt[:40]], SamplingParams(max_tokens=8)) == stepped
    assert outs[0] != outs[20]


def test_cow_of_a_fork_runs_as_one_copy():
    from fllm_b200.models.decoder import KVCache
    from fllm_b200.runtime.scheduler import ScheduledStep
    calls = []
    kv = KVCache(1, 8, 1, 4, 8, "cpu", torch.float32)
    ops = SimpleNamespace(kv_copy_blocks=lambda pools, pairs: calls.append((len(pools), list(pairs))))
    kv.copy_blocks(ScheduledStep(cow=[(0, 1), (2, 3)]).cow, ops)
    assert calls == [(1, [(0, 1), (2, 3)])]


def test_a_stage_without_caches_copies_nothing():
    from fllm_b200.models.decoder import KVCache
    from fllm_b200.models.row_cache import RowCache
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    for kv in (KVCache(0, 4, 2, 16, 64, "cpu"), RowCache([], 4, 16, "cpu")):
        assert kv.pools() == []
        kv.copy_blocks([(0, 1), (1, 2)], RefOps())
        kv.compact(i32([[0, 1]]), i32([3]), i32([[1, 2]]), i32([2]), RefOps())


@pytest.mark.parametrize("first", [0, 20])
@pytest.mark.parametrize("how", ["import", "swap"])
def test_blocks_freed_behind_a_window_stay_absent_when_the_sequence_comes_back(first, how):
    """A sequence that is handed over, or comes back from the host, has holes where its window had passed. Fresh blocks hold other text there, which
    must not be found under this text's name."""
    from fllm_b200.config import EngineConfig, preset
    from fllm_b200.runtime import LLMEngine, SamplingParams
    from fllm_b200.runtime.scheduler import ScheduledStep
    cfg = preset("qwen3-tiny")
    cfg.sliding_window, cfg.window_first = 24, first
    make = lambda: LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=64, max_model_len=256, preemption="swap"), device="cpu")
    prompt = [(7 * i) % 50 + 1 for i in range(120)]
    other = prompt[:70] + [3, 9, 4]
    params = SamplingParams(max_tokens=6)
    want = [make().generate([p], params)[0] for p in (prompt, other)]
    eng = make()
    if how == "import":
        blob, _ = eng.prefill_only(prompt, params)
        eng = make()
        eng.kv.store.normal_()                          # blocks that were others' before
        rid = eng.import_request(blob)
        live = blob["live_blocks"]
    else:
        rid = eng.add_request(prompt, params)
        while not eng.requests[rid].output:
            eng.step()
        eng.drain()
        assert eng.scheduler._preempt_one(ScheduledStep(), None) and eng.requests[rid].swapped
        live = eng.scheduler.swapper.parked[eng.requests[rid].seq_id][1]
        eng.blocks.reset_prefix_cache()
        eng.kv.store.normal_()
        eng.step()
        eng.drain()
    r = eng.requests[rid]
    head = -(-first // 16)
    assert live == list(range(head)) + [6, 7]
    table = eng.blocks.table(r.seq_id)
    assert [i for i, b in enumerate(table) if b >= 0] == live and eng.blocks.num_used() == len(live)
    assert eng.blocks.np_table(r.seq_id).tolist() == table
    got = {}
    follow = eng.add_request(other, params)
    while eng.has_unfinished():
        for e in eng.step():
            got.setdefault(e.request_id, []).extend(e.token_ids)
    assert got[follow] == want[1] and r.output == want[0]
    assert eng.blocks.num_used() == 0


def test_trees_without_a_step_batch_take_any_window_below_one():
    c = so.setup([5], [9], 2, 2, 64, device="cpu", words=1, trees=[so.grow(5, 1)])
    tree = lambda **kw: RefOps().attention_tree(c.q, c.k, c.v, c.tables, c.row_seq, c.positions, c.masks.view(-1), c.base, 2, 2, 64, 0.125, **kw)
    assert torch.equal(tree(window=-3), tree())
    for kw in (dict(first=-1), dict(first=2), dict(window=-3, meta=c.meta)):
        with pytest.raises(ValueError):
            tree(**kw)


def test_a_forked_sequence_writes_into_a_block_of_its_own():
    """Two sequences share a partly filled block and go on with different tokens: the engine's step copies it for one of them, both read what they would
    have alone."""
    import copy
    from fllm_b200.config import EngineConfig, preset
    from fllm_b200.runtime import LLMEngine, SamplingParams
    cfg = preset("qwen3-tiny")
    make = lambda: LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=64, max_model_len=256), device="cpu")
    prompt = [(7 * i) % 50 + 1 for i in range(40)]
    params = SamplingParams(max_tokens=8)

    def start(eng):
        rid = eng.add_request(prompt, params)
        r = eng.requests[rid]
        while len(r.output) < 2:
            eng.step()
        eng.drain()
        return r
    want = []
    for turn in (0, 1):                                  # alone: the first as it is, the second with another last token
        eng = make()
        r = start(eng)
        if turn:
            r.output[-1] = 17
        while eng.has_unfinished():
            eng.step()
        want.append(list(r.output))
    eng = make()
    parent = start(eng)
    child = copy.copy(parent)
    child.request_id, child.seq_id, child.output = "child", next(eng._seq_ids), list(parent.output)
    child.output[-1] = 17
    eng.blocks.fork(parent.seq_id, child.seq_id)
    eng.scheduler.running.append(child)
    eng.requests["child"] = child
    shared = list(eng.blocks.table(parent.seq_id))
    assert parent.num_computed % 16 and shared == eng.blocks.table(child.seq_id)
    calls = []
    copies = eng.ops.kv_copy_blocks
    eng.ops.kv_copy_blocks = lambda pools, pairs: (calls.append((len(pools), list(pairs))), copies(pools, pairs))
    eng.step()
    eng.drain()
    tables = [eng.blocks.table(r.seq_id) for r in (parent, child)]
    (pools, ((src, dst),)), = calls
    assert pools == 1 and eng.blocks.stats["cow"] == 1 and src == shared[-1] and {src, dst} == {t[len(shared) - 1] for t in tables}
    assert all(t[:len(shared) - 1] == shared[:-1] for t in tables)
    while eng.has_unfinished():
        eng.step()
    assert [parent.output, child.output] == want and want[0] != want[1] and len(calls) == 1
    assert eng.blocks.num_used() == 0
