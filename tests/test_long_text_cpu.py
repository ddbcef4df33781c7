"""Caches held in 4 bits and attention over selected blocks without a GPU: what their statements say, and engines that are served by them."""
import math

import pytest
import torch

from fllm_b200.config import EngineConfig, preset
from fllm_b200.models.decoder import KVCache
from fllm_b200.models.weights import init_random_weights
from fllm_b200.ops.blocks import NOT_FINITE, bounds_width, code_bounds
from fllm_b200.ops.kv4 import is_kv4, kv4_decode, kv4_encode, kv4_width
from fllm_b200.ops.reference import RefOps
from fllm_b200.runtime import LLMEngine, SamplingParams


def _prompts(vocab, lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("D", [64, 128, 256])
def test_encoding(D):
    """Half a step at most, ends of the range within reach, exact rows of one value; rows that are not finite read as NaN."""
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(200, D, generator=g) * torch.exp2(torch.randint(-20, 20, (200, 1), generator=g).float())).bfloat16()
    x[0], x[1], x[2] = 3.0, 0.0, -5.5
    rows = kv4_encode(x)
    assert rows.shape == (200, kv4_width(D)) and rows.dtype == torch.uint8 and is_kv4(rows, D) and not is_kv4(rows, 2 * D)
    y = kv4_decode(rows).double()
    step = rows[:, D // 2:D // 2 + 2].contiguous().view(torch.bfloat16).double()
    low = rows[:, D // 2 + 2:].contiguous().view(torch.bfloat16).double()
    assert torch.equal(low[:, 0], x.double().amin(1)) and torch.equal(y[:3], x[:3].double())
    # fp32 rounds z + s c once more: 2^-24 of the row's largest
    assert ((y - x.double()).abs() <= step / 2 * (1 + 2.0 ** -22) + 2.0 ** -23 * x.double().abs().amax(1, keepdim=True)).all()
    assert (step <= (x.double().amax(1, keepdim=True) - low) / 15 * (1 + 2.0 ** -7)).all()
    codes = torch.stack([rows[:, :D // 2] & 15, rows[:, :D // 2] >> 4], -1).flatten(1).double()
    assert torch.equal((low + step * codes).float().double(), y)
    for bad in (math.nan, math.inf, -math.inf):
        z = x[5:6].clone()
        z[0, 3] = bad
        assert torch.isnan(kv4_decode(kv4_encode(z))).all()
    wide = torch.zeros(1, D).bfloat16()
    wide[0, 0], wide[0, 1] = 3e38, -3e38
    assert torch.isnan(kv4_decode(kv4_encode(wide))).all()


def test_widths():
    assert [kv4_width(d) for d in (64, 128, 256)] == [36, 68, 132]
    for d in (32, 96, 512):
        with pytest.raises(ValueError):
            kv4_width(d)


def test_bounds_hold_every_key_and_scores_every_product():
    g = torch.Generator().manual_seed(3)
    k = torch.randn(50, 2, 16, 64, generator=g) * torch.exp2(torch.randint(-10, 10, (50, 2, 1, 1), generator=g).float())
    k[0, 0] = 0.0
    b = code_bounds(k)
    e = b[..., 128].double()
    hi, lo = (b[..., i:i + 64].double() * torch.exp2(e)[..., None] for i in (0, 64))
    assert (k.double().amax(2) <= hi).all() and (k.double().amin(2) >= lo).all() and b.abs().max() <= 127
    assert int(b[0, 0, 128]) == -120 and (b[0, 0, :128] == 0).all()
    assert (b[..., :128].abs().amax(-1)[e > -120] >= 64).all()
    q = torch.randn(4, 64, generator=g)                  # of a group of four heads
    u, w = q.clamp(min=0).sum(0).double(), (-q).clamp(min=0).sum(0).double()
    score = (hi * u - lo * w).sum(-1)
    assert (score >= torch.einsum("hd,bktd->bkht", q.double(), k.double()).sum(2).amax(-1) - 1e-9).all()
    k[3, 1, 2, 5], k[4, 0, 0, 0] = math.nan, 3e38
    b = code_bounds(k)
    assert int(b[3, 1, 128]) == NOT_FINITE and int(b[4, 0, 128]) == NOT_FINITE and int(b[3, 0, 128]) != NOT_FINITE


def _first_logits(eng, prompt):
    rows = []
    eng.add_request(prompt, SamplingParams(max_tokens=1))
    while eng.has_unfinished():
        step = eng.scheduler.schedule()
        logits = eng.decoder.forward(eng._build_batch(step))
        if logits.shape[0]:
            rows.append(logits[-1].float())
        eng._commit(step, eng.decoder.greedy_tokens(logits).tolist())
    return rows[-1]


def _engine(w, cfg, **more):
    args = dict(max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256, num_kv_blocks=64)
    return LLMEngine(cfg, EngineConfig(**{**args, **more}), device="cpu", weights=w)


def test_engine_with_a_4_bit_cache():
    """Chunked prompts, prefix hits, forks of blocks and preemption keep the tokens; the logits follow those over a bf16 cache: a row's values are off by
    half of 1/15 of its range at most, a tenth of their size in the mean, and what attention averages less."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    a, b = _prompts(cfg.vocab_size, (70, 45))
    eng = _engine(w, cfg, kv_cache_dtype="int4")
    assert eng.kv.store.dtype == torch.uint8 and eng.kv.store.shape[-1] == cfg.head_dim // 2 + 4
    assert KVCache.bytes_per_block(2, 4, 16, 128, four_bit=True) == 2 * 2 * 4 * 16 * 68
    x, y = _first_logits(_engine(w, cfg), a), _first_logits(eng, a)
    err = (x - y).abs().max() / x.abs().max()
    assert 0 < err < 0.3, err
    sp = SamplingParams(max_tokens=10)
    want = [_engine(w, cfg, kv_cache_dtype="int4", enable_prefix_caching=False).generate([p], sp)[0] for p in (a, b)]
    eng = _engine(w, cfg, kv_cache_dtype="int4", max_num_batched_tokens=32)
    assert [eng.generate([p], sp)[0] for p in (a, b)] == want and [eng.generate([p], sp)[0] for p in (a, b)] == want
    tight = _engine(w, cfg, kv_cache_dtype="int4", num_kv_blocks=13, max_model_len=128, watermark=0.0, enable_prefix_caching=False, preemption="swap", swap_space_gb=0.25)
    roomy = _engine(w, cfg, kv_cache_dtype="int4", max_model_len=128, enable_prefix_caching=False)
    four = _prompts(cfg.vocab_size, (40, 44, 48, 52))
    assert tight.generate(four, SamplingParams(max_tokens=12)) == roomy.generate(four, SamplingParams(max_tokens=12))
    assert tight.scheduler.swapper.stats["swapped_in"] > 0


def test_blocks_are_handed_over_between_kinds_of_caches():
    """A prompt's blocks from a 4-bit engine to another, from bf16 to 4-bit (encoded: what that engine itself would hold of the same rows in the first layer)
    and back (rounded); e4m3 and bf16 do not take each other's."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    p = _prompts(cfg.vocab_size, (50,))[0]
    mk = lambda kind, **kw: _engine(w, cfg, kv_cache_dtype=kind, **kw)
    sp = SamplingParams(max_tokens=8)
    kinds = {k: mk(k).prefill_only(p, sp)[0] for k in ("bf16", "int4", "fp8_e4m3")}

    def finish(eng, blob):
        rid, toks = eng.import_request(blob), list(blob["output"])
        while eng.has_unfinished():
            toks += [t for ev in eng.step() if ev.request_id == rid for t in ev.token_ids]
        return toks
    assert finish(mk("int4"), kinds["int4"]) == mk("int4").generate([p], sp)[0]
    for src, dst in (("bf16", "int4"), ("int4", "bf16")):
        eng = mk(dst, sparse_blocks=8)
        eng.import_request(kinds[src])
        table = [eng.blocks.table(r.seq_id) for r in eng.requests.values()][0][:3]
        got, kv = eng.kv.store[:, :, table], kinds[src]["kv"][:, :, :3]
        assert torch.equal(got, kv4_encode(kv) if dst == "int4" else kv4_decode(kv).bfloat16())
        for layer in range(cfg.num_layers):                 # of the full blocks
            keys = eng.kv.k(layer)[table]
            assert torch.equal(eng.kv.bounds[layer][table], code_bounds(kv4_decode(keys) if dst == "int4" else keys.float()))
        assert len(finish(mk(dst), kinds[src])) == 8
    for src, dst in (("fp8_e4m3", "bf16"), ("bf16", "fp8_e4m3"), ("fp8_e4m3", "int4"), ("int4", "fp8_e4m3")):
        with pytest.raises(ValueError):
            mk(dst).import_request(kinds[src])
    short = dict(kinds["bf16"], kv=kinds["bf16"]["kv"][..., :32])
    with pytest.raises(ValueError):
        mk("int4").import_request(short)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_engine_with_selected_blocks(kind):
    """Texts within the blocks that are read: the tokens of an engine that reads all. Longer ones: chunks and prefix hits, preemption and the tiers, which bring
    blocks back, keep the tokens."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    sp = SamplingParams(max_tokens=12)
    p = _prompts(cfg.vocab_size, (150, 100, 180))
    mk = lambda **kw: _engine(w, cfg, kv_cache_dtype=kind, **kw)
    assert [mk(sparse_blocks=13).generate([x], sp)[0] for x in p] == [mk().generate([x], sp)[0] for x in p]
    few = dict(sparse_blocks=4, sparse_lead=1, sparse_tail=2)
    want = [mk(**few, enable_prefix_caching=False, max_num_batched_tokens=256).generate([x], sp)[0] for x in p]
    eng = mk(**few, max_num_batched_tokens=48)
    assert [eng.generate([x], sp)[0] for x in p] == want and [eng.generate([x], sp)[0] for x in p] == want
    logits = [_first_logits(mk(**kw), p[2]) for kw in (few, {})]
    assert not torch.equal(*logits)
    tight = mk(**few, num_kv_blocks=26, watermark=0.0, enable_prefix_caching=False, preemption="swap", swap_space_gb=0.25)
    assert tight.generate(p, sp) == mk(**few, enable_prefix_caching=False).generate(p, sp)
    assert tight.scheduler.swapper.stats["swapped_in"] > 0
    tier = mk(**few, num_kv_blocks=16, watermark=0.0, kv_tier_host_gb=0.01)
    assert [tier.generate([x], sp)[0] for x in p] == want and [tier.generate([x], sp)[0] for x in p] == want
    assert tier.blocks.stats["tier_restored"] > 0


def test_copies_and_compaction_keep_the_bounds():
    ops = RefOps()
    for kind in ("bf16", "int4"):
        kv = KVCache(2, 9, 3, 16, 64, "cpu", "int4" if kind == "int4" else torch.bfloat16, (4, 1, 2))
        if kind == "int4":
            kv.store.copy_(kv4_encode(torch.randn(*kv.store.shape[:-1], 64)))
        else:
            kv.store.normal_()
        every = torch.arange(9)
        kv.find_bounds(every, ops)
        fresh = lambda: torch.stack([code_bounds(kv4_decode(kv.k(i)) if kind == "int4" else kv.k(i).float()) for i in range(2)])
        assert torch.equal(kv.bounds, fresh())
        kv.copy_blocks([(1, 5), (5, 6)], ops)
        kv.copy_block(2, 7)
        assert torch.equal(kv.bounds, fresh())
        # a tree behind 28 tokens: rows 28 to 33 are moved to, of which 31 ends block 4
        kv.compact(torch.tensor([[3, 4, 8]], dtype=torch.int32), torch.tensor([28], dtype=torch.int32), torch.tensor([[0, 2, 5, 7, 9, 12]], dtype=torch.int32),
                   torch.tensor([6], dtype=torch.int32), ops)
        assert torch.equal(kv.bounds[:, 4], fresh()[:, 4])


@pytest.mark.parametrize("bad", [dict(kv_cache_dtype="int3"), dict(sparse_blocks=2), dict(sparse_blocks=4, sparse_tail=0), dict(sparse_blocks=4, sparse_lead=-1)])
def test_engine_refusals(bad):
    cfg = preset("qwen3-tiny")
    with pytest.raises(ValueError):
        LLMEngine(cfg, EngineConfig(num_kv_blocks=8, max_model_len=64, **bad), device="cpu")


def test_engine_refuses_models_without_such_layers():
    cfg = preset("qwen3-tiny")
    cfg.head_dim = 32
    with pytest.raises(ValueError, match="head dims"):
        LLMEngine(cfg, EngineConfig(num_kv_blocks=8, max_model_len=64, kv_cache_dtype="int4"), device="cpu")


def test_command_line_flags():
    import argparse
    from fllm_b200.cli import _add_engine_flags, build_engine
    p = argparse.ArgumentParser()
    _add_engine_flags(p)
    args = p.parse_args(["--model", "qwen3-tiny", "--device", "cpu", "--kv-cache-type", "int4", "--sparse-blocks", "6", "--sparse-lead", "2", "--sparse-tail", "1", "--ctx",
                         "128", "--kv-blocks", "16"])
    eng = build_engine(args)
    eng = eng[0] if isinstance(eng, tuple) else eng
    assert eng.kv.sparse == (6, 2, 1) and eng.kv.four_bit and eng.kv.bounds.shape[-1] == bounds_width(eng.model_cfg.head_dim)


def test_blocks_that_are_handed_over_are_as_many_as_are_named():
    """Fewer or more blocks than the request names, of the pool's kind or of another: refused, and nothing stays allocated."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    p = _prompts(cfg.vocab_size, (50,))[0]
    for src in ("bf16", "int4"):
        blob = _engine(w, cfg, kv_cache_dtype=src).prefill_only(p, SamplingParams(max_tokens=4))[0]
        for dst in ("bf16", "int4"):
            eng = _engine(w, cfg, kv_cache_dtype=dst)
            free = eng.blocks.num_free()
            for kv in (blob["kv"][:, :, :1], blob["kv"][:, :, [0, 1, 2, 3, 3]]):
                with pytest.raises(ValueError, match="blocks"):
                    eng.import_request(dict(blob, kv=kv))
                assert eng.blocks.num_free() == free and not eng.requests


def test_e4m3_blocks_come_back():
    """Blocks of an e4m3 cache are handed over, and swapped, like those of other kinds."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    mk = lambda **kw: _engine(w, cfg, kv_cache_dtype="fp8_e4m3", max_model_len=128, enable_prefix_caching=False, **kw)
    p = _prompts(cfg.vocab_size, (40, 44, 48, 52))
    sp = SamplingParams(max_tokens=12)
    blob = mk().prefill_only(p[0], sp)[0]
    eng = mk()
    rid, toks = eng.import_request(blob), list(blob["output"])
    while eng.has_unfinished():
        toks += [t for ev in eng.step() if ev.request_id == rid for t in ev.token_ids]
    assert toks == mk().generate([p[0]], sp)[0]
    tight = mk(num_kv_blocks=13, watermark=0.0, preemption="swap", swap_space_gb=0.25)
    assert tight.generate(p, sp) == mk().generate(p, sp) and tight.scheduler.swapper.stats["swapped_in"] > 0


def test_the_tiers_bring_blocks_back_without_more_where_no_bounds_are_kept(monkeypatch):
    """No tensor is made for bounds that an engine does not have."""
    cfg = preset("qwen3-tiny")
    w = init_random_weights(cfg, "cpu")
    p, sp = _prompts(cfg.vocab_size, (150, 100, 180)), SamplingParams(max_tokens=4)
    looked = []
    monkeypatch.setattr(KVCache, "find_bounds", lambda self, blocks, ops: looked.append(len(blocks)))
    for sparse in (0, 4):
        eng = _engine(w, cfg, sparse_blocks=sparse, num_kv_blocks=16, watermark=0.0, kv_tier_host_gb=0.01)
        for _ in range(2):
            for x in p:
                eng.generate([x], sp)
        assert eng.blocks.stats["tier_restored"] > 0
        assert len(looked) == (eng.blocks.stats["tier_restored"] if sparse else 0)


def test_texts_of_too_many_blocks_are_refused_before_any_step():
    """The kernel that chooses blocks holds the scores of MOST_BLOCKS of them; the PyTorch operators have no such limit."""
    from types import SimpleNamespace

    from fllm_b200.ops.blocks import MOST_BLOCKS
    cfg = preset("qwen3-tiny")
    check = lambda ops, **kw: LLMEngine._check_cache_kind(SimpleNamespace(cfg=EngineConfig(sparse_blocks=8, **kw), model_cfg=cfg, ops=ops))
    native, plain = SimpleNamespace(k=None), SimpleNamespace()
    check(native, max_model_len=16 * MOST_BLOCKS)
    check(native, max_model_len=32 * MOST_BLOCKS, block_size=32)
    check(plain, max_model_len=16 * MOST_BLOCKS + 1)
    for bad in (dict(max_model_len=16 * MOST_BLOCKS + 1), dict(max_model_len=64 * MOST_BLOCKS, block_size=32)):
        with pytest.raises(ValueError, match="blocks"):
            check(native, **bad)
