"""Engines with a cache held in 4 bits and with attention over selected blocks on the kernels: against the PyTorch operators, with and without graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _prompts(vocab, lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


def _cfg(head_dim):
    from fllm_b200.config import preset
    cfg = preset("qwen3-tiny")
    cfg.head_dim = head_dim
    return cfg


def _step_logits(cfg, eng, ops, kind, sparse, prompt):
    from fllm_b200.models.decoder import Decoder, KVCache, StepBatch
    n = len(prompt)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    b = StepBatch(i32(prompt), i32(list(range(n))), i32(list(range(n))), i32([0] * n), i32([list(range(40))]), i32([n - 1]), num_seqs=1, num_tokens=n,
                  max_kv_len=n, max_q_len=n, min_q_len=n, seq_lens=i32([n]), q_starts=i32([0, n]))
    kv = KVCache(cfg.num_layers, 44, cfg.num_kv_heads, 16, cfg.head_dim, "cuda", kind, sparse)
    return Decoder(cfg, eng.weights, kv, ops, eng.spec).forward(b).float()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("sparse", [None, (40, 1, 2)])
def test_model_follows_the_pytorch_operators(head_dim, kind, sparse):
    """A prompt in one step. (Rows of activations that differ in the last bit may meet another code; a block that scores almost as well as another may be
    chosen instead of it: the lists here hold all blocks, so that the logits can be compared. Choices themselves are compared with equal inputs elsewhere.)"""
    from fllm_b200.config import EngineConfig
    from fllm_b200.ops.reference import RefOps
    from fllm_b200.runtime import LLMEngine
    cfg = _cfg(head_dim)
    eng = LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=64, max_model_len=256), device="cuda:0")
    prompt = _prompts(cfg.vocab_size, (300,))[0]
    dtype = "int4" if kind == "int4" else torch.bfloat16
    mine, plain = (_step_logits(cfg, eng, ops, dtype, sparse, prompt) for ops in (eng.ops, RefOps()))
    assert (mine - plain).abs().max() <= (0.05 if kind == "bf16" else 0.1) * plain.abs().max()
    assert eng.ops.check_status() == 0


@pytest.mark.parametrize("kind", ["bf16", "int4", "fp8_e4m3"])
@pytest.mark.parametrize("sparse", [0, 5])
def test_served(kind, sparse):
    """Chunked prompts, captured decode steps, prefix hits: a request alone gives the same tokens from every engine; eager steps, whose attention may be cut
    into other parts (sums in another order, after which a random model may go another way), give the first; requests together run."""
    from fllm_b200.config import EngineConfig
    from fllm_b200.models.weights import init_random_weights
    from fllm_b200.runtime import LLMEngine, SamplingParams
    cfg = _cfg(64)
    w = init_random_weights(cfg, "cuda:0")
    mk = lambda **kw: LLMEngine(cfg, EngineConfig(max_num_seqs=8, max_num_batched_tokens=64, max_model_len=512, num_kv_blocks=160, kv_cache_dtype=kind,
                                                  sparse_blocks=sparse, **kw), device="cuda:0", weights=w)
    p = _prompts(cfg.vocab_size, (150, 33, 280))
    sp = SamplingParams(max_tokens=40)
    graphs, eager = mk(), mk(use_cuda_graphs=False)
    a = [graphs.generate([x], sp)[0] for x in p]
    assert a == [mk().generate([x], sp)[0] for x in p] and graphs.stats.graph_steps > 0
    assert [t[0] for t in a] == [eager.generate([x], sp)[0][0] for x in p]
    assert [len(t) for t in graphs.generate(p, sp)] == [40] * 3
    assert graphs.ops.check_status() == 0 and eager.ops.check_status() == 0
    if sparse:
        assert int((graphs.kv.bounds[0] != 0).any(-1).any(-1).sum()) > 10


def test_a_list_of_all_blocks_serves_what_plain_attention_does():
    from fllm_b200.config import EngineConfig
    from fllm_b200.models.weights import init_random_weights
    from fllm_b200.runtime import LLMEngine
    cfg = _cfg(128)
    w = init_random_weights(cfg, "cuda:0")
    prompt = _prompts(cfg.vocab_size, (200,))[0]
    rows = []
    for sparse in (0, 30):
        eng = LLMEngine(cfg, EngineConfig(max_num_seqs=4, num_kv_blocks=64, max_model_len=256), device="cuda:0", weights=w)
        rows.append(_step_logits(cfg, eng, eng.ops, torch.bfloat16, (sparse, 1, 2) if sparse else None, prompt))
    assert (rows[0] - rows[1]).abs().max() <= 0.05 * rows[0].abs().max()


def test_blocks_are_handed_over_between_kinds_of_caches():
    from fllm_b200.config import EngineConfig
    from fllm_b200.models.weights import init_random_weights
    from fllm_b200.ops.blocks import code_bounds
    from fllm_b200.ops.kv4 import kv4_decode, kv4_encode
    from fllm_b200.runtime import LLMEngine, SamplingParams
    cfg = _cfg(64)
    w = init_random_weights(cfg, "cuda:0")
    mk = lambda kind, **kw: LLMEngine(cfg, EngineConfig(max_num_seqs=4, max_model_len=256, num_kv_blocks=64, kv_cache_dtype=kind, **kw), device="cuda:0", weights=w)
    p = _prompts(cfg.vocab_size, (90,))[0]
    for src, dst in (("bf16", "int4"), ("int4", "bf16")):
        blob, _ = mk(src).prefill_only(p, SamplingParams(max_tokens=6))
        eng = mk(dst, sparse_blocks=8)
        rid, toks = eng.import_request(blob), list(blob["output"])
        table = [eng.blocks.table(r.seq_id) for r in eng.requests.values()][0][:5]
        kv = blob["kv"][:, :, :5].cuda()
        assert torch.equal(eng.kv.store[:, :, table], kv4_encode(kv) if dst == "int4" else kv4_decode(kv).bfloat16())
        keys = eng.kv.k(1)[table]
        assert torch.equal(eng.kv.bounds[1][table], code_bounds(kv4_decode(keys) if dst == "int4" else keys.float()))
        while eng.has_unfinished():
            toks += [t for ev in eng.step() if ev.request_id == rid for t in ev.token_ids]
        assert len(toks) == 6 and eng.ops.check_status() == 0


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_copies_and_compaction(kind):
    from fllm_b200.models.decoder import KVCache
    from fllm_b200.ops.kv4 import kv4_encode
    from fllm_b200.ops.native import NativeOps
    from fllm_b200.ops.reference import RefOps
    ops, sides = NativeOps(torch.device("cuda:0")), []
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(3, 2, 12, 4, 16, 128, generator=g, device="cuda").bfloat16()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    for o in (ops, RefOps()):
        kv = KVCache(3, 12, 4, 16, 128, "cuda", "int4" if kind == "int4" else torch.bfloat16, (4, 1, 2))
        kv.store.copy_(kv4_encode(x) if kind == "int4" else x)
        kv.find_bounds(torch.arange(12, device="cuda"), o)
        kv.copy_blocks([(1, 5), (5, 6)], o)
        kv.compact(i32([[3, 4, 8], [0, 2, 9]]), i32([28, 12]), i32([[0, 2, 5, 7, 9, 12], [1, 2, 3, 4, 5, 6]]), i32([6, 4]), o)
        sides.append(kv)
    assert torch.equal(sides[0].store, sides[1].store) and torch.equal(sides[0].bounds, sides[1].bounds) and ops.check_status() == 0
