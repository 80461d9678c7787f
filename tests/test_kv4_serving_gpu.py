"""The 4-bit cache behind the connector: pushed to another instance, offloaded and onboarded, matched as a prefix."""

import pytest
import torch

from test_pd_serving_gpu import _prompts, run_colocated

from kvbm_b200.models.llama import LlamaConfig, LlamaModel
from kvbm_b200.serving.engine import EngineConfig, LLMEngine, Request
from kvbm_b200.serving.pd import PdConfig

pytestmark = pytest.mark.gpu


def _cfg():
    return LlamaConfig(hidden=256, layers=3, heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512,
                       max_position=512)


def _run(eng, req):
    eng.add_request(req)
    while eng.has_unfinished() or eng._delayed:
        eng.step()
    torch.cuda.synchronize()
    return req


def _rows(pool, blocks, n):
    """The first n tokens' rows of a request's blocks, all layers."""
    ids = torch.tensor(blocks[: -(-n // 16)], device="cuda")
    return [pool.layer_view(l)[ids].transpose(1, 2).flatten(0, 1)[:n] for l in range(pool.config.num_layers)]


def test_prefill_is_pushed_into_another_instance():
    """The decode instance's pool holds the bytes that the prefill wrote, and goes on from them as one engine does."""
    model = LlamaModel(_cfg(), "cuda", seed=5)
    cfg = PdConfig(model=model.cfg, concurrency=4, prompt_len=72, gen_len=6, kv_bits=4)
    prompts = _prompts(4, [72, 50, 33, 16], model.cfg.vocab)
    dec, pre, reqs = run_colocated(model, cfg, prompts, layer_batch=2)
    assert dec.engine.pool.dtype == pre.engine.pool.dtype == torch.uint8
    assert dec.leader.cd_stats["dispatched"] == 4 and dec.leader.cd_stats["received"] == 4
    moved = sum((p.numel() + 15) // 16 for p in prompts)
    assert pre.worker.take_push_timings()[1] * cfg.prompt_blocks == moved * cfg.kv_bytes_per_request()
    scratch = model.allocate_pool(16, 16, kv_bits=4)
    for r, p in zip(reqs, prompts):
        n = p.numel()
        ids = list(range(1, 1 + (n + 15) // 16))
        model.prefill(p.cuda(), scratch, torch.tensor(ids, dtype=torch.int32, device="cuda"))
        for a, b in zip(_rows(scratch, ids, n - 1), _rows(dec.engine.pool, r.block_ids, n - 1)):
            assert torch.equal(a, b)  # (decode computes the last prompt position again)
        assert r.output.numel() == cfg.gen_len
    for inst in (dec, pre):
        inst.shutdown()


def test_offloaded_blocks_are_onboarded():
    from kvbm_b200.connector.leader import ConnectorLeader
    from kvbm_b200.connector.worker import ConnectorWorker
    from kvbm_b200.engine.leader import InstanceLeader, ParallelWorkers
    from kvbm_b200.logical.manager import BlockManager, Tier
    from kvbm_b200.utils.config import KvbmConfig

    model = LlamaModel(_cfg(), "cuda", seed=3)
    kcfg = KvbmConfig.load({"cache": {"host": {"num_blocks": 32}}}, env={}, system_toml=None)
    leader = ConnectorLeader(InstanceLeader(BlockManager(32, 16, "lineage", Tier.G2), ParallelWorkers([])), 16)
    worker = ConnectorWorker(kcfg, block_size=16)
    eng = LLMEngine(model, EngineConfig(num_gpu_blocks=40, max_num_seqs=2, max_model_len=256, max_tokens=4,
                                        use_graphs=False, kv_bits=4), leader, worker)
    worker.register_layout(eng.pool)
    prompt = _prompts(1, [80], model.cfg.vocab)[0]
    a = _run(eng, Request("a", prompt, max_tokens=4))
    before = [x.clone() for x in _rows(eng.pool, a.block_ids, 64)]
    for _ in range(10):  # the worker reports the offload; the leader registers the blocks
        eng.step()
    with torch.inference_mode():
        eng.pool._flat().fill_(255)
    b = Request("b", prompt, max_tokens=4)
    eng.add_request(b)
    eng.step()
    assert b.num_external_tokens == 64
    while eng.has_unfinished() or eng._delayed:
        eng.step()
    torch.cuda.synchronize()
    for x, y in zip(before, _rows(eng.pool, b.block_ids, 64)):
        assert torch.equal(x, y)
    worker.shutdown()


def test_cached_prefix_is_matched():
    """A second request over a prompt whose blocks are in the pool prefills the rest alone, and leaves them as they are."""
    model = LlamaModel(_cfg(), "cuda", seed=4)
    eng = LLMEngine(model, EngineConfig(num_gpu_blocks=40, max_num_seqs=2, max_model_len=256, max_tokens=4,
                                        use_graphs=False, kv_bits=4, prefix_caching=True))
    prompt = _prompts(1, [80], model.cfg.vocab)[0]
    a = _run(eng, Request("a", prompt, max_tokens=4))
    before = [x.clone() for x in _rows(eng.pool, a.block_ids, 64)]
    prefilled = eng.stats["prefill_tokens"]
    b = _run(eng, Request("b", prompt, max_tokens=4))
    assert b.num_cached_tokens == 64 and eng.stats["prefill_tokens"] - prefilled == 16
    assert b.block_ids[:4] == a.block_ids[:4]
    for x, y in zip(before, _rows(eng.pool, b.block_ids, 64)):
        assert torch.equal(x, y)


def test_more_requests_enter_a_decode_batch_than_one_launch_takes():
    from types import SimpleNamespace as NS

    from kvbm_b200.serving.engine import DecodeBatch

    n = 8200
    batch = DecodeBatch(NS(device=torch.device("cuda", 0)), NS(config=NS(page_size=16)), n + 3, 2, 4, 1, dummy_block=9)
    batch.enter([(i, [i, i + 1][: 1 + i % 2], -1, i % 17, 1) for i in range(n)])
    want = torch.tensor([[i, i + 1 if i % 2 else 9] for i in range(n)] + [[9, 9]] * 3, dtype=torch.int32)
    assert torch.equal(batch.block_table.cpu(), want)
    assert batch.pos.tolist() == [i % 17 for i in range(n)] + [0] * 3
    assert batch.active.tolist() == [1] * n + [0] * 3
