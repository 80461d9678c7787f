"""What surrounds the 4-bit cache's operators in the model harness and the serving stack, without a GPU."""

import pytest
import torch

from kvbm_b200.models.llama import LlamaConfig, LlamaModel


def _model():
    """The harness without its weights: what its bookkeeping needs, on the CPU."""
    m = object.__new__(LlamaModel)
    m.cfg = LlamaConfig(hidden=64, layers=1, heads=2, kv_heads=1, head_dim=64, intermediate=64, vocab=16)
    m.device = torch.device("cpu")
    m._decode_scratch, m._outgrown, m._scratch_captured, m._scratch_stream = None, [], False, None
    m._decode_counters, m._counters_captured = None, False
    return m


def test_scratch_of_growing_batches_is_let_go():
    m, made = _model(), set()
    for batch in range(1, 257):
        s = m.decode_scratch(batch, 4)
        assert s.numel() >= batch * 2 * 4 * 66
        made.add(s.data_ptr())
        assert m.decode_scratch(1, 4) is s  # a smaller step uses the same
    assert m._outgrown == [] and len(made) < 20
    assert m._decode_scratch.numel() <= 1.5 * 256 * 2 * 4 * 66


def test_scratch_of_a_captured_step_is_kept():
    m = _model()
    m.decode_scratch(1, 1)
    m._capturing = lambda: True
    mine = m.decode_scratch(1, 1)
    m._capturing = lambda: False
    for batch in range(2, 200):
        m.decode_scratch(batch, 1)
    assert [s is mine for s in m._outgrown] == [True]


class _Pool:
    dtype = torch.uint8


class _FakeModel:
    """The engine's view of a model, on the CPU."""

    device = torch.device("cpu")

    class cfg:
        kv_heads, heads, head_dim, layers = 2, 4, 64, 1

    def allocate_pool(self, n, page, kv_bits=16):
        assert kv_bits == 4
        return _Pool()

    def prefill(self, tokens, pool, ids, **kw):
        return torch.tensor([7])

    def decode_step(self, tok, pos, *a):
        return pos.long() % 100


def _engine(monkeypatch, **kw):
    from test_serving_engine_cpu import FakeEvent, FakeStream

    from kvbm_b200.serving import engine as E

    monkeypatch.setattr(torch.cuda, "Event", FakeEvent)
    monkeypatch.setattr(torch.cuda, "Stream", FakeStream)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    monkeypatch.setattr(E.llama_ops, "decode_splits", lambda *a, **k: 1)
    return E, E.LLMEngine(_FakeModel(), E.EngineConfig(num_gpu_blocks=8, max_num_seqs=2, max_model_len=64, max_tokens=4,
                                                       use_graphs=False, kv_bits=4), **kw)


def test_engine_raises_when_an_attention_launch_gave_up(monkeypatch):
    """The status is read in every step: NaN does not go on as tokens."""
    from kvbm_b200.ops import _lib

    class Lib:
        status = 0

        def kvbm_kv4_status(self, device, reset):
            was, self.status = self.status, 0 if reset else self.status
            return was

        kvbm_error_string = None

    lib = Lib()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    E, eng = _engine(monkeypatch)
    eng.add_request(E.Request("a", torch.arange(5, dtype=torch.int32), max_tokens=4))
    eng.step()
    lib.status = 3
    with pytest.raises(_lib.KvbmCudaError, match="status 3"):
        eng.step()
    eng.step()
    lib.status = 3
    with pytest.raises(_lib.KvbmCudaError, match="status 3"):
        eng.check()


def test_engine_refuses_a_16_bit_pool_for_4_bits(monkeypatch):
    from kvbm_b200.serving import engine as E

    _engine(monkeypatch)
    pool = _Pool()
    cfg = dict(num_gpu_blocks=8, max_num_seqs=2, max_model_len=64, max_tokens=4, use_graphs=False)
    for bits in (4, 16):  # a pool that is passed in says what it holds
        assert E.LLMEngine(_FakeModel(), E.EngineConfig(kv_bits=bits, **cfg), pool=pool).pool is pool
    pool.dtype = torch.bfloat16
    with pytest.raises(ValueError, match="kv_bits"):
        E.LLMEngine(_FakeModel(), E.EngineConfig(kv_bits=4, **cfg), pool=pool)
    with pytest.raises(ValueError, match="kv_bits"):
        E.LLMEngine(_FakeModel(), E.EngineConfig(kv_bits=8, **cfg), pool=pool)


def test_fp8_on_the_wire_is_refused_for_a_pool_of_bytes():
    """At setup, not with the first push in the middle of a request."""
    from kvbm_b200.connector.worker import ConnectorWorker

    w = object.__new__(ConnectorWorker)
    w.g1 = _Pool()
    with pytest.raises(ValueError, match="wire_dtype"):
        w.enable_disagg(1, None, mailbox_slots=4, wire_dtype="fp8")


def test_disaggregation_in_4_bits_counts_its_bytes():
    from kvbm_b200.serving.pd import PdConfig

    model = LlamaConfig(hidden=64, layers=3, heads=4, kv_heads=2, head_dim=128, intermediate=64, vocab=16)
    a, b = PdConfig(model=model, prompt_len=40), PdConfig(model=model, prompt_len=40, kv_bits=4)
    assert a.kv_bytes_per_request() == 3 * 3 * 2 * 16 * 2 * 256 and b.kv_bytes_per_request() == 3 * 3 * 2 * 16 * 2 * 80
    with pytest.raises(ValueError, match="kv_bits"):
        PdConfig(kv_bits=8)
    with pytest.raises(ValueError, match="wire_dtype"):
        PdConfig(kv_bits=4, wire_dtype="fp8")


def test_prefill_refuses_too_few_blocks():
    class Pool:
        dtype = torch.bfloat16

        class config:
            page_size = 16

    m, ids = _model(), torch.tensor([3, 1], dtype=torch.int32)
    for start, n in ((0, 33), (30, 3), (32, 1)):
        with pytest.raises(ValueError, match="do not hold"):
            m.prefill(torch.zeros(n, dtype=torch.int32), Pool(), ids, start_pos=start)
