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
