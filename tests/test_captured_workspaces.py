"""Workspaces that grow keep what a captured launch was given, without a GPU."""

from test_kv4_serving import _model

from kvbm_b200.ops import _lib, llama_ops


def test_a_captured_step_keeps_its_tickets():
    m = _model()
    m.decode_counters(2)
    m._capturing = lambda: True
    mine = m.decode_counters(2)
    assert m.decode_counters(2) is mine
    own = m.decode_counters(5)  # more than there are: the graph's, and nobody else's
    assert own.numel() >= 5 and own is not mine and m._decode_counters is mine
    m._capturing = lambda: False
    more = m.decode_counters(9)
    assert more is not own and more.numel() >= 9 and not more.any()
    assert any(t is mine for t in m._outgrown)
    m.decode_counters(30)
    assert len(m._outgrown) == 1  # `more` was never captured


def test_a_captured_step_that_needs_more_scratch_gets_its_own():
    m = _model()
    m.decode_scratch(1, 1)
    before = m._decode_scratch
    m._capturing = lambda: True
    assert m.decode_scratch(50, 4).numel() >= 50 * 2 * 4 * 66
    assert m._decode_scratch is before and not m._outgrown


def test_a_captured_gemm_keeps_its_workspace(monkeypatch):
    w = llama_ops.GemmWorkspace("cpu")
    w.reserve(100, 3)
    monkeypatch.setattr(_lib, "capturing", lambda device: True)
    ws, tickets = w.reserve(90, 2)
    assert ws is w.ws and tickets is w.tickets
    own = w.reserve(500, 3)
    assert own[0].numel() >= 500 and w.ws is ws and w.tickets is tickets
    monkeypatch.setattr(_lib, "capturing", lambda device: False)
    more = w.reserve(100, 7)
    assert more[1].numel() >= 7 and more[0].numel() >= 100 and not more[0].any() and not more[1].any()
    assert any(t is ws for t in w._kept) and any(t is tickets for t in w._kept)
    w.reserve(1000, 20)
    assert len(w._kept) == 2
