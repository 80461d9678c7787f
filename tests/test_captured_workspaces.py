"""Workspaces that grow keep what a captured launch was given, without a GPU."""

from test_kv4_serving import _model


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
