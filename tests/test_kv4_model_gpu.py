"""The 4-bit cache and the q/k head norms on the model's and the serving engine's paths."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

from kvbm_b200.models.llama import KvPush, LlamaConfig, LlamaModel
from kvbm_b200.ops import kv4_ops, kv_ops
from kvbm_b200.physical.layout import KvBlockLayout, KvLayout, LayoutConfig
from kvbm_b200.serving.engine import EngineConfig, LLMEngine, Request


def _cfg(**kw):
    return LlamaConfig(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=1024,
                       max_position=1024, **kw)


def _check_greedy(model, seq, first, tol):
    ref = model.reference_forward(torch.tensor(seq, device=model.device))
    for pos in range(first - 1, len(seq) - 1):
        row = ref[pos]
        assert float(row[seq[pos + 1]]) >= float(row.max()) - tol * float(row.abs().max()), pos


def _randomise_norms(model):
    g = torch.Generator(device="cuda").manual_seed(7)
    for L in model.layers:
        for k in ("qn", "kn"):
            L[k].copy_(1 + 0.3 * torch.randn(L[k].shape, device="cuda", generator=g))


def test_qk_norm_model_matches_reference():
    """Prefill in two chunks and decode steps of a model with head norms over a 16-bit pool (the bf16 model's
    tolerance of the plain harness)."""
    model = LlamaModel(_cfg(qk_norm=True), "cuda", seed=3)
    _randomise_norms(model)
    pool = model.allocate_pool(16)
    T = 45
    prompt = torch.randint(0, 1024, (T,), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(1))
    ids = torch.tensor([3, 7, 1, 12, 5], dtype=torch.int32, device="cuda")
    model.prefill(prompt[:20], pool, ids)
    tok = model.prefill(prompt[20:], pool, ids, start_pos=20)
    seq = prompt.tolist() + [int(tok)]
    for step in range(5):
        pos = torch.tensor([T + step], dtype=torch.int32, device="cuda")
        nxt = model.decode_step(torch.tensor([seq[-1]], device="cuda"), pos, pool, ids.view(1, -1), pos + 1, splits=2)
        seq.append(int(nxt))
    _check_greedy(model, seq, T, 0.05)


def _copy_as_values(src4, dst16, ids, n):
    """The rows of a 4-bit pool as the bf16 values they stand for, into a 16-bit pool."""
    page = src4.config.page_size
    p = torch.arange(n, device="cuda")
    slots = ids.long()[p // page] * page + p % page
    for l in range(src4.config.num_layers):
        k, v = kv4_ops.kv4_gather(src4.layer_view(l), slots)
        dst16.layer_view(l)[slots // page, 0, slots % page] = k
        dst16.layer_view(l)[slots // page, 1, slots % page] = v
    return slots


def _near(got, want, moved):
    """4-bit rows' values beside the bf16 rows of another computation, whose elements are up to ``moved`` away:
    quantising adds half a step, of a scale up to 2^-7 above a fifteenth of the range, the range taken from the moved
    elements; the values' own rounding to bf16 is at most 2^-8 of the largest."""
    g = want.float().unflatten(-1, (-1, 32))
    moved = moved.unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    top, span = g.abs().amax(-1, keepdim=True), g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
    bound = moved + (span + 2 * moved) / 30 * (1 + 2.0 ** -6) + 2.0 ** -8 * (top + moved) * (1 + 2.0 ** -6)
    assert ((got.float().unflatten(-1, (-1, 32)) - g).abs() <= bound).all()


def _behind_attention(x):
    """How far an element lies from another computation's behind an attention that two kernels computed, or that read
    keys a rounding apart. About a dozen roundings to bf16 lie between (weights, output, projection, residual, norms,
    gate, up, down, qkv), half a step of 2^-8 at most each and in each of the two: up to 24 x 2^-8 < 2^-3 of the
    group's largest element."""
    return x.float().unflatten(-1, (-1, 32)).abs().amax(-1).div(8).repeat_interleave(32, -1)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("order", [KvBlockLayout.OPERATIONAL_NHD, KvBlockLayout.OPERATIONAL_HND])
def test_model_over_a_4_bit_pool(norm, order):
    """A 4-bit pool holds what quantising the 16-bit pool would give; a prefill over its prefix and a decode step
    over it are those of a 16-bit pool that holds the same values."""
    model = LlamaModel(_cfg(qk_norm=norm), "cuda", seed=5)
    if norm:
        _randomise_norms(model)
    p4, p16 = model.allocate_pool(16, block_layout=order, kv_bits=4), model.allocate_pool(16, block_layout=order)
    assert p4.config.bytes_per_block * 256 == p16.config.bytes_per_block * 80
    prompt = torch.randint(0, 1024, (77,), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(2))
    ids = torch.tensor([9, 2, 14, 4, 11, 6], dtype=torch.int32, device="cuda")

    def same_rows(first, last):
        p = torch.arange(first, last, device="cuda")
        s = ids.long()[p // 16] * 16 + p % 16
        for l in range(2):
            a, b = p4.layer_view(l)[s // 16, :, s % 16], p16.layer_view(l)[s // 16, :, s % 16]
            if norm:  # one kernel wrote both
                assert torch.equal(a[:, 0], kv4_ops.pack_rows(b[:, 0], False))
                assert torch.equal(a[:, 1], kv4_ops.pack_rows(b[:, 1], True))
                continue
            # The 16-bit rotation fuses a product and a sum, the 4-bit one rounds both: a pair (a, b) gives
            # a cos - b sin in fp32 within 2^-23 (|a cos| + |b sin|) of each other, and in bf16 within a step of that,
            # 2^-7 of it; a rotation keeps the pair's length, at most sqrt 2 times the row's largest element.
            k = b[:, 0].float()
            far = (2.0 ** -7 * 1.5 * k.abs().amax(-1, keepdim=True)).expand_as(k)
            k4, v4 = kv4_ops.kv4_gather(p4.layer_view(l), s)
            if l == 0:
                _near(k4, b[:, 0], far)
                assert torch.equal(a[:, 1], kv4_ops.pack_rows(b[:, 1], True))
            else:
                _near(k4, b[:, 0], _behind_attention(b[:, 0]))
                _near(v4, b[:, 1], _behind_attention(b[:, 1]))

    t4, t16 = model.prefill(prompt[:50], p4, ids), model.prefill(prompt[:50], p16, ids)
    assert not norm or torch.equal(t4, t16)
    same_rows(0, 50)
    _copy_as_values(p4, p16, ids, 50)
    t4, t16 = model.prefill(prompt[50:], p4, ids, start_pos=50), model.prefill(prompt[50:], p16, ids, start_pos=50)
    assert not norm or torch.equal(t4, t16)  # the same bf16 prefix went into the same attention
    same_rows(50, 77)
    _copy_as_values(p4, p16, ids, 77)
    pos = torch.tensor([77], dtype=torch.int32, device="cuda")
    for p in (p4, p16):
        model.decode_step(t16, pos, p, ids.view(1, -1), pos + 1, splits=2)
    slot = ids[77 // 16].long() * 16 + 77 % 16
    same = slot // 16, 0, slot % 16
    if norm:
        assert torch.equal(p4.layer_view(0)[same], kv4_ops.pack_rows(p16.layer_view(0)[same], False))
    k4, v4 = kv4_ops.kv4_gather(p4.layer_view(1), slot.view(1))
    b = p16.layer_view(1)[slot // 16, :, slot % 16]
    _near(k4[0], b[0], _behind_attention(b[0]))
    _near(v4[0], b[1], _behind_attention(b[1]))


@pytest.mark.parametrize("bits", [4, 16])
def test_decode_steps_of_several_sizes(bits):
    """A captured step keeps its scratch when a larger step needs more; a table may have more rows than the batch."""
    model = LlamaModel(_cfg(), "cuda", seed=8)
    pool = model.allocate_pool(128, kv_bits=bits)
    g = torch.Generator("cuda").manual_seed(4)
    prompt = torch.randint(0, 1024, (300,), device="cuda", dtype=torch.int32, generator=g)
    ids = torch.arange(32, dtype=torch.int32, device="cuda")
    model.prefill(prompt, pool, ids)
    table = F.pad(ids, (0, 224)).repeat(40, 1)  # wide enough for requests that are cut
    tok, pos = torch.full((1,), 7, device="cuda"), torch.full((1,), 299, dtype=torch.int32, device="cuda")

    def step(B, rows):
        return model.decode_step(tok.expand(B).contiguous(), pos.expand(B).contiguous(), pool, table[:rows],
                                 pos.expand(B) + 1, splits=4)

    eager = step(1, 1)
    assert torch.equal(step(1, 40), eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(1, 1)
        with torch.cuda.graph(graph, stream=side):
            got = step(1, 1)
    torch.cuda.current_stream().wait_stream(side)
    small = model._decode_scratch
    step(40, 40)
    assert model._decode_scratch.numel() > small.numel() and any(s is small for s in model._outgrown)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, eager)


def test_4_bit_pools_refuse_what_they_cannot_do():
    model = LlamaModel(_cfg(), "cuda", seed=1)
    p4, p16 = model.allocate_pool(4, kv_bits=4), model.allocate_pool(4)
    ids = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="16-bit pools"):
        model.prefill(tok, p4, ids, kv_push=KvPush(p16, ids))
    with pytest.raises(ValueError, match="bf16 pools"):
        KvPush(p4, ids)
    with pytest.raises(ValueError, match="kv_bits"):
        model.allocate_pool(4, kv_bits=8)
    with pytest.raises(ValueError, match="not cast"):
        kv_ops.kv_transfer(p4, [0], p16, [0])
    with pytest.raises(ValueError, match="head_dim"):
        LlamaConfig(head_dim=96).kv_layout_config(4, dtype=torch.uint8)


@pytest.mark.parametrize("engine", ["tile", "tma", "auto"])
def test_4_bit_pools_move_between_tiers_and_layouts(engine):
    cfg = LayoutConfig.for_model(8, 3, 4, kv4_ops.row_bytes(128), 16, torch.uint8)
    g1 = KvLayout.allocate(cfg, "fully_contiguous", KvBlockLayout.OPERATIONAL_NHD)
    hnd = KvLayout.allocate(cfg, "layer_separate", KvBlockLayout.OPERATIONAL_HND, zero=True)
    g2 = KvLayout.allocate(cfg, "fully_contiguous", KvBlockLayout.OPERATIONAL_NHD, location="pinned", zero=True)
    back = KvLayout.allocate(cfg, "fully_contiguous", KvBlockLayout.OPERATIONAL_NHD, zero=True)
    g1._flat().random_(0, 256)
    kv_ops.kv_transfer(g1, [1, 4, 6], hnd, [0, 7, 3], engine=engine)
    kv_ops.kv_transfer(g1, [1, 4, 6], g2, [2, 5, 0], engine=engine)
    kv_ops.kv_transfer(g2, [2, 5, 0], back, [6, 1, 4], engine=engine)
    torch.cuda.synchronize()
    for l in range(3):
        a = g1.layer_view(l)
        assert torch.equal(hnd.layer_view(l)[[0, 7, 3]], a[[1, 4, 6]])
        assert torch.equal(back.layer_view(l)[[6, 1, 4]], a[[1, 4, 6]])
    # a tensor-parallel rank's heads
    half = KvLayout.allocate(LayoutConfig.for_model(8, 3, 2, kv4_ops.row_bytes(128), 16, torch.uint8),
                             "fully_contiguous", KvBlockLayout.OPERATIONAL_NHD, zero=True)
    kv_ops.kv_transfer(g1, [3], half, [5], src_head_offset=2, num_heads=2, engine="tile")
    torch.cuda.synchronize()
    for l in range(3):
        assert torch.equal(half.layer_view(l)[5], g1.layer_view(l)[3][:, :, 2:])


@pytest.mark.parametrize("graphs", [False, True])
def test_serving_engine_with_a_4_bit_pool(graphs):
    """Requests of several lengths through prefill chunks and a decode batch; near-greedy against the reference with
    a quantised cache's tolerance: 4 bits in groups of 32 move a normal element by 0.27 / sqrt(12) = 8 % of its
    standard deviation, four times the 2 % (2^-8 times some rounding steps) that the bf16 harness is given 5 % for."""
    model = LlamaModel(_cfg(), "cuda", seed=6)
    eng = LLMEngine(model, EngineConfig(num_gpu_blocks=64, max_num_seqs=4, max_num_batched_tokens=48, max_model_len=256,
                                        max_tokens=8, use_graphs=graphs, kv_bits=4))
    assert eng.pool.dtype == torch.uint8
    eng.warmup()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1024, (n,), generator=g, dtype=torch.int32).pin_memory() for n in (5, 16, 61, 100, 33, 2)]
    reqs = [Request(f"r{i}", p, max_tokens=6) for i, p in enumerate(prompts)]
    for r in reqs:
        eng.add_request(r)
    for _ in range(100):
        if not eng.has_unfinished():
            break
        eng.step()
    torch.cuda.synchronize()
    assert not eng.has_unfinished()
    for p, r in zip(prompts, reqs):
        _check_greedy(model, p.tolist() + r.output.tolist(), len(p), 0.2)
    eng.release_graphs()
