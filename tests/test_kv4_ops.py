"""The 4-bit cache's row format and the refusals of its operators, without a GPU."""

import math

import pytest
import torch

from kvbm_b200.ops import kv4_ops, table_ops

BF = torch.bfloat16


@pytest.mark.parametrize("hd,row", [(64, 48), (128, 80), (256, 160)])
def test_row_bytes(hd, row):
    assert kv4_ops.row_bytes(hd) == row and row % 16 == 0


@pytest.mark.parametrize("value", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_hold_every_element_within_half_a_step(hd, value):
    g = torch.Generator().manual_seed(hd + value)
    x = (torch.randn(50, 3, hd, generator=g) * torch.logspace(-3, 3, 50)[:, None, None]).to(BF)
    x[7] = 1.5  # a group of equal values is exact
    rows = kv4_ops.pack_rows(x, value)
    assert rows.shape == (50, 3, kv4_ops.row_bytes(hd)) and rows.dtype == torch.uint8
    back = kv4_ops.unpack_rows(rows, value).double().unflatten(-1, (-1, 32))
    ref = x.double().unflatten(-1, (-1, 32))
    span = ref.amax(-1) - ref.amin(-1)
    # scale = span / 15 rounded up to bf16 (8 bits: by at most 2^-7), the element within half of it, and the
    # fp32 product and sum round by 2^-24 of at most 15 scale and the largest element
    step = span / 15 * (1 + 2.0 ** -7)
    bound = step / 2 + 2.0 ** -23 * (span + ref.abs().amax(-1))
    assert ((back - ref).abs() <= bound.unsqueeze(-1)).all()
    assert torch.equal(back[7], ref[7])
    low = ref.argmin(-1, keepdim=True)  # the least element is exact
    assert torch.equal(back.gather(-1, low), ref.gather(-1, low))


def test_rows_keep_code_order():
    x = torch.arange(128).remainder(16).to(BF).expand(1, 128).clone()
    x[0, ::32], x[0, 15::32] = 0, 15
    k, v = kv4_ops.pack_rows(x, False)[0], kv4_ops.pack_rows(x, True)[0]
    for d in range(128):
        g, b, i = d // 32, d % 32 // 4, d % 4
        n = 4 * (4 * b + g) + i
        assert (int(k[d // 2]) >> (4 * (d % 2))) & 15 == d % 16
        assert (int(v[n // 2]) >> (4 * (n % 2))) & 15 == d % 16


def test_rows_with_infinities_and_extremes():
    big = torch.finfo(BF).max
    x = torch.zeros(5, 64, dtype=BF)
    x[0, 3], x[1, 40], x[2, 5] = math.inf, math.nan, -math.inf
    x[3, :32] = torch.linspace(-1, 1, 32).to(BF) * big
    x[4, :32] = 2.0 ** -130
    back = kv4_ops.unpack_rows(kv4_ops.pack_rows(x, True), True)
    assert back[0, :32].isnan().all() and (back[0, 32:] == 0).all()
    assert back[1, 32:].isnan().all() and back[2, :32].isnan().all()
    assert back[3].isfinite().all() and float((back[3] - x[3].float()).abs().max()) <= big / 15 * (1 + 2.0 ** -6)
    assert torch.equal(back[4], x[4].float())


def _pool(nb=4, page=16, heads=2, row=80, dtype=torch.uint8):
    return torch.zeros(nb, 2, page, heads, row, dtype=dtype)


def _write_args(T=3, hq=4, hkv=2, hd=128, **kw):
    a = dict(qkv=torch.zeros(T, hq + 2 * hkv, hd, dtype=BF), positions=torch.zeros(T, dtype=torch.int32),
             cos_sin=torch.zeros(32, hd), hq=hq, hkv=hkv, kv=_pool(heads=hkv, row=kv4_ops.row_bytes(hd) if hd in
                                                                  (64, 128, 256) else 80),
             slots=torch.zeros(T, dtype=torch.int64))
    return {**a, **kw}


@pytest.mark.parametrize("change,message", [
    (dict(qkv=torch.zeros(3, 8, 128)), "bf16"),
    (dict(hq=5), "8 heads"),
    (dict(hd=96), "head_dim"),
    (dict(qkv=torch.zeros(3, 128, 8, dtype=BF).transpose(1, 2)), "contiguous heads"),
    (dict(qkv=torch.zeros(1, 8, 128, dtype=BF).expand(3, 8, 128)), "overlap"),
    (dict(kv=_pool(row=48)), "cache holds"),
    (dict(kv=_pool(heads=1)), "cache holds"),
    (dict(kv=_pool(row=128, dtype=torch.float16)), "4-bit cache"),
    (dict(kv=_pool()[:, 0]), "num_blocks, 2, page"),
    (dict(kv=_pool(row=96)[..., :80][..., ::1][:, :, :, :, 8:]), "aligned|cache holds"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "slots"),
    (dict(cos_sin=torch.zeros(32, 24)), "rot"),
    (dict(cos_sin=torch.zeros(32, 144)), "rot"),
    (dict(q_weight=torch.zeros(64, dtype=BF)), "q_weight"),
    (dict(k_weight=torch.zeros(128)), "k_weight"),
    (dict(k_out=torch.zeros(3, 2, 128, dtype=BF)), "k_out needs q_out"),
    (dict(q_out=torch.zeros(3, 2, 128, dtype=BF)), "q_out"),
    ({}, "CUDA tensors"),
])
def test_write_refusals(change, message):
    hd = change.pop("hd", 128)
    with pytest.raises(ValueError, match=message):
        kv4_ops.qk_norm_rope_kv_write(**{**_write_args(hd=hd), **change})


def _attn_args(**kw):
    a = dict(q=torch.zeros(2, 8, 128, dtype=BF), kv=_pool(), block_table=torch.zeros(2, 3, dtype=torch.int32),
             seq_lens=torch.zeros(2, dtype=torch.int32), softmax_scale=1.0)
    return {**a, **kw}


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(2, 8, 128)), "bf16"),
    (dict(q=torch.zeros(2, 7, 128, dtype=BF)), "multiple"),
    (dict(q=torch.zeros(2, 8, 64, dtype=BF)), "do not hold"),
    (dict(q=torch.zeros(2, 128, 8, dtype=BF).transpose(1, 2)), "contiguous heads"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), "block_table"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "seq_lens"),
    (dict(ctas=-1), "ctas"),
    (dict(scratch=torch.zeros(10, dtype=torch.float64)), "scratch"),
    (dict(out=torch.zeros(2, 8, 64, dtype=BF)), "out"),
    ({}, "CUDA tensors"),
])
def test_attention_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        kv4_ops.paged_decode_attn_kv4(**_attn_args(**change))


@pytest.mark.parametrize("change,message", [
    (dict(kv=_pool(row=64)), "rows of 48"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots"),
    (dict(k_out=torch.zeros(3, 2, 64, dtype=BF)), "k_out"),
    ({}, "CUDA tensors"),
])
def test_gather_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        kv4_ops.kv4_gather(**{**dict(kv=_pool(), slots=torch.zeros(3, dtype=torch.int64)), **change})


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("change,message", [
    (dict(query_lens=torch.tensor([1, 2])), "query_lens"),
    (dict(context_lens=_i32(1)), "context_lens"),
    (dict(block_ids=torch.zeros(2, 2, dtype=torch.int32)), "block_ids"),
    (dict(block_counts=_i32(1, 2, 3)), "block_counts"),
    (dict(page=0), "page"),
    (dict(num_tokens=-1), "num_tokens"),
    (dict(max_blocks=None), "max_blocks"),
    (dict(rows=_i32(0, 1)), "rows"),
    (dict(table=torch.zeros(1, 4, dtype=torch.int32)), "1 rows for 2"),
    (dict(table=torch.zeros(2, 5, dtype=torch.int32)), "differs"),
    (dict(table=torch.zeros(2, 4)), "block table"),
    (dict(query_lens=torch.zeros(8193, dtype=torch.int32), context_lens=torch.zeros(8193, dtype=torch.int32)), "8192"),
    ({}, "CUDA tensors"),
])
def test_table_refusals(change, message):
    a = dict(query_lens=_i32(1, 2), context_lens=_i32(0, 5), block_ids=_i32(0, 1, 2), page=16, max_blocks=4)
    with pytest.raises(ValueError, match=message):
        table_ops.batch_tables(**{**a, **change})


@pytest.mark.parametrize("change,message", [
    (dict(positions=torch.zeros(2)), "positions"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "3 rows for 2"),
    (dict(block_table=torch.zeros(2, 4)), "block table"),
    (dict(page=0), "page"),
    (dict(out=torch.zeros(3, dtype=torch.int64)), "out"),
    ({}, "CUDA tensors"),
])
def test_slot_map_refusals(change, message):
    a = dict(block_table=torch.zeros(2, 4, dtype=torch.int32), positions=_i32(1, 2), page=16)
    with pytest.raises(ValueError, match=message):
        table_ops.slot_map(**{**a, **change})
