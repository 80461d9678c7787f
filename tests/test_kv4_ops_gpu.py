"""GPU numerics of the 4-bit cache's operators against plain forms in 64 bits."""

import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

from kvbm_b200.ops import _lib, kv4_ops, table_ops
from kvbm_b200.physical.layout import KvBlockLayout, KvLayout, LayoutConfig

BF = torch.bfloat16
HALF_STEP = 2.0 ** -8  # of a bf16, relative


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _empty_pool(nb, page, heads, hd, bits=4, order="nhd", fill=0):
    width, dtype = (kv4_ops.row_bytes(hd), torch.uint8) if bits == 4 else (hd, BF)
    if order == "hnd":
        return torch.full((nb, 2, heads, page, width), fill, dtype=dtype, device="cuda").transpose(2, 3)
    return torch.full((nb, 2, page, heads, width), fill, dtype=dtype, device="cuda")


# ------------------------------------------------------------------ tables


def _plain_tables(q, c, ids, page, max_blocks, T, counts=None, pad=0):
    table, seq, cu, pos, slots = [], [], [0], [], []
    at = 0
    for b in range(len(q)):
        qb, cb = max(q[b], 0), max(c[b], 0)
        n = max(counts[b], 0) if counts is not None else -(-(qb + cb) // page)
        mine = ids[at: at + n][:max_blocks]
        at += n
        table.append(mine + [pad] * (max_blocks - len(mine)))
        seq.append(qb + cb)
        cu.append(cu[-1] + qb)
        for p in range(cb, cb + qb):
            pos.append(p)
            ok = p // page < len(mine) and mine[p // page] >= 0
            slots.append(mine[p // page] * page + p % page if ok else -1)
    pos, slots = pos[:T], slots[:T]
    return table, seq, cu, pos + [0] * (T - len(pos)), slots + [-1] * (T - len(slots))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("q,c,page,max_blocks,T,counts,n_ids", [
    ([], [], 16, 4, 5, None, 0),                              # no request at all
    ([1], [0], 16, 1, 1, None, 1),
    ([0, 0, 3], [0, 33, 0], 16, 4, 7, None, 4),               # nothing new, an empty one, a padded batch
    ([5, -2, 17], [-4, 16, 15], 16, 3, 22, None, 5),          # negative lengths count as 0
    ([40, 9], [100, 3], 16, 4, 49, None, 20),                 # 9 blocks needed, a table of 4
    ([40, 9], [100, 3], 16, 16, 20, None, 20),                # fewer places than tokens
    ([4, 4, 4], [60, 0, 12], 16, 8, 12, [2, 5, 1], 8),        # reserved ahead, and too few
    ([4, 4, 4], [60, 0, 12], 1, 70, 12, None, 70),            # ids run out
    ([7] * 300, list(range(300)), 32, 12, 2200, None, 3000),  # more requests than threads
    ([3000, 1, 1], [1, 5000, 0], 128, 64, 3002, None, 80),
])
def test_batch_tables(q, c, page, max_blocks, T, counts, n_ids):
    ids = torch.randperm(max(n_ids, 1), generator=torch.Generator().manual_seed(n_ids))[:n_ids].tolist()
    if n_ids > 3:
        ids[2] = -1  # a block that is not there
    got = table_ops.batch_tables(_i32(q), _i32(c), _i32(ids), page=page, max_blocks=max_blocks, num_tokens=T,
                                 block_counts=_i32(counts) if counts else None, pad_block=9)
    want = _plain_tables(q, c, ids, page, max_blocks, T, counts, pad=9)
    for g, w, name in zip(got, want, got._fields):
        assert g.tolist() == w, name


def test_batch_tables_into_rows_of_a_persistent_table():
    table = torch.full((6, 8), -7, dtype=torch.int32, device="cuda")[:, :5]  # strided rows
    got = table_ops.batch_tables(_i32([1, 2, 1]), _i32([16, 0, 3]), _i32([4, 5, 6, 7]), page=16, num_tokens=4,
                                 table=table, rows=_i32([4, 1, 99]), pad_block=2)
    assert got.block_table.data_ptr() == table.data_ptr()
    assert table.tolist() == [[-7] * 5, [6, 2, 2, 2, 2], [-7] * 5, [-7] * 5, [4, 5, 2, 2, 2], [-7] * 5]
    assert got.slots.tolist() == [80, 96, 97, 115]


@pytest.mark.parametrize("B", [1, 256, 8192])
def test_batch_tables_largest_batches(B):
    g = torch.Generator().manual_seed(B)
    q = torch.randint(0, 3, (B,), generator=g).tolist()
    c = torch.randint(0, 40, (B,), generator=g).tolist()
    n = sum(-(-(a + b) // 16) for a, b in zip(q, c))
    ids = torch.randperm(n + 1, generator=g)[:n].tolist()
    got = table_ops.batch_tables(_i32(q), _i32(c), _i32(ids), page=16, max_blocks=3, num_tokens=sum(q) + 3)
    for a, w in zip(got, _plain_tables(q, c, ids, 16, 3, sum(q) + 3)):
        assert a.tolist() == w


@pytest.mark.parametrize("page", [1, 16, 64])
def test_slot_map(page):
    table = torch.randperm(7 * 9, generator=torch.Generator().manual_seed(page)).int().view(7, 9).cuda()
    table[2, 0] = -1
    pos = _i32([0, 5 * page, 0, 9 * page, -1, 9 * page - 1, 2 ** 31 - 1])
    want = [int(table[i, p // page]) * page + p % page if 0 <= p < 9 * page and int(table[i, p // page]) >= 0 else -1
            for i, p in enumerate(pos.tolist())]
    assert table_ops.slot_map(table, pos, page=page).tolist() == want
    one = table_ops.slot_map(table[3], torch.arange(9 * page, dtype=torch.int32, device="cuda"), page=page)
    assert one.tolist() == [int(table[3, p // page]) * page + p % page for p in range(9 * page)]
    wide = torch.zeros(7, 20, dtype=torch.int32, device="cuda")
    wide[:, :9] = table
    assert table_ops.slot_map(wide[:, :9], pos, page=page).tolist() == want
    assert table_ops.slot_map(table[:0], pos[:0], page=page).numel() == 0


# ------------------------------------------------------------------- write


def _cos_sin(n, rot):
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    f = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    return torch.cat([f.cos(), f.sin()], -1).float().cuda()


def _heads64(qkv, pos, cs, hq, hkv, qw, kw, eps):
    """Normalised and rotated q and k in 64 bits, and the size the rotation's rounding is relative to."""
    rot = cs.shape[1]
    x = qkv.double()
    c, s = cs.double()[pos.long()][:, None, : rot // 2], cs.double()[pos.long()][:, None, rot // 2:]

    def turn(y, w):
        if w is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        out = torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1)
        size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), y[..., rot:].abs()], -1)
        return out, size

    return turn(x[:, :hq], qw), turn(x[:, hq: hq + hkv], kw)


def _close(got, want, size):
    # one rounding to bf16, after about a dozen in fp32 relative to the terms' sizes (128 squares summed in a
    # tree of 3 + log2 steps, a root, a quotient, two products and a sum): below 2^-19 of them
    err = (got.double() - want).abs()
    assert (err <= HALF_STEP * want.abs() + 2.0 ** -19 * size + 2.0 ** -133).all(), float(err.max())


@pytest.mark.parametrize("T,hq,hkv,hd,rot,page,bits,order,norm,out", [
    (1, 32, 8, 128, 128, 16, 4, "nhd", True, "q"),
    (50, 8, 2, 128, 128, 16, 4, "hnd", True, None),
    (33, 5, 1, 64, 32, 32, 4, "nhd", True, "qk"),
    (19, 3, 3, 256, 256, 1, 4, "hnd", True, "qk"),
    (70, 7, 3, 128, 48, 64, 16, "hnd", True, "qk"),
    (21, 4, 2, 256, 128, 16, 16, "nhd", "k", None),
    (9, 0, 4, 64, 64, 16, 4, "nhd", "q", None),
    (300, 12, 2, 128, 128, 16, 4, "nhd", False, "q"),
    (17, 1, 1, 64, 16, 16, 16, "nhd", True, None),
])
def test_qk_norm_rope_kv_write(T, hq, hkv, hd, rot, page, bits, order, norm, out):
    g = _gen(T * hd)
    nb = -(-T // page) + 2
    kv = _empty_pool(nb, page, hkv, hd, bits, order, fill=3)
    before = kv.clone()
    wide = torch.randn(T, (hq + 2 * hkv) * hd + 24, device="cuda", generator=g).to(BF)  # rows with a gap behind them
    qkv = wide[:, : (hq + 2 * hkv) * hd].view(T, hq + 2 * hkv, hd)
    orig = wide.clone()
    pos = torch.randint(0, 500, (T,), device="cuda", generator=g).int()
    slots = torch.randperm(nb * page, device="cuda", generator=g)[:T]
    cs = _cos_sin(500, rot)
    qw = (1 + 0.3 * torch.randn(hd, device="cuda", generator=g)).to(BF) if norm in (True, "q") else None
    kw = (1 + 0.3 * torch.randn(hd, device="cuda", generator=g)).to(BF) if norm in (True, "k") else None
    if T > 8:
        pos[3] = 500      # outside the table: left alone
        pos[4] = -1
        slots[5] = -1     # not written
        slots[6] = nb * page
    o = orig[:, : (hq + 2 * hkv) * hd].view(T, hq + 2 * hkv, hd)
    (q64, q_size), (k64, k_size) = _heads64(o, pos.clamp(0, 499), cs, hq, hkv, qw, kw, 1e-6)
    q_out = torch.full((T, hq, hd), 5.0, device="cuda", dtype=BF) if out else None
    k_out = torch.full((T, hkv, hd), 5.0, device="cuda", dtype=BF) if out == "qk" else None
    kv4_ops.qk_norm_rope_kv_write(qkv, pos, cs, hq, hkv, kv, slots, q_weight=qw, k_weight=kw, eps=1e-6, q_out=q_out,
                                  k_out=k_out)
    torch.cuda.synchronize()
    live = torch.ones(T, dtype=torch.bool, device="cuda")
    if T > 8:
        live[3:5] = False
    if out:
        assert torch.equal(wide, orig)
        assert (q_out[~live] == 5).all() and (k_out is None or (k_out[~live] == 5).all())
        q, k = q_out, k_out
    else:
        assert torch.equal(wide[:, (hq + 2 * hkv) * hd:], orig[:, (hq + 2 * hkv) * hd:])
        assert torch.equal(qkv[:, hq + hkv:], o[:, hq + hkv:]) and torch.equal(qkv[~live], o[~live])
        q, k = qkv[:, :hq], qkv[:, hq: hq + hkv]
    _close(q[live], q64[live], q_size[live])
    if k is not None:
        _close(k[live], k64[live], k_size[live])
    stored = live.clone()
    if T > 8:
        stored[5:7] = False
    s = slots[stored]
    touched = torch.zeros(nb, page, dtype=torch.bool, device="cuda")
    touched[s // page, s % page] = True
    keep = ~touched[:, None, :, None, None].expand_as(kv)
    assert torch.equal(kv[keep], before[keep])  # every other row is as it was
    rows_k, rows_v = kv[s // page, 0, s % page], kv[s // page, 1, s % page]
    v = o[stored][:, hq + hkv:]
    if bits == 16:
        assert torch.equal(rows_v, v)
        _close(rows_k, k64[stored], k_size[stored])
        assert k is None or torch.equal(rows_k, k[stored])
    else:
        assert torch.equal(rows_v, kv4_ops.pack_rows(v, True))
        if k is not None:
            assert torch.equal(rows_k, kv4_ops.pack_rows(k[stored], False))
        else:
            back = kv4_ops.unpack_rows(rows_k, False).double()
            span = (k64[stored].unflatten(-1, (-1, 32)).amax(-1) - k64[stored].unflatten(-1, (-1, 32)).amin(-1))
            # half a step of the rounded-up scale, and the bf16 rounding of the element and of the range's ends
            bound = span / 30 * (1 + 2.0 ** -7) + 2.0 ** -7 * k64[stored].unflatten(-1, (-1, 32)).abs().amax(-1)
            err = (back - k64[stored]).abs().unflatten(-1, (-1, 32)).amax(-1)
            assert (err <= bound).all()


def test_write_poisoned_and_constant_groups():
    hkv, hd, page = 2, 128, 16
    kv = _empty_pool(2, page, hkv, hd)
    x = torch.randn(8, 3 * hkv, hd, device="cuda", generator=_gen(1)).to(BF)
    x[0, 4, 3], x[1, 5, 40], x[2, 4, 127] = math.inf, math.nan, -math.inf
    x[3, 4] = 0.75
    x[4, 4] = 0.0
    x[5, 4, :32] = torch.linspace(-1, 1, 32).to(BF) * 1e38
    x[6, 4] = torch.finfo(BF).tiny / 4
    kv4_ops.qk_norm_rope_kv_write(x.clone(), torch.zeros(8, dtype=torch.int32, device="cuda"), _cos_sin(1, hd), hkv, hkv,
                                  kv, torch.arange(8, device="cuda"))
    assert torch.equal(kv[0, 1, :8], kv4_ops.pack_rows(x[:, 2 * hkv:], True))
    k, v = kv4_ops.kv4_gather(kv, torch.arange(8, device="cuda"))
    assert v[0, 0, :32].isnan().all() and v[0, 0, 32:].isfinite().all()
    assert torch.equal(v[3, 0], x[3, 4]) and torch.equal(v[4, 0], x[4, 4]) and torch.equal(v[6, 0], x[6, 4])


@pytest.mark.parametrize("order", ["nhd", "hnd"])
@pytest.mark.parametrize("T,heads,hd,page", [(0, 2, 64, 16), (1, 1, 64, 1), (77, 8, 128, 16), (130, 3, 256, 32)])
def test_gather(T, heads, hd, page, order):
    nb = -(-T // page) + 1
    kv = _empty_pool(nb, page, heads, hd, order=order)
    x = torch.randn(nb, 2, page, heads, hd, device="cuda", generator=_gen(T)).to(BF)
    kv[:, 0], kv[:, 1] = kv4_ops.pack_rows(x[:, 0], False), kv4_ops.pack_rows(x[:, 1], True)
    slots = torch.randint(0, nb * page, (T,), device="cuda", generator=_gen(T + 1))  # repeats allowed
    if T > 3:
        slots[1], slots[2] = -1, nb * page
    k, v = kv4_ops.kv4_gather(kv, slots)
    ok = (slots >= 0) & (slots < nb * page)
    s = slots[ok]
    for got, o in ((k, 0), (v, 1)):
        rows = kv[s // page, o, s % page]
        assert torch.equal(got[ok], kv4_ops.unpack_rows(rows, bool(o)).to(BF))
        assert not got[~ok].any() and got.shape == (T, heads, hd)


# --------------------------------------------------------------- attention


def _filled(B, lens, heads, hd, page, order="nhd", seed=0, spread=1.0):
    """A pool whose live rows hold data and all others 0xff, its table, and the values in 64 bits."""
    nb = max(1, -(-max(max(lens), 1) // page))
    kv = _empty_pool(B * nb + 2, page, heads, hd, order=order, fill=255)
    g = _gen(seed)
    table = (torch.randperm(B * nb, device="cuda", generator=g) + 2).int().view(B, nb)
    x = torch.randn(B, nb * page, 2, heads, hd, device="cuda", generator=g)
    x[..., 5] *= 4 * spread
    x[:, :, 1] += 0.3
    x = x.to(BF)
    vals = []
    for b in range(B):
        rk, rv = kv4_ops.pack_rows(x[b, :, 0], False), kv4_ops.pack_rows(x[b, :, 1], True)
        for j in range(-(-lens[b] // page)):
            n = min(page, lens[b] - j * page)
            kv[int(table[b, j]), 0, :n] = rk[j * page: j * page + n]
            kv[int(table[b, j]), 1, :n] = rv[j * page: j * page + n]
        vals.append(_values(rk[: lens[b]], rv[: lens[b]]))
    return kv, table, vals


def _attn64(q, vals, scale):
    """The result in 64 bits, and what its error is measured against (see _check_attn)."""
    B, hq, hd = q.shape
    out, size = torch.zeros(2, B, hq, hd, dtype=torch.float64, device="cuda")
    for b, (k, v, err) in enumerate(vals):
        if k.shape[0]:
            rep = hq // k.shape[1]
            kk, vv, ee = (x.repeat_interleave(rep, 1) for x in (k, v, err))
            p = torch.softmax(torch.einsum("hd,nhd->hn", q[b].double(), kk) * scale, -1)
            out[b] = torch.einsum("hn,nhd->hd", p, vv)
            size[b] = torch.einsum("hn,nhd->hd", p, ee)
    return out, size


def _values(rk, rv):
    """k and v of 4-bit rows in 64 bits, and how far a token's p v may be off, for p = 1.

    Scores are sums in fp32 of exact products: p is off by less than 2^-10 of itself at the tests' sizes of scores, and
    so is p v. The kernel sums p zero in fp32, and codes times weights fp16(p scale) on tensor cores: 2^-11 of
    p (v - zero). Those sums are kept in fp32 but may be cut instead of rounded, and every other code is taken out of
    c0 + 16 c1, at most 255, as a sixteenth of a difference: 2^-20 of 16 p scale, and as much again for the rest.
    """
    hd = {48: 64, 80: 128, 160: 256}[rv.shape[-1]]
    par = rv[..., hd // 2: hd // 2 + hd // 8].contiguous().view(BF).double().unflatten(-1, (-1, 2))
    s, zero = (x.repeat_interleave(32, -1) for x in (par[..., 0], par[..., 1]))
    v = kv4_ops.unpack_rows(rv, True).double()
    off = 2.0 ** -10 * v.abs() + 2.0 ** -11 * (v - zero).abs() + 2.0 ** -15 * s
    return kv4_ops.unpack_rows(rk, False).double(), v, off


def _check_attn(got, q, vals, scale):
    want, size = _attn64(q, vals, scale)
    # the result is rounded to bf16 once, by half a step of what is rounded
    bound = HALF_STEP * (want.abs() + size) + size + 1e-30
    err = (got.double() - want).abs()
    assert (err <= bound).all(), (float((err - bound).max()), float(err.max()))


@pytest.mark.parametrize("lens,hkv,group,hd,page,order,ctas", [
    ([1], 1, 1, 64, 16, "nhd", 0),
    ([1, 2, 15, 16, 17, 31, 33], 2, 4, 128, 16, "nhd", 1),
    ([0, 300, 5, 64, 65], 2, 7, 64, 32, "hnd", 3),           # an empty request
    ([0, 0], 1, 3, 128, 16, "nhd", 2),                        # nothing but empty ones
    ([129, 1000], 3, 5, 128, 64, "hnd", 0),
    ([77, 700, 3], 1, 8, 256, 16, "nhd", 5),
    ([40, 41], 2, 1, 256, 1, "nhd", 2),                       # pages of one token
    ([100, 513], 2, 2, 128, 8, "hnd", 4),                     # pages that end inside a tile
    ([257, 90], 1, 16, 64, 16, "nhd", 3),                     # more query heads than a CTA takes
    ([333, 47], 1, 13, 128, 16, "hnd", 7),
    ([2100], 8, 4, 128, 16, "nhd", 400),                       # more CTAs than it has work for
    ([5], 4, 6, 64, 128, "nhd", 9),
        ([3000, 2500], 1, 4, 64, 16, "nhd", 0),                   # 8 streams of tokens, many CTAs a request
        ([700, 0, 900, 1], 3, 3, 128, 32, "hnd", 2),              # CTAs that begin and end inside requests
        ([150] * 9, 12, 2, 64, 16, "nhd", 5),                     # more KV heads than a CTA has warps
        ([6000], 5, 4, 128, 16, "nhd", 0),
        ([20000], 8, 2, 64, 16, "nhd", 0),                        # one request in 74 parts
        ([60000] + [5, 0, 17] * 13, 1, 8, 64, 16, "nhd", 0),      # a request in many parts among short ones
        ([700, 30, 1200, 5, 90, 2000] * 5, 4, 4, 128, 16, "nhd", 0),  # cuts that move behind short requests
        ([64, 100, 31], 6, 2, 64, 32, "nhd", 0),                  # pairs of heads, 6 of them
        ([640, 100, 3100], 4, 6, 64, 16, "nhd", 0),
])
def test_paged_decode_attention(lens, hkv, group, hd, page, order, ctas):
    B = len(lens)
    kv, table, vals = _filled(B, lens, hkv, hd, page, order, seed=sum(lens) + hd)
    q = 2 * torch.randn(B, hkv * group, hd, device="cuda", generator=_gen(9))
    q = q.to(BF)
    seq = _i32(lens)
    for _ in range(2):  # a call leaves nothing to the next
        got = kv4_ops.paged_decode_attn_kv4(q, kv, table, seq, 1 / math.sqrt(hd), ctas=ctas)
        _check_attn(got, q, vals, 1 / math.sqrt(hd))
    for b, n in enumerate(lens):
        assert n or not got[b].any()
    assert kv4_ops.kv4_status() == 0


def test_attention_strided_query_table_and_caller_buffers():
    lens, hkv, group, hd, page = [90, 200, 17], 2, 4, 128, 16
    kv, table, vals = _filled(3, lens, hkv, hd, page, seed=4)
    wide = torch.randn(3, 8 + 2 * hkv, hd, device="cuda", generator=_gen(1)).to(BF)
    q = wide[:, :8]
    big = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    big[:, : table.shape[1]] = table
    scratch = torch.full((kv4_ops.kv4_decode_scratch(3, 8, hkv, hd, table.shape[1] * page, 4),), math.nan, device="cuda")
    out = torch.empty(3, 8, hd, dtype=BF, device="cuda")
    got = kv4_ops.paged_decode_attn_kv4(q, kv, big[:, : table.shape[1]], _i32(lens), 0.1, ctas=4, scratch=scratch, out=out)
    assert got.data_ptr() == out.data_ptr()
    _check_attn(got, q, vals, 0.1)
    # a table wider than the sequences need, and lengths beyond the table's width
    _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, big, _i32(lens), 0.1), q, vals, 0.1)
    full = table[:, :1].contiguous()
    vals1 = [tuple(x[:16] for x in v) for v in vals]
    _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, full, _i32([90, 2 ** 31 - 1, 17]), 0.1), q, vals1, 0.1)
    none = kv4_ops.paged_decode_attn_kv4(q, kv, table[:, :0], _i32(lens), 0.1)
    assert not none.any()
    assert kv4_ops.paged_decode_attn_kv4(q[:0], kv, table[:0], _i32([]), 0.1).shape == (0, 8, hd)


def test_attention_pages_outside_the_pool_hold_no_tokens():
    lens, hkv, hd, page = [64, 64, 64], 2, 128, 16
    kv, table, vals = _filled(3, lens, hkv, hd, page, seed=6)
    table[0, 1], table[1, 0], table[2] = -1, kv.shape[0], 2 ** 30
    keep = [torch.arange(64, device="cuda") // 16 != 1, torch.arange(64, device="cuda") // 16 != 0,
            torch.zeros(64, dtype=torch.bool, device="cuda")]
    q = torch.randn(3, 8, hd, device="cuda", generator=_gen(2)).to(BF)
    got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), 0.2, ctas=2)
    _check_attn(got, q, [tuple(x[m] for x in v) for v, m in zip(vals, keep)], 0.2)
    assert not got[2].any()


@pytest.mark.parametrize("scale", [0.0, 1e-4, 3.0, -0.5])
def test_attention_scales(scale):
    """Equal weights, and weights that sit on one token; q elements of very different size."""
    lens, hkv, group, hd = [200, 33], 1, 4, 128
    kv, table, vals = _filled(2, lens, hkv, hd, 16, seed=8)
    q = (torch.randn(2, 4, hd, device="cuda", generator=_gen(3)) *
         torch.logspace(-4, 0, hd, device="cuda")).to(BF)
    got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), scale)
    _check_attn(got, q, vals, scale)


def test_attention_one_token_far_above_many():
    """A first token of almost all weight in front of many of little: their sum still counts."""
    n, hd = 4096, 64
    kv, table, _ = _filled(1, [n], 1, hd, 16, seed=10)
    x = torch.zeros(n, 2, 1, hd, device="cuda")
    x[0, 0, 0, 0], x[1:, 1] = 8.0, 1.0
    x[0, 1] = -1.0
    x = x.to(BF)
    rk, rv = kv4_ops.pack_rows(x[:, 0], False), kv4_ops.pack_rows(x[:, 1], True)
    for j in range(n // 16):
        kv[int(table[0, j]), 0], kv[int(table[0, j]), 1] = rk[16 * j: 16 * j + 16], rv[16 * j: 16 * j + 16]
    q = torch.zeros(1, 1, hd, device="cuda", dtype=BF)
    q[0, 0, 0] = 1.0
    vals = [_values(rk, rv)]
    for ctas in (1, 8):
        got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32([n]), 1.0, ctas=ctas)
        _check_attn(got, q, vals, 1.0)


def test_attention_poison_shows_only_where_it_is():
    lens, hkv, hd = [40, 40], 2, 128
    kv, table, vals = _filled(2, lens, hkv, hd, 16, seed=12)
    blk = int(table[0, 1])
    kv[blk, 0, 3, 1] = 255  # one K row of request 0, KV head 1
    q = torch.randn(2, 4, hd, device="cuda", generator=_gen(4)).to(BF)
    got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), 0.1, ctas=3)
    assert got[0, 2:].isnan().all()
    want, _ = _attn64(q, vals, 0.1)
    assert got[0, :2].isfinite().all() and got[1].isfinite().all()
    assert (got[1].double() - want[1]).abs().max() < 0.1


def test_offsets_beyond_32_bits():
    """Blocks more than 4 GiB into the pool, for each kernel that addresses it."""
    hkv, hd, page = 2, 128, 16
    row = kv4_ops.row_bytes(hd)
    stride = 2 * page * hkv * row
    far = 2 ** 32 // stride + 3
    flat = torch.zeros((far + 2) * stride, dtype=torch.uint8, device="cuda")
    kv = flat.view(far + 2, 2, page, hkv, row)
    x = torch.randn(30, 3 * hkv, hd, device="cuda", generator=_gen(5)).to(BF)
    slots = (torch.tensor([far, 1], device="cuda")[torch.arange(30, device="cuda") // 16] * page
             + torch.arange(30, device="cuda") % 16)
    q, k = torch.empty(30, hkv, hd, dtype=BF, device="cuda"), torch.empty(30, hkv, hd, dtype=BF, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(x, torch.arange(30, dtype=torch.int32, device="cuda"), _cos_sin(32, hd), hkv, hkv, kv,
                                  slots, q_out=q, k_out=k)
    kg, vg = kv4_ops.kv4_gather(kv, slots)
    assert torch.equal(vg, kv4_ops.unpack_rows(kv4_ops.pack_rows(x[:, 2 * hkv:], True), True).to(BF))
    vals = [_values(kv4_ops.pack_rows(k, False), kv4_ops.pack_rows(x[:, 2 * hkv:], True))]
    got = kv4_ops.paged_decode_attn_kv4(q[29:], kv, _i32([[far, 1]]), _i32([30]), 0.1, ctas=2)
    _check_attn(got, q[29:], vals, 0.1)


# ------------------------------------------------------- all of them together


def _run_together(B=5, hq=8, hkv=2, hd=128, page=16):
    """Two ragged steps of a batch: tables, write, decode attention over what was written."""
    g = _gen(42)
    pool = KvLayout.allocate(LayoutConfig.for_model(64, 2, hkv, kv4_ops.row_bytes(hd), page, torch.uint8),
                             "fully_contiguous", KvBlockLayout.OPERATIONAL_NHD)
    kv = pool.layer_view(1)
    cs = _cos_sin(512, hd)
    prompt = [33, 1, 16, 100, 47]
    owned = [-(-(n + 1) // page) for n in prompt]
    ids = _i32(torch.randperm(64, generator=torch.Generator().manual_seed(1))[: sum(owned)].tolist())
    T = sum(prompt) + 6  # a padded batch
    x = torch.randn(T, hq + 2 * hkv, hd, device="cuda", generator=g).to(BF)
    y = torch.randn(B, hq + 2 * hkv, hd, device="cuda", generator=g).to(BF)
    w = (1 + 0.1 * torch.randn(2, hd, device="cuda", generator=g)).to(BF)
    return pool, kv, cs, prompt, owned, ids, T, x, y, w


def _steps(kv, cs, prompt, owned, ids, T, x, y, w, hq=8, hkv=2, hd=128, page=16):
    B = len(prompt)
    t = table_ops.batch_tables(_i32(prompt), _i32([0] * B), ids, page=page, max_blocks=10, num_tokens=T,
                               block_counts=_i32(owned))
    q1 = torch.empty(T, hq, hd, dtype=BF, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(x, t.positions, cs, hq, hkv, kv, t.slots, q_weight=w[0], k_weight=w[1], q_out=q1)
    pos = t.seq_lens  # the next token's position
    slots = table_ops.slot_map(t.block_table, pos, page=page)
    q2 = torch.empty(B, hq, hd, dtype=BF, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(y, pos, cs, hq, hkv, kv, slots, q_weight=w[0], k_weight=w[1], q_out=q2)
    out = kv4_ops.paged_decode_attn_kv4(q2, kv, t.block_table, pos + 1, 1 / math.sqrt(hd), ctas=2)
    return t, q2, out


def test_operators_together():
    pool, kv, cs, prompt, owned, ids, T, x, y, w = _run_together()
    t, q2, out = _steps(kv, cs, prompt, owned, ids, T, x, y, w)
    page, vals, at, blk = 16, [], 0, 0
    for b, n in enumerate(prompt):
        mine = ids[blk: blk + owned[b]].long()
        blk += owned[b]
        assert t.block_table[b, : owned[b]].tolist() == mine.tolist()
        p = torch.arange(n + 1, device="cuda")
        k, v = kv4_ops.kv4_gather(kv, mine[p // page] * page + p % page)
        raw = torch.cat([x[at: at + n], y[b: b + 1]])
        assert torch.equal(v, kv4_ops.unpack_rows(kv4_ops.pack_rows(raw[:, 10:], True), True).to(BF))
        (_, _), (k64, _) = _heads64(raw, p, cs, 8, 2, w[0], w[1], 1e-6)
        span = k64.unflatten(-1, (-1, 32)).amax(-1) - k64.unflatten(-1, (-1, 32)).amin(-1)
        err = (k.double() - k64).abs().unflatten(-1, (-1, 32)).amax(-1)
        # half a step, the element's and the range's bf16 roundings, and the read-back's
        assert (err <= span / 30 * (1 + 2.0 ** -7) + 3 * HALF_STEP * k64.unflatten(-1, (-1, 32)).abs().amax(-1)).all()
        rows = kv[mine[p // page], :, p % page]
        vals.append(_values(rows[:, 0], rows[:, 1]))
        at += n
    _check_attn(out, q2, vals, 1 / math.sqrt(128))


def test_operators_together_captured_and_on_another_stream():
    pool, kv, cs, prompt, owned, ids, T, x, y, w = _run_together()
    _, _, want = _steps(kv, cs, prompt, owned, ids, T, x, y, w)
    want = want.clone()
    args = (_i32(prompt), _i32([0] * 5), ids, _i32(owned))

    def step(stream=None):
        t = table_ops.batch_tables(args[0], args[1], args[2], page=16, max_blocks=10, num_tokens=T,
                                   block_counts=args[3], stream=stream)
        q1 = torch.empty(T, 8, 128, dtype=BF, device="cuda")
        kv4_ops.qk_norm_rope_kv_write(x, t.positions, cs, 8, 2, kv, t.slots, q_weight=w[0], k_weight=w[1], q_out=q1,
                                      stream=stream)
        slots = table_ops.slot_map(t.block_table, t.seq_lens, page=16, stream=stream)
        q2 = torch.empty(5, 8, 128, dtype=BF, device="cuda")
        kv4_ops.qk_norm_rope_kv_write(y, t.seq_lens, cs, 8, 2, kv, slots, q_weight=w[0], k_weight=w[1], q_out=q2,
                                      stream=stream)
        return t, q1, q2, slots

    kv.zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    t, q1, q2, slots = step(stream=s)
    got = kv4_ops.paged_decode_attn_kv4(q2, kv, t.block_table, _i32([n + 1 for n in prompt]), 1 / math.sqrt(128),
                                        ctas=2, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    kv.zero_()
    graph = torch.cuda.CUDAGraph()
    seq = _i32([n + 1 for n in prompt])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        t, q1, q2, slots = step()
        got = kv4_ops.paged_decode_attn_kv4(q2, kv, t.block_table, seq, 1 / math.sqrt(128), ctas=2)
    for _ in range(2):
        kv.zero_()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def _unfused(x, w, cos_sin, rot, eps):
    """The formula in fp32, each operation rounded by itself, the squares summed in the kernel's order."""
    y = x.float()
    s = y * y
    if s.shape[-1] == 256:
        s = s[..., :128] + s[..., 128:]
    if x.shape[-1] > 64:
        s = s.unflatten(-1, (32, 4))
        s = ((s[..., 0] + s[..., 1]) + s[..., 2]) + s[..., 3]
    while s.shape[-1] > 1:
        n = s.shape[-1] // 2
        s = s[..., :n] + s[..., n:]
    y = y * torch.rsqrt(s / x.shape[-1] + eps) * w.float()
    c, n = cos_sin[:, None, :rot // 2], cos_sin[:, None, rot // 2:]
    a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    return torch.cat([a * c - b * n, b * c + a * n, y[..., rot:]], -1).bfloat16()


@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 16), (128, 128), (128, 48), (256, 256), (256, 64)])
def test_write_rounds_as_the_unfused_formula(hd, rot):
    """k decides the codes of the cache, so it is the same bit for bit as each operation by itself."""
    tokens, hq, hkv, page = 193, 6, 3, 16
    gen = torch.Generator().manual_seed(hd + rot)
    qkv = torch.randn(tokens, hq + 2 * hkv, hd, generator=gen).bfloat16().cuda()
    wq, wk = ((1 + 0.2 * torch.randn(hd, generator=gen)).bfloat16().cuda() for _ in range(2))
    angle = 6.0 * torch.rand(tokens, rot // 2, generator=gen)
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).cuda()
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    slots = torch.arange(tokens, device="cuda")
    kv = torch.zeros(13, 2, page, hkv, kv4_ops.row_bytes(hd), dtype=torch.uint8, device="cuda")
    q = torch.empty(tokens, hq, hd, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(tokens, hkv, hd, dtype=torch.bfloat16, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(qkv, positions, cos_sin, hq, hkv, kv, slots, q_weight=wq, k_weight=wk, eps=1e-6,
                                  q_out=q, k_out=k)
    assert torch.equal(q, _unfused(qkv[:, :hq], wq, cos_sin, rot, 1e-6))
    want = _unfused(qkv[:, hq:hq + hkv], wk, cos_sin, rot, 1e-6)
    assert torch.equal(k, want)
    rows = kv[:, 0].reshape(-1, hkv, kv4_ops.row_bytes(hd))[:tokens].cpu()
    assert torch.equal(rows, kv4_ops.pack_rows(want.cpu(), False))


def test_write_without_query_heads():
    """K and V alone: with a q_out of no heads qkv stays as it is."""
    gen = _gen(11)
    qkv = torch.randn(5, 4, 128, device="cuda", generator=gen).bfloat16()
    before = qkv.clone()
    cos_sin = torch.cat([torch.full((8, 64), 0.6, device="cuda"), torch.full((8, 64), 0.8, device="cuda")], -1)
    positions = torch.arange(5, dtype=torch.int32, device="cuda")
    slots = torch.arange(5, device="cuda")
    kv = _empty_pool(1, 16, 2, 128)
    k = torch.empty(5, 2, 128, dtype=BF, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(qkv, positions, cos_sin, 0, 2, kv, slots, k_out=k,
                                  q_out=torch.empty(5, 0, 128, dtype=BF, device="cuda"))
    assert torch.equal(qkv, before)
    kv4_ops.qk_norm_rope_kv_write(qkv, positions, cos_sin, 0, 2, _empty_pool(1, 16, 2, 128), slots)
    assert torch.equal(qkv[:, :2], k) and torch.equal(qkv[:, 2:], before[:, 2:])
    assert torch.equal(kv[0, 0, :5], kv4_ops.pack_rows(k, False))
    assert torch.equal(kv[0, 1, :5], kv4_ops.pack_rows(before[:, 2:], True))


def test_a_pool_without_blocks():
    """Nothing is written, rows are zeros, attention has no tokens."""
    kv = _empty_pool(0, 16, 2, 128)
    qkv = torch.randn(3, 8, 128, device="cuda", generator=_gen(12)).bfloat16()
    slots = torch.tensor([0, -1, 7], device="cuda")
    cos_sin = torch.ones(4, 128, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(qkv, torch.arange(3, dtype=torch.int32, device="cuda"), cos_sin, 4, 2, kv, slots)
    k, v = kv4_ops.kv4_gather(kv, slots)
    assert not k.any() and not v.any()
    out = kv4_ops.paged_decode_attn_kv4(qkv[:, :4], kv, torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
                                        torch.full((3,), 20, dtype=torch.int32, device="cuda"), 0.1)
    assert not out.any()


def test_attention_scratch_of_requests_that_are_cut():
    lens, hkv, hd, page = [3000, 5, 0, 700], 2, 128, 16
    kv, table, vals = _filled(4, lens, hkv, hd, page, seed=6)
    q = torch.randn(4, 8, hd, device="cuda", generator=_gen(2)).to(BF)
    need = kv4_ops.kv4_decode_scratch(4, 8, hkv, hd, table.shape[1] * page)
    assert need > 0 and kv4_ops.kv4_decode_scratch(4, 8, hkv, hd, 64) == 0
    for fill in (math.nan, 3e38):
        scratch = torch.full((need,), fill, device="cuda")
        _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), 0.1, scratch=scratch), q, vals, 0.1)
    with pytest.raises(ValueError, match="are needed"):
        kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), 0.1, scratch=scratch[4:])


def test_launches_are_counted():
    kv, table, _ = _filled(1, [40], 2, 64, 16)
    q = torch.zeros(1, 4, 64, dtype=BF, device="cuda")
    wide = torch.zeros(1, 400, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    for t, n in ((table, 1), (wide, 2)):
        assert (kv4_ops.kv4_decode_scratch(1, 4, 2, 64, t.shape[1] * 16) > 0) == (n == 2)
        before = _lib.launch_count()
        kv4_ops.paged_decode_attn_kv4(q, kv, t, _i32([40]), 0.1)
        assert _lib.launch_count() - before == n


def _held(x, page=16):
    """A pool with the rows of bf16 x [n, 2, heads, hd] as one request's, its table, the values in 64 bits and V's
    scales [n, heads, hd]."""
    n, _, heads, hd = x.shape
    nb = -(-n // page)
    rk, rv = kv4_ops.pack_rows(x[:, 0], False), kv4_ops.pack_rows(x[:, 1], True)
    kv = _empty_pool(nb, page, heads, hd, fill=255)
    for o, rows in ((0, rk), (1, rv)):
        at = torch.arange(n, device="cuda")
        kv[at // page, o, at % page] = rows
    scales = rv[..., hd // 2: hd // 2 + hd // 8].contiguous().view(BF).double()[..., ::2].repeat_interleave(32, -1)
    return kv, torch.arange(nb, dtype=torch.int32, device="cuda").view(1, nb), [_values(rk, rv)], scales


def _spread_values(kind, n, heads, hd):
    """V whose scales differ, and K that make some tokens' scores the lowest by far."""
    x = torch.randn(n, 2, heads, hd, device="cuda", generator=_gen(hd + n))
    if kind == "one group":              # a group of channels far above its neighbours
        x[:, 1, :, :32] *= 1e10
    elif kind == "one group 60 times":
        x[:, 1, :, :32] *= 60
    elif kind == "one group far below":
        x[:, 1, :, 32:] *= 1e-12
    elif kind == "later tokens":         # what was summed before has to be brought down
        x[n // 2:, 1] *= 2.0 ** 15
    elif kind == "later tokens of a group":
        x[n // 3:, 1, :, :32] *= 1e9
    elif kind == "first tokens that hardly count":  # they alone set how the weights are held, at first
        x[:40, 1] *= 1e20
        x[:40, 0, :, 0] = -800.0
        x[40:, 0, :, 0] = 20.0
    elif kind == "a light token among others":
        x[5, 1] *= 1e15
        x[5, 0, :, 0] = -800.0
    elif kind == "a group of equal elements":
        x[:, 1, :, 32:64] = 0.5
    elif kind == "equal elements at first":
        x[:500, 1, :, :32] = 0.25
        x[500:, 1, :, :32] *= 1e-7
    elif kind == "tiny":
        x[:, 1] *= 1e-33
    return x.to(BF)


@pytest.mark.parametrize("group,hd", [(4, 128), (7, 64), (2, 256), (8, 128), (6, 256), (1, 64)])
@pytest.mark.parametrize("kind", ["one group", "one group 60 times", "one group far below", "later tokens",
                                  "later tokens of a group", "first tokens that hardly count",
                                  "a light token among others", "a group of equal elements",
                                  "equal elements at first", "tiny"])
def test_attention_values_of_very_different_size(kind, group, hd):
    """Each group of V against its own size. Beside what `_values` allows, a weight may be off by 2^-26 of the largest
    that the head gives the group, times a code of up to 15."""
    n, heads = 700, 2
    kv, table, vals, scales = _held(_spread_values(kind, n, heads, hd))
    q = torch.randn(1, heads * group, hd, device="cuda", generator=_gen(group)).to(BF)
    q[..., 0] = 1.0
    scale = 1 / math.sqrt(hd)
    want, size = _attn64(q, vals, scale)
    k = vals[0][0].repeat_interleave(group, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), k) * scale, -1)
    largest = (p.t().unsqueeze(-1) * scales.repeat_interleave(group, 1)).amax(0)
    size = size + 15 * n * 2.0 ** -26 * largest
    for ctas in (1, 4):
        got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32([n]), scale, ctas=ctas)
        # rounded to bf16 once
        assert ((got.double() - want).abs() <= HALF_STEP * (want.abs() + size) + size + 2.0 ** -133).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_one_token_far_above_many_whose_values_vary(hd):
    """As above where the many tokens' values fill their groups, so that their weights are held in 16 bits."""
    n = 4096
    x = torch.randn(n, 2, 1, hd, device="cuda", generator=_gen(hd))
    x[:, 0] = 0.0
    x[0, 0, 0, 0] = 8.0
    kv, table, vals, _ = _held(x.to(BF))
    q = torch.zeros(1, 1, hd, device="cuda", dtype=BF)
    q[0, 0, 0] = 1.0
    for ctas in (1, 8):
        _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32([n]), 1.0, ctas=ctas), q, vals, 1.0)


def test_attention_poisoned_value_shows_only_where_it_is():
    """A V row with a NaN in one group: this group of the heads that read it, and no other result."""
    lens, hkv, hd = [40, 40], 2, 128
    kv, table, vals = _filled(2, lens, hkv, hd, 16, seed=13)
    x = torch.randn(1, hd, device="cuda", generator=_gen(1)).to(BF)
    x[0, 70] = math.nan
    kv[int(table[0, 1]), 1, 3, 1] = kv4_ops.pack_rows(x, True)[0]
    q = torch.randn(2, 4, hd, device="cuda", generator=_gen(4)).to(BF)
    got = kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32(lens), 0.1, ctas=3)
    assert got[0, 2:, 64:96].isnan().all()
    assert got[0, 2:, :64].isfinite().all() and got[0, 2:, 96:].isfinite().all()
    assert got[0, :2].isfinite().all()
    _check_attn(got[1:], q[1:], vals[1:], 0.1)


def _in_threads(calls, rounds):
    """Each of `calls` over and over in a thread of its own; what they raised."""
    errors = []

    def work(call):
        try:
            for _ in range(rounds):
                call()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


def test_attention_calls_of_several_threads():
    """Launches of one kernel that take different amounts of shared memory (a request with a short table 8 warps a CTA,
    four with long ones 6) do not get in each other's way."""
    kv, table, vals = _filled(1, [40], 6, 128, 16, "hnd")
    one = torch.randn(1, 6, 128, device="cuda", generator=_gen(1)).to(BF)
    wide = torch.zeros(4, 400, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    outs = []

    def call(t):
        q, seq = one.expand(t.shape[0], 6, 128).contiguous(), _i32([40] * t.shape[0])
        out, scratch = torch.empty_like(q), torch.empty(1 << 20, device="cuda")
        outs.append(out)
        return lambda: kv4_ops.paged_decode_attn_kv4(q, kv, t, seq, 0.1, out=out, scratch=scratch)

    assert not _in_threads([call(table), call(wide), call(table), call(wide)], 500)
    for out in outs:
        for row in out:
            _check_attn(row[None], one, vals, 0.1)


def test_table_calls_of_several_threads():
    def call(B):
        q, c, ids = torch.ones(B, dtype=torch.int32, device="cuda"), _i32([0] * B), torch.arange(B, dtype=torch.int32, device="cuda")
        return lambda: table_ops.batch_tables(q, c, ids, page=16, max_blocks=1)

    assert not _in_threads([call(8192), call(3500), call(8192), call(3500)], 500)


def test_strides_of_dimensions_of_one_do_not_matter():
    """One token, one request, one block, page or head may lie at any pitch: it is not used."""
    hd, hkv, page = 128, 2, 16
    kv, table, vals = _filled(1, [30], hkv, hd, page)
    q = torch.randn(1, 8, hd, device="cuda", generator=_gen(3)).to(BF)
    odd = torch.zeros(1, 8 * hd + 3, dtype=BF, device="cuda")
    odd[:, : 8 * hd] = q.flatten(1)
    view = odd.as_strided((1, 8, hd), (8 * hd + 3, hd, 1))
    assert view.stride(0) % 8
    _check_attn(kv4_ops.paged_decode_attn_kv4(view, kv, table, _i32([30]), 0.1), q, vals, 0.1)
    x = torch.randn(1, 8, hd, device="cuda", generator=_gen(4)).to(BF)
    odd[:, : 8 * hd] = x.flatten(1)
    where, cs, slot = _i32([0]), _cos_sin(1, hd), torch.tensor([5], device="cuda")
    a, b = _empty_pool(1, page, hkv, hd), _empty_pool(1, page, hkv, hd)
    qa, qb = torch.empty(2, 1, 4, hd, dtype=BF, device="cuda")
    kv4_ops.qk_norm_rope_kv_write(x, where, cs, 4, hkv, a, slot, q_out=qa)
    kv4_ops.qk_norm_rope_kv_write(view, where, cs, 4, hkv, b, slot, q_out=qb)
    assert torch.equal(a, b) and torch.equal(qa, qb)
    # one block of one head, as a slice of bytes at odd pitches
    flat = torch.zeros(3 * page * 80 + 40, dtype=torch.uint8, device="cuda")
    one = flat.as_strided((1, 2, page, 1, 80), (24, page * 80, 80, 7, 1))
    rows = torch.empty(1, 2, page, 1, 80, dtype=torch.uint8, device="cuda")
    rows.copy_(kv[int(table[0, 0]), :, :, :1][None])
    one.copy_(rows)
    at = torch.arange(page, device="cuda")
    for got, want in zip(kv4_ops.kv4_gather(one, at), kv4_ops.kv4_gather(rows, at)):
        assert torch.equal(got, want)
    q1 = q[:, :4].contiguous()
    _check_attn(kv4_ops.paged_decode_attn_kv4(q1, one, _i32([[0]]), _i32([page]), 0.1), q1,
                [tuple(x[:page, :1] for x in vals[0])], 0.1)


@pytest.mark.parametrize("hkv,order", [(3, "nhd"), (2, "hnd")])
def test_a_copy_that_is_given_up_is_reported(hkv, order):
    """With a limit of 0 no copy is waited for: the launch lets those under way arrive and ends, its results are NaN, and
    the host reads status 3. The next launch, with the usual limit, is right."""
    lens, hd = [3000, 0, 700], 128
    kv, table, vals = _filled(3, lens, hkv, hd, 16, order, seed=3)
    q = torch.randn(3, 4 * hkv, hd, device="cuda", generator=_gen(5)).to(BF)
    seq = _i32(lens)
    kv4_ops.kv4_status()
    kv4_ops.set_kv4_wait_limit_ns(0)
    try:
        got = kv4_ops.paged_decode_attn_kv4(q, kv, table, seq, 0.1)
        torch.cuda.synchronize()
    finally:
        kv4_ops.set_kv4_wait_limit_ns(None)
    assert kv4_ops.kv4_status(reset=False) == 3
    assert got[0].isnan().all() and got[2].isnan().all()
    with pytest.raises(_lib.KvbmCudaError, match="status 3"):
        kv4_ops.check_kv4_status("cuda")
    kv4_ops.check_kv4_status()  # cleared
    _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, table, seq, 0.1), q, vals, 0.1)
    assert kv4_ops.kv4_status() == 0


@pytest.mark.parametrize("exponent", [10, 14, 24, 32, 60, 125])
@pytest.mark.parametrize("group,hd", [(4, 128), (7, 64), (3, 256)])
def test_attention_large_scores(group, hd, exponent):
    """Scores of up to 1e38 are finite, and beside those of other tokens: all the weight lies on the largest ones."""
    n, heads = 50, 2
    x = torch.randn(n, 2, heads, hd, device="cuda", generator=_gen(8))
    x[:, 0, :, 0] = torch.linspace(-1, 2, n, device="cuda")[torch.randperm(n, device="cuda", generator=_gen(9)), None]
    kv, table, vals, _ = _held(x.to(BF))
    q = torch.zeros(1, heads * group, hd, dtype=BF, device="cuda")
    q[..., 0] = 2.0 ** exponent
    q[0, 1, 0] = -(2.0 ** exponent)
    q[0, 2, 0] = 2.0 ** (exponent - 6)
    for ctas in (1, 2):
        _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32([n]), 1.0, ctas=ctas), q, vals, 1.0)


@pytest.mark.parametrize("group,hd", [(4, 128), (7, 64)])
def test_attention_large_negative_scores_in_front(group, hd):
    """A tile whose scores are far below zero leaves nothing behind when ordinary ones follow."""
    n, heads = 100, 2
    x = torch.randn(n, 2, heads, hd, device="cuda", generator=_gen(8))
    x[:, 0] = 0.0
    x[:64, 0, :, 0] = -torch.linspace(1, 2, 64, device="cuda")[:, None]
    x[64:, 0, :, 1] = torch.randn(36, heads, device="cuda", generator=_gen(9))
    kv, table, vals, _ = _held(x.to(BF))
    q = torch.zeros(1, heads * group, hd, dtype=BF, device="cuda")
    q[..., 1] = 1.0
    for e in (8, 20, 40, 100):
        q[..., 0] = 2.0 ** e
        for ctas in (1, 2):
            _check_attn(kv4_ops.paged_decode_attn_kv4(q, kv, table, _i32([n]), 1.0, ctas=ctas), q, vals, 1.0)


def test_attention_a_warp_that_starts_again_keeps_no_other_waiting():
    """Two warps share the copies of two heads. One of them does its tiles again in fp32, for milliseconds: the other's
    wait for the next request's copies, which the first issues, begins when that is done."""
    n, hd = 3000, 128
    x = torch.randn(n, 2, 8, hd, device="cuda", generator=_gen(3))
    x[:, 1, 0, :32] *= 1e6  # the first head's
    kv, table, vals, _ = _held(x.to(BF))
    q = torch.randn(1, 16, hd, device="cuda", generator=_gen(4)).to(BF)
    kv4_ops.kv4_status()
    kv4_ops.set_kv4_wait_limit_ns(1_000_000)
    try:
        got = kv4_ops.paged_decode_attn_kv4(q.expand(3, 16, hd).contiguous(), kv, table.expand(3, -1).contiguous(),
                                            _i32([n] * 3), 0.1, ctas=1)
        torch.cuda.synchronize()
    finally:
        kv4_ops.set_kv4_wait_limit_ns(None)
    assert kv4_ops.kv4_status() == 0
    for row in got:
        _check_attn(row[None], q, vals, 0.1)
