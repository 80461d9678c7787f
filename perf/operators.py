"""The operators of a 4-bit paged KV cache, for measuring: block tables and slots from request lengths,
q/k head norms + RoPE + cache write, the cache's read back into bf16 rows, decode attention over it.

Each case is one call as a serving step makes it. ``run`` computes it in plain torch, or with the
kernels of ``kvbm_b200.ops`` when ``own`` is true.

A 4-bit row is ``hd/2`` bytes of codes, then (scale, zero) in bf16 for each group of 32 elements, padded
to 16 bytes; an element is ``zero + code * scale``. K keeps code d in nibble d; V keeps the code of
element 32 g + 4 b + i in nibble 4 (NG b + g) + i, NG = hd / 32.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

GROUP = 32


def listed():
    return [
        # four short requests enter an engine between two decode steps: latency is all there is
        {"name": "tables-admit-4", "op": "tables", "batch": 4, "tokens": 64, "max_len": 400, "page": 16,
         "max_blocks": 64, "reserved": True, "rows": 32},
        # a full continuous-batching step: 8,192 new tokens of 256 requests, contexts up to 16,384
        {"name": "tables-step-256", "op": "tables", "batch": 256, "tokens": 8192, "max_len": 16384, "page": 16,
         "max_blocks": 1024, "reserved": False, "rows": 0},
        # the slots of one decode step of a 32-slot batch
        {"name": "slots-decode-32", "op": "slots", "batch": 32, "max_len": 8448, "page": 16},
        # one decode step of a 32-slot batch, Llama-3-8B heads, rotated q apart, K/V into 4 bits
        {"name": "write-decode-32-kv4", "op": "write", "tokens": 32, "hq": 32, "hkv": 8, "hd": 128, "rot": 128,
         "page": 16, "bits": 4, "order": "nhd", "norm": True, "pad": 0, "keep_k": False},
        # a prefill chunk of 8,192 tokens into 4 bits, rotated q and k kept for the chunk's own attention
        {"name": "write-prefill-8192-kv4", "op": "write", "tokens": 8192, "hq": 32, "hkv": 8, "hd": 128, "rot": 128,
         "page": 16, "bits": 4, "order": "nhd", "norm": True, "pad": 0, "keep_k": True},
        # a padded odd chunk of a model with 64-wide heads, partial rotation, into a 16-bit head-first cache
        {"name": "write-odd-1237-kv16", "op": "write", "tokens": 1237, "hq": 14, "hkv": 2, "hd": 64, "rot": 32,
         "page": 32, "bits": 16, "order": "hnd", "norm": True, "pad": 37, "keep_k": True},
        # a short cached prefix read back for the attention of the rest of the prompt
        {"name": "read-77", "op": "read", "tokens": 77, "hkv": 8, "hd": 128, "page": 16, "order": "nhd"},
        # a long cached prefix, Llama-3-8B heads
        {"name": "read-16384", "op": "read", "tokens": 16384, "hkv": 8, "hd": 128, "page": 16, "order": "nhd"},
        # one request with a short context: the latency of a single token
        {"name": "attn-1x300", "op": "attn", "batch": 1, "max_len": 300, "spread": False, "hq": 32, "hkv": 8,
         "hd": 128, "page": 16, "order": "nhd"},
        # one request with a very long context: the work has to be split over it
        {"name": "attn-1x131072", "op": "attn", "batch": 1, "max_len": 131072, "spread": False, "hq": 32, "hkv": 8,
         "hd": 128, "page": 16, "order": "nhd"},
        # the decode batch of the framework's serving benchmark
        {"name": "attn-32x8448", "op": "attn", "batch": 32, "max_len": 8448, "spread": False, "hq": 32, "hkv": 8,
         "hd": 128, "page": 16, "order": "nhd"},
        # a ragged batch, 7 query heads of width 64 on each KV head, an empty slot among them, head-first pages of 32
        {"name": "attn-61x9000-ragged", "op": "attn", "batch": 61, "max_len": 9000, "spread": True, "hq": 28, "hkv": 4,
         "hd": 64, "page": 32, "order": "hnd"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "slots", "write", "write", "read", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 64])
    order = rng.choice(["nhd", "hnd"])
    hd = rng.choice([64, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "tables":
        batch = _log(rng, 1, 256)
        max_len = _log(rng, 64, 16384)
        return {"op": op, "batch": batch, "tokens": _log(rng, batch, 8192), "max_len": max_len, "page": page,
                "max_blocks": -(-max_len // page) + rng.randrange(4), "reserved": rng.random() < 0.5,
                "rows": rng.choice([0, batch + rng.randrange(32)])}
    if op == "slots":
        return {"op": op, "batch": _log(rng, 1, 512), "max_len": _log(rng, 64, 16384), "page": page}
    if op == "write":
        keep = rng.random() < 0.5
        tokens = _log(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "hq": hkv * rng.choice([1, 3, 4, 7, 8] if hkv < 8 and hd < 256 else [1, 2, 3]),
                "hkv": hkv, "hd": hd, "rot": hd // rng.choice([1, 1, 2]), "page": page, "bits": rng.choice([4, 4, 16]),
                "order": order, "norm": rng.random() < 0.7, "pad": rng.randrange(tokens) if rng.random() < 0.3 else 0,
                "keep_k": keep}
    if op == "read":
        return {"op": op, "tokens": _log(rng, 1, 16384), "hkv": hkv, "hd": hd, "page": page, "order": order}
    batch = _log(rng, 1, 128)
    cap = 32 * 8448 * 8 * 128 // (batch * hkv * hd)
    return {"op": op, "batch": batch, "max_len": _log(rng, 16, max(17, min(131072, cap))), "spread": rng.random() < 0.6,
            "hq": hkv * rng.choice([1, 2, 4, 5, 7, 8]), "hkv": hkv, "hd": hd, "page": page, "order": order}


def _row_bytes(hd):
    return -(-(hd // 2 + 4 * (hd // GROUP)) // 16) * 16


def work(case):
    op = case["op"]
    if op == "tables":
        B, T = case["batch"], case["tokens"]
        ids = B * (case["max_len"] // (2 * case["page"]) + 1)
        return {"bytes": 4 * (2 * B + ids) + 4 * B * case["max_blocks"] + 4 * (2 * B + 1) + 12 * T, "flops": 0}
    if op == "slots":
        return {"bytes": case["batch"] * (4 + 4 + 8), "flops": 0}
    if op == "write":
        T, hq, hkv, hd = case["tokens"], case["hq"], case["hkv"], case["hd"]
        row = _row_bytes(hd) if case["bits"] == 4 else 2 * hd
        n = 2 * T * (hq + 2 * hkv) * hd + T * (4 * case["rot"] + 12) + 2 * T * hq * hd
        n += 2 * T * hkv * hd if case["keep_k"] else 0
        n += (T - case["pad"]) * 2 * hkv * row
        if case["bits"] == 4:  # the values are read back
            n += 2 * T * hkv * 2 * hd
        return {"bytes": n, "flops": T * (hq + hkv) * hd * 7}
    if op == "read":
        rows = case["tokens"] * 2 * case["hkv"]
        return {"bytes": rows * (_row_bytes(case["hd"]) + 2 * case["hd"]) + 8 * case["tokens"], "flops": 2 * rows * case["hd"]}
    total = case["batch"] * case["max_len"] * (0.5 if case["spread"] else 1)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    return {"bytes": int(total * (2 * hkv * _row_bytes(hd) + 4 / case["page"]) + case["batch"] * 4 * hq * hd),
            "flops": int(total * 4 * hq * hd)}


# ---------------------------------------------------------------- the inputs


def _pool(blocks, page, heads, width, order, dtype, dev):
    """[blocks, 2, page, heads, width], token-first or head-first in memory."""
    if order == "hnd":
        return torch.zeros(blocks, 2, heads, page, width, dtype=dtype, device=dev).transpose(2, 3)
    return torch.zeros(blocks, 2, page, heads, width, dtype=dtype, device=dev)


def _rows(x, value):
    """bf16 [..., hd] -> uint8 rows [..., row bytes]."""
    hd = x.shape[-1]
    ng = hd // GROUP
    codes, scale, zero = _quantise(x)
    if value:  # element (g, b, i) goes to nibble (b, g, i)
        codes = codes.reshape(*x.shape[:-1], ng, 8, 4).transpose(-3, -2)
    codes = codes.reshape(*x.shape[:-1], hd // 2, 2).to(torch.uint8)
    packed = codes[..., 0] | (codes[..., 1] << 4)
    par = torch.stack([scale, zero], -1).to(torch.bfloat16).flatten(-2).view(torch.uint8)
    pad = torch.zeros(*x.shape[:-1], _row_bytes(hd) - hd // 2 - 4 * ng, dtype=torch.uint8, device=x.device)
    return torch.cat([packed, par, pad], -1)


def _quantise(x):
    """codes, scale, zero in fp32 of bf16 values: groups of 32, scale rounded up to bf16, zero the group's least."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = (0.5 * hi - 0.5 * lo) / torch.full_like(lo, 7.5)  # a true quotient: by a number, torch takes its reciprocal
    up = ((s.contiguous().view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)
    up = torch.where(s < 2.0 ** -126, torch.zeros_like(s), up)
    # a quotient, not a product with 1 / scale: bf16 values lie exactly between two codes often enough
    codes = ((0.5 * g - 0.5 * lo) / torch.where(up > 0, 0.5 * up, 1.0)).round().clamp(0, 15)
    return codes, up.squeeze(-1), lo.squeeze(-1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def ints(lo, hi, *shape):
        return torch.randint(lo, max(lo + 1, hi), shape, device=dev, generator=gen)

    op, st = case["op"], dict(case)
    if op == "tables":
        B, T, page = case["batch"], case["tokens"], case["page"]
        q = torch.ones(B, dtype=torch.int64, device=dev)
        if T > B:  # most of the step's tokens belong to a few prefills; one request may bring none
            cuts = torch.sort(ints(0, T - B + 1, B)).values
            q += torch.diff(cuts, prepend=torch.zeros(1, dtype=torch.int64, device=dev))
            q[-1] = 0 if B > 2 else q[-1]
        ctx = ints(0, case["max_len"], B)
        ctx = torch.minimum(ctx, torch.clamp(case["max_len"] - q, min=0))
        need = (ctx + q + page - 1) // page
        counts = torch.minimum(need + ints(0, 4, B), torch.full_like(need, case["max_blocks"])) if case["reserved"] else need
        n = int(counts.sum())
        st["query_lens"], st["context_lens"] = q.int(), ctx.int()
        st["block_ids"] = torch.randperm(n, device=dev, generator=gen).int()
        st["block_counts"] = counts.int() if case["reserved"] else None
        st["table"] = st["table_rows"] = None
        if case["rows"]:
            st["table"] = torch.full((case["rows"], case["max_blocks"]), -7, dtype=torch.int32, device=dev)
            st["table_rows"] = torch.randperm(case["rows"], device=dev, generator=gen)[:B].int()
        return st
    if op == "slots":
        B, page = case["batch"], case["page"]
        nb = -(-case["max_len"] // page)
        st["block_table"] = torch.randperm(B * nb, device=dev, generator=gen).int().view(B, nb)
        st["positions"] = ints(0, case["max_len"], B).int()
        return st
    if op == "write":
        T, hq, hkv, hd, page = (case[k] for k in ("tokens", "hq", "hkv", "hd", "page"))
        blocks = -(-T // page) + 3
        st["qkv"] = (1.5 * rnd(T, hq + 2 * hkv, hd)).bfloat16()
        st["positions"] = (torch.arange(T, device=dev) + ints(0, 8000, 1)).int()
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"])
        f = torch.arange(16384, dtype=torch.float64, device=dev)[:, None] * inv
        st["cos_sin"] = torch.cat([f.cos(), f.sin()], -1).float()
        st["q_weight"] = (1 + 0.2 * rnd(hd)).bfloat16() if case["norm"] else None
        st["k_weight"] = (1 + 0.2 * rnd(hd)).bfloat16() if case["norm"] else None
        st["slots"] = torch.randperm(blocks * page, device=dev, generator=gen)[:T]
        st["slots"][T - case["pad"]:] = -1
        width, dtype = (_row_bytes(hd), torch.uint8) if case["bits"] == 4 else (hd, torch.bfloat16)
        st["kv"] = _pool(blocks, page, hkv, width, case["order"], dtype, dev)
        st["eps"] = 1e-6
        return st
    hkv, hd, page = case["hkv"], case["hd"], case["page"]
    if op == "read":
        B, lens = 1, torch.tensor([case["tokens"]], device=dev)
    else:
        B = case["batch"]
        lens = torch.full((B,), case["max_len"], device=dev)
        if case["spread"]:
            lens = ints(1, case["max_len"] + 1, B)
            if B > 3:
                lens[B // 3] = 0
    nb = -(-int(case["tokens"] if op == "read" else case["max_len"]) // page)
    st["kv"] = _pool(B * nb + 1, page, hkv, _row_bytes(hd), case["order"], torch.uint8, dev)
    table = torch.randperm(B * nb, device=dev, generator=gen).view(B, nb) + 1
    pos = torch.arange(nb * page, device=dev).view(nb, page)
    chan = 1 + 3 * (rnd(2, hkv, hd) > 2).float()  # a few channels stand out, as in trained models
    for b in range(B):
        x = rnd(nb, 2, page, hkv, hd) * chan[None, :, None]
        x[:, 1] += 0.25
        x = x.bfloat16()
        rows = torch.stack([_rows(x[:, 0], False), _rows(x[:, 1], True)], 1)
        live = (pos < lens[b])[:, None, :, None, None]  # behind the last token lies what was there before
        st["kv"][table[b]] = torch.where(live, rows, torch.full_like(rows, 255))
    if op == "read":
        t = torch.arange(case["tokens"], device=dev)
        st["slots"] = table[0][t // page] * page + t % page
        return st
    st["block_table"] = table.int()
    st["seq_lens"] = lens.int()
    st["q"] = (1.5 * rnd(B, case["hq"], hd)).bfloat16()
    st["scale"] = 1 / math.sqrt(hd)
    st["counters"] = torch.zeros(B * case["hq"], dtype=torch.int32, device=dev)
    return st


# ---------------------------------------------------------------- one pass


def run(state):
    op = state["op"]
    if own:
        from kvbm_b200.ops import kv4_ops, table_ops

        if op == "tables":
            t = table_ops.batch_tables(state["query_lens"], state["context_lens"], state["block_ids"],
                                       page=state["page"], max_blocks=state["max_blocks"], num_tokens=state["tokens"],
                                       block_counts=state["block_counts"], table=state["table"],
                                       rows=state["table_rows"])
            return [t.block_table, t.seq_lens, t.cu_query, t.positions, t.slots]
        if op == "slots":
            return [table_ops.slot_map(state["block_table"], state["positions"], page=state["page"])]
        if op == "write":
            qkv = state["qkv"]
            q_out = torch.empty(qkv.shape[0], state["hq"], state["hd"], dtype=qkv.dtype, device=qkv.device)
            k_out = torch.empty(qkv.shape[0], state["hkv"], state["hd"], dtype=qkv.dtype, device=qkv.device) \
                if state["keep_k"] else None
            kv4_ops.qk_norm_rope_kv_write(qkv, state["positions"], state["cos_sin"], state["hq"], state["hkv"],
                                          state["kv"], state["slots"], q_weight=state["q_weight"],
                                          k_weight=state["k_weight"], eps=state["eps"], q_out=q_out, k_out=k_out)
            out = [q_out] + ([k_out] if state["keep_k"] else [])
            if state["bits"] == 16:
                return out + [state["kv"]]
            return out + list(kv4_ops.kv4_gather(state["kv"], state["slots"]))
        if op == "read":
            return list(kv4_ops.kv4_gather(state["kv"], state["slots"]))
        return [kv4_ops.paged_decode_attn_kv4(state["q"], state["kv"], state["block_table"], state["seq_lens"],
                                              state["scale"])]
    if op == "tables":
        return _plain_tables(state)
    if op == "slots":
        t, p, page = state["block_table"], state["positions"].long(), state["page"]
        return [t.gather(1, (p // page)[:, None])[:, 0].long() * page + p % page]
    if op == "write":
        return _plain_write(state)
    if op == "read":
        k, v = _plain_read(state["kv"], state["slots"], state["hd"])
        return [k.bfloat16(), v.bfloat16()]
    return _plain_attn(state)


def _plain_tables(st):
    page, T, nb = st["page"], st["tokens"], st["max_blocks"]
    q, ctx = st["query_lens"].long(), st["context_lens"].long()
    seq = ctx + q
    counts = (seq + page - 1) // page if st["block_counts"] is None else st["block_counts"].long()
    cu = torch.cat([torch.zeros_like(q[:1]), q.cumsum(0)])
    first = counts.cumsum(0) - counts
    j = torch.arange(nb, device=q.device)
    have = j[None] < counts[:, None]
    ids = st["block_ids"].long()
    table = torch.where(have, ids[torch.where(have, first[:, None] + j, 0)], 0)
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = t < cu[-1]
    b = torch.where(live, b, 0)
    pos = torch.where(live, ctx[b] + t - cu[b], 0)
    col = pos // page
    ok = live & (col < nb) & (col < counts[b])
    slot = torch.where(ok, table[b, torch.where(ok, col, 0)] * page + pos % page, -1)
    if st["table"] is not None:
        st["table"][st["table_rows"].long()] = table.int()
        table = st["table"]
    return [table.int(), seq.int(), cu.int(), pos.int(), slot]


def _plain_write(st):
    hq, hkv, hd, rot = st["hq"], st["hkv"], st["hd"], st["rot"]
    x = st["qkv"].float()
    cs = st["cos_sin"][st["positions"].long()][:, None]
    c, s = cs[..., : rot // 2], cs[..., rot // 2:]

    def turn(y, w):
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + st["eps"]) * w.float()
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1).bfloat16()

    q = turn(x[:, :hq], st["q_weight"])
    k = turn(x[:, hq: hq + hkv], st["k_weight"])
    v = st["qkv"][:, hq + hkv:]
    out = [q, k] if st["keep_k"] else [q]
    live = (st["slots"] >= 0)
    if st["bits"] == 16:
        n = x.shape[0] - st["pad"]
        at = st["slots"][:n]
        page = st["page"]
        st["kv"][at // page, 0, at % page] = k[:n]
        st["kv"][at // page, 1, at % page] = v[:n]
        return out + [st["kv"]]

    def held(y):
        codes, scale, zero = _quantise(y)
        z = (codes * scale[..., None] + zero[..., None]).flatten(-2)
        return torch.where(live[:, None, None], z, 0.0).bfloat16()

    return out + [held(k), held(v)]


def _plain_values(rows, hd, value):
    """uint8 rows [..., row bytes] -> fp32 [..., hd]."""
    ng = hd // GROUP
    by = rows[..., : hd // 2]
    codes = torch.stack([by & 15, by >> 4], -1).flatten(-2).float()
    if value:
        codes = codes.unflatten(-1, (8, ng, 4)).transpose(-3, -2).flatten(-3)
    par = rows[..., hd // 2: hd // 2 + 4 * ng].contiguous().view(torch.bfloat16).float().unflatten(-1, (ng, 2))
    return (codes.unflatten(-1, (ng, GROUP)) * par[..., :1] + par[..., 1:]).flatten(-2)


def _plain_read(kv, slots, hd):
    page = kv.shape[2]
    rows = kv[slots // page, :, slots % page]
    return _plain_values(rows[:, 0], hd, False), _plain_values(rows[:, 1], hd, True)


def _plain_attn(st):
    hd, hkv, hq = st["hd"], st["hkv"], st["hq"]
    q = st["q"].float()
    B = q.shape[0]
    rows = st["kv"][st["block_table"].long()]  # [B, blocks, 2, page, heads, row]
    k = _plain_values(rows[:, :, 0].flatten(1, 2), hd, False)
    v = _plain_values(rows[:, :, 1].flatten(1, 2), hd, True)
    live = torch.arange(k.shape[1], device=q.device)[None] < st["seq_lens"][:, None]
    s = torch.einsum("bhgd,bnhd->bhgn", q.view(B, hkv, hq // hkv, hd), k) * st["scale"]
    s = torch.where(live[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    v = torch.where(live[:, :, None, None], v, 0.0)
    o = torch.einsum("bhgn,bnhd->bhgd", p, v) / torch.where(l > 0, l, 1.0)
    return [o.reshape(B, hq, hd).bfloat16()]


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    op, page = case["op"], case["page"]
    if op == "tables":
        q, ctx, ids = (st[k].cpu().numpy().astype(np.int64) for k in ("query_lens", "context_lens", "block_ids"))
        B, nb, T = len(q), case["max_blocks"], case["tokens"]
        table = np.zeros((B, nb), np.int32)
        pos, slot = np.zeros(T, np.int32), np.full(T, -1, np.int64)
        t = o = 0
        for b in range(B):
            n = -(-(q[b] + ctx[b]) // page) if st["block_counts"] is None else int(st["block_counts"][b])
            mine = ids[o: o + n][:nb]
            table[b, : len(mine)] = mine
            p = np.arange(ctx[b], ctx[b] + q[b])
            at = np.full(len(p), -1, np.int64)
            ok = p // page < len(mine)
            at[ok] = mine[p[ok] // page] * page + p[ok] % page
            room = max(0, min(len(p), T - t))
            pos[t: t + room], slot[t: t + room] = p[:room], at[:room]
            t, o = t + len(p), o + n
        if st["table"] is not None:
            full = st["table"].cpu().numpy()
            full[st["table_rows"].cpu().numpy()] = table
            table = full
        cu = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        return [table, (q + ctx).astype(np.int32), cu, pos, slot]
    if op == "slots":
        t, p = st["block_table"].cpu().numpy().astype(np.int64), st["positions"].cpu().numpy().astype(np.int64)
        return [t[np.arange(len(p)), p // page] * page + p % page]
    hd, hkv = case["hd"], case["hkv"]
    if op == "write":
        hq, half = case["hq"], case["rot"] // 2
        x = st["qkv"].double()
        ang = st["cos_sin"].double()[st["positions"].long()].unsqueeze(1)
        heads = x[:, : hq + hkv].clone()
        if case["norm"]:
            heads /= (heads.pow(2).sum(-1, keepdim=True) / hd + st["eps"]).sqrt()
            heads[:, :hq] *= st["q_weight"].double()
            heads[:, hq:] *= st["k_weight"].double()
        first, second = heads[..., :half].clone(), heads[..., half: 2 * half].clone()
        heads[..., :half] = first * ang[..., :half] - second * ang[..., half:]
        heads[..., half: 2 * half] = first * ang[..., half:] + second * ang[..., :half]
        q, k, v = heads[:, :hq], heads[:, hq:], x[:, hq + hkv:]
        out = [q, k] if case["keep_k"] else [q]
        if case["bits"] == 16:
            kv = st["kv"].double()
            n = case["tokens"] - case["pad"]
            flat = st["slots"][:n]
            kv[flat // page, 0, flat % page] = k[:n]
            kv[flat // page, 1, flat % page] = v[:n]
            return out + [kv]

        def held(y):
            g = y.reshape(*y.shape[:-1], hd // GROUP, GROUP)
            least = g.min(-1, keepdim=True).values
            step = (g.max(-1, keepdim=True).values - least) / 15
            mant, expo = torch.frexp(step)  # up to 8 significant bits
            step = torch.ldexp(torch.ceil(mant * 256) / 256, expo)
            safe = torch.where(step > 0, step, 1.0)
            near = least + torch.round((g - least) / safe).clamp(0, 15) * step
            return torch.where((st["slots"] >= 0)[:, None, None], near.reshape(y.shape), 0.0)

        return out + [held(k.bfloat16().double()), held(v)]

    lane = torch.arange(hd, device=st["kv"].device)
    nib_v = 4 * ((hd // GROUP) * (lane % GROUP // 4) + lane // GROUP) + lane % 4

    def value(rows, nib):
        code = (rows[..., nib // 2].int() >> (4 * (nib % 2)).int()) & 15
        w = rows[..., hd // 2:].int()
        at = 4 * (lane // GROUP)

        def half(k):  # a bf16 is the upper half of an fp32
            bits = (w[..., at + k] << 16) | (w[..., at + k + 1] << 24)
            return bits.contiguous().view(torch.float32).double()

        return half(0) * code + half(2)

    if op == "read":
        rows = st["kv"][st["slots"] // page, :, st["slots"] % page]
        return [value(rows[:, 0], lane), value(rows[:, 1], nib_v)]
    B, hq = case["batch"], case["hq"]
    out = torch.zeros(B, hq, hd, dtype=torch.float64, device=st["q"].device)
    for b, n in enumerate(st["seq_lens"].tolist()):
        if n:
            rows = st["kv"][st["block_table"][b, : -(-n // page)].long()]
            k = value(rows[:, 0].reshape(-1, hkv, rows.shape[-1])[:n], lane)
            v = value(rows[:, 1].reshape(-1, hkv, rows.shape[-1])[:n], nib_v)
            for h in range(hkv):
                a = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                w = torch.softmax(st["q"][b, a].double() @ k[:, h].T * st["scale"], -1)
                out[b, a] = w @ v[:, h]
    return [out]
