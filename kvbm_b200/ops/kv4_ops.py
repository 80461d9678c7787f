"""Python entry points of the 4-bit paged KV cache (sm_100a, libkvbm_cuda.so).

A 4-bit cache is a uint8 pool whose ``head_dim`` is :func:`row_bytes` of the model's: 48, 80 or 160 bytes for
64, 128 or 256 elements, against 128, 256 or 512 in bf16. Groups of 32 elements share a scale and a zero (the
group's least value), both bf16; an element is ``zero + code * scale`` and off by at most half a scale. Since a
row is plain bytes, the pool is offloaded, onboarded, resharded by heads and pushed like any other.

``kv`` below is one layer of a pool, ``[num_blocks, 2, page, heads, row]``: ``KvLayout.layer_view(layer)`` or any
tensor of that shape with unit inner stride and the other strides multiples of 16 bytes (token-first, head-first
and universal pools alike). Block ids and slots outside the pool are checked on the device: such a page holds no
tokens, such a slot is not written and reads as zeros.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

GROUP = 32
_HEAD_DIM = {48: 64, 80: 128, 160: 256}  # by row bytes
_ROW_BYTES = {hd: row for row, hd in _HEAD_DIM.items()}


def row_bytes(head_dim: int) -> int:
    """Bytes of one K or V row of ``head_dim`` (64, 128 or 256) elements in 4 bits."""
    row = _ROW_BYTES.get(head_dim)
    if row is not None:
        return row
    raise ValueError(f"a 4-bit cache takes head_dim 64, 128 or 256, not {head_dim}")


def _cache_args(kv: torch.Tensor, device, bits: int = 4) -> tuple:
    if kv.dim() != 5 or kv.shape[1] != 2:
        raise ValueError(f"the cache must be [num_blocks, 2, page, heads, row], not {tuple(kv.shape)}")
    if kv.device != device:
        raise ValueError(f"the cache is on {kv.device}, expected {device}")
    if kv.dtype != (torch.uint8 if bits == 4 else torch.bfloat16):
        raise ValueError(f"a {bits}-bit cache is {torch.uint8 if bits == 4 else torch.bfloat16}, not {kv.dtype}")
    nb, _, page, heads, row = kv.shape
    block, outer, token, head, unit = kv.stride()
    # a dimension of one may come with any stride
    block, token, head = block if nb > 1 else 0, token if page > 1 else 0, head if heads > 1 else 0
    ptr = kv.data_ptr()
    if bits == 16:
        block, outer, token, head = 2 * block, 2 * outer, 2 * token, 2 * head
    if (unit != 1 and row > 1) or (ptr | block | outer | token | head) & 15:
        raise ValueError("cache rows need unit stride and 16-byte aligned starts")
    return (ptr, block, outer, token, head, page, nb), heads, row


def _vec(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, device) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} [{n}] on {device}")


def _weight(w: torch.Tensor | None, name: str, hd: int, device) -> int | None:
    if w is None:
        return None
    _vec(w, name, torch.bfloat16, hd, device)
    ptr = w.data_ptr()
    if ptr & 15:
        raise ValueError(f"{name} must be 16-byte aligned")
    return ptr


def _rows_out(o: torch.Tensor | None, name: str, shape: tuple, device) -> int | None:
    if o is None:
        return None
    ptr = o.data_ptr()
    if o.shape != shape or o.dtype != torch.bfloat16 or not o.is_contiguous() or o.device != device or ptr & 15:
        raise ValueError(f"{name} must be a contiguous bf16 {list(shape)} on {device}")
    return ptr


def qk_norm_rope_kv_write(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, hq: int, hkv: int,
                          kv: torch.Tensor, slots: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None, eps: float = 1e-6, q_out: torch.Tensor | None = None,
                          k_out: torch.Tensor | None = None, stream=None) -> None:
    """RMSNorm of every q and k head, RoPE and the write of k and v into a paged cache, in one pass.

    qkv: bf16 [T, hq + 2 * hkv, hd], hd 64, 128 or 256, heads contiguous (rows may be strided). ``q_weight`` /
    ``k_weight`` (bf16 [hd]) scale the normalised head; without one that norm is left out. ``cos_sin`` is fp32
    [max_position, rot]: cos then sin of the rotate-half convention over the first ``rot`` (a multiple of 16)
    elements. ``kv`` is bf16 (hd wide) or uint8 (:func:`row_bytes` wide: 4 bits); the cache takes k and v as
    rounded to bf16, at ``slots`` (int64 [T], distinct; one outside the pool is not written). Norm and rotation
    are fp32, every operation rounded by itself.

    Without ``q_out`` q and k are rotated in place in ``qkv``. With ``q_out`` (bf16 [T, hq, hd]) ``qkv`` stays as
    it is: the rotated q go there and k to the cache and, if given, to ``k_out`` (bf16 [T, hkv, hd]). A token
    whose position is outside ``cos_sin`` is left alone altogether.
    """
    dev = qkv.device
    if qkv.dim() != 3 or qkv.dtype != torch.bfloat16:
        raise ValueError("qkv must be bf16 [T, hq + 2 * hkv, hd]")
    T, H, hd = qkv.shape
    if hq < 0 or hkv < 1 or H != hq + 2 * hkv:
        raise ValueError(f"qkv has {H} heads, expected {hq} + 2 * {hkv}")
    if hd not in (64, 128, 256):
        raise ValueError(f"qk_norm_rope_kv_write takes head_dim 64, 128 or 256, not {hd}")
    token_stride, head_stride, unit = qkv.stride()
    if unit != 1 or (H > 1 and head_stride != hd) or (T > 1 and token_stride & 7) or qkv.data_ptr() & 15:
        raise ValueError("qkv needs contiguous heads and 16-byte aligned tokens")
    if T > 1 and token_stride < H * hd and q_out is None:
        raise ValueError("tokens of qkv that overlap cannot be rotated in place")
    bits = 16 if kv.dtype == torch.bfloat16 else 4
    cache, heads, row = _cache_args(kv, dev, bits)
    if heads != hkv or row != (hd if bits == 16 else row_bytes(hd)):
        raise ValueError(f"the cache holds {heads} heads of {row}, expected {hkv} of "
                         f"{hd if bits == 16 else row_bytes(hd)}")
    _vec(positions, "positions", torch.int32, T, dev)
    _vec(slots, "slots", torch.int64, T, dev)
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.device != dev \
            or cos_sin.data_ptr() & 15:
        raise ValueError("cos_sin must be a contiguous fp32 [max_position, rot] on the same device")
    max_pos, rot = cos_sin.shape
    if rot < 16 or rot > hd or rot % 16:
        raise ValueError(f"rot {rot} must be a multiple of 16 up to head_dim {hd}")
    if k_out is not None and q_out is None:
        raise ValueError("k_out needs q_out")
    qw = _weight(q_weight, "q_weight", hd, dev)
    kw = _weight(k_weight, "k_weight", hd, dev)
    qo = _rows_out(q_out, "q_out", (T, hq, hd), dev)
    if q_out is not None and hq == 0:
        qo = qkv.data_ptr()  # an empty tensor has no address, and none would mean in place: nothing is written there
    ko = _rows_out(k_out, "k_out", (T, hkv, hd), dev)
    with _lib.on_device(dev, stream) as st:
        _lib.call("kvbm_qk_norm_rope_kv_write", qkv.data_ptr(), token_stride, T, hq, hkv, hd, rot,
                  positions.data_ptr(), cos_sin.data_ptr(), max_pos, qw, kw, eps, bits, *cache, slots.data_ptr(),
                  qo, ko, st)


def kv4_gather(kv: torch.Tensor, slots: torch.Tensor, *, k_out: torch.Tensor | None = None,
               v_out: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows of a 4-bit cache at ``slots`` (int64 [T]) as bf16 [T, heads, head_dim]."""
    dev = kv.device
    cache, heads, row = _cache_args(kv, dev)
    hd = _HEAD_DIM.get(row)
    if hd is None:
        raise ValueError(f"a 4-bit cache has rows of 48, 80 or 160 bytes, not {row}")
    T = slots.numel()
    _vec(slots, "slots", torch.int64, T, dev)
    shape = (T, heads, hd)
    _rows_out(k_out, "k_out", shape, dev)
    _rows_out(v_out, "v_out", shape, dev)
    with _lib.on_device(dev, stream) as st:
        if k_out is None:
            k_out = kv.new_empty(shape, dtype=torch.bfloat16)
        if v_out is None:
            v_out = torch.empty_like(k_out)
        _lib.call("kvbm_kv4_gather", *cache, heads, hd, slots.data_ptr(), T, k_out.data_ptr(), v_out.data_ptr(), st)
    return k_out, v_out


@functools.lru_cache(maxsize=256)
def _decode_plan(batch: int, hq: int, hkv: int, hd: int, max_tokens: int, ctas: int, device: int) -> tuple:
    """(floats of scratch, SMs) of a launch of these sizes."""
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    out = (C.c_int64 * 2)()
    _lib.check(_lib.load().kvbm_paged_decode_attn_kv4_plan(batch, hq, hkv, hd, min(max_tokens, 2 ** 31 - 1), ctas, sms,
                                                           out), "kvbm_paged_decode_attn_kv4_plan")
    return int(out[0]), sms


def kv4_decode_scratch(batch: int, hq: int, hkv: int, head_dim: int, max_tokens: int, ctas: int = 0,
                       device=None) -> int:
    """Floats of scratch that :func:`paged_decode_attn_kv4` takes for these sizes (``max_tokens``: the block
    table's width in tokens); 0 where requests are too short to be cut."""
    dev = torch.device(device if device is not None else "cuda")
    return _decode_plan(batch, hq, hkv, head_dim, max_tokens, ctas,
                        dev.index if dev.index is not None else torch.cuda.current_device())[0]


def paged_decode_attn_kv4(q: torch.Tensor, kv: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                          softmax_scale: float, *, ctas: int = 0, scratch: torch.Tensor | None = None,
                          out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of one token per request over a 4-bit paged cache. q: bf16 [B, Hq, hd]; returns the same.

    Hq is a multiple of the cache's heads. ``block_table`` (int32 [B, max_blocks]) and ``seq_lens`` (int32 [B])
    as for the 16-bit kernel; a length beyond the table counts as the table's, one of 0 or less gives zeros, and a
    page whose id is outside the pool holds no tokens. The work is cut evenly over ``ctas`` CTAs (0: as many as
    the GPU holds at a time), whatever the lengths; results of requests that several CTAs share go through
    ``scratch`` (fp32, :func:`kv4_decode_scratch` entries; made here if not given, nothing in it outlives the
    call). Launches that may overlap need a scratch each. A launch whose copies do not arrive gives up: its results
    are NaN, and :func:`check_kv4_status` raises.
    """
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise ValueError("q must be bf16 [B, Hq, hd]")
    dev = q.device
    B, hq, hd = q.shape
    cache, hkv, row = _cache_args(kv, dev)
    if row != row_bytes(hd):
        raise ValueError(f"the cache's rows of {row} bytes do not hold head_dim {hd}")
    if hq < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads are not a multiple of the cache's {hkv}")
    row_stride, head_stride, unit = q.stride()
    if unit != 1 or (hq > 1 and head_stride != hd) or (B > 1 and row_stride & 7) or q.data_ptr() & 15:
        raise ValueError("q needs contiguous heads and 16-byte aligned rows")
    if B > 65535:
        raise ValueError(f"at most 65,535 requests, got {B}")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype != torch.int32 or \
            block_table.device != dev or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{B}, max_blocks] with unit inner stride on {dev}")
    _vec(seq_lens, "seq_lens", torch.int32, B, dev)
    max_blocks = block_table.shape[1]
    if ctas < 0:
        raise ValueError("ctas must not be negative")
    if scratch is not None and (scratch.dtype != torch.float32 or scratch.device != dev
                                or not scratch.is_contiguous() or scratch.data_ptr() % 16):
        raise ValueError(f"scratch must be 16-byte aligned fp32 on {dev}")
    _rows_out(out, "out", (B, hq, hd), dev)
    with _lib.on_device(dev, stream) as st:
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if B == 0:
            return out
        need, sms = _decode_plan(B, hq, hkv, hd, max_blocks * kv.shape[2], ctas, dev.index)
        if scratch is None:
            if need > 0:
                scratch = torch.empty(need, dtype=torch.float32, device=dev)
        elif scratch.numel() < need:
            raise ValueError(f"scratch holds {scratch.numel()} floats, {need} are needed")
        _lib.call("kvbm_paged_decode_attn_kv4", q.data_ptr(), row_stride, *cache, block_table.data_ptr() or None,
                  block_table.stride(0), max_blocks, seq_lens.data_ptr(), B, hq, hkv, hd, softmax_scale, ctas, sms,
                  scratch.data_ptr() if need > 0 else None, out.data_ptr(), st)
        if need > 0:
            _lib.count_launches(1)
    return out


def _index(device) -> int:
    dev = torch.device(device) if device is not None else None
    return dev.index if dev is not None and dev.index is not None else torch.cuda.current_device()


def kv4_status(reset: bool = True, device=None) -> int:
    """0, or the error a :func:`paged_decode_attn_kv4` launch recorded on ``device`` (None: the current one) since the
    last reset; 3: a wait for a copy timed out, and the launch's results are NaN. Synchronizes the device."""
    dev = _index(device)
    torch.cuda.synchronize(dev)
    return int(_lib.load().kvbm_kv4_status(dev, 1 if reset else 0))


def check_kv4_status(device=None) -> None:
    """Raise (and clear the status) if a :func:`paged_decode_attn_kv4` launch on ``device`` recorded an error. A host
    read of mapped memory without synchronization: it sees the launches that the host has waited for."""
    st = int(_lib.load().kvbm_kv4_status(_index(device), 1))
    if st:
        raise _lib.KvbmCudaError(f"decode attention over a 4-bit cache failed on the device: status {st} "
                                 "(a wait for a copy timed out; the results of that launch are NaN)")


def set_kv4_wait_limit_ns(ns: int | None) -> None:
    """After how long a launch from here on gives a copy up: 0 at once, None the default of one second."""
    _lib.load().kvbm_kv4_set_wait_limit_ns(-1 if ns is None else int(ns))


# ------------------------------------------------------------- rows on the host


def pack_rows(x: torch.Tensor, value: bool) -> torch.Tensor:
    """bf16 [..., head_dim] as 4-bit rows (uint8 [..., row_bytes]) in plain torch: what the write kernel stores.
    ``value`` selects the V order of the codes."""
    hd = x.shape[-1]
    row, ng = row_bytes(hd), hd // GROUP
    g = x.to(torch.bfloat16).float().unflatten(-1, (ng, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = (0.5 * hi - 0.5 * lo) / torch.full_like(lo, 7.5)
    up = ((s.contiguous().view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)
    up = torch.where(s < 2.0 ** -126, torch.zeros_like(s), up)
    c = ((0.5 * g - 0.5 * lo) / torch.where(up > 0, 0.5 * up, torch.ones_like(up))).round().clamp(0, 15)
    fine = g.isfinite().all(-1, keepdim=True)
    c = torch.where(fine, c, 0.0)
    if value:
        c = c.unflatten(-1, (8, 4)).transpose(-3, -2)  # (group, 8, 4) -> (8, group, 4)
    c = c.reshape(*x.shape[:-1], hd // 2, 2).to(torch.uint8)
    par = torch.cat([up, torch.where(fine, lo, 0.0)], -1).contiguous().view(torch.int32) >> 16
    par[..., :1] = torch.where(fine, par[..., :1], 0x7FC0)  # the same NaN on every device
    par = par.to(torch.int16).flatten(-2).view(torch.uint8)
    pad = torch.zeros(*x.shape[:-1], row - hd // 2 - 4 * ng, dtype=torch.uint8, device=x.device)
    return torch.cat([c[..., 0] | (c[..., 1] << 4), par, pad], -1)


def unpack_rows(rows: torch.Tensor, value: bool) -> torch.Tensor:
    """4-bit rows (uint8 [..., row_bytes]) as fp32 [..., head_dim], in plain torch."""
    hd = _HEAD_DIM.get(rows.shape[-1])
    if hd is None:
        raise ValueError(f"a 4-bit cache has rows of 48, 80 or 160 bytes, not {rows.shape[-1]}")
    ng = hd // GROUP
    c = torch.stack([rows[..., : hd // 2] & 15, rows[..., : hd // 2] >> 4], -1).flatten(-2).double()
    if value:
        c = c.unflatten(-1, (8, ng, 4)).transpose(-3, -2).flatten(-3)
    par = rows[..., hd // 2: hd // 2 + 4 * ng].contiguous().view(torch.bfloat16).double().unflatten(-1, (ng, 2))
    # the product is exact in 64 bits: one rounding, as the kernels' fused multiply-add has
    return (c.unflatten(-1, (ng, GROUP)) * par[..., :1] + par[..., 1:]).flatten(-2).float()
