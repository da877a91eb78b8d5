"""Host side of the committed prefix's attention: the paged key / value cache and the attention over it.

* ``kv_cache_write`` -- new keys and values into cache slots, as they are or quantised to 8 bits;
* ``kv_cache_read`` -- slots back as rows of the model's type;
* ``paged_attention`` -- new rows (a prefill chunk, single tokens, a draft tree's nodes) over each
  sequence's pages; with ``causal=False`` and a tree's nodes it gives the prefix half that
  ``tree_attn_merge`` merges with.

A cache is [blocks, page, Hkv, D] of the model's type (bf16 or fp16), or of ``torch.float8_e4m3fn`` with a
byte [blocks, page, Hkv] (uint8) per slot and head: byte c, 1 to 254, stands for the scale 2^(c - 127).  Slot n is row
n % page of block n / page.  The blocks of a cache may be strided (two halves of one allocation); within a
block it is contiguous.  No call synchronises with the host.
"""
from __future__ import annotations

import torch

from chain_flow_amd import _lib

_TYPES = (torch.bfloat16, torch.float16)


def _laid(t, want):
    """Whether a tensor's strides behind the first are as wanted; those over a single element may be anything."""
    got = t.stride()[1:]
    return got == want or all(n == 1 or g == w for n, g, w in zip(t.shape[1:], got, want))


def _check_cache(k_cache, v_cache, k_exp, v_exp, dtype):
    """-> (blocks, page, Hkv, D, block strides of k and v) of a cache that serves rows of ``dtype``."""
    shape = k_cache.shape
    blocks, page, Hkv, D = shape
    kind = k_cache.dtype
    if v_cache.shape != shape or v_cache.dtype != kind:
        raise ValueError("k_cache and v_cache must share one shape and type")
    if not blocks * page * Hkv:
        raise ValueError(f"a cache of shape {tuple(shape)} holds nothing")
    if D != 128 and D != 256 and D != 64:
        raise ValueError(f"head width {D} is not 64, 128 or 256")
    if kind == torch.float8_e4m3fn:
        for e in (k_exp, v_exp):
            if e is None or e.dtype != torch.uint8 or e.shape != shape[:3] or not e.is_contiguous():
                raise ValueError(f"an 8-bit cache needs contiguous uint8 k_exp and v_exp [{blocks}, {page}, {Hkv}]")
    elif kind != dtype or k_exp is not None or v_exp is not None:
        raise ValueError(f"the cache must be {dtype} without exponents, or float8_e4m3fn with them")
    row = Hkv * D
    inner = page * row
    want = (row, D, 1)
    bs_k, bs_v = (inner, inner) if blocks == 1 else (k_cache.stride(0), v_cache.stride(0))
    if (not _laid(k_cache, want) or not _laid(v_cache, want) or bs_k < inner or bs_v < inner or (bs_k | bs_v) % 16
            or (k_cache.data_ptr() | v_cache.data_ptr()) % 16):
        raise ValueError("cache blocks must be contiguous [page, Hkv, D], on strides of 16 elements and 16-byte "
                         "boundaries")
    return blocks, page, Hkv, D, bs_k, bs_v


def _rows(t):
    """Rows [T, heads, D] with contiguous heads whose vector loads are aligned (copied where they are not), and
    their stride."""
    T, h, D = t.shape
    ld = t.stride(0) if T > 1 else h * D
    if not _laid(t, (D, 1)) or ld < h * D or ld % 8 or t.data_ptr() % 16:
        t, ld = _lib.aligned(t.contiguous()), h * D
    return t, ld


def kv_cache_write(key, value, k_cache, v_cache, slots, *, k_exp=None, v_exp=None, status=None) -> None:
    """key, value [T, Hkv, D] bf16 or fp16 (rows may be strided) into ``slots`` [T] of the cache, in place.

    With an 8-bit cache each (row, head) gets the least power-of-two scale, from 2^-126 up, that brings its
    largest finite magnitude to 448 or below; its elements are rounded to e4m3 once (nearest even; they end
    at 240 where 256 times the scale exceeds the type's largest value, so that what was finite reads back
    finite), NaN and infinities are stored as NaN.

    A negative slot is a padding row (skipped).  A slot past the cache is skipped and sets ``status`` (int32
    [1] on the device, zeroed by the caller), if given, to 1.  Slots of one call must differ: rows that share
    one race, and what the slot then holds is undefined (a host tensor's are checked here)."""
    if key.dtype not in _TYPES or value.dtype != key.dtype or value.shape != key.shape:
        raise ValueError("key and value must be bf16 or fp16 tensors of one shape [T, Hkv, D]")
    blocks, page, Hkv, D, bs_k, bs_v = _check_cache(k_cache, v_cache, k_exp, v_exp, key.dtype)
    T = key.shape[0]
    if key.shape != (T, Hkv, D) or slots.shape != (T,):
        raise ValueError(f"key and value must be [T, {Hkv}, {D}] and slots [T]")
    dev = _lib.device_of(key, value, k_cache, v_cache, k_exp, v_exp, status=status)
    if not slots.is_cuda:
        used = slots[slots >= 0]
        if used.unique().numel() != used.numel() or (used >= blocks * page).any():
            raise ValueError(f"slots must be distinct and below {blocks * page}")
    slots = _lib.index32(slots, dev)
    key, ld_k = _rows(key)
    value, ld_v = _rows(value)
    _lib.check(_lib.lib().cfh_kv_write(
        key.data_ptr(), ld_k, value.data_ptr(), ld_v, T, Hkv, D, key.dtype == torch.bfloat16, k_cache.data_ptr(), bs_k,
        v_cache.data_ptr(), bs_v, _lib.ptr(k_exp), _lib.ptr(v_exp), blocks, page, slots.data_ptr(), _lib.ptr(status),
        _lib.stream_of(dev)), "cfh_kv_write")


def kv_cache_read(k_cache, v_cache, slots, *, dtype=None, k_exp=None, v_exp=None, status=None):
    """``slots`` [T] of the cache as rows -> (key, value) [T, Hkv, D] of ``dtype`` (default: the cache's type, bf16
    for an 8-bit cache); 8-bit elements are multiplied by their scale and rounded to nearest even.  A negative
    slot, and one past the cache (which sets ``status``), gives a zero row."""
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype == torch.float8_e4m3fn else k_cache.dtype
    if dtype not in _TYPES:
        raise ValueError("rows are read as bf16 or fp16")
    blocks, page, Hkv, D, bs_k, bs_v = _check_cache(k_cache, v_cache, k_exp, v_exp, dtype)
    if slots.dim() != 1:
        raise ValueError("slots must be [T]")
    dev = _lib.device_of(k_cache, v_cache, k_exp, v_exp, status=status)
    slots = _lib.index32(slots, dev)
    T = slots.shape[0]
    key = k_cache.new_empty((T, Hkv, D), dtype=dtype)
    value = torch.empty_like(key)
    _lib.check(_lib.lib().cfh_kv_read(
        k_cache.data_ptr(), bs_k, v_cache.data_ptr(), bs_v, _lib.ptr(k_exp), _lib.ptr(v_exp), blocks, page,
        slots.data_ptr(), T, Hkv, D, dtype == torch.bfloat16, key.data_ptr(), value.data_ptr(), _lib.ptr(status),
        _lib.stream_of(dev)), "cfh_kv_read")
    return key, value


def paged_attention(query, k_cache, v_cache, block_table, seq_lens, cu_q, *, scale: float, causal: bool = True,
                    k_exp=None, v_exp=None, max_len: int | None = None, out=None, status=None):
    """query [T, H, D] (rows may be strided; H a multiple of Hkv) over the cache: sequence s has the query rows
    cu_q[s] .. cu_q[s + 1] (ascending) and seq_lens[s] tokens in blocks block_table[s]; row i of its n sees token j where
    j < len and, if ``causal``, j <= len - n + i (the rows' own keys and values are the cache's last n, written
    before the call).  -> (out [T, H, D] of the query's type, lse [H, T] fp32: ``tree_attn_merge``'s prefix_lse).

    A row that sees no token gives 0 and -inf.  Rows of no sequence stay as they were in ``out`` (0 without it); their
    lse is -inf.  Lengths, tables and bounds are read on the device only: a negative length or one past the table, and
    rows that see a token of a block outside the cache, give NaN; a sequence whose rows do not lie in the query is
    skipped, and where a bound falls below the one before it that sequence and all behind it are; each sets ``status``
    (int32 [1], zeroed by the caller), if given, to 1.  ``max_len``: an upper bound of the lengths (default: what the
    table holds); it only plans how the work is split."""
    if query.dtype not in _TYPES:
        raise ValueError("query must be bf16 or fp16")
    blocks, page, Hkv, D, bs_k, bs_v = _check_cache(k_cache, v_cache, k_exp, v_exp, query.dtype)
    T, H, Dq = query.shape
    if Dq != D or H % Hkv:
        raise ValueError(f"query must be [T, H, {D}] with H a multiple of {Hkv}")
    S = seq_lens.shape[0]
    if seq_lens.shape != (S,) or cu_q.shape != (S + 1,) or block_table.dim() != 2 or block_table.shape[0] != S:
        raise ValueError("seq_lens must be [S], cu_q [S + 1] and block_table [S, blocks]")
    dev = _lib.device_of(query, k_cache, v_cache, k_exp, v_exp, status=status)
    fresh = out is None
    if fresh:
        out = query.new_empty((T, H, D))
        o_ld = H * D
    else:
        o_ld = out.stride(0) if T > 1 else H * D
        if (out.shape != query.shape or out.dtype != query.dtype or out.get_device() != dev or not _laid(out, (D, 1))
                or o_ld < H * D or o_ld % 8 or out.data_ptr() % 16):
            raise ValueError(f"out must be a {query.dtype} [{T}, {H}, {D}] tensor on cuda:{dev} with contiguous heads, "
                             "16-byte aligned")
    table = block_table
    if table.dtype != torch.int32 or table.get_device() != dev:
        table = _lib.index32(table, dev)
    width = table.shape[1]
    if table.stride(1) != 1 or table.stride(0) < width:
        table = table.contiguous()
    lens, cu = _lib.index32(seq_lens, dev), _lib.index32(cu_q, dev)
    most = width * page
    most = most if max_len is None else max(0, min(int(max_len), most))
    query, q_ld = _rows(query)
    L = _lib.lib()
    nws = L.cfh_paged_attn_ws_bytes(T, H, Hkv, D, S, most)
    lse = query.new_empty((H, T), dtype=torch.float32)
    if not S:
        lse.fill_(float("-inf"))
        return out.zero_() if fresh else out, lse
    ws = query.new_empty(nws, dtype=torch.uint8) if nws > 0 else None
    _lib.check(L.cfh_paged_attn_fresh(
        query.data_ptr(), q_ld, T, H, Hkv, D, query.dtype == torch.bfloat16, k_cache.data_ptr(), bs_k, v_cache.data_ptr(),
        bs_v, _lib.ptr(k_exp), _lib.ptr(v_exp), blocks, page, table.data_ptr(), max(table.stride(0), width), width,
        lens.data_ptr(), cu.data_ptr(), S, float(scale), bool(causal), most, out.data_ptr(), o_ld, lse.data_ptr(), _lib.ptr(ws),
        _lib.ptr(status), fresh, _lib.stream_of(dev)), "cfh_paged_attn")
    return out, lse
