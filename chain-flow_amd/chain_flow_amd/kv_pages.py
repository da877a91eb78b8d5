"""Host side of the paged cache's book-keeping: which pages a sequence holds, and how many sequences hold a page.

A pool is three int32 tensors on the device, updated in place by both calls:

* ``block_table`` [S, W]: the pages of each sequence, as ``paged_attention`` reads them (-1: none);
* ``room`` [S]: the tokens that a sequence's pages are for; it holds the first ceil(room / page) entries of its row;
* ``ref`` [blocks]: the sequences that hold a page; 0: free.

``kv_pages_resize`` gives every sequence the pages for its new room (room for a draft tree before a verify, only for what
was accepted behind it, none when a request ends); ``kv_pages_fork`` lets sequences share the pages of others (several
answers to one prompt).  Empty pools are zeros, with a table of -1.  No call synchronises with the host, and the
pages that a call takes depend on the pool and the call alone.
"""
from __future__ import annotations

import torch

from chain_flow_amd import _lib
from chain_flow_amd.kv_cache import _check_pool


def _check_pages(block_table, room, ref, page, status):
    """-> (S, W, row stride, blocks, device index) of a pool's book-keeping."""
    i32 = torch.int32
    if block_table.dtype != i32 or room.dtype != i32 or ref.dtype != i32:
        raise ValueError("block_table, room and ref must be int32: they are updated in place")
    shape = block_table.shape
    if len(shape) != 2 or ref.dim() != 1 or room.shape != shape[:1]:
        raise ValueError("block_table must be [S, W], room [S] and ref [blocks]")
    S, W = shape
    blocks = ref.shape[0]
    ld, one = block_table.stride()
    if S < 2:
        ld = W
    if (one != 1 and W > 1) or ld < W or not room.is_contiguous() or not ref.is_contiguous() or not blocks:
        raise ValueError("block_table must have contiguous rows, room and ref be contiguous, and ref hold a page")
    if page < 1:
        raise ValueError(f"a page of {page} tokens")
    return S, W, ld, blocks, _lib.device_of(block_table, room, ref, status=status)


def kv_pages_fork(block_table, room, ref, src, dst, *, page: int, status=None) -> None:
    """For each i, sequence dst[i] lets go of the pages it holds and shares those of sequence src[i], with its room
    (src[i] = -1: it holds none).  ``src`` and ``dst`` [n]; dst[i] = -1 is padding.  Nothing is copied: a shared last page
    is, when ``kv_pages_resize`` lets one of its holders grow.  (So rows are written behind the room that was shared: a
    sequence with room for more than it holds is resized to its length before it is shared.)

    Destinations must differ, and no source may be another pair's destination: such pairs, and ones whose sequences or rooms do
    not lie in the table, are skipped and set ``status`` (int32 [1], zeroed by the caller), if given, to 1 (host tensors
    are checked here)."""
    S, W, ld, blocks, dev = _check_pages(block_table, room, ref, page, status)
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError("src and dst must be [n]")
    if not src.is_cuda and not dst.is_cuda:
        pairs = [(a, b) for a, b in zip(src.tolist(), dst.tolist()) if b != -1]
        to = [b for _, b in pairs]
        if (len(set(to)) != len(to) or any(not -1 <= a < S or not 0 <= b < S for a, b in pairs)
                or any(a != b and a in set(to) for a, b in pairs)):
            raise ValueError(f"destinations must differ, sources be none of them, and both lie in the {S} sequences")
    src, dst = _lib.index32(src, dev), _lib.index32(dst, dev)
    _lib.check(_lib.lib().cfh_kv_fork(
        block_table.data_ptr(), ld, W, room.data_ptr(), S, ref.data_ptr(), blocks, page, src.data_ptr(), dst.data_ptr(),
        src.shape[0], _lib.ptr(status), _lib.stream_of(dev)), "cfh_kv_fork")


def kv_pages_resize(block_table, room, ref, new_room, *, page: int, k_cache=None, v_cache=None, k_exp=None, v_exp=None,
                    status=None) -> None:
    """Every sequence gets the pages for ``new_room`` [S] tokens (negative: it is left as it is): pages behind are let go
    of (free once no sequence holds them; the call's own takes may have them), missing ones taken, the lowest free ones
    first, in order of the sequences and of their places.  ``room`` becomes ``new_room``.

    Where a sequence grows and its last page is filled in part (by room % page tokens) and shared, it gets a copy of its
    own, but for the last of the growing ones if no other sequence holds the page.  The copy's rows are copied
    in ``k_cache`` and ``v_cache`` (one cache, or those of several layers [layers, blocks, page, Hkv, D]; with their
    exponents); without them only the table changes, which is enough where nothing is shared.

    Where the free pages end, that sequence and all behind it that need one are left as they were and set ``status``
    (int32 [1], zeroed by the caller), if given, to 1; so do rooms that do not lie in the table.  At most 4,096 sequences."""
    S, W, ld, blocks, dev = _check_pages(block_table, room, ref, page, status)
    if new_room.shape != (S,):
        raise ValueError(f"new_room must be [{S}]")
    pool = None
    if k_cache is not None or v_cache is not None:
        if k_cache is None or v_cache is None:
            raise ValueError("k_cache and v_cache go together")
        pool = _check_pool(k_cache, v_cache, k_exp, v_exp)
        if pool.blocks != blocks or pool.page != page:
            raise ValueError(f"the cache must have {blocks} blocks of {page} tokens, as ref and page say")
        _lib.device_of(k_cache, v_cache, k_exp, v_exp, block_table)
    new_room = _lib.index32(new_room, dev)
    L = _lib.lib()
    nws = L.cfh_kv_resize_ws_bytes(S, W, blocks)
    ws = block_table.new_empty(nws // 4) if nws > 0 else None
    _lib.check(L.cfh_kv_resize(
        pool, block_table.data_ptr(), ld, W, room.data_ptr(), S, ref.data_ptr(), blocks, page, new_room.data_ptr(),
        _lib.ptr(ws), _lib.ptr(status), _lib.stream_of(dev)), "cfh_kv_resize")
