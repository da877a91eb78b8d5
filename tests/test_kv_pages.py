"""The pages' oracle against the rules it stands for, and the calls' refusals (CPU only)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.kv_cache import _check_pool, kv_cache_commit
from chain_flow_amd.kv_pages import kv_pages_fork, kv_pages_resize
from oracle import kv_pages as okp


def test_oracle_keeps_its_invariants_and_every_sequence_its_tokens():
    """Random forks, growth and shrinking: each sequence reads back its own tokens through its table, whoever
    shares them."""
    rng = np.random.default_rng(0)
    S, W, page, blocks = 6, 9, 4, 60
    table, room, ref = np.full((S, W), -1), np.zeros(S, dtype=int), np.zeros(blocks, dtype=int)
    cache = np.zeros((1, blocks, page), dtype=int)
    own = [[] for _ in range(S)]
    stamp = 1
    for _ in range(300):
        if rng.random() < 0.3:
            dst = rng.permutation(S)[:2]
            src = [rng.choice([v for v in range(-1, S) if v not in dst]) for _ in dst]
            assert not okp.fork(table, room, ref, src, dst, page)
            for a, b in zip(src, dst):
                own[b] = list(own[a]) if a >= 0 else []
        else:
            new = np.where(rng.random(S) < 0.3, -1, rng.integers(0, W * page + 1, S))
            assert not okp.resize(table, room, ref, new, page, [cache])
            for s, n in enumerate(new):
                if n < 0:
                    continue
                while len(own[s]) < n:                                # written behind the old room
                    i = len(own[s])
                    cache[0, table[s, i // page], i % page] = stamp
                    own[s].append(stamp)
                    stamp += 1
                own[s] = own[s][:n]
        okp.check(table, room, ref, page)
        for s in range(S):
            assert [cache[0, table[s, i // page], i % page] for i in range(room[s])] == own[s]


def test_oracle_refuses_from_where_the_free_pages_end():
    table, room, ref = np.full((4, 5), -1), np.zeros(4, dtype=int), np.zeros(7, dtype=int)
    assert okp.resize(table, room, ref, [9, 12, 8, 4], 4)
    assert room.tolist() == [9, 12, 0, 0] and (ref == 0).sum() == 1        # (one page is left, but the fourth comes behind the third)
    okp.check(table, room, ref, 4)


def test_commit_oracle_moves_each_row():
    rng = np.random.default_rng(1)
    table = rng.permutation(12)[:8].reshape(2, 4)
    cache = np.arange(12 * 5).reshape(1, 12, 5).copy()
    old = cache.copy()
    assert not okp.commit([cache], table, [3, 0], np.array([[0, 2, 5, 9], [4, 7, 0, 0]]), [4, 2], 5)
    for s, base, p in ((0, 3, [0, 2, 5, 9]), (1, 0, [4, 7])):
        for i, v in enumerate(p):
            assert cache[0, table[s, (base + i) // 5], (base + i) % 5] == old[0, table[s, (base + v) // 5], (base + v) % 5]
    assert okp.commit([cache], table, [3, 0], np.array([[0, 2, 2, 9], [4, 20, 0, 0]]), [4, 2], 5)


def _pool(S=3, W=4, blocks=10):
    return torch.full((S, W), -1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32), torch.zeros(blocks, dtype=torch.int32)


def test_pages_refusals_without_a_device():
    table, room, ref = _pool()
    ids = torch.zeros(2, dtype=torch.int32)
    for t, r, f, page in ((table.long(), room, ref, 4), (table[0], room, ref, 4), (table, room[:2], ref, 4), (table, room, ref[:0], 4),
                          (table.t(), torch.zeros(4, dtype=torch.int32), ref, 4), (table, room, torch.zeros(20, dtype=torch.int32)[::2], 4),
                          (table, room, ref, 0), (table, room, ref.float(), 4)):
        with pytest.raises(ValueError):
            kv_pages_fork(t, r, f, ids, ids, page=page)
        with pytest.raises(ValueError):
            kv_pages_resize(t, r, f, torch.zeros(3, dtype=torch.int32), page=page)
    with pytest.raises(ValueError, match="one GPU"):
        kv_pages_fork(table, room, ref, ids, ids, page=4)
    L, p = _lib.lib(), 4096      # stand-in addresses: never dereferenced, the checks fail first
    assert L.cfh_kv_resize_ws_bytes(3, 4, 10) == 48 + 64 + 40 and L.cfh_kv_resize_ws_bytes(3, 4, 100) == 48 + 64 + 48
    assert L.cfh_kv_resize_ws_bytes(-1, 4, 10) == L.cfh_kv_resize_ws_bytes(3, 4, 0) == -1

    def fork(ld=4, W=4, S=3, blocks=10, page=4, n=2, src=p):
        return L.cfh_kv_fork(p, ld, W, p, S, p, blocks, page, src, p, n, None, None)
    assert fork(n=0) == 0 and fork(ld=3) == fork(n=-1) == fork(blocks=0) == fork(page=0) == fork(src=None) == 1
    assert fork(n=65536) == fork(W=1 << 30, ld=1 << 30) == 2

    def resize(ld=4, W=4, S=3, blocks=10, page=4, ws=p, room=p):
        return L.cfh_kv_resize(None, p, ld, W, room, S, p, blocks, page, p, ws, None, None)
    assert resize(S=0) == 0 and resize(ld=3) == resize(S=-1) == resize(ws=None) == resize(ws=p + 8) == resize(room=None) == 1
    assert resize(S=4097) == resize(W=1 << 29, ld=1 << 29) == 2


def test_pool_refusals_without_a_device():
    k = torch.zeros(2, 5, 4, 2, 64, dtype=torch.bfloat16)
    e = torch.zeros(2, 5, 4, 2, dtype=torch.uint8)
    f = torch.zeros(2, 5, 4, 2, 64).to(torch.float8_e4m3fn)
    pool = _check_pool(k, k, None, None)
    assert (pool.layers, pool.blocks, pool.page, pool.heads, pool.dim, pool.ls_k, pool.bs_v) == (2, 5, 4, 2, 64, 2560, 512)
    both = torch.zeros(2, 5, 2, 4, 2, 64, dtype=torch.float16)              # keys and values of a block side by side
    pool = _check_pool(both[:, :, 0], both[:, :, 1], None, None)
    assert (pool.bs_k, pool.ls_k) == (1024, 5120)
    pool = _check_pool(f, f, e, e)
    assert pool.ls_k_exp == 40 and _check_pool(f[0], f[0], e[0], e[0]).ls_k_exp == 0
    for args in ((k, k[:, :4], None, None), (k, k.half(), None, None), (k.float(), k.float(), None, None), (k, k, e, e),
                 (f, f, e, None), (f, f, e.int(), e.int()), (f, f, e[:, :4], e[:, :4]), (f, f, e[:1].expand(2, -1, -1, -1), e),
                 (k[:, :0], k[:, :0], None, None), (k[..., :32], k[..., :32], None, None),
                 (k.transpose(2, 3), k.transpose(2, 3), None, None), (k[0, 0], k[0, 0], None, None),
                 (k[:1].expand(2, -1, -1, -1, -1), k, None, None),
                 (k.flatten()[8:8 + 1024].view(2, 4, 2, 64), k.flatten()[4:1028].view(2, 4, 2, 64), None, None)):
        with pytest.raises(ValueError):
            _check_pool(*args)
    lens, path = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 5, dtype=torch.int32)
    table = torch.zeros(3, 4, dtype=torch.int32)
    for args in ((table, lens[:2], path, lens), (table, lens, path[0], lens), (table[:2], lens, path, lens),
                 (table, lens, path, lens[:2]), (table, lens[None], path, lens)):
        with pytest.raises(ValueError):
            kv_cache_commit(k, k, *args)
    with pytest.raises(ValueError, match="one GPU"):
        kv_cache_commit(k, k, table, lens, path, lens)
    L, p = _lib.lib(), 4096
    good = _lib.KvPool(p, p, None, None, 2560, 2560, 512, 512, 0, 0, 2, 5, 4, 2, 64)

    def commit(S=3, P=5, p_ld=5, W=4, t_ld=4, path=p, **kw):
        pool = _lib.KvPool(*(getattr(good, n) for n, _ in good._fields_))
        for n, v in kw.items():
            setattr(pool, n, v)
        return L.cfh_kv_commit(pool, p, t_ld, W, p, path, p_ld, P, p, S, None, None)
    assert commit(S=0) == commit(P=0) == 0
    assert commit(p_ld=4) == commit(t_ld=3) == commit(S=-1) == commit(path=None) == commit(k=None) == commit(k_exp=p) == 1
    assert commit(bs_k=511) == commit(bs_v=520) == commit(ls_k=2552) == commit(ls_v=512) == commit(ls_k=2544) == commit(k=p + 8) == commit(layers=0) == 1
    assert commit(dim=96) == commit(blocks=1 << 30) == commit(S=65536) == 2


def test_pages_end_within_32_bits():
    """A page is copied in pieces of 16 KB whose ends are 32-bit numbers: the largest pages, whose last piece would end behind
    them, are refused by every call that takes a pool."""
    L, p = _lib.lib(), 4096

    def calls(page):
        pool = _lib.KvPool(p, p, None, None, 0, 0, page * 64, page * 64, 0, 0, 1, 1, page, 1, 64)
        return (L.cfh_kv_resize(pool, p, 4, 4, p, 0, p, 1, page, p, p, None, None),
                L.cfh_kv_commit(pool, p, 4, 4, p, p, 5, 5, p, 0, None, None))
    last = (2 ** 30 - 16384) // 64
    assert calls(last) == (0, 0) and (last * 128 + 16383) // 16384 * 16384 < 2 ** 31
    assert calls(last + 1) == calls((2 ** 30 - 1) // 64) == (2, 2)
