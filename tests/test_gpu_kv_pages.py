"""The paged cache's pages and accepted rows on the GPU against the step-by-step oracle: tables, rooms, holders and
cache contents bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.kv_cache import kv_cache_commit
from chain_flow_amd.kv_pages import kv_pages_fork, kv_pages_resize
from oracle import kv_pages as okp


def _i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def _cache(layers, blocks, page, Hkv, D, kind, dev, seed=0):
    """(keyword arguments of a call, byte arrays of the oracle)."""
    g = torch.Generator().manual_seed(seed)
    es = 1 if kind == "fp8" else 2
    raw = [torch.randint(0, 256, (layers, blocks, page, Hkv * D * es), dtype=torch.uint8, generator=g) for _ in range(2)]
    exps = [torch.randint(1, 255, (layers, blocks, page, Hkv), dtype=torch.uint8, generator=g) for _ in range(2)] if es == 1 else []
    dtype = {"fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16, "fp16": torch.float16}[kind]
    kv = [r.to(dev).view(dtype).view(layers, blocks, page, Hkv, D) for r in raw]
    kw = dict(k_cache=kv[0], v_cache=kv[1])
    if exps:
        kw.update(k_exp=exps[0].to(dev), v_exp=exps[1].to(dev))
    return kw, [r.numpy().copy() for r in raw + exps]


def _same(kw, arrays):
    got = [kw[n] for n in ("k_cache", "v_cache", "k_exp", "v_exp") if n in kw]
    return all(np.array_equal(g.contiguous().view(torch.uint8).cpu().numpy().reshape(a.shape), a) for g, a in zip(got, arrays))


def _pool(S, W, blocks, dev):
    return (np.full((S, W), -1), np.zeros(S, dtype=int), np.zeros(blocks, dtype=int)), \
        (torch.full((S, W), -1, dtype=torch.int32, device=dev), torch.zeros(S, dtype=torch.int32, device=dev),
         torch.zeros(blocks, dtype=torch.int32, device=dev))


def _equal(host, dev):
    return all(np.array_equal(h, d.cpu().numpy()) for h, d in zip(host, dev))


@pytest.mark.gpu
@pytest.mark.parametrize("S,W,page,blocks,layers,Hkv,D,kind", [
    (1, 1, 1, 1, 1, 1, 64, "bf16"), (5, 9, 4, 61, 2, 2, 64, "fp16"), (17, 7, 16, 140, 3, 3, 128, "fp8"),
    (40, 12, 3, 300, 1, 1, 256, "fp8"), (9, 6, 48, 70, 2, 4, 256, "bf16"), (64, 5, 64, 330, 1, 8, 256, "bf16")])
def test_random_forks_and_resizes(cuda, S, W, page, blocks, layers, Hkv, D, kind):
    """Rounds of forks and resizes, some of which run out of pages."""
    rng = np.random.default_rng(S)
    host, dev = _pool(S, W, blocks, cuda)
    kw, arrays = _cache(layers, blocks, page, Hkv, D, kind, cuda)
    refused = 0
    for turn in range(25):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        if rng.random() < 0.4 and S > 1:
            n = int(rng.integers(1, S // 2 + 1))
            dst = rng.permutation(S)[:n]
            rest = [v for v in range(-1, S) if v not in dst]
            src = rng.choice(rest, n)
            dst = np.where(rng.random(n) < 0.1, -1, dst)
            bad = okp.fork(*host, src, dst, page)
            kv_pages_fork(*dev, _i32(src, cuda), _i32(dst, cuda), page=page, status=status)
        else:
            new = np.where(rng.random(S) < 0.3, -1, np.minimum(rng.integers(0, W * page + 1, S), host[1] + rng.integers(-page, 2 * page + 1, S)))
            new = np.where(new < -1, 0, new)
            bad = okp.resize(*host, new, page, arrays)
            kv_pages_resize(*dev, _i32(new, cuda), page=page, status=status, **kw)
        torch.cuda.synchronize()
        refused += bad
        assert int(status) == bad and _equal(host, dev) and _same(kw, arrays), turn
        okp.check(*host, page)
    print(f"[pages] S={S}: {refused} calls refused a sequence, {int((host[2] > 1).sum())} pages shared at the end", flush=True)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1000, 1025, 4096])
def test_many_sequences_and_pages(cuda, S):
    """More sequences than threads of the planning workgroup, more free pages than one step of its search, shared last
    pages of several families, and a pool that ends in the middle."""
    rng = np.random.default_rng(S)
    W, page, blocks = 24, 4, 9 * S
    host, dev = _pool(S, W, blocks, cuda)
    for turn in range(4):
        new = rng.integers(0, W * page + 1, S) if turn == 3 else rng.integers(0, 40, S)
        bad = okp.resize(*host, new, page)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        kv_pages_resize(*dev, _i32(new, cuda), page=page, status=status)
        assert int(status) == bad and _equal(host, dev)
        dst = np.flatnonzero(rng.random(S) < 0.4)
        src = rng.choice(np.setdiff1d(np.arange(S), dst)[:7], len(dst))
        bad = okp.fork(*host, src, dst, page)
        kv_pages_fork(*dev, _i32(src, cuda), _i32(dst, cuda), page=page, status=status)
        torch.cuda.synchronize()
        assert not bad and _equal(host, dev)
        print(f"[pages] S={S} turn {turn}: {int((host[2] == 0).sum())} free", flush=True)


@pytest.mark.gpu
def test_all_holders_of_a_shared_last_page_grow_at_once(cuda):
    """All but the last get copies; where the pages end between them, it and the ones behind are refused."""
    page, W = 8, 3
    for blocks in (2, 3, 4, 5, 9):
        host, dev = _pool(5, W, blocks, cuda)
        kw, arrays = _cache(2, blocks, page, 2, 64, "bf16", cuda, seed=blocks)
        for new in ([13, 0, 0, 0, 0], None, [20 if blocks > 6 else 16, 15, 14, 16, 14]):
            status = torch.zeros(1, dtype=torch.int32, device=cuda)
            if new is None:
                bad = okp.fork(*host, [0, 0, 0, 0], [1, 2, 3, 4], page)
                kv_pages_fork(*dev, _i32([0, 0, 0, 0], cuda), _i32([1, 2, 3, 4], cuda), page=page, status=status)
            else:
                bad = okp.resize(*host, new, page, arrays)
                kv_pages_resize(*dev, _i32(new, cuda), page=page, status=status, **kw)
            torch.cuda.synchronize()
            assert int(status) == bad and _equal(host, dev) and _same(kw, arrays), (blocks, new)
        print(f"[pages] {blocks} pages: rooms {host[1].tolist()}", flush=True)


@pytest.mark.gpu
def test_refused_pairs_and_rooms_leave_their_sequences(cuda):
    page = 4
    host, dev = _pool(6, 4, 30, cuda)
    okp.resize(*host, [10, 5, 3, 0, 16, 7], page)
    kv_pages_resize(*dev, _i32([10, 5, 3, 0, 16, 7], cuda), page=page)
    assert _equal(host, dev)
    for src, dst in (([0, 1], [3, 3]), ([0, 3], [3, 5]), ([6, 0], [3, 5]), ([-2, 0], [3, 5]), ([0, 1], [6, 3]), ([0, 1], [-2, 3]),
                     ([2 ** 31 - 1, 1], [3, 0])):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        assert okp.fork(*host, src, dst, page)
        kv_pages_fork(*dev, _i32(src, cuda), _i32(dst, cuda), page=page, status=status)
        assert int(status) == 1 and _equal(host, dev), (src, dst)
    for new in ([17, -1, -1, -1, -1, -1], [2 ** 31 - 1] + [3] * 5, [1, 2, 3, 4, 2 ** 30, 6]):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        assert okp.resize(*host, new, page)
        kv_pages_resize(*dev, _i32(new, cuda), page=page, status=status)
        assert int(status) == 1 and _equal(host, dev), new
    # a room the table cannot hold is refused, whoever wrote it; entries that are no page count for none
    for room in (17, -3, 2 ** 31 - 1):
        t = [d.clone() for d in dev]
        t[1][2] = room
        before = [d.clone() for d in t]
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        kv_pages_resize(*t, _i32([-1, -1, 9, -1, -1, -1], cuda), page=page, status=status)
        assert int(status) == 1 and all(torch.equal(a, b) for a, b in zip(t, before))
        kv_pages_fork(*t, _i32([2], cuda), _i32([3], cuda), page=page, status=status)
        assert all(torch.equal(a, b) for a, b in zip(t, before))
    for entry in (-1, 30, 2 ** 31 - 1):
        t = [d.clone() for d in dev]
        t[0][0, 0] = entry
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        kv_pages_resize(*t, _i32([0, -1, -1, -1, -1, -1], cuda), page=page, status=status)
        torch.cuda.synchronize()
        assert int(status) == 1 and int(t[1][0]) == 0
    # the page that would be copied is none: the sequence is left
    t = [d.clone() for d in dev]
    assert host[1][1] % page
    t[0][1, okp.held(host[1][1], page) - 1] = 99
    before = [d.clone() for d in t]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv_pages_resize(*t, _i32([-1, 9, -1, -1, -1, -1], cuda), page=page, status=status)
    assert int(status) == 1 and all(torch.equal(a, b) for a, b in zip(t, before))


@pytest.mark.gpu
def test_strided_tables_and_host_indices(cuda):
    page = 4
    host, _ = _pool(4, 5, 20, cuda)
    big = torch.full((4, 9), -5, dtype=torch.int32, device=cuda)
    table = big[:, 2:7]
    table.fill_(-1)
    room, ref = torch.zeros(4, dtype=torch.int32, device=cuda), torch.zeros(20, dtype=torch.int32, device=cuda)
    okp.resize(*host, [9, 0, 20, 1], page)
    kv_pages_resize(table, room, ref, torch.tensor([9, 0, 20, 1]), page=page)
    okp.fork(*host, [2, -1], [1, 0], page)
    kv_pages_fork(table, room, ref, torch.tensor([2, -1]), torch.tensor([1, 0]), page=page)
    assert _equal(host, (table, room, ref)) and (big[:, [0, 1, 7, 8]] == -5).all()
    for src, dst in (([0, 1], [3, 3]), ([0, 3], [3, 2]), ([4], [0]), ([0], [4]), ([-2], [0])):
        with pytest.raises(ValueError, match="destinations"):
            kv_pages_fork(table, room, ref, torch.tensor(src), torch.tensor(dst), page=page)
    assert _equal(host, (table, room, ref))


def _commit_case(rng, S, W, page, P, dev, extra=3):
    blocks = S * W + extra
    table = rng.permutation(blocks)[: S * W].reshape(S, W)
    lens = rng.integers(0, max(W * page - 2 * P, 1), S)
    nodes = 2 * P
    path = np.full((S, P), -1)
    count = np.zeros(S, dtype=int)
    for s in range(S):
        most = min(nodes, W * page - int(lens[s]))
        count[s] = rng.integers(0, min(P, most) + 1)
        path[s, : count[s]] = np.sort(rng.permutation(most)[: count[s]])
    return blocks, table, lens, path, count


@pytest.mark.gpu
@pytest.mark.parametrize("S,W,page,P,layers,Hkv,D,kind", [
    (1, 1, 1, 1, 1, 1, 64, "bf16"), (3, 5, 16, 6, 1, 1, 64, "fp8"), (7, 4, 48, 40, 3, 3, 128, "fp8"), (2, 9, 64, 200, 2, 8, 256, "fp16"),
    (48, 6, 16, 8, 5, 2, 128, "bf16"), (5, 40, 3, 60, 2, 5, 64, "fp8"), (1, 30, 5, 65, 16, 4, 256, "bf16"), (4, 30, 16, 64, 1, 1, 256, "fp8")])
def test_commit_moves_accepted_rows(cuda, S, W, page, P, layers, Hkv, D, kind):
    rng = np.random.default_rng(S * P)
    blocks, table, lens, path, count = _commit_case(rng, S, W, page, P, cuda)
    kw, arrays = _cache(layers, blocks, page, Hkv, D, kind, cuda, seed=P)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    print(f"[commit] S={S} P={P} moves {int(count.sum())} rows", flush=True)
    for _ in range(2):
        assert not okp.commit(arrays, table, lens, path, count, page)
        kv_cache_commit(kw["k_cache"], kw["v_cache"], _i32(table, cuda), _i32(lens, cuda), _i32(path, cuda), _i32(count, cuda),
                        k_exp=kw.get("k_exp"), v_exp=kw.get("v_exp"), status=status)
        torch.cuda.synchronize()
        assert _same(kw, arrays) and int(status) == 0


@pytest.mark.gpu
def test_commit_of_one_layer_views_and_blocks_side_by_side(cuda):
    """A [blocks, page, Hkv, D] cache, keys and values of a block in one allocation, a table and paths with strides."""
    rng = np.random.default_rng(3)
    blocks, table, lens, path, count = _commit_case(rng, 4, 3, 8, 6, cuda)
    both = torch.randn(2, blocks, 2, 8, 2, 64, device=cuda).half()
    k, v = both[:, :, 0], both[:, :, 1]
    arrays = [x.cpu().numpy().copy() for x in (k, v)]
    okp.commit(arrays, table, lens, path, count, 8)
    wide = lambda x: torch.cat([_i32(x, cuda), _i32(x, cuda)], 1)[:, : x.shape[1]]                 # noqa: E731
    kv_cache_commit(k, v, wide(table), _i32(lens, cuda), wide(path), torch.tensor(count))
    assert all(np.array_equal(x.cpu().numpy(), a) for x, a in zip((k, v), arrays))
    okp.commit([a[1:] for a in arrays], table, lens, path, count, 8)
    kv_cache_commit(k[1], v[1], _i32(table, cuda), _i32(lens, cuda), _i32(path, cuda).long(), _i32(count, cuda))
    torch.cuda.synchronize()
    assert all(np.array_equal(x.cpu().numpy(), a) for x, a in zip((k, v), arrays))


@pytest.mark.gpu
def test_commit_refuses_a_sequence_at_a_time(cuda):
    page, W, P = 8, 3, 5
    rng = np.random.default_rng(4)
    table = rng.permutation(12)[:9].reshape(3, 3)
    good = np.array([[1, 2, 4, 7, 9], [0, 3, -1, -1, -1], [2, 5, 6, -1, -1]])
    for s, path, lens, count, page_id in ((0, [1, 2, 2, 7, 9], 4, 5, None), (0, [-1, 2, 4, 7, 9], 4, 5, None), (0, [1, 9, 4, 7, 9], 4, 5, None),
                                          (0, good[0], 4, 6, None), (0, good[0], -1, 5, None), (0, good[0], 15, 5, None),
                                          (0, [1, 2, 4, 7, 2 ** 31 - 1], 4, 5, None), (0, good[0], 2 ** 31 - 1, 5, None),
                                          (0, good[0], 4, 5, -1), (0, good[0], 4, 5, 12), (0, good[0], 4, 2 ** 31 - 1, None)):
        kw, arrays = _cache(2, 12, page, 1, 64, "fp8", cuda, seed=7)
        t, p, ln, n = table.copy(), good.copy(), np.array([4, 9, 0]), np.array([5, 2, 3])
        p[s], ln[s], n[s] = path, lens, count
        if page_id is not None:
            t[s, 1] = page_id
        assert okp.commit(arrays, t, ln, p, n, page)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        kv_cache_commit(kw["k_cache"], kw["v_cache"], _i32(t, cuda), _i32(ln, cuda), _i32(p, cuda), _i32(n, cuda), k_exp=kw["k_exp"],
                        v_exp=kw["v_exp"], status=status)
        torch.cuda.synchronize()
        assert int(status) == 1 and _same(kw, arrays), (path, lens, count, page_id)


@pytest.mark.gpu
def test_pages_behind_4_gib(cuda):
    """Copies and moved rows whose offsets pass 32 bits, in bytes and (of the last layer) in elements."""
    layers, blocks, page, Hkv, D = 2, 70001, 16, 8, 256
    print("[pages] behind 4 GiB", flush=True)
    k, v = (torch.zeros(layers, blocks, page, Hkv, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    table = torch.full((2, 3), -1, dtype=torch.int32, device=cuda)
    room, ref = torch.zeros(2, dtype=torch.int32, device=cuda), torch.ones(blocks, dtype=torch.int32, device=cuda)
    free = [69990, 69995, 70000]
    ref[free] = 0
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv_pages_resize(table, room, ref, _i32([21, 0], cuda), page=page, status=status)
    assert table[0].tolist() == free[:2] + [-1]
    for c in (k, v):
        for p in free[:2]:
            c[:, p] = torch.randn(layers, page, Hkv, D, device=cuda).to(torch.bfloat16)
    kv_pages_fork(table, room, ref, _i32([0], cuda), _i32([1], cuda), page=page, status=status)
    kv_pages_resize(table, room, ref, _i32([-1, 26], cuda), page=page, k_cache=k, v_cache=v, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0 and table[1].tolist() == [free[0], free[2], -1]
    for c in (k, v):
        assert torch.equal(c[:, free[2], :5], c[:, free[1], :5]) and not c[:, free[2], 5:].any()
    rows = torch.randn(layers, 5, Hkv, D, device=cuda).to(torch.bfloat16)
    k[:, free[2], 5:10], v[:, free[2], 5:10] = rows, rows * 2
    kv_cache_commit(k, v, table[1:], _i32([21], cuda), _i32([[1, 4]], cuda), _i32([2], cuda), status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for c, r in ((k, rows), (v, rows * 2)):
        assert torch.equal(c[:, free[2], 5:7], r[:, [1, 4]]) and torch.equal(c[:, free[2], 7:10], r[:, 2:])


@pytest.mark.gpu
def test_pages_in_a_graph(cuda):
    """A captured step -- grow, commit, shrink, fork -- replayed over pools that change between replays."""
    page, W, S, blocks, P = 4, 12, 6, 80, 3
    rng = np.random.default_rng(5)
    host, dev = _pool(S, W, blocks, cuda)
    kw, arrays = _cache(2, blocks, page, 1, 64, "bf16", cuda)
    grow, back = (torch.zeros(S, dtype=torch.int32, device=cuda) for _ in range(2))
    path, count = torch.zeros(S, P, dtype=torch.int32, device=cuda), torch.zeros(S, dtype=torch.int32, device=cuda)
    src, dst = (torch.zeros(2, dtype=torch.int32, device=cuda) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(S, dtype=torch.int32, device=cuda)

    def step():
        lens.copy_(dev[1])
        kv_pages_resize(*dev, grow, page=page, status=status, **kw)
        kv_cache_commit(kw["k_cache"], kw["v_cache"], dev[0], lens, path, count, status=status)
        kv_pages_resize(*dev, back, page=page, status=status, **kw)
        kv_pages_fork(*dev, src, dst, page=page, status=status)

    state = [t.clone() for t in (*dev, kw["k_cache"], kw["v_cache"])]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, s in zip((*dev, kw["k_cache"], kw["v_cache"]), state):
        t.copy_(s)
    for turn in range(6):
        n0 = host[1].copy()
        c = rng.integers(0, P + 1, S)
        n_back = np.minimum(n0 + c, W * page - 8)
        g = np.minimum(n0 + 7, W * page)
        c = n_back - n0
        p = np.array([np.concatenate([np.sort(rng.permutation(min(7, max(g[s] - n0[s], 0)))[: max(c[s], 0)]),
                                      np.full(P - max(c[s], 0), -1)]) for s in range(S)])
        pair = rng.permutation(S)[:4]
        for t, v in ((grow, g), (back, n_back), (path, p), (count, c), (src, pair[:2]), (dst, pair[2:])):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        bad = okp.resize(*host, g, page, arrays)
        bad |= okp.commit(arrays, host[0], n0, p, c, page)
        bad |= okp.resize(*host, n_back, page, arrays)
        bad |= okp.fork(*host, pair[:2], pair[2:], page)
        status.zero_()
        graph.replay()
        torch.cuda.synchronize()
        print(f"[pages graph] replay {turn}: rooms {host[1].tolist()}", flush=True)
        assert int(status) == bad and _equal(host, dev) and _same(kw, arrays)
