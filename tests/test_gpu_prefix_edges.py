"""Edges of the committed prefix's calls on the GPU: saturated bounds, bounds that fall, rows of no sequence in fresh
outputs, probabilities far below the largest one, dimensions of size one, captured calls."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.gdn import gdn_prefill
from chain_flow_amd.kv_cache import paged_attention
from conftest import rel_err, to64
from oracle import kv_cache as okv
from test_gpu_gdn_seq import TOL
from test_gpu_gdn_seq import Case as GdnCase
from test_gpu_kv_cache import BF, F8, FP, Case, close


def poison(cuda, *nbytes):
    """NaNs in the blocks that the allocator hands out next."""
    held = [torch.full((max(n, 1),), 0xFF, dtype=torch.uint8, device=cuda) for n in nbytes]
    torch.cuda.synchronize()
    del held


def check_first(c, out, lse, S, causal=True):
    """The rows of the first S sequences of an attention case against the oracle."""
    T = c.cu[S]
    ref = okv.attention(to64(c.q[:T]), c.ok[:S], c.ov[:S], c.lens[:S], c.cu[:S + 1], c.scale, causal)
    close(out[:T].contiguous(), lse[:, :T].contiguous(), *ref, max(c.lens[:S] + [1]), c.dtype)


def wide(c, tokens):
    """The case's table with room for `tokens` tokens a sequence: a call of that max_len is planned in pieces."""
    table = torch.full((c.table.shape[0], max(c.table.shape[1], -(-tokens // c.page))), -1, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table
    return table


# ---------------------------------------------------------------- saturated bounds
@pytest.mark.gpu
@pytest.mark.parametrize("H,bounds", [(256, [0, 5, 2 ** 40, 2 ** 40]),                             # many rows a sequence
                                      (32, [0, 1, 2, 3, 3, 3, 3, 3, 3, 3, 3, 2 ** 40, 2 ** 40])])  # few
def test_attention_bounds_past_32_bits_skip_their_sequences_only(cuda, H, bounds):
    """Bounds that 32 bits do not hold, times many heads a kv head: those sequences are skipped, the others are not."""
    S, good = len(bounds) - 1, next(i for i, b in enumerate(bounds) if b > 100) - 1
    news = np.diff(np.minimum(bounds, bounds[good] + 1)).tolist()
    c = Case(cuda, BF, BF, news, [40 + 3 * i for i in range(S)], H, 1, 64, 16, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(c.q, 7.0)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(cuda)  # noqa: E731
    o, lse = paged_attention(c.q, c.k, c.v, i32(c.table), i32(c.lens), torch.tensor(bounds), scale=c.scale, out=out, status=status)
    assert status.item() == 1 and (o[bounds[good]:] == 7).all()
    check_first(c, o, lse, good)


# ---------------------------------------------------------------- bounds that fall
FALLS = [
    # news, bounds, sequences before the fall
    ([100, 50, 50], [0, 100, -1000, 200], 1),
    ([100, 50, 50], [0, 100, 60, 200], 1),
    ([3, 2, 3], [0, 3, -7, 8], 1),
    ([60, 1, 1, 90, 4], [0, 60, 61, 62, 20, 156], 3),
    ([40, 30, 20], [0, 40, 70, -1], 2),
    ([40, 30], [40, 0, 70], 0),
    ([1] * 100 + [50], [*range(90), 3, *range(91, 101), 150], 89),
    ([1] * 600 + [50], [*range(401), 3, *range(402, 601), 650], 400),
    ([0] * 700 + [30] + [1] * 300, [0] * 701 + [30 + i for i in range(200)] + [1 + i for i in range(101)], 900),
]


@pytest.mark.gpu
@pytest.mark.parametrize("state", [torch.float32, BF])
@pytest.mark.parametrize("news,bounds,good", FALLS)
def test_prefill_stops_where_the_bounds_fall(cuda, news, bounds, good, state):
    """The sequences before the first bound that falls below the one before it, and their slots, are what they are by
    themselves; from it on sequences are skipped, their rows and slots left as they were, and the status word is set."""
    c = GdnCase(cuda, news, state=state, seed=3)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((sum(news), 4, 64), 7.0, dtype=BF, device=cuda)
    poison(cuda, 1 << 24)
    print(f"[prefill falls] {len(news)} sequences, {good} before it", flush=True)
    o, st = c.run(out=out, status=status, cu=bounds)
    assert status.item() == 1 and (o[bounds[good] if good else 0:] == 7).all()
    others = np.setdiff1d(np.arange(len(news) + 3), c.slots.numpy()[:good])
    assert torch.equal(st.cpu()[others], c.state[others])
    if good:
        c.cu, c.slots = c.cu[:good + 1], c.slots[:good]
        ref, rst = c.oracle()
        T = bounds[good]
        assert rel_err(to64(o[:T]), ref[:T]) < TOL[BF] and rel_err(to64(st), rst) < TOL[state]


# ---------------------------------------------------------------- attention where bounds fall
@pytest.mark.gpu
@pytest.mark.parametrize("most", [100, 3000])
@pytest.mark.parametrize("news,bounds,good", FALLS)
def test_attention_stops_where_the_bounds_fall(cuda, news, bounds, good, most):
    """As the delta rule's.  Whole and in pieces."""
    rng = np.random.default_rng(len(news))
    lens = (np.asarray(news) + rng.integers(0, 30 if len(news) > 9 else 900, len(news))).tolist()
    c = Case(cuda, BF, BF, news, lens, 4, 2, 64, 16, seed=2)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(c.q, 7.0)
    print(f"[attention falls] {len(news)} sequences, {good} before it", flush=True)
    o, lse = c.run(cu=bounds, out=out, status=status, table=wide(c, most), max_len=most)
    assert status.item() == 1 and (o[bounds[good] if good else 0:] == 7).all()
    if good:
        assert c.cu[:good + 1].tolist() == bounds[:good + 1]
        check_first(c, o, lse, good)


# ---------------------------------------------------------------- rows of no sequence in fresh outputs
OUTSIDE = [
    # rows of the query, bounds, rows that sequences cover
    (21, [3, 7, 16], (3, 16)),                # before, behind
    (300, [0, 130, 131, 290], (0, 290)),
    (9, [4, 4], (4, 4)),                      # one sequence of no rows
    (40, [-5, 10, 30, 50], (10, 30)),         # sequences that are skipped
    (40, [-5, 50], (0, 0)),
    (40, [41, 50], (0, 0)),
    (40, [0, 20, 5, 40], (0, 20)),            # a fall
    (700, [2 + i for i in range(601)], (2, 602)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,bounds,cover", OUTSIDE)
def test_prefill_rows_of_no_sequence_are_zero_in_a_fresh_out(cuda, T, bounds, cover):
    S = len(bounds) - 1
    c = GdnCase(cuda, [T], seed=6)
    c.state = torch.zeros(S + 1, 4, 64, 128)
    c.slots = torch.arange(S, dtype=torch.int32)
    a, b = cover
    out = torch.full((T, 4, 64), 7.0, dtype=BF, device=cuda)
    want = c.run(cu=bounds, out=out)[0]
    assert (want[:a] == 7).all() and (want[b:] == 7).all()
    poison(cuda, T * 4 * 64 * 2)
    o, _ = c.run(cu=bounds)
    assert (o[:a] == 0).all() and (o[b:] == 0).all() and torch.equal(o[a:b], want[a:b])


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[5], [70], [3, 70, 1, 64], [1] * 9])
def test_prefill_rows_of_a_padding_sequence_are_zero_in_a_fresh_out(cuda, news):
    """Each sequence in turn a padding one (slot -1), short and long; and no sequence at all."""
    for s in range(len(news)):
        c = GdnCase(cuda, news, seed=7)
        c.slots[s] = -1
        poison(cuda, sum(news) * 4 * 64 * 2)
        o, _ = c.run()
        at = slice(c.cu[s], c.cu[s + 1])
        assert (o[at] == 0).all() and o.isfinite().all()
    c = GdnCase(cuda, news, seed=7)
    c.slots = c.slots[:0]
    poison(cuda, sum(news) * 4 * 64 * 2)
    assert (c.run(cu=[0])[0] == 0).all()


@pytest.mark.gpu
def test_decode_rows_of_padding_are_zero_in_a_fresh_out(cuda):
    c = GdnCase(cuda, [1] * 5, seed=8, slots=[4, -1, 0, -1, 6])
    poison(cuda, 5 * 4 * 64 * 2)
    o, st = c.run(decode=True)
    ref, rst = c.oracle()
    assert (o[1] == 0).all() and (o[3] == 0).all()
    live = [0, 2, 4]
    assert rel_err(to64(o[live]), ref[live]) < TOL[BF] and rel_err(to64(st), rst) < 1e-5


# ---------------------------------------------------------------- fresh attention outputs
@pytest.mark.gpu
@pytest.mark.parametrize("most", [100, 4000])
@pytest.mark.parametrize("T,bounds,cover", OUTSIDE)
def test_attention_rows_of_no_sequence_are_zero_in_a_fresh_out(cuda, T, bounds, cover, most):
    """Without `out`, rows that no sequence has (or a skipped one) are 0, and their lse is -inf with and without it."""
    S = len(bounds) - 1
    c = Case(cuda, BF, BF, [0] * S, [20 + i % 50 for i in range(S)], 4, 2, 64, 16, seed=4)
    q = torch.randn(T, 4, 64, device=cuda).to(BF)
    a, b = cover
    for given in (False, True):
        poison(cuda, *[T * 4 * 64 * 2] * 2, *[T * 4 * 4] * 2)
        out = torch.full_like(q, 7.0) if given else None
        o, lse = c.run(q=q, cu=bounds, out=out, table=wide(c, most), max_len=most)
        rest = torch.cat([o[:a], o[b:]])
        assert (rest == (7 if given else 0)).all()
        assert (lse[:, :a] == -np.inf).all() and (lse[:, b:] == -np.inf).all()
        assert o[a:b].isfinite().all() and (lse[:, a:b] > -np.inf).all() or min(c.lens) < max(np.diff(bounds))
        assert not o[a:b].isnan().any() and not lse[:, a:b].isnan().any()


@pytest.mark.gpu
def test_attention_of_no_sequences_is_zero(cuda):
    c = Case(cuda, BF, BF, [0], [20], 4, 2, 64, 16, seed=5)
    q = torch.randn(5, 4, 64, device=cuda).to(BF)
    poison(cuda, 5 * 4 * 64 * 2, 5 * 4 * 4)
    o, lse = c.run(q=q, cu=[0], lens=[], table=c.table[:0])
    assert (o == 0).all() and (lse == -np.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("most", [100, 3000])
def test_the_plain_c_call_leaves_rows_of_no_sequence(cuda, most):
    """cfh_paged_attn itself writes no row of out or lse that no sequence has; in the others it is the Python call."""
    c = Case(cuda, BF, BF, [4, 30], [50, 90], 4, 2, 64, 16, seed=13)
    q = torch.randn(50, 4, 64, device=cuda).to(BF)
    bounds, table = [7, 11, 41], wide(c, most).to(cuda)
    o, lse = c.run(q=q, cu=bounds, table=table, max_len=most)
    out, lse2 = torch.full_like(q, 7.0), torch.full((4, 50), 7.0, device=cuda)
    lens, cu = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (c.lens, bounds))
    L = _lib.lib()
    ws = torch.empty(max(1, L.cfh_paged_attn_ws_bytes(50, 4, 2, 64, 2, most)), dtype=torch.uint8, device=cuda)
    blocks, stride = c.k.shape[0], c.k.stride(0)
    rc = L.cfh_paged_attn(q.data_ptr(), 256, 50, 4, 2, 64, 1, c.k.data_ptr(), stride, c.v.data_ptr(), stride, None, None, blocks,
                          16, table.data_ptr(), table.shape[1], table.shape[1], lens.data_ptr(), cu.data_ptr(), 2, c.scale, 1, most,
                          out.data_ptr(), 256, lse2.data_ptr(), ws.data_ptr(), None, _lib.stream_handle())
    torch.cuda.synchronize()
    assert rc == 0
    assert (out[:7] == 7).all() and (out[41:] == 7).all() and (lse2[:, :7] == 7).all() and (lse2[:, 41:] == 7).all()
    assert torch.equal(out[7:41], o[7:41]) and torch.equal(lse2[:, 7:41], lse[:, 7:41])


# ---------------------------------------------------------------- probabilities far below the largest
@pytest.mark.gpu
@pytest.mark.parametrize("cache", [FP, F8])
@pytest.mark.parametrize("T,D,split", [(1, 64, False), (40, 64, False), (40, 128, False), (40, 256, False), (1, 128, True)])
def test_many_small_probabilities_beside_a_large_one(cuda, T, D, split, cache):
    """fp16: one token takes nearly all the weight (the first, as a prompt's first token does) and each of 60,000 others
    2^-25.5 of it; together they are 1.3e-3 of the result.  A probability enters the product with v as fp16 scaled by
    2^7, so it loses at most 2^-25 2^-7, and a row at most L 2^-32 |v|."""
    L = 60000
    c = Case(cuda, FP, cache, [T], [L], 2, 1, D, 64, seed=9)
    k, v = (t.view(torch.uint8 if cache == F8 else FP) for t in (c.k, c.v))
    one = 0x38 if cache == F8 else 1.0                                      # (the byte of e4m3's 1)
    blk = c.table[0].long().to(cuda)
    k[blk], v[blk] = 0, one
    if cache == F8:
        c.ke[blk], c.ve[blk] = 127, 127
    k[blk[0], 0, 0, 0] = one
    v[blk[0], 0] = 0
    c.ok, c.ov = [np.zeros((L, 1, D))], [np.ones((L, 1, D))]
    c.ok[0][0, 0, 0], c.ov[0][0] = 1.0, 0.0
    c.q.zero_()
    c.q[:, :, 0] = 25.5 * np.log(2.0) / c.scale
    out, lse = c.run(causal=False, max_len=L if split else 1)
    ref, rlse, weight, reach = okv.attention(to64(c.q), c.ok, c.ov, c.lens, c.cu, c.scale, False)
    u, score = 2.0 ** -11, (D * 2.0 ** -24 * reach).T[..., None]
    bound = u * np.abs(ref) + (u + 2 * score + L * 2.0 ** -23) * weight + 2.0 ** -24 + L * 2.0 ** -32
    off = np.abs(to64(out) - ref) / bound
    print(f"[small probabilities] {cache} T={T} D={D}: {to64(out).max():.3e} for {ref.max():.3e}, {off.max():.3f} of its bound", flush=True)
    assert off.max() <= 1.0 and np.abs(to64(lse) - rlse).max() <= score.max() + L * 2.0 ** -24 + 2.0 ** -22 * np.abs(rlse).max()


# ---------------------------------------------------------------- dimensions of size one
@pytest.mark.gpu
def test_attention_strides_of_size_one_do_not_count(cuda):
    """One kv head kept as [blocks, 1, page, D], one query head behind a wider stride: contiguous all the same."""
    c = Case(cuda, BF, BF, [3, 1], [40, 9], 1, 1, 64, 16, seed=10)
    want = c.run()
    c.k, c.v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k, c.v))
    c.k, c.v = (t.as_strided(t.shape, (1024, 64, 4096, 1)) for t in (c.k, c.v))
    out = torch.zeros(4, 64, dtype=BF, device=cuda).as_strided((4, 1, 64), (64, 8, 1))
    got = c.run(q=c.q.as_strided(c.q.shape, (64, 8, 1)), out=out)
    assert got[0].data_ptr() == out.data_ptr()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------- captured, with bounds that change between replays
@pytest.mark.gpu
@pytest.mark.parametrize("S", [5, 300, 700])
def test_a_captured_call_follows_its_bounds(cuda, S):
    """One graph of an attention (whose out and lse it makes) and a prefill; before each replay the bounds are others:
    all rows, none, rows of no sequence on either side, a fall, ends outside the query.  Every replay equals the eager
    calls."""
    news = [1 + i % 3 for i in range(S)]
    news[S // 2] = 60
    T = sum(news)
    c = Case(cuda, BF, BF, [0] * S, [70 + i % 9 for i in range(S)], 4, 2, 64, 16, seed=11)
    g = GdnCase(cuda, [T], H=1, HV=2, V=16, seed=12)
    state = torch.randn(S, 2, 16, 128, device=cuda)
    q = torch.randn(T, 4, 64, device=cuda).to(BF)
    d = lambda t: t.to(cuda)  # noqa: E731
    x, a, b, A, dt, slots = d(g.x), d(g.a), d(g.b), d(g.A), d(g.dt), torch.arange(S, dtype=torch.int32, device=cuda)
    table, lens = wide(c, 3000).to(cuda), torch.tensor(c.lens, dtype=torch.int32, device=cuda)
    whole = torch.tensor([0, *np.cumsum(news)], dtype=torch.int32)
    fall, low, late = whole.clone(), whole - 3, whole + 3
    fall[S // 3:] -= 7
    cu = whole.to(cuda)
    st, status = state.clone(), torch.zeros(1, dtype=torch.int32, device=cuda)

    def step(st, status):
        o, lse = paged_attention(q, c.k, c.v, table, lens, cu, scale=c.scale, status=status)
        return o, lse, gdn_prefill(x, a, b, A, dt, st, slots, cu, num_q_heads=1, status=status)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(st, status)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(st, status)
    for name, bounds in (("whole", whole), ("fall", fall), ("none", whole * 0 + 5), ("low", low), ("whole", whole),
                         ("late", late)):
        print(f"[captured bounds] S={S} {name}", flush=True)
        cu.copy_(bounds)
        st.copy_(state)
        status.zero_()
        graph.replay()
        got = [t.clone() for t in (*outs, st, status)]
        est, estat = state.clone(), torch.zeros_like(status)
        want = (*step(est, estat), est, estat)
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(got, want)), name
        assert status.item() == (name in ("fall", "low", "late")) and all(t.isfinite().all() for t in (got[0], got[2]))
