"""GPU parity of the gated delta rule over committed tokens (gdn_prefill, gdn_decode) against the float64 oracle.

Bounds.  fp32 states: 1e-5 norm-relative, as the tree scan's: fp32 products and sums, or products of values split
into two bf16 parts, which drop at most 2^-17 of a factor.  bf16 states and outputs are rounded once, at most 2^-8 of
each value, so 2^-8 + 1e-5 norm-relative."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.gdn import gdn_decode, gdn_prefill, tree_gdn_vllm
from conftest import rel_err, to64
from oracle import gdn as ogdn

BF = torch.bfloat16
TOL = {torch.float32: 1e-5, BF: 2.0 ** -8 + 1e-5}


class Case:
    def __init__(self, cuda, news, H=2, HV=4, V=64, state=torch.float32, seed=0, gate=-3.0, spread=1.0, kscale=1.0, slots=None):
        g = torch.Generator().manual_seed(seed)
        T, K = sum(news), 128
        self.H, self.cuda, self.news = H, cuda, news
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        x = r(T, 2 * H * K + HV * V)
        self.x = (x * torch.sigmoid(x) * kscale).to(BF)                     # SiLU rows: keys share a direction
        self.a, self.b = (r(T, HV) * spread).to(BF), (r(T, HV) * 1.5).to(BF)
        self.A, self.dt = torch.log(1 + 15 * torch.rand(HV, generator=g)), r(HV) * 0.5 + gate
        S = len(news)
        self.state = (r(S + 3, HV, V, K) * 0.2).to(state)
        self.slots = torch.randperm(S + 3, generator=g)[:S].to(torch.int32) if slots is None else torch.tensor(slots, dtype=torch.int32)
        self.cu = np.concatenate([[0], np.cumsum(news)]).astype(int)

    def oracle(self, initial=None, l2=True, scale=128 ** -0.5):
        return ogdn.gdn_sequences(to64(self.x), to64(self.a), to64(self.b), to64(self.A), to64(self.dt), to64(self.state),
                                  self.slots.tolist(), self.cu.tolist(), self.H, scale, initial, l2)

    def run(self, decode=False, state=None, **kw):
        st = self.state.to(self.cuda) if state is None else state
        d = lambda t: t.to(self.cuda)  # noqa: E731
        args = (d(self.x), d(self.a), d(self.b), d(self.A), d(self.dt), st, d(self.slots))
        if decode:
            o = gdn_decode(*args, num_q_heads=self.H, **kw)
        else:
            o = gdn_prefill(*args, d(torch.tensor(kw.pop("cu", self.cu), dtype=torch.int32)), num_q_heads=self.H, **kw)
        torch.cuda.synchronize()
        return o, st

    def check(self, o, st, ref, rst, what=""):
        eo, es = rel_err(to64(o), ref), rel_err(to64(st), rst)
        print(f"  {what} out err {eo:.2e} state err {es:.2e}", flush=True)
        assert eo < TOL[BF] and es < TOL[st.dtype]
        # And no row of the state is worse off by more than chance, 8 times that bound of what went into it.  With
        # T = (I + L)^-1, T_jl = -beta_j D_jl k_j^T [prod_(l < m < j) (I - beta_m k_m k_m^T)] k_l, products of
        # contractions, so |T| <= 1 and an error of d_j is one of the R_l's, |R_l| <= |v_l| + |S0 row|: what the row's
        # own final norm is plays no part (equal keys and update rates of 1 leave it as small as its last v).
        rows = np.maximum(np.linalg.norm(rst, axis=-1), np.linalg.norm(to64(self.state), axis=-1))
        v = np.abs(to64(self.x)[:, -rows.shape[1] * rows.shape[2]:]).reshape(-1, *rows.shape[1:])
        for s, slot in enumerate(self.slots.tolist()):
            if slot >= 0 and self.cu[s] < self.cu[s + 1]:
                rows[slot] = np.maximum(rows[slot], v[self.cu[s]:self.cu[s + 1]].max(0))
        d = np.linalg.norm(to64(st) - rst, axis=-1) / rows
        print(f"  worst row at {d.max() / (8 * TOL[st.dtype]):.3f} of its bound", flush=True)
        assert d.max() < 8 * TOL[st.dtype]


NEWS = [[1], [2], [15, 16, 17], [63], [64], [65], [128, 127, 129, 1], [200, 3]]


@pytest.mark.gpu
@pytest.mark.parametrize("state", [torch.float32, BF])
@pytest.mark.parametrize("news", NEWS)
def test_prefill_matches_oracle(cuda, news, state):
    c = Case(cuda, news, state=state, seed=len(news) + news[0])
    print(f"[gdn prefill] {news} {state}", flush=True)
    o, st = c.run()
    c.check(o, st, *c.oracle())
    others = np.setdiff1d(np.arange(len(news) + 3), c.slots.numpy())
    assert torch.equal(st.cpu()[others], c.state[others])


@pytest.mark.gpu
@pytest.mark.parametrize("H,HV,V", [(1, 1, 16), (1, 4, 32), (3, 3, 48), (16, 32, 128), (2, 4, 256)])
def test_prefill_head_layouts(cuda, H, HV, V):
    c = Case(cuda, [70, 5] if H < 16 else [70], H=H, HV=HV, V=V, seed=3)
    print(f"[gdn prefill heads] {H}/{HV}x{V}", flush=True)
    c.check(*c.run(), *c.oracle())


@pytest.mark.gpu
@pytest.mark.parametrize("gate,spread", [(-12.0, 1.0), (0.0, 1.0), (4.0, 3.0), (30.0, 1.0), (-3.0, 12.0)])
def test_prefill_decays_from_none_to_all(cuda, gate, spread):
    """Decays of 1 - 1e-5 a token, of everything within a token, and tokens of either side by side (a logarithm of
    -500 next to one of -1e-4): no difference of large sums may decide a small one."""
    c = Case(cuda, [150, 64], seed=4, gate=gate, spread=spread)
    print(f"[gdn decay] gate {gate} spread {spread}", flush=True)
    o, st = c.run()
    assert torch.isfinite(o).all() and torch.isfinite(st).all()
    c.check(o, st, *c.oracle())


@pytest.mark.gpu
def test_prefill_without_normalisation_and_its_own_scale(cuda):
    c = Case(cuda, [90], seed=5, kscale=0.12)
    c.check(*c.run(use_qk_l2norm=False, scale=0.5), *c.oracle(l2=False, scale=0.5))


@pytest.mark.gpu
def test_prefill_equal_keys(cuda):
    """The same key at every token with update rates near 1: the triangular system's largest entries."""
    c = Case(cuda, [130], seed=6)
    K = 128
    c.x[:, c.H * K:2 * c.H * K] = c.x[0, c.H * K:2 * c.H * K]
    c.b[:] = 6.0
    c.check(*c.run(), *c.oracle())


@pytest.mark.gpu
@pytest.mark.parametrize("state", [torch.float32, BF])
@pytest.mark.parametrize("S,H,HV,V", [(1, 2, 4, 128), (7, 16, 32, 128), (70, 1, 2, 48)])
def test_decode_matches_oracle(cuda, S, H, HV, V, state):
    c = Case(cuda, [1] * S, H=H, HV=HV, V=V, state=state, seed=7)
    print(f"[gdn decode] S={S} {H}/{HV}x{V} {state}", flush=True)
    c.check(*c.run(decode=True), *c.oracle())


@pytest.mark.gpu
def test_every_update_rate_rounds_as_the_exact_sigmoid(cuda):
    """beta = bf16(sigmoid(b)) for every finite bf16 b: with a zero state and q = k, o is beta (v) up to rounding, so
    a wrong side of a rounding border shows as a step of 2^-8."""
    b = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    b = b[torch.isfinite(b.float())]
    n = b.numel() // 4096 * 4096
    b = b[:n].view(-1, 1)
    want = torch.sigmoid(b.double()).to(torch.float64)
    beta = torch.from_numpy(ogdn._round_bf16(want.numpy()))
    K, V = 128, 16
    st = torch.zeros(4096, 1, V, K, device=cuda)
    for lo in range(0, n, 4096):
        x = torch.zeros(4096, 2 * K + V, dtype=BF)
        x[:, K] = 1.0
        x[:, 2 * K:] = 1.0
        st.zero_()
        gdn_decode(x.to(cuda), torch.zeros(4096, 1, dtype=BF, device=cuda), b[lo:lo + 4096].to(cuda), torch.zeros(1, device=cuda),
                   torch.zeros(1, device=cuda), st, torch.arange(4096, dtype=torch.int32, device=cuda), num_q_heads=1,
                   use_qk_l2norm=False)
        assert torch.equal(st[:, 0, 0, 0].cpu().double(), beta[lo:lo + 4096, 0].float().double()), lo


@pytest.mark.gpu
@pytest.mark.parametrize("state", [torch.float32, BF])
def test_prefill_in_pieces_then_decode_then_a_draft_tree(cuda, state):
    """A prompt in two calls, two decoded tokens, then a chain draft tree from the same slot: each step continues the
    one before (against the oracle over the whole, to what one rounding of the state a call allows)."""
    N = 6
    c = Case(cuda, [100 + 30 + 2 + N], H=2, HV=4, V=64, state=state, seed=8)
    c.slots = torch.tensor([1], dtype=torch.int32)
    full, fst = c.oracle()
    st = torch.cat([c.state, c.state.new_zeros((N, *c.state.shape[1:]))]).to(cuda)
    d = lambda t: t.to(cuda)  # noqa: E731
    at, outs = 0, []
    for n in (100, 30, 1, 1):
        r = slice(at, at + n)
        rows = (d(c.x[r]), d(c.a[r]), d(c.b[r]), d(c.A), d(c.dt), st, d(c.slots))
        if n == 1:
            outs.append(gdn_decode(*rows, num_q_heads=c.H))
        else:
            outs.append(gdn_prefill(*rows, torch.tensor([0, n], dtype=torch.int32, device=cuda), num_q_heads=c.H))
        at += n
    r = slice(at, at + N)
    outs.append(tree_gdn_vllm(d(c.x[r]), d(c.a[r]), d(c.b[r]), d(c.A), d(c.dt), st, torch.arange(4, 4 + N),
                              torch.arange(-1, N - 1), num_q_heads=c.H, prefix_slot=1))
    torch.cuda.synchronize()
    tol = 1e-5 if state == torch.float32 else (4 + N) * 2.0 ** -8
    eo, es = rel_err(to64(torch.cat(outs)), full), rel_err(to64(st)[4 + N - 1], fst[1])
    print(f"[gdn run] {state} out {eo:.2e} state {es:.2e}", flush=True)
    assert eo < 2.0 ** -8 + tol and es < tol


@pytest.mark.gpu
@pytest.mark.parametrize("decode", [False, True])
def test_padding_refused_and_shared_slots(cuda, decode):
    """Slot -1: nothing read or written.  A slot outside the state, or of two sequences: NaN rows, the slot as it was,
    the status word; the other sequences as without them."""
    news = [1] * 6 if decode else [70, 3, 64, 5, 1, 66]
    c = Case(cuda, news, seed=9, slots=[4, -1, 99, 2, 2, 6])
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((sum(news), 4, 64), 7.0, dtype=BF, device=cuda)
    o, st = c.run(decode, out=out, status=status)
    assert o is out and status.item() == 1
    rows = [slice(c.cu[s], c.cu[s + 1]) for s in range(6)]
    assert (out[rows[1]] == 7).all() and all(out[rows[s]].isnan().all() for s in (2, 3, 4))
    ok = Case(cuda, news, seed=9, slots=[4, -1, -1, -1, -1, 6])
    ref, rst = ok.oracle()
    for s in (0, 5):
        assert rel_err(to64(out[rows[s]]), ref[rows[s]]) < TOL[BF]
    assert rel_err(to64(st), rst) < 1e-5
    others = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(st.cpu()[others], c.state[others])
    status.zero_()
    ok.run(decode, status=status)
    assert status.item() == 0


@pytest.mark.gpu
def test_prefill_rows_of_no_sequence_empty_and_foreign_bounds(cuda):
    """Rows before the first and behind the last sequence stay; an empty sequence leaves its slot (also with initial
    false); bounds outside the rows skip the sequence and set status."""
    c = Case(cuda, [3, 70, 0, 20, 7], seed=10)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    sub = Case(cuda, [3, 70, 0, 20, 7], seed=10)
    sub.news, sub.cu, sub.slots = [70, 0, 20], c.cu[1:5], c.slots[1:4]
    ref, rst = sub.oracle(initial=[True, False, False])
    out = torch.full((100, 4, 64), 7.0, dtype=BF, device=cuda)
    o, st = sub.run(out=out, status=status, initial=torch.tensor([True, False, False]))
    assert status.item() == 0 and (out[:3] == 7).all() and (out[93:] == 7).all()
    assert rel_err(to64(out[3:93]), ref[3:93]) < TOL[BF] and rel_err(to64(st), rst) < 1e-5
    out.fill_(7.0)
    o, st2 = sub.run(out=out, status=status, cu=[3, 73, 73, 101])
    assert status.item() == 1 and (out[73:] == 7).all()
    assert torch.equal(st2[c.slots[3].item()].cpu(), c.state[c.slots[3].item()])


@pytest.mark.gpu
def test_prefill_and_decode_in_one_graph(cuda):
    """Captured together and replayed on new rows, with eager work between: every replay equals the eager calls."""
    c = Case(cuda, [130, 40], seed=11)
    d = lambda t: t.to(cuda)  # noqa: E731
    x, a, b, A, dt, slots = d(c.x), d(c.a), d(c.b), d(c.A), d(c.dt), d(c.slots)
    cu = torch.tensor(c.cu, dtype=torch.int32, device=cuda)
    st = d(c.state)

    def step(st):
        o = gdn_prefill(x, a, b, A, dt, st, slots, cu, num_q_heads=c.H)
        return o, gdn_decode(x[:2], a[:2], b[:2], A, dt, st, slots, num_q_heads=c.H)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(st)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(st)
    for i in range(4):
        x.copy_(torch.randn(x.shape, device=cuda))
        st.copy_(c.state)
        graph.replay()
        got, gst = [o.clone() for o in outs], st.clone()
        est = d(c.state)
        want = step(est)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(gst, est), i


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["q", "k", "v", "a", "b"])
@pytest.mark.parametrize("at", [0, 5, 22, 70, 127])
def test_a_row_that_is_not_finite_leaves_the_rows_before_it(cuda, where, at):
    """NaN or infinity in one row's q, k, v or gates: the rows before it are what they are without it, it and (but for q)
    the rows after it are NaN where it reaches: the whole value head, or with v its own column; the other sequence and
    the other heads as without it."""
    clean = Case(cuda, [150, 40], seed=12)
    ref, rst = clean.run()
    c = Case(cuda, [150, 40], seed=12)
    K, h = 128, 1                                                          # q/k head 1: value heads 2 and 3
    hit = torch.zeros(4, 64, dtype=torch.bool)
    if where == "q":
        c.x[at, h * K + 3] = float("nan")
        hit[2:] = True
    elif where == "k":
        c.x[at, (c.H + h) * K + 7] = float("inf")
        hit[2:] = True
    elif where == "v":
        c.x[at, 2 * c.H * K + 2 * 64 + 9] = float("nan")
        hit[2, 9] = True
    else:
        (c.a if where == "a" else c.b)[at, 3] = float("nan")
        hit[3] = True
    o, st = c.run()
    assert torch.equal(o[:at], ref[:at]) and torch.equal(o[150:], ref[150:])
    after = o[at:150].cpu()
    assert torch.equal(after[:, ~hit], ref[at:150].cpu()[:, ~hit])
    assert after[0][hit].isnan().all()
    if where == "q":
        assert torch.equal(o[at + 1:], ref[at + 1:]) and torch.equal(st, rst)
    else:
        assert after[:, hit].isnan().all()
        s = st[c.slots[0]].cpu()
        assert s[hit].isnan().all() and torch.equal(s[~hit], rst[c.slots[0]].cpu()[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("n,S", [(8, 1), (9, 1), (10, 1), (11, 1), (16, 8), (17, 8), (24, 8), (25, 8)])
def test_rows_in_turn_and_chunks_at_the_rule_between_them(cuda, n, S):
    """Row counts on either side of the one up to which the rows go one after another."""
    c = Case(cuda, [n] * S, H=16 if S == 8 else 2, HV=32 if S == 8 else 4, V=128, seed=13)
    c.check(*c.run(), *c.oracle())


@pytest.mark.gpu
def test_index_tensors_of_64_bits(cuda):
    """int64 slots and bounds; a value past 32 bits is outside, not what its low half says; floats are refused."""
    c = Case(cuda, [30, 4], seed=14)
    ref, rst = c.oracle()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    c.slots = c.slots.long()
    o, st = c.run(status=status)
    c.check(o, st, ref, rst)
    assert status.item() == 0
    c.slots[1] += 2 ** 32
    o, st = c.run(status=status)
    assert status.item() == 1 and o[30:].isnan().all() and not o[:30].isnan().any()
    c.slots = c.slots.double()
    with pytest.raises(ValueError, match="integers"):
        c.run()


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Prefills on two streams together give what each gives alone (workspaces are the call's own)."""
    cases = [Case(cuda, [300, 70], H=4, HV=8, V=128, seed=15 + i) for i in range(2)]
    alone = [c.run() for c in cases]
    args = []
    for c in cases:
        cu = torch.tensor(c.cu, dtype=torch.int32).to(cuda)
        args.append([t.to(cuda) for t in (c.x, c.a, c.b, c.A, c.dt)] + [c.slots.to(cuda), cu])
    states = [[c.state.to(cuda) for _ in range(6)] for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for r in range(6):
        for i, s in enumerate(streams):
            x, a, b, A, dt, slots, cu = args[i]
            with torch.cuda.stream(s):
                got[i].append(gdn_prefill(x, a, b, A, dt, states[i][r], slots, cu, num_q_heads=4))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i][0]) for o in got[i]) and all(torch.equal(t, alone[i][1]) for t in states[i])


@pytest.mark.gpu
def test_many_sequences(cuda):
    """As many sequences as a call takes, of 0 to 2 rows and one long one."""
    g = torch.Generator().manual_seed(17)
    for S, many in ((4096, 0), (500, 6000)):
        news = torch.randint(0, 3, (S,), generator=g).tolist()
        news[S // 2] += many
        c = Case(cuda, news, H=1, HV=1, V=16, seed=18)
        c.check(*c.run(), *c.oracle())
    with pytest.raises(ValueError, match="4096"):
        gdn_prefill(c.x.to(cuda), c.a.to(cuda), c.b.to(cuda), c.A.to(cuda), c.dt.to(cuda), c.state.to(cuda),
                    torch.zeros(4097, dtype=torch.int32, device=cuda), torch.zeros(4098, dtype=torch.int32, device=cuda),
                    num_q_heads=1)


@pytest.mark.gpu
@pytest.mark.parametrize("state", [torch.float32, BF])
@pytest.mark.parametrize("news", [[1] * 63 + [300], [200] + [1] * 40 + [65, 10, 11], [3, 64, 0, 1, 129, 24, 25, 2], [11, 10, 12] * 7])
def test_short_and_long_sequences_in_one_call(cuda, news, state):
    """Each sequence by the form for its own length, whatever the others': decode rows beside prompts; with a padding
    entry, a foreign slot and a shared one of either length, and rows of no sequence."""
    c = Case(cuda, news, state=state, seed=19)
    ref, rst = c.oracle()
    c.check(*c.run(), ref, rst)
    long, short = int(np.argmax(news)), int(np.argmin([n or 99 for n in news]))
    for s in (long, short):
        for bad in (-1, len(news) + 3):
            keep = c.slots.clone()
            c.slots[s] = bad
            status = torch.zeros(1, dtype=torch.int32, device=cuda)
            out = torch.full((sum(news), c.A.shape[0], 64), 7.0, dtype=BF, device=cuda)
            o, st = c.run(status=status, out=out)
            at = slice(c.cu[s], c.cu[s + 1])
            assert status.item() == (bad != -1)
            assert (o[at] == 7).all() if bad == -1 else o[at].isnan().all()
            assert torch.equal(st[keep[s]].cpu(), c.state[keep[s]])
            rows = torch.ones(sum(news), dtype=torch.bool)
            rows[at] = False
            assert rel_err(to64(o.cpu()[rows]), ref[rows.numpy()]) < TOL[BF]
            c.slots = keep


@pytest.mark.gpu
def test_bounds_with_one_sequence_of_no_rows(cuda):
    """One sequence that has no rows of a query that has: nothing but the status of its slot."""
    c = Case(cuda, [90], seed=20)
    for slot, want in ((0, 0), (9, 1), (-1, 0)):
        c.slots = torch.tensor([slot], dtype=torch.int32)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.full((90, 4, 64), 7.0, dtype=BF, device=cuda)
        o, st = c.run(status=status, out=out, cu=[40, 40])
        assert status.item() == want and (o == 7).all() and torch.equal(st.cpu(), c.state)
