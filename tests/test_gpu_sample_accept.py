"""The sampled acceptance on the GPU against the float64 oracle, which adds one token's weight after the other: tokens, paths
and lengths equal, logprobs within one fp32 rounding (half a step of 2^-24, relative) of the 64-bit value's neighbourhood.

A draw compares a running sum with u times the total.  Two orders of adding the same float64 weights differ by at most V eps
of the total, V 2^-52: over a row's borders together the chance that a u falls between them is below V^2 2^-52, 1.4e-5 for
248,320 tokens, and none of the seeds here has one."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.tree_verify import tree_sample_accept
from oracle import tree_verify as otv


def _tree(n, rng):
    return np.array([int(rng.integers(max(-1, i - 9), i)) for i in range(n)], dtype=np.int64)


def _case(ns, V, dtype, seed, scale=2.5):
    """Requests of ns drafts over rows with a few likely tokens; drafts among their parent row's likely ones."""
    rng = np.random.default_rng(seed)
    R, D = sum(n + 1 for n in ns), sum(ns)
    x = rng.normal(size=(R, V)) * scale
    for r in range(R):
        x[r, rng.integers(0, V, 4)] += 4 * scale
    x = torch.from_numpy(x).to(dtype)
    cu_d, cu_r = np.cumsum(ns), np.cumsum([n + 1 for n in ns])
    par = np.concatenate([_tree(n, rng) for n in ns] + [np.zeros(0, np.int64)])
    draft = np.zeros(D, dtype=np.int64)
    xs = x.double().numpy()
    for b, n in enumerate(ns):
        for i in range(n):
            d = cu_d[b] - n + i
            row = cu_r[b] - (n + 1) + par[d] + 1
            draft[d] = np.argsort(-xs[row], kind="stable")[rng.integers(0, min(3, V))]
    return x, cu_d, cu_r, draft, par, rng


def _check(x, cu_d, cu_r, draft, par, spec, u, T, k, P, dev, tokens=True):
    t = lambda v, d: None if v is None else torch.tensor(np.asarray(v), dtype=d, device=dev)      # noqa: E731
    got = tree_sample_accept(x.to(dev) if not x.is_cuda else x, cu_d, cu_r, draft, par, spec, t(u, torch.float32),
                             t(T, torch.float32), top_k=t(k, torch.int32), top_p=t(P, torch.float32))
    torch.cuda.synchronize()
    f32 = lambda v: None if v is None else np.asarray(v, dtype=np.float32).astype(np.float64)      # noqa: E731
    ref = otv.sampled_descent(x.double().cpu().numpy(), cu_d, cu_r, draft, par, spec, f32(u), f32(T), k, f32(P))
    for g, r in zip(got[:3], ref[:3]):
        assert np.array_equal(g.cpu().numpy(), r)
    # one rounding to fp32 (2^-24 of the value), and the log of a quotient whose 64-bit sums may be off by V 2^-52
    lp = got[3].double().cpu().numpy()
    assert (np.abs(lp - ref[3]) <= np.abs(ref[3]) * 2.0 ** -24 + x.shape[1] * 2.0 ** -51).all()
    return ref


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 511, 1000, 8192, 8200, 32000, 65535, 65543, 248320])
def test_matches_the_oracle_over_vocabularies(cuda, V, dtype):
    ns = [5, 0, 3, 9, 1] if V < 100000 else [5, 0]
    x, cu_d, cu_r, draft, par, rng = _case(ns, V, dtype, V)
    B = len(ns)
    print(f"[sample accept] V={V} {dtype}", flush=True)
    for k, P in ((None, None), ([3, 0, 50, 1, V + 5][:B], [0.9, 0.5, 1.0, 0.99, 0.0][:B])):
        _check(x, cu_d, cu_r, draft, par, max(ns), rng.random(x.shape[0]), [1.0, 0.6, 0.0, 1.7, 0.9][:B], k, P, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_trees_with_filters(cuda, seed):
    rng = np.random.default_rng(seed)
    ns = [int(v) for v in rng.integers(0, 41, 7)]
    x, cu_d, cu_r, draft, par, rng = _case(ns, 3001, torch.bfloat16 if seed % 2 else torch.float16, seed, scale=1.5)
    T = rng.choice([0.0, 0.3, 0.7, 1.0, 1.5], 7)
    print(f"[sample accept] trees {ns}", flush=True)
    ref = _check(x, cu_d, cu_r, draft, par, max(ns) + seed, rng.random(x.shape[0]), T, rng.integers(0, 60, 7),
                 rng.random(7) * 1.2, cuda)
    assert ref[2].max() >= 1


@pytest.mark.gpu
@pytest.mark.parametrize("V", [70000, 248320])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_whose_value_counts_pass_16_bits(cuda, V, dtype):
    """Constant rows, rows masked to the type's lowest value, and rows of two values: a value's count is above 65,535,
    in either half of the values or both."""
    lowest = torch.finfo(dtype).min
    x = torch.full((7, V), 1.5, dtype=dtype)
    x[1] = lowest
    x[1, 123], x[1, V - 1] = 2.0, 1.0
    x[2] = -3.25
    x[3, ::2] = -1.5
    x[4] = float("-inf")
    x[4, 69999] = -7.0
    x[5] = lowest
    x[6, : V // 2] = 1.25
    rng = np.random.default_rng(V)
    print(f"[sample accept] counts over 16 bits V={V} {dtype}", flush=True)
    for T, k, P in ((1.0, 0, 1.0), (0.8, 66000, 0.97), (50.0, 0, 0.5)):
        _check(x, np.zeros(7, np.int64), np.arange(1, 8), [], [], 0, rng.random(7), [T] * 7, [k] * 7, [P] * 7, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_infinities_nan_and_nothing(cuda, dtype):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(9, 600, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[0] = -inf
    x[1] = nan
    x[2, ::3], x[2, 1::3] = nan, -inf
    x[3, 17], x[3, 500] = inf, inf
    x[4] = 0.0
    x[4, ::2] = -0.0
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).max
    x[7] = -inf
    x[7, 599] = torch.finfo(dtype).min
    u = [0.3, 0.3, 0.99, 0.7, 0.5, 0.25, 0.75, 0.9, 0.1]
    print(f"[sample accept] odd rows {dtype}", flush=True)
    for T in (1.0, 0.0, 1e-30, 1e30, inf):
        _check(x, np.zeros(9, np.int64), np.arange(1, 10), [], [], 0, u, [T] * 9, None, None, cuda)
        _check(x, np.zeros(9, np.int64), np.arange(1, 10), [], [], 0, u, [T] * 9, [5] * 9, [0.9] * 9, cuda)
    # a row without a token in the middle of a walk ends it
    x = torch.full((3, 16), -1.0).to(dtype)
    x[0, 4] = 60.0
    x[1] = nan
    ref = _check(x, [2], [3], [4, 5], [-1, 0], 2, [0.5] * 3, [1.0], None, None, cuda)
    assert ref[2][0] == 1 and ref[0][0].tolist() == [4, -1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V", [(1, 65536), (24, 65605), (25, 65605), (130, 65541), (3, 262144), (2, 530000)])
def test_long_rows_counted_whole_and_in_parts(cuda, R, V, dtype):
    """Few long rows are counted by several workgroups, more of them by one each: odd rows and drawn tokens in the first part,
    the last one and the last logits behind whole vectors."""
    inf, nan = float("inf"), float("nan")
    rng = np.random.default_rng(R + V)
    x = torch.randn(R, V, generator=torch.Generator().manual_seed(R)).mul(3).to(dtype)
    odd = [lambda r: r.fill_(0.0)[::2].fill_(-0.0), lambda r: r.fill_(-2.0)[V - 1:].fill_(9.0), lambda r: r.fill_(nan),
           lambda r: r.fill_(-inf)[:1].fill_(-5.0), lambda r: r.fill_(-1.0)[::3].fill_(nan), lambda r: r[::5].fill_(inf),
           lambda r: r[V // 2:].fill_(torch.finfo(dtype).min), lambda r: r.fill_(-0.5)[V - 3:].fill_(-0.25)]
    for i in range(R if R < 24 else 0, R):
        if i % 3 == 0:
            odd[i // 3 % len(odd)](x[i])
    if R < 24:
        odd[1](x[0])
    T = rng.choice([0.0, 0.7, 1.0, 40.0], R)
    print(f"[sample accept] long rows {R} x {V} {dtype}", flush=True)
    _check(x, np.zeros(R, np.int64), np.arange(1, R + 1), [], [], 0, rng.random(R), T, rng.integers(0, 2 * V, R),
           rng.random(R) * 1.3, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [5000, 60001, 70001])
def test_rows_masked_here_and_there(cuda, V, dtype):
    """A constrained request's logits: most or some of them -inf, the type's lowest value, a large negative number or the row's
    own lowest one, in no runs; temperatures from ones that drop what is masked to ones at which it counts as much as the rest."""
    lowest, far = torch.finfo(dtype).min, torch.tensor(-1.0e4).to(dtype).item()
    g = torch.Generator().manual_seed(V)
    rows = [(m, d) for m in (float("-inf"), lowest, far, -3.5, -0.0) for d in (0.03, 0.5, 0.97, 0.9999)] + [(float("nan"), 0.6)]
    R = len(rows) + (6 if V == 70001 else 0)       # (more than 24 long rows are counted whole)
    x = torch.randn(R, V, generator=g).mul(2).to(dtype)
    x[-1], x[-2] = x[-1].abs() + 1, -x[-2].abs() - 1
    for i, (m, d) in enumerate(rows):
        x[i] = torch.where(torch.rand(V, generator=g) < d, torch.tensor(m).to(dtype), x[i])
    rng = np.random.default_rng(V)
    print(f"[sample accept] masked rows {R} x {V} {dtype}", flush=True)
    for n in (R, 20):
        for T in (1.0, 0.0, 3.0e4, 1e38):
            k = rng.integers(0, 2 * V, n) * (rng.random(n) < 0.7)
            _check(x[:n], np.zeros(n, np.int64), np.arange(1, n + 1), [], [], 0, rng.random(n), [T] * n, k,
                   np.where(rng.random(n) < 0.5, 1.0, rng.random(n)), cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [4096, 8203, 32768])
def test_many_rows_of_every_kind(cuda, V, dtype):
    """More rows than CUs: narrower counts, which clustered and constant rows leave."""
    R = 264
    g = torch.Generator().manual_seed(V)
    x = torch.randn(R, V, generator=g).to(dtype)
    kinds = [lambda r: r.mul_(2.5), lambda r: r.mul_(0.3).sub_(6), lambda r: r.mul_(0.01).add_(3), lambda r: r.fill_(-1.25),
             lambda r: r[::2].fill_(torch.finfo(dtype).min), lambda r: r[: V // 2].fill_(float("-inf")), lambda r: r.fill_(0.0)[::3].fill_(-0.0),
             lambda r: r.fill_(float("-inf")), lambda r: r[::7].fill_(float("nan")), lambda r: r.fill_(-2.0)[1::2].fill_(-1.0),
             lambda r: r.fill_(7.0)[5:9].fill_(8.0)]
    for i in range(R):
        kinds[i % len(kinds)](x[i])
    rng = np.random.default_rng(V)
    print(f"[sample accept] rows of every kind {R} x {V} {dtype}", flush=True)
    T = rng.choice([0.0, 0.5, 1.0, 30.0], R)
    _check(x, np.zeros(R, np.int64), np.arange(1, R + 1), [], [], 0, rng.random(R), T, rng.integers(0, V, R) * (rng.random(R) < 0.6),
           np.where(rng.random(R) < 0.4, 1.0, rng.random(R)), cuda)


@pytest.mark.gpu
def test_uniforms_at_and_past_their_ends(cuda):
    x = torch.randn(8, 501, generator=torch.Generator().manual_seed(4)).bfloat16()
    u = [0.0, -1.0, float("nan"), 1.0, 7.0, float("inf"), 1 - 2.0 ** -24, 2.0 ** -30]
    print("[sample accept] uniforms", flush=True)
    for P in (None, [0.9] * 8, [1e-9] * 8, [-1.0] * 8, [float("nan")] * 8):
        _check(x, np.zeros(8, np.int64), np.arange(1, 9), [], [], 0, u, [1.0] * 8, None, P, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 0), (8, 1), (5, 3)])
def test_strided_and_unaligned_rows(cuda, pad, shift):
    x, cu_d, cu_r, draft, par, rng = _case([4, 2], 1003, torch.float16, 9)
    big = torch.full((x.shape[0] * (1003 + pad) + shift,), 99.0, dtype=torch.float16, device=cuda)
    view = big[shift:].view(x.shape[0], 1003 + pad)[:, :1003]
    view.copy_(x.to(cuda))
    print(f"[sample accept] pad {pad} shift {shift}", flush=True)
    _check(view, cu_d, cu_r, draft, par, 4, rng.random(x.shape[0]), [1.0, 0.5], [0, 9], None, cuda)


@pytest.mark.gpu
def test_device_counts_padding_requests_and_refused_ones(cuda):
    """Counts on the device: padding requests emit nothing, ones that do not fit are refused with the status set, and the
    others are as if alone; rows behind the last request are left out."""
    x, cu_d, cu_r, draft, par, rng = _case([3, 2, 4], 700, torch.bfloat16, 12)
    x = torch.cat([x, x[:3]]).to(cuda)
    u = torch.rand(x.shape[0], device=cuda)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)                              # noqa: E731
    dr, pa = ints(draft.tolist()), ints(par.tolist())

    def call(cd, cr, T):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        got = tree_sample_accept(x, ints(cd), ints(cr), dr, pa, 4, u, torch.tensor(T, device=cuda), status=status)
        torch.cuda.synchronize()
        return [g.cpu().numpy() for g in got], int(status)
    print("[sample accept] device counts", flush=True)
    ref, st = call([3, 5, 9], [4, 7, 12], [1.0, 0.7, 0.9])
    assert st == 0
    want = otv.sampled_descent(x.double().cpu().numpy(), [3, 5, 9], [4, 7, 12], draft, par, 4, u.double().cpu().numpy(),
                               [float(np.float32(t)) for t in (1.0, 0.7, 0.9)])
    assert all(np.array_equal(g, w) for g, w in zip(ref[:3], want[:3]))
    got, st = call([3, 3, 5, 9, 9], [4, 4, 7, 12, 12], [1.0, 9.0, 0.7, 0.9, 9.0])                  # padding among them
    assert st == 0 and all(np.array_equal(g[[0, 2, 3]], r) for g, r in zip(got, ref))
    assert (got[0][[1, 4]] == -1).all() and (got[2][[1, 4]] == 0).all() and (got[3][[1, 4]] == 0).all()
    for cd, cr, good in (([3, 5, 9], [4, 7, 13], 2), ([3, 5, 10], [4, 7, 13], 2), ([3, 5, 9], [4, 6, 12], 1),
                         ([3, 5, 4], [4, 7, 6], 2), ([-1, 5, 9], [4, 7, 12], 0), ([3, 5, 9], [4, 7, 2 ** 31 - 1], 2),
                         ([3, 1, 9], [4, 2, 12], 1)):
        got, st = call(cd, cr, [1.0, 0.7, 0.9])
        assert st == 1
        assert all(np.array_equal(g[:good], r[:good]) for g, r in zip(got, ref))
        assert (got[0][good] == -1).all() and got[2][good] == 0
    # walks over parents and drafts that name no node stay in the tree
    pa2 = ints([5, -7, 0, 2 ** 31 - 1, -1, 3, 3, 3, -1])
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = tree_sample_accept(x, ints([3, 5, 9]), ints([4, 7, 12]), dr, pa2, 4, u, torch.ones(3, device=cuda), status=status)
    assert int(got[2][0]) == 0 and int(status) == 0


@pytest.mark.gpu
def test_many_requests(cuda):
    """More requests than one look of a wave at the counts holds (64), and more than one at the bounds (256)."""
    for B in (65, 300):
        x, cu_d, cu_r, draft, par, rng = _case([1] * B, 130, torch.bfloat16, B)
        print(f"[sample accept] {B} requests", flush=True)
        _check(x, cu_d, cu_r, draft, par, 1, rng.random(x.shape[0]), rng.choice([0.0, 0.8, 1.2], B),
               rng.integers(0, 20, B), rng.random(B) + 0.2, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5000, 70001])
def test_graph_replays_follow_their_inputs(cuda, V):
    x, cu_d, cu_r, draft, par, rng = _case([6, 3], V, torch.bfloat16, 21)
    ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=cuda)                  # noqa: E731
    xg, u = x.to(cuda), torch.rand(x.shape[0], device=cuda)
    args = (ints(cu_d), ints(cu_r), ints(draft), ints(par), 6, u, torch.tensor([1.0, 0.7], device=cuda))
    tree_sample_accept(xg, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):    # (as the draft graphs: captures of one mode go together)
        out = tree_sample_accept(xg, *args)
    for i in range(4):
        print(f"[sample accept] replay {i}", flush=True)
        u.copy_(torch.rand(x.shape[0]))
        xg.copy_(x.roll(i, 1))
        want = [w.clone() for w in tree_sample_accept(xg, *args)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_refusals(cuda):
    x = torch.zeros(3, 8, dtype=torch.bfloat16, device=cuda)
    u, T = torch.zeros(3, device=cuda), torch.ones(1, device=cuda)
    ok = ([2], [3], [1, 2], [-1, 0], 2)
    tree_sample_accept(x, *ok, u, T)
    for bad in ((u[:2], T), (u.double(), T), (u.cpu(), T), (u, T.half()), (u, torch.ones(2, device=cuda)), (u, 1.0), ([0.5] * 3, T)):
        with pytest.raises(ValueError):
            tree_sample_accept(x, *ok, *bad)
    for kw in (dict(top_k=T), dict(top_p=u), dict(top_p=T.int()), dict(status=T)):
        with pytest.raises(ValueError):
            tree_sample_accept(x, *ok, u, T, **kw)
    with pytest.raises(ValueError, match="inconsistent"):
        tree_sample_accept(x, [2], [4], [1, 2], [-1, 0], 2, u, T)
    with pytest.raises(ValueError, match="integers"):
        tree_sample_accept(x, torch.tensor([2.0]), *ok[1:], u, T)
