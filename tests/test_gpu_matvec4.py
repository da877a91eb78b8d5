"""The 4-bit head on the GPU against float64: quantised weights equal, products within the roundings.

A product's whole numbers and fp16 values multiply exactly in fp32.  A group's G terms are added in fp32 in some order: off by
at most G 2^-23 of the sum of their magnitudes (2^-23 a step also where a unit truncates); the scaled groups by as much a group, one more for the scaling; then one rounding to fp16, 2^-11 of the value (2^-25 below its normal range)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import to64
from chain_flow_amd.config import flownet
from chain_flow_amd.drafter import Drafter
from chain_flow_amd.head import QuantHead, ShortlistHead, matvec4, quantize4, row_topk
from chain_flow_amd.weights import make_weights, synthetic_context
from oracle import beam as obeam
from oracle import head as ohead


def _weights(n, K, group, seed, dev):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (n, K // 2), dtype=torch.uint8, generator=g)
    s = (torch.exp2(torch.randn(n, K // group, generator=g)) * 0.02).half()
    return w.to(dev), s.to(dev), ohead.dequant4(ohead.unpack4(w.numpy()), to64(s))


def _close(y, x, W, group):
    x, y = np.asarray(x, dtype=np.float64), to64(y)
    K = W.shape[1]
    ref, mag = x @ W.T, np.abs(x) @ np.abs(W).T
    tol = np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 + (group + K / group + 2) * 2.0 ** -23 * mag
    worst = float((np.abs(y - ref) / tol).max()) if y.size else 0.0
    assert worst <= 1.0, worst
    return worst


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,n,K", [(1, 1, 128), (1, 17, 128), (3, 15, 256), (2, 16, 384), (5, 129, 640), (16, 1000, 640), (17, 33, 1024),
                                   (8, 8191, 2560), (1, 62642, 2560), (4, 4099, 5376), (16, 2049, 4096), (16, 300, 5376), (40, 500, 1152),
                                   (2, 40, 65536), (7, 64, 20480), (9, 2048, 128)])
def test_products_match_float64(cuda, M, n, K, group):
    w, s, W = _weights(n, K, group, M + n, cuda)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).half()
    y = matvec4(x.to(cuda), w, s)
    torch.cuda.synchronize()
    print(f"[matvec4] M={M} n={n} K={K} G={group}: {_close(y, x.numpy(), W, group):.2f} of the bound", flush=True)


@pytest.mark.gpu
def test_strided_rows_gathered_columns_and_given_outputs(cuda):
    w, s, W = _weights(77, 640, 64, 1, cuda)
    x = torch.randn(9, 3, 512, generator=torch.Generator().manual_seed(2)).half()
    t = torch.randn(11, 128, generator=torch.Generator().manual_seed(3)).half()
    ids = torch.tensor([3, -1, 10, 99, 0, -7, 2 ** 31 - 1, 5, 5], dtype=torch.int32)
    full = np.concatenate([x[:, 1].double().numpy(), t.double().numpy()[np.clip(ids.numpy(), 0, 10)]], 1)
    wide = torch.stack([ids, ids + 1 - 1, ids * 0], 1).flatten().contiguous()
    out = torch.full((9, 77), 7.0, dtype=torch.float16, device=cuda)
    print("[matvec4] gathered columns", flush=True)
    got = matvec4(x.to(cuda)[:, 1], w, s, table=t.to(cuda), ids=wide.to(cuda), ids_stride=3, out=out)
    torch.cuda.synchronize()
    assert got is out
    _close(out, full, W, 64)
    odd = torch.zeros(9 * 640 + 1, dtype=torch.float16, device=cuda)[1:].view(9, 640)     # rows no vector load can read
    odd.copy_(torch.from_numpy(full).half())
    _close(matvec4(odd, w, s), full, W, 64)
    big = torch.zeros(78 * 320 + 8, dtype=torch.uint8, device=cuda)
    big[8:8 + 77 * 320].view(77, 320).copy_(w)                                              # weights off their alignment
    _close(matvec4(odd, big[8:8 + 77 * 320].view(77, 320), s.t().contiguous().t()), full, W, 64)
    assert matvec4(odd[:0], w, s).shape == (0, 77) and matvec4(odd, w[:0], s[:0]).shape == (9, 0)
    for bad in (dict(out=out[:8]), dict(out=out.float()), dict(out=torch.zeros(77, 9, dtype=torch.float16, device=cuda).t())):
        with pytest.raises(ValueError):
            matvec4(odd, w, s, **bad)
    with pytest.raises(ValueError, match="one GPU"):
        matvec4(odd, w, s.cpu())


@pytest.mark.gpu
def test_what_is_not_finite_stays_in_its_row_and_column(cuda):
    w, s, W = _weights(50, 256, 32, 5, cuda)
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(6)).half()
    clean = matvec4(x.to(cuda), w, s)
    x[1, 30], x[3, 200] = float("nan"), float("inf")
    s[7, 2] = float("nan")
    s[9, 0] = float("inf")
    print("[matvec4] NaN and infinities", flush=True)
    y = matvec4(x.to(cuda), w, s).cpu()
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any() and torch.isnan(y[:, 7]).all()
    rows, cols = [0, 2, 4], [c for c in range(50) if c not in (7, 9)]
    assert torch.equal(y[rows][:, cols], clean.cpu()[rows][:, cols])
    # results past fp16's range are infinite, as a conversion's
    s2 = torch.full_like(s, 60000.0)
    assert torch.isinf(matvec4(torch.full((1, 256), 60000.0, dtype=torch.float16, device=cuda), torch.full_like(w, 0xff), s2)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_weights_equal_the_oracles(cuda, group):
    g = torch.Generator().manual_seed(group)
    w = (torch.randn(300, 512, generator=g) * torch.exp(torch.randn(300, 1, generator=g) * 2)).half()
    w[5] = 0
    w[6] = 6e-8
    w[7, ::2] = 65504.0
    w2 = torch.randn(300, 256, generator=g).half()
    rows = torch.randperm(300, generator=g)[:121]
    q, s = quantize4(w.to(cuda), group, rows.to(cuda), w2.to(cuda))
    torch.cuda.synchronize()
    full = np.concatenate([to64(w), to64(w2)], 1)[rows.numpy()]
    oq, os_ = ohead.quantize4(full, group)
    print(f"[quantize4] G={group}", flush=True)
    assert np.array_equal(to64(s), os_)
    got = ohead.unpack4(q.cpu().numpy())
    # (a quotient within fp32's half step of a border between two whole numbers may fall on either)
    near = np.abs(np.abs(full / np.maximum(np.repeat(os_, group, 1), 1e-300)) % 1 - 0.5) < 2.0 ** -20
    assert ((got == oq) | near).all() and (np.abs(got - oq) <= 1).all() and (got != oq).mean() < 1e-3
    bad = w.clone()
    bad[1, 3], bad[2, 100] = float("nan"), float("-inf")
    q, s = quantize4(bad.to(cuda), group)
    s = s.cpu()
    want = torch.zeros(300, 512 // group, dtype=torch.bool)
    want[1, 3 // group] = want[2, 100 // group] = True
    assert torch.equal(torch.isnan(s), want)
    with pytest.raises(ValueError, match="rows"):
        quantize4(w.to(cuda), group, torch.tensor([300]))


@pytest.mark.gpu
def test_head_of_4_bits(cuda):
    """Logits and top-k against the dequantised rows; near the fp16 head's logits by the scales' half steps."""
    cfg = flownet(512, layers=1, flow_steps=1)
    W = make_weights(cfg, 4096, init="test", base_seed=7)
    sl = torch.randperm(4096, generator=torch.Generator().manual_seed(3))[:1999].sort().values
    args = [W["lm_head.weight"].half().to(cuda), sl, W["markov.w1.weight"], W["markov.w2.weight"]]
    head, full = QuantHead(*args, group=32), ShortlistHead(*args)
    h = (torch.randn(11, 512, generator=torch.Generator().manual_seed(4))).half()
    prev = torch.randint(-1, 4096, (11, 2), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    print("[4-bit head]", flush=True)
    D = ohead.dequant4(ohead.unpack4(head.weight.cpu().numpy()), to64(head.scale))
    w1 = to64(head.w1)
    x = np.concatenate([to64(h), w1[np.clip(prev[:, 0].numpy(), 0, None)]], 1)
    lg = head.logits(h.to(cuda), prev.to(cuda).view(-1), 2)
    _close(lg, x, D, 32)
    x0 = np.concatenate([to64(h), np.zeros((11, head.r))], 1)
    _close(head.logits(h.to(cuda)), x0, D, 32)
    # against the fp16 head: each weight off by half a scale, each fp16 sum by its roundings
    slack = np.abs(x) @ np.repeat(to64(head.scale), 32, 1).T / 2
    ref = full.logits(h[:8].to(cuda), prev[:8].to(cuda).view(-1), 2)
    assert (np.abs(to64(lg[:8]) - to64(ref)) <= slack[:8] + 2e-3 * (1 + np.abs(to64(ref)))).all()
    vals, ids, lse = head.topk(h.to(cuda), 5, prev.to(cuda).view(-1), 2)
    torch.cuda.synchronize()
    ls = torch.log_softmax(lg.double(), 1)
    order = torch.sort(ls, dim=1, descending=True, stable=True)
    assert torch.equal(ids.long(), order.indices[:, :5]) and (vals.double() - order.values[:, :5]).abs().max() < 1e-4
    assert torch.equal(head.map(ids).cpu(), sl[ids.cpu().long()])


@pytest.mark.gpu
@pytest.mark.parametrize("M,n", [(1, 1), (2, 15), (3, 511), (1, 512), (4, 513), (1, 62642), (5, 4099), (300, 2049), (2, 300001)])
@pytest.mark.parametrize("k", [1, 4, 16])
def test_split_top_k(cuda, M, n, k):
    """A row's top k over many workgroups: ids equal to a stable sort's (lower column first among equals), -1 past the numbers."""
    x = (torch.randn(M, n, generator=torch.Generator().manual_seed(n)) * 4).half()
    x[0] = x[0].mul(2).round().div(2)              # many equal ones
    if n > 20:
        x[0, 5], x[0, n - 1], x[M - 1, 3] = float("nan"), float("-inf"), float("-inf")
    if M > 2:
        x[1] = float("-inf")
        x[2] = float("nan")
    print(f"[split top-k] {M} x {n} k {k}", flush=True)
    vals, ids, lse = (t.cpu() for t in row_topk(x.to(cuda), k, split=True))
    assert torch.equal(ids, row_topk(x.to(cuda), k)[1].cpu())
    v = to64(x)
    for m in range(M):
        order = np.argsort(np.where(np.isnan(v[m]), np.inf, -v[m]), kind="stable")
        order = order[: int((~np.isnan(v[m])).sum())][:k]
        assert ids[m, : len(order)].tolist() == order.tolist() and (ids[m, len(order):] == -1).all()
        if np.isnan(v[m]).all() or np.isneginf(v[m]).all():
            assert not torch.isfinite(lse[m])
        elif np.isnan(v[m]).any():
            assert torch.isnan(lse[m])
        else:
            top = v[m].max()
            want = top + np.log(np.exp(v[m] - top).sum())
            # exponentials within 2^-22, n of them added in fp32 by 8 a lane, lanes and sets, the log and a sum: below 2^-17 of 1
            tol = 2.0 ** -17 + abs(want) * 2.0 ** -22
            assert abs(float(lse[m]) - want) <= tol
            got = vals[m, : len(order)].double().numpy()
            want = v[m][order] - want
            assert (np.abs(got - want)[np.isfinite(want)] <= tol + np.abs(want[np.isfinite(want)]) * 2.0 ** -23).all()


@pytest.mark.gpu
def test_drafter_with_a_head_of_4_bits(cuda):
    """Chain and tree drafts over the 4-bit head equal the oracle's search over the dequantised rows, but for near ties."""
    cfg = flownet(512, layers=1, flow_steps=2)
    W = make_weights(cfg, 4096, init="test", base_seed=1)
    W["lm_head.weight"] = (W["lm_head.weight"].float() * 8).half()
    sl = torch.randperm(4096, generator=torch.Generator().manual_seed(2))[:1024].sort().values.to(torch.int32)
    dr = Drafter(cfg, {k: v.to(cuda) for k, v in W.items()}, sl.to(cuda), device=cuda, head_bits=4, head_group=32)
    ctx = synthetic_context(2, cfg.context_size, 512, seed=1)
    pred = dr.predict_hidden(ctx.to(cuda))
    known0 = torch.tensor([int(sl[7]), int(sl[100])])
    print("[4-bit drafts]", flush=True)
    chains = dr.beam_chains(None, known0.to(cuda), 5, 4, pred=pred).cpu().numpy()
    tree = dr.beam_tree(None, known0.to(cuda), 4, 4, 3, pred=pred).cpu()
    assert tree.shape == (2, 2 * 12) and set(tree[:, :12].flatten().tolist()) <= set(sl.tolist())
    D = ohead.dequant4(ohead.unpack4(dr.head.weight.cpu().numpy()), to64(dr.head.scale))
    W64 = {k: v.double().numpy() for k, v in W.items()}
    sl64 = sl.long().numpy()
    w1 = to64(dr.head.w1)

    def score(h, prev):
        x = np.concatenate([np.asarray(h, dtype=np.float64), w1[np.clip(prev, 0, None)]], 1)
        return (x @ D.T).astype(np.float16).astype(np.float64)
    resid = lambda lp, nl: ohead.path_residual(W64, W64["embed_tokens.weight"], lp, nl, cfg.path_order)    # noqa: E731
    ref, trace = obeam.beam_chains(to64(pred), known0.numpy(), sl64, 4, 5, cfg.path_order, score, resid, return_trace=True)
    near = any((ohead.margins(t["lp"], 4) <= 1e-2).any() or (ohead.margins(t["cand"], 4) <= 1e-2).any() for t in trace)
    assert np.array_equal(chains, ref) or near
    with pytest.raises(ValueError, match="one pass"):
        Drafter(cfg, W, sl, device=cuda, head_bits=4, twopass_m=64)


@pytest.mark.gpu
def test_products_in_a_graph(cuda):
    w, s, W = _weights(700, 2560, 64, 8, cuda)
    x = torch.randn(20, 2560, device=cuda).half()
    matvec4(x, w, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = matvec4(x, w, s)
    for i in range(4):
        x.copy_(torch.randn(20, 2560))
        want = matvec4(x, w, s).clone()
        graph.replay()
        torch.cuda.synchronize()
        print(f"[matvec4 graph] replay {i}", flush=True)
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_head_first_used_in_a_graph(cuda):
    """Logits without previous tokens, captured before any eager use: eager calls before the first replay are right."""
    g = torch.Generator().manual_seed(3)
    lm, w1, w2 = (torch.randn(*s, generator=g).half().to(cuda) for s in ((500, 256), (500, 128), (500, 128)))
    h = torch.randn(3, 256, generator=g).half().to(cuda)
    head = QuantHead(lm, None, w1, w2)
    matvec4(h, *quantize4(lm))                     # (loads the library)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = head.logits(h)
    eager = head.logits(h).clone()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        print(f"[4-bit head in a graph] replay {i}", flush=True)
        assert torch.equal(y, eager) and torch.equal(head.logits(h), eager)
    _close(eager, np.concatenate([to64(h), np.zeros((3, 128))], 1),
           ohead.dequant4(ohead.unpack4(head.weight.cpu().numpy()), to64(head.scale)), 64)


@pytest.mark.gpu
def test_drafts_over_4_bits_in_a_graph(cuda):
    cfg = flownet(512, layers=1, flow_steps=2)
    W = make_weights(cfg, 2048, init="test", base_seed=3)
    dr = Drafter(cfg, {k: v.to(cuda) for k, v in W.items()}, None, device=cuda, head_bits=4)
    pred = dr.predict_hidden(synthetic_context(3, cfg.context_size, 512, seed=2).to(cuda))
    known = torch.tensor([3, 500, 2000], device=cuda)
    draft = lambda: (dr.beam_chains(None, known, 5, 4, pred=pred), dr.beam_tree(None, known, 4, 4, 3, pred=pred))   # noqa: E731
    draft()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out = draft()
    for i in range(3):
        known.copy_(torch.tensor([7 * i + 1, 40 * i, 2047 - i]))
        want = [w.clone() for w in draft()]
        graph.replay()
        torch.cuda.synchronize()
        print(f"[4-bit drafts in a graph] replay {i}", flush=True)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 3, 16])
def test_split_top_k_takes_both_zeros_as_equal(cuda, k):
    """-0 and +0 are equal numbers: the lower column comes first, within 512 columns and between."""
    g = torch.Generator().manual_seed(k)
    x = -(torch.rand(4, 1700, generator=g) + 0.5).half()
    x[0, 3], x[0, 7] = -0.0, 0.0                                   # -0 before +0, at the cut of k = 1
    x[1, 600], x[1, 5], x[1, 601] = 0.0, -0.0, -0.0
    at = torch.randperm(1700, generator=g)[:60]
    x[2, at] = torch.where(torch.rand(60, generator=g) < 0.5, -0.0, 0.0).half()
    x[3] = torch.where(torch.rand(1700, generator=g) < 0.9, -0.0, 0.0).half()
    vals, ids, _ = (t.cpu() for t in row_topk(x.to(cuda), k, split=True))
    print(f"[split top-k] zeros, k {k}: {ids[:, 0].tolist()}", flush=True)
    want = np.argsort(-to64(x), axis=1, kind="stable")[:, :k]
    assert ids.tolist() == want.tolist()
    full = row_topk(x.to(cuda), k)
    assert torch.equal(ids, full[1].cpu()) and (vals - full[0].cpu()).abs().max() < 1e-5


@pytest.mark.gpu
def test_split_top_k_of_columns_without_a_number(cuda):
    """A NaN anywhere makes a row's log-sum-exp NaN, as a softmax's, also where 512 columns hold nothing else."""
    x = torch.randn(6, 2000, generator=torch.Generator().manual_seed(1)).half()
    x[0, 512:1024] = float("nan")
    x[1, 512:1024] = float("-inf")
    x[1, 700] = float("nan")
    x[2, 1536:] = float("nan")
    x[3, 10] = float("nan")
    x[4, 512:1024] = float("-inf")                                 # (no NaN: finite)
    print("[split top-k] sets of NaN", flush=True)
    vals, ids, lse = (t.cpu() for t in row_topk(x.to(cuda), 4, split=True))
    assert torch.isnan(lse).tolist() == [True] * 4 + [False] * 2 and torch.isnan(vals[:4]).all() and torch.isfinite(vals[4:]).all()
    v = to64(x)
    assert ids.tolist() == np.argsort(np.where(np.isnan(v), np.inf, -v), axis=1, kind="stable")[:, :4].tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,n,K", [(1, 40, 128), (4, 129, 5376), (16, 33, 640), (3, 8191, 2560)])
def test_products_beside_large_columns(cuda, M, n, K, group):
    """The bound holds with the weights' own magnitudes: a weight of zero takes nothing from a column, however large it is,
    and rows of x far from zero lose nothing to what their weights cancel."""
    g = torch.Generator().manual_seed(M * K + group)
    for size in (1000.0, 8000.0, 60000.0):
        w, s, W = _weights(n, K, group, M + n, "cpu")
        x = torch.randn(M, K, generator=g).half()
        at = torch.arange(K) % group == int(size) % group              # a column a group, of either sign, whose weights are 0
        x[:, at] = torch.where(torch.rand(M, int(at.sum()), generator=g) < 0.5, -size, size).half()
        u = torch.from_numpy(ohead.unpack4(w.numpy()).astype(np.uint8))
        u[:, at] = 8
        w = u[:, ::2] | u[:, 1::2] << 4
        W = ohead.dequant4(u.numpy(), to64(s))
        assert np.array_equal(ohead.unpack4(w.numpy()), u.numpy())
        y = matvec4(x.to(cuda), w.to(cuda), s.to(cuda))
        print(f"[matvec4] columns of {size:.0f}, M={M} n={n} K={K} G={group}: {_close(y, x.numpy(), W, group):.2f} of the bound", flush=True)
    x = (torch.randn(M, K, generator=g) + 200).half()
    s = (s.float() * 2.0 ** -6).half()
    W = ohead.dequant4(u.numpy(), to64(s))
    y = matvec4(x.to(cuda), w.to(cuda), s.to(cuda))
    print(f"[matvec4] rows around 200, M={M} n={n} K={K} G={group}: {_close(y, x.numpy(), W, group):.2f} of the bound", flush=True)


@pytest.mark.gpu
def test_drafts_over_4_bits_equal_the_oracles(cuda):
    """Chains and trees over the 4-bit head, token for token and parent for parent.  No two candidates of the search are within
    0.05 of each other (hiddens are chosen so; logits of up to 32 are rounded by 2^-7 at most), so nothing else passes."""
    cfg = flownet(512, layers=1, flow_steps=2)
    W = make_weights(cfg, 4096, init="test", base_seed=1)
    W["lm_head.weight"] = (W["lm_head.weight"].float() * 8).half()
    sl = torch.randperm(4096, generator=torch.Generator().manual_seed(2))[:1024].sort().values.to(torch.int32)
    dr = Drafter(cfg, {k: v.to(cuda) for k, v in W.items()}, sl.to(cuda), device=cuda, head_bits=4, head_group=32)
    pred = torch.randn(2, 8, 512, generator=torch.Generator().manual_seed(2203)).half()
    known0 = torch.tensor([int(sl[7]), int(sl[100])])
    print("[4-bit drafts] against the oracle's search", flush=True)
    chains = dr.beam_chains(None, known0.to(cuda), 5, 4, pred=pred.to(cuda)).cpu()
    tree = dr.beam_tree(None, known0.to(cuda), 4, 4, 4, pred=pred.to(cuda)).cpu()
    D = ohead.dequant4(ohead.unpack4(dr.head.weight.cpu().numpy()), to64(dr.head.scale))
    W64 = {k: to64(v) for k, v in W.items()}
    sl64, w1 = sl.long().numpy(), to64(dr.head.w1)

    def score(h, prev):
        x = np.concatenate([np.asarray(h, dtype=np.float64), w1[np.clip(prev, 0, None)]], 1)
        return (x @ D.T).astype(np.float16).astype(np.float64)
    resid = lambda lp, nl: ohead.path_residual(W64, W64["embed_tokens.weight"], lp, nl, cfg.path_order)    # noqa: E731
    args = (to64(pred), known0.numpy(), sl64, 4)
    ref, trace = obeam.beam_chains(*args, 5, cfg.path_order, score, resid, return_trace=True)
    ref_tree, more = obeam.beam_tree(*args, 4, 4, cfg.path_order, score, resid, return_trace=True)
    assert min(ohead.margins(t[what], 4).min() for t in trace + more for what in ("lp", "cand")) > 0.05
    assert chains.tolist() == ref.tolist()
    assert tree.tolist() == ref_tree.tolist()
