"""The sampled acceptance's oracle, pinned by the rules it stands for (CPU only), and the call's refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.tree_verify import _counts_fit, tree_sample_accept
from oracle import tree_verify as otv


def _probs(x, T, k=None, P=None):
    """Probabilities by a plain sort and softmax."""
    order = np.argsort(-x, kind="stable")
    w = np.exp((x[order] - x.max()) / T)
    if k:
        w[k:] = 0
    if P is not None:
        c = np.cumsum(w)
        w[1:][c[:-1] >= P * c[-1]] = 0
    p = np.zeros(len(x))
    p[order] = w / w.sum()
    return p


@pytest.mark.parametrize("T,k,P", [(1.0, None, None), (0.6, 5, None), (1.3, None, 0.7), (0.9, 9, 0.5), (2.0, 1, 0.01)])
def test_drawn_tokens_are_distributed_as_the_filtered_softmax(T, k, P):
    """Over n evenly spaced u every token is drawn p n times, off by at most one at each end of its interval."""
    x = np.random.default_rng(0).normal(size=23) * 2
    x[5] = x[11]
    p, n = _probs(x, T, k, P), 20000
    got = np.zeros(23)
    for i in range(n):
        tok, lp = otv.sampled_token(x, T, k, P, (i + 0.5) / n)
        got[tok] += 1
        assert abs(lp - np.log(p[tok])) < 1e-12
    assert (np.abs(got - p * n) <= 1.0 + 1e-6).all()


def test_small_uniforms_draw_the_likeliest_and_ties_go_to_the_lower_index():
    x = np.array([1.0, 3.0, -2.0, 3.0, 2.0])
    assert [otv.sampled_token(x, 1.0, 2, None, u)[0] for u in (0.0, 0.49, 0.5, 0.99)] == [1, 1, 3, 3]
    assert otv.sampled_token(x, 0.0, None, None, 0.9) == (1, 0.0)
    assert otv.sampled_token(np.array([-0.0, 0.0]), 1.0, 1, None, 0.5)[0] == 0


def test_rows_of_infinities_and_nan():
    inf, nan = np.inf, np.nan
    assert otv.sampled_token(np.array([-inf, nan]), 1.0, None, None, 0.3) == (-1, 0.0)
    assert otv.sampled_token(np.array([nan, -inf, -5.0]), 1.0, None, None, 0.9)[0] == 2
    assert otv.sampled_token(np.array([3.0, inf, 1.0, inf]), 1.0, None, None, 0.7)[0] == 3


def test_certain_drafts_accept_as_the_recursive_rule():
    """Two children of the root: the first accepted with p(x1), the second with p(x2) / (1 - p(x1)) if it is not, else a
    token of the rest: summed over u, the walk takes each with exactly its p."""
    x = np.random.default_rng(1).normal(size=(3, 12))
    p = _probs(x[0], 1.0)
    n, took = 5000, np.zeros(3)
    for i in range(n):
        out, path, ln, _ = otv.sampled_descent(x, [2], [3], [4, 7], [-1, -1], 2, [(i + 0.5) / n, 0.5, 0.5], [1.0])
        took[path[0, 0]] += 1
        assert ln[0] == (path[0, 0] >= 0) and out[0, 0] == (x[0].argsort()[::-1][np.searchsorted(
            np.cumsum(np.sort(p)[::-1]), (i + 0.5) / n, side="right")])
    assert abs(took[0] / n - p[4]) <= 1 / n + 1e-9 and abs(took[1] / n - p[7]) <= 1 / n + 1e-9


def test_a_greedy_request_walks_as_the_greedy_descent():
    rng = np.random.default_rng(2)
    x = rng.normal(size=(7, 9))
    par, draft = [-1, -1, 0, 1, 1, 3], rng.integers(0, 9, 6)
    draft[1] = x[0].argmax()
    draft[4] = x[2].argmax()
    ref = otv.greedy_descent(otv.first_argmax(x), [6], [7], draft, par, 4)
    got = otv.sampled_descent(x, [6], [7], draft, par, 4, rng.random(7), [0.0])
    assert all(np.array_equal(a, b) for a, b in zip(ref, got)) and (got[3] == 0).all()


def test_host_counts():
    assert _counts_fit([2, 2, 5], [3, 4, 8], 8, 5, 3)
    assert _counts_fit([2, 2, 2], [3, 3, 4], 9, 2, 2)                # (the second: padding)
    assert not _counts_fit([2, 2, 5], [3, 4, 8], 7, 5, 3)            # more rows than there are
    assert not _counts_fit([2, 2, 5], [3, 4, 8], 8, 4, 3)            # more drafts
    assert not _counts_fit([2, 2, 5], [3, 4, 8], 8, 5, 2)            # longer than max_spec_len
    assert not _counts_fit([2, 1], [3, 3], 8, 5, 3) and not _counts_fit([2], [2], 8, 5, 3)


def test_refusals_without_a_device():
    logits = torch.zeros(3, 8, dtype=torch.bfloat16)
    args = ([2], [3], [1, 2], [-1, 0], 2, torch.zeros(3), torch.ones(1))
    for bad in (logits.float(), logits[:, ::2], logits[0], logits[:0]):
        with pytest.raises(ValueError):
            tree_sample_accept(bad, *args)
    with pytest.raises(ValueError, match="negative"):
        tree_sample_accept(logits, *args[:4], -1, *args[5:])
    with pytest.raises(ValueError, match="one length"):
        tree_sample_accept(logits, [2], [3], [1, 2], [-1], 2, *args[5:])
    with pytest.raises(ValueError, match="one GPU"):
        tree_sample_accept(logits, *args)
    L, p = _lib.lib(), 4096      # stand-in addresses: never dereferenced, the checks fail first

    def call(logits=p, ld=8, V=8, rows=3, drafts=2, B=1, spec=2, u=p, T=p, path=p, ws=p, ids=p):
        return L.cfh_tree_sample_accept(logits, ld, V, rows, 1, p, p, ids, p, drafts, B, spec, u, T, None, None, p, path, p,
                                        p, ws, None, None)
    assert call(B=0) == 0
    assert call(logits=None) == call(ld=7) == call(V=0) == call(rows=0) == call(drafts=-1) == call(B=-1) == 1
    assert call(spec=-1) == call(u=None) == call(T=None) == call(path=None) == call(ws=None) == call(ids=None) == 1
    assert call(V=(1 << 24) + 1, ld=1 << 25) == 2
    assert L.cfh_tree_sample_ws_bytes(5, 64) >= 40 and L.cfh_tree_sample_ws_bytes(-1, 64) == L.cfh_tree_sample_ws_bytes(5, 0) == -1
