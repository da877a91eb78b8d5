"""The committed prefix's calls without a GPU: what their host side refuses and plans."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.kv_cache import kv_cache_read, kv_cache_write


def test_gdn_calls_into_fresh_outputs_check_their_arguments():
    """As the calls into outputs that hold something (stand-in addresses, never dereferenced); rows of zeros are written
    16 bytes at a time."""
    L = _lib.lib()
    p = 4096

    def dec(fn, S=3, out=p, K=128, slots=p):
        return fn(p, p, p, p, p, p, 1, 9, slots, S, 2, 4, K, 128, 1, 0.1, out, None, None)
    assert dec(L.cfh_gdn_decode_fresh, S=0) == 0 and dec(L.cfh_gdn_decode_fresh, K=64) == 2
    assert dec(L.cfh_gdn_decode_fresh, slots=None) == 1 and dec(L.cfh_gdn_decode_fresh, out=p + 8) == 1

    def pre(S=3, T=20, cu=p, out=p, ws=p):
        return L.cfh_gdn_prefill_fresh(p, p, p, p, p, p, 1, 9, p, cu, None, S, T, 2, 4, 128, 128, 1, 0.1, out, ws, None, None)
    assert pre(T=0) == 0 and pre(S=0) == 0 and pre(cu=None) == 1 and pre(out=p + 8) == 1 and pre(ws=None, T=200) == 1


def test_attention_into_fresh_outputs_checks_its_arguments():
    L = _lib.lib()
    p = 4096

    def attn(S=2, T=3, out=p, lse=p, cu=p, max_len=80):
        return L.cfh_paged_attn_fresh(p, 1024, T, 8, 4, 128, 1, p, 16 * 512, p, 16 * 512, None, None, 7, 16, p, 5, 5, p, cu,
                                      S, 0.1, 1, max_len, out, 1024, lse, p, None, 1, None)
    assert attn(T=0) == 0 and attn(S=0) == 0
    assert attn(out=p + 8) == 1 and attn(lse=None) == 1 and attn(cu=None) == 1 and attn(max_len=-1) == 1


@pytest.mark.parametrize("shape,strides", [((4, 8, 1, 64), (512, 64, 512, 1)),      # [blocks, Hkv, page, D] seen as pages
                                           ((4, 1, 2, 64), (128, 999, 64, 1)), ((1, 8, 2, 64), (7, 128, 64, 1)),
                                           ((4, 1, 1, 64), (64, 1, 3, 1))])
def test_strides_of_dimensions_of_size_one_do_not_count(shape, strides):
    """A cache that is contiguous but for what a stride over one element says passes (as far as a CPU's goes); one that
    is not, with more than one element there, does not."""
    k = torch.zeros(4096, dtype=torch.bfloat16).as_strided(shape, strides)
    rows = torch.zeros(3, shape[2], 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one GPU"):
        kv_cache_read(k, k, torch.arange(3))
    with pytest.raises(ValueError, match="one GPU"):
        kv_cache_write(rows, rows, k, k, torch.arange(3))
    wide = torch.zeros(1 << 14, dtype=torch.bfloat16).as_strided((4, 8, 2, 64), (1024, 64, 512, 1))
    with pytest.raises(ValueError, match="contiguous"):
        kv_cache_read(wide, wide, torch.arange(3))


def test_prefill_plan_places_every_chunk_in_the_workspace():
    """The split that the launches use: the rows of a sequence that go one after another stay in the rule's range and grow
    with the work, chunks of longer sequences lie apart and inside the workspace, and no more sequences are long than
    have workgroups."""
    L = _lib.lib()
    rng = np.random.default_rng(1)
    plan = (ctypes.c_int32 * 5)()
    seen = set()
    for _ in range(2000):
        HV, V = int(rng.choice([1, 2, 8, 32])), int(rng.choice([16, 64, 128, 256]))
        edges = [0, 1, 8, 9, 10, 11, 15, 16, 17, 18, 63, 64, 65, 128, 129, 500]
        news = rng.choice(edges, size=int(rng.choice([1, 2, 5, 40, 300])), p=None if rng.random() < 0.5 else
                          np.r_[[0.3, 0.3], [0.4 / 14] * 14])
        cu = np.concatenate([[int(rng.integers(0, 30))], news]).cumsum()
        T, S = int(cu[-1] + rng.integers(0, 30)), len(news)
        assert L.cfh_gdn_prefill_plan(T, S, HV, V, plan) == 0
        few, step, plus, nlong, places = plan
        seen.add(few)
        assert 9 <= few <= 16
        at = [c for s, n in enumerate(news) if n > few for c in range(cu[s] // step + plus * s, cu[s] // step + plus * s - (-n // 64))]
        assert len(set(at)) == len(at) and max(at, default=-1) < places
        assert sum(n > few for n in news) <= nlong or T <= few
        if T > few:
            assert places * HV * 34048 <= L.cfh_gdn_prefill_ws_bytes(T, S, HV)
    assert {9, 16} <= seen
    assert L.cfh_gdn_prefill_plan(5, 0, 1, 16, plan) == 1 and L.cfh_gdn_prefill_plan(5, 4097, 1, 16, plan) == 2
