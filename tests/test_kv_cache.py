"""The paged cache and the committed GDN without a GPU: the oracle against torch's own e4m3 and against plain
identities, and every refusal that is decided on the host (ValueError from Python, status codes from the C ABI)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.gdn import gdn_decode, gdn_prefill
from chain_flow_amd.kv_cache import kv_cache_read, kv_cache_write, paged_attention
from conftest import to64
from oracle import gdn as ogdn
from oracle import kv_cache as okv

BF, FP, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def test_e4m3_grid_is_torchs_cast():
    x = torch.cat([torch.arange(256, dtype=torch.uint8).view(F8).float(), torch.randn(4000) * 50,
                   torch.randn(4000) * 0.01, torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 0.0])])
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert np.array_equal(okv.grid_e4m3(to64(x)), to64(x.to(F8).float()))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_oracle_quantise_reads_back_within_half_a_step(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 64, generator=g) * torch.exp2(torch.randint(-12, 13, (64, 1), generator=g).float())
    x[0], x[1, 3], x[2] = 0.0, torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = to64(x.to(dtype))
    q, E = okv.quantise(x, "bf16" if dtype == BF else "fp16")
    back = q * np.ldexp(1.0, E)[:, None]
    assert np.isfinite(back.astype(np.float32)).all() and np.abs(back).max() <= torch.finfo(dtype).max
    # 2^-4 of the value, or half of e4m3's smallest step times the scale
    assert (np.abs(back - x) <= np.maximum(np.abs(x) * 2.0 ** -4, np.ldexp(2.0 ** -10, E)[:, None])).all()
    assert (np.abs(x).max(-1) <= np.ldexp(448.0, E)).all() and (E >= -126).all()


def test_oracle_sequence_is_the_tree_of_a_chain():
    """A chain draft tree's nodes over fp32 slots go through the same recurrence as a sequence of its rows."""
    rng = np.random.default_rng(2)
    N, H, HV, K, V = 5, 1, 2, 128, 16
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, a, b, A, dt, st = f(N, 2 * H * K + HV * V), f(N, HV), f(N, HV), f(HV), f(HV), f(N + 1, HV, V, K) * 0.1
    o, ns = ogdn.tree_gdn_vllm(x, a, b, A, dt, st, np.arange(1, N + 1), np.arange(-1, N - 1), 0, H, HV, K, V,
                               K ** -0.5, state_bf16=False)
    o2, ns2 = ogdn.gdn_sequences(x, a, b, A, dt, st, [0], [0, N], H, K ** -0.5)
    assert np.allclose(o, o2, rtol=0, atol=1e-5) and np.allclose(ns[N], ns2[0], rtol=0, atol=1e-5)


def test_kv_argument_checks_without_a_device():
    """The C ABI's checks return before any launch (stand-in addresses, never dereferenced)."""
    L = _lib.lib()
    p = 4096

    def write(ld=512, T=3, Hkv=4, D=128, kc=p, bs=16 * 512, ke=None, ve=None, blocks=7, page=16, slots=p, key=p):
        return L.cfh_kv_write(key, ld, p, ld, T, Hkv, D, 1, kc, bs, p, bs, ke, ve, blocks, page, slots, None, None)
    assert write(T=0) == 0
    assert write(D=96) == 2 and write(blocks=1 << 28, page=16) == 2
    assert write(ld=504) == 1 and write(ld=516) == 1 and write(bs=16 * 512 - 16) == 1 and write(bs=16 * 512 + 8) == 1
    assert write(kc=None) == 1 and write(kc=p + 8) == 1 and write(key=p + 2) == 1 and write(slots=None) == 1
    assert write(ke=p) == 1 and write(T=-1) == 1 and write(page=0) == 1 and write(Hkv=0) == 1

    def read(T=3, D=128, bs=16 * 512, key=p, ke=None, ve=None):
        return L.cfh_kv_read(p, bs, p, bs, ke, ve, 7, 16, p, T, 4, D, 1, key, p, None, None)
    assert read(T=0) == 0 and read(D=32) == 2 and read(bs=100) == 1 and read(key=None) == 1 and read(ve=p) == 1

    def attn(T=3, H=8, Hkv=4, D=128, S=2, max_blocks=5, ld=5, q_ld=1024, page=16, q=p, cu=p, max_len=80, table=p):
        return L.cfh_paged_attn(q, q_ld, T, H, Hkv, D, 1, p, page * Hkv * D, p, page * Hkv * D, None, None, 7, page,
                                table, ld, max_blocks, p, cu, S, 0.1, 1, max_len, p, H * D, p, p, None, None)
    assert attn(T=0) == 0 and attn(S=0) == 0
    assert attn(H=6) == 1 and attn(Hkv=0) == 1 and attn(ld=4) == 1 and attn(q_ld=1016) == 1 and attn(q_ld=1028) == 1
    assert attn(q=p + 4) == 1 and attn(cu=None) == 1 and attn(max_len=-1) == 1 and attn(table=None) == 1
    assert attn(D=100) == 2 and attn(max_blocks=1 << 28, ld=1 << 28) == 2
    assert L.cfh_paged_attn_ws_bytes(-1, 8, 4, 128, 2, 80) == -1 and L.cfh_paged_attn_ws_bytes(3, 6, 4, 128, 2, 80) == -1


def test_gdn_sequence_argument_checks_without_a_device():
    L = _lib.lib()
    p = 4096

    def dec(S=3, H=2, HV=4, K=128, V=128, nslots=9, x=p, slots=p):
        return L.cfh_gdn_decode(x, p, p, p, p, p, 1, nslots, slots, S, H, HV, K, V, 1, 0.1, p, None, None)
    assert dec(S=0) == 0 and dec(K=64) == 2 and dec(S=4097) == 2 and dec(HV=3) == 1 and dec(V=24) == 1
    assert dec(nslots=0) == 1 and dec(x=None) == 1 and dec(x=p + 2) == 1 and dec(slots=None) == 1 and dec(S=-1) == 1

    def pre(S=3, T=20, cu=p, HV=4, ws=p):
        return L.cfh_gdn_prefill(p, p, p, p, p, p, 1, 9, p, cu, None, S, T, 2, HV, 128, 128, 1, 0.1, p, ws, None, None)
    assert pre(T=0) == 0 and pre(S=0) == 0 and pre(cu=None) == 1 and pre(HV=5) == 1 and pre(S=5000) == 2
    assert L.cfh_gdn_prefill_ws_bytes(-1, 1, 4) == -1 and L.cfh_gdn_prefill_ws_bytes(64, 1, 0) == -1


def _cache(dtype=BF, blocks=4, page=8, Hkv=2, D=64):
    c = torch.zeros(blocks, page, Hkv, D, dtype=torch.float32).to(dtype)
    e = torch.full((blocks, page, Hkv), 127, dtype=torch.uint8)
    return c, c.clone(), e, e.clone()


@pytest.mark.parametrize("why,change", [
    ("one shape", dict(value=torch.zeros(3, 2, 64, dtype=FP))),
    ("one shape", dict(key=torch.zeros(3, 2, 64), value=torch.zeros(3, 2, 64))),
    ("must be torch.bfloat16", dict(cache=FP)),
    ("needs contiguous uint8", dict(cache=F8)),
    ("without exponents", dict(k_exp=torch.zeros(4, 8, 2, dtype=torch.uint8))),
    ("slots", dict(slots=torch.zeros(2, dtype=torch.int32))),
    ("must be", dict(key=torch.zeros(3, 4, 64, dtype=BF), value=torch.zeros(3, 4, 64, dtype=BF))),
    ("head width", dict(D=96, key=torch.zeros(3, 2, 96, dtype=BF), value=torch.zeros(3, 2, 96, dtype=BF))),
    ("one GPU", dict()),
])
def test_kv_write_refuses(why, change):
    k, v, _, _ = _cache(change.pop("cache", BF), D=change.pop("D", 64))
    args = dict(key=torch.zeros(3, 2, 64, dtype=BF), value=torch.zeros(3, 2, 64, dtype=BF),
                slots=torch.arange(3, dtype=torch.int32), k_exp=None) | change
    with pytest.raises(ValueError, match=why):
        kv_cache_write(args["key"], args["value"], k, v, args["slots"], k_exp=args["k_exp"])


def test_cache_layout_refusals():
    k, v, ke, ve = _cache(F8)
    with pytest.raises(ValueError, match="rows are read"):
        kv_cache_read(k, v, torch.arange(3), dtype=torch.float32, k_exp=ke, v_exp=ve)
    with pytest.raises(ValueError, match="uint8"):
        kv_cache_read(k, v, torch.arange(3), k_exp=ke, v_exp=ve[:2])
    k, v, _, _ = _cache()
    with pytest.raises(ValueError, match="share one shape"):
        kv_cache_read(k, v[:2], torch.arange(3))
    with pytest.raises(ValueError, match="contiguous"):
        kv_cache_read(k.transpose(1, 2), v.transpose(1, 2), torch.arange(3))
    with pytest.raises(ValueError, match=r"\[T\]"):
        kv_cache_read(k, v, torch.zeros(2, 2, dtype=torch.int32))


@pytest.mark.parametrize("why,change", [
    ("bf16 or fp16", dict(query=torch.zeros(3, 4, 64))),
    ("H a multiple", dict(query=torch.zeros(3, 3, 64, dtype=BF))),
    ("H a multiple", dict(query=torch.zeros(3, 4, 128, dtype=BF))),
    ("the cache must be torch.float16", dict(query=torch.zeros(3, 4, 64, dtype=FP))),
    ("cu_q", dict(cu=torch.zeros(4, dtype=torch.int32))),
    ("block_table", dict(table=torch.zeros(3, 2, dtype=torch.int32))),
    ("one GPU", dict()),
])
def test_paged_attention_refuses(why, change):
    k, v, _, _ = _cache()
    args = dict(query=torch.zeros(3, 4, 64, dtype=BF), table=torch.zeros(2, 2, dtype=torch.int32),
                lens=torch.zeros(2, dtype=torch.int32), cu=torch.zeros(3, dtype=torch.int32)) | change
    with pytest.raises(ValueError, match=why):
        paged_attention(args["query"], k, v, args["table"], args["lens"], args["cu"], scale=1.0)


@pytest.mark.parametrize("why,change", [
    ("width", dict(x=torch.zeros(3, 500, dtype=BF))),
    ("bf16", dict(x=torch.zeros(3, 2 * 128 + 2 * 32, dtype=FP))),
    ("no multiple", dict(H=3)),
    ("multiple of 16", dict(state=torch.zeros(4, 2, 32, 64))),
    ("multiple of 16", dict(state=torch.zeros(4, 2, 24, 128))),
    ("contiguous bf16 or fp32", dict(state=torch.zeros(4, 2, 32, 128, dtype=FP))),
    (r"\[T, HV\]", dict(a=torch.zeros(3, 1, dtype=BF))),
    ("slots", dict(slots=torch.zeros(2, 1, dtype=torch.int32))),
    ("one GPU", dict()),
])
def test_gdn_sequences_refuse(why, change):
    args = dict(x=torch.zeros(3, 2 * 128 + 2 * 32, dtype=BF), a=torch.zeros(3, 2, dtype=BF), H=1,
                state=torch.zeros(4, 2, 32, 128), slots=torch.arange(3, dtype=torch.int32)) | change
    call = (args["x"], args["a"], torch.zeros(3, 2, dtype=BF), torch.zeros(2), torch.zeros(2), args["state"], args["slots"])
    with pytest.raises(ValueError, match=why):
        gdn_decode(*call, num_q_heads=args["H"])
    with pytest.raises(ValueError, match=why):
        gdn_prefill(*call, torch.tensor([0, 1, 2, 3]), num_q_heads=args["H"])


def test_gdn_prefill_refuses_its_own_arguments():
    call = (torch.zeros(3, 2 * 128 + 2 * 32, dtype=BF), torch.zeros(3, 2, dtype=BF), torch.zeros(3, 2, dtype=BF),
            torch.zeros(2), torch.zeros(2), torch.zeros(4, 2, 32, 128), torch.arange(2, dtype=torch.int32))
    for kw, cu in ((dict(), torch.tensor([0, 3])), (dict(initial=torch.zeros(3, dtype=torch.bool)), torch.tensor([0, 1, 3])),
                   (dict(initial=torch.zeros(2)), torch.tensor([0, 1, 3]))):
        with pytest.raises(ValueError):
            gdn_prefill(*call, cu, num_q_heads=1, **kw)


@pytest.mark.parametrize("shape", [(0, 16, 2, 64), (4, 0, 2, 64), (4, 16, 0, 64)])
def test_caches_that_hold_nothing_are_refused(shape):
    k = torch.zeros(shape, dtype=BF)
    with pytest.raises(ValueError, match="holds nothing"):
        kv_cache_read(k, k, torch.arange(3))
    with pytest.raises(ValueError, match="holds nothing"):
        paged_attention(torch.zeros(3, 4, 64, dtype=BF), k, k, torch.zeros(2, 2, dtype=torch.int32),
                        torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), scale=1.0)


def test_gdn_prefill_workspace_covers_every_split():
    """The chunks of sequences of more than `few` rows, at the places either rule gives them, fit the workspace and do
    not overlap; decode-like calls of many sequences need no more than their rows do."""
    rng = np.random.default_rng(0)
    per = _lib.lib().cfh_gdn_prefill_ws_bytes(64, 1, 1) // 2
    for _ in range(300):
        few = int(rng.integers(9, 17))
        news = rng.choice([0, 1, few, few + 1, 63, 64, 65, 128, 129, 500], size=int(rng.integers(1, 40)))
        cu = np.concatenate([[int(rng.integers(0, 3))], news]).cumsum()
        T, S = int(cu[-1] + rng.integers(0, 3)), len(news)
        slots = _lib.lib().cfh_gdn_prefill_ws_bytes(T, S, 1) // per
        by_rows = T // (few + 1) + 1 < T // 64 + S
        used = []
        for s, n in enumerate(news):
            start = cu[s] // (few + 1) if by_rows else cu[s] // 64 + s
            if n > few:
                used += range(start, start + -(-int(n) // 64))
        assert len(set(used)) == len(used)
        if T > few:
            assert max(used, default=0) < slots
    assert _lib.lib().cfh_gdn_prefill_ws_bytes(4096, 4096, 1) // per <= 4096 // 10 + 1
