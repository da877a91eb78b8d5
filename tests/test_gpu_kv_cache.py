"""GPU parity of the paged cache (rows written, quantised and read back) and of the attention over it, against the
float64 oracle.

Bounds of the attention.  A score's fp32 error is at most D * 2^-24 * reach (reach: |scale| sum |q| |k|), which
moves a probability by twice that relatively; a probability is rounded once to the 2-byte type before its product
with v (u = 2^-8 bf16, 2^-11 fp16; fp16 loses at most 2^-25 below its normal range), the output once more.  So
|o - ref| <= u |o| + (u + 2 D 2^-24 reach + L 2^-23) sum p |v|, and |lse - ref| <= D 2^-24 reach + L 2^-24 + 2^-22 |lse|."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.kv_cache import kv_cache_read, kv_cache_write, paged_attention
from chain_flow_amd.tree_verify import tree_attn_merge
from conftest import to64
from oracle import kv_cache as okv

BF, FP, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAME = {BF: "bf16", FP: "fp16"}


def empty_cache(dtype, blocks, page, Hkv, D, cuda, packed=False):
    """A cache whose every place holds NaN (as memory that was never written may)."""
    if dtype == F8:
        bytes_ = torch.full((2, blocks, page, Hkv, D), 0x7F, dtype=torch.uint8, device=cuda)
        k, v = bytes_.view(F8)
        ke, ve = (torch.full((blocks, page, Hkv), 255, dtype=torch.uint8, device=cuda) for _ in range(2))
        return k, v, ke, ve
    if packed:          # keys and values of a block side by side in one allocation
        kv = torch.full((blocks, 2, page, Hkv, D), float("nan"), dtype=dtype, device=cuda)
        return kv[:, 0], kv[:, 1], None, None
    k, v = torch.full((2, blocks, page, Hkv, D), float("nan"), dtype=dtype, device=cuda)
    return k, v, None, None


# ---------------------------------------------------------------- rows in and out
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T,Hkv,D,page,packed", [(1, 1, 64, 16, False), (37, 4, 256, 16, True), (130, 3, 128, 7, False),
                                                 (5, 8, 64, 1, False)])
def test_write_and_read_two_byte_rows(cuda, dtype, T, Hkv, D, page, packed):
    """2-byte rows come back bit for bit, from strided sources; places not written keep their bytes."""
    g = torch.Generator().manual_seed(T)
    blocks = -(-T // page) + 2
    kv = torch.randn(T, 2 * Hkv + 1, D, generator=g).to(dtype).to(cuda)
    key, value = kv[:, :Hkv], kv[:, Hkv:2 * Hkv]
    kc, vc, _, _ = empty_cache(dtype, blocks, page, Hkv, D, cuda, packed)
    slots = torch.randperm(blocks * page, generator=g)[:T].to(torch.int32)
    print(f"[kv rows] {dtype} T={T} Hkv={Hkv} D={D} page={page}", flush=True)
    kv_cache_write(key, value, kc, vc, slots.to(cuda))
    k2, v2 = kv_cache_read(kc, vc, slots.to(cuda))
    assert torch.equal(k2, key) and torch.equal(v2, value)
    rest = np.setdiff1d(np.arange(blocks * page), slots.numpy())
    assert kc.reshape(-1, Hkv, D)[rest].isnan().all() and vc.reshape(-1, Hkv, D)[rest].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (3, 128), (2, 256)])
def test_write_quantises_as_the_oracle_bit_for_bit(cuda, dtype, Hkv, D):
    """Elements, exponents and the rows read back, with rows of zeros, of the smallest and the largest values, next
    to the 448 border, with NaN and infinities; no tolerance: a power-of-two scale leaves one rounding."""
    g = torch.Generator().manual_seed(D)
    T, page = 50, 16
    x = torch.randn(T, Hkv, D, generator=g) * torch.exp2(torch.randint(-14, 14, (T, Hkv, 1), generator=g).float())
    x = x.to(dtype)
    fin = torch.finfo(dtype)
    x[0] = 0
    x[1, 0, 5], x[2, 0, 0], x[3] = fin.max, -fin.max, fin.smallest_normal
    x[4, 0, :4] = torch.tensor([448.0, -447.0, 18.0, 2.0 ** -10])
    x[5, 0] = torch.linspace(-450, 450, D).to(dtype)
    x[6, 0, 1], x[6, 0, 2], x[7, -1, 3] = float("nan"), float("inf"), float("-inf")
    x[8, 0] = float("nan")
    x[9, 0] = torch.finfo(dtype).tiny / 8
    y = x.flip(0).contiguous()
    kc, vc, ke, ve = empty_cache(F8, 5, page, Hkv, D, cuda)
    slots = torch.randperm(5 * page, generator=g)[:T].to(torch.int32).to(cuda)
    print(f"[kv quantise] {dtype} Hkv={Hkv} D={D}", flush=True)
    kv_cache_write(x.to(cuda), y.to(cuda), kc, vc, slots, k_exp=ke, v_exp=ve)
    k2, v2 = kv_cache_read(kc, vc, slots, dtype=dtype, k_exp=ke, v_exp=ve)
    for rows, c, e, back in ((x, kc, ke, k2), (y, vc, ve, v2)):
        q, E = okv.quantise(to64(rows), NAME[dtype])
        at = slots.long().cpu()
        assert np.array_equal(e.cpu().reshape(-1, Hkv)[at].numpy().astype(int), E + 127)
        assert np.array_equal(to64(c.float()).reshape(-1, Hkv, D)[at], q, equal_nan=True)
        ref = torch.from_numpy(q * np.ldexp(1.0, E)[..., None]).to(dtype)
        assert torch.equal(back.cpu().nan_to_num(7.0), ref.nan_to_num(7.0))
        assert torch.isfinite(back.cpu()[torch.isfinite(rows)]).all()


@pytest.mark.gpu
def test_every_e4m3_byte_reads_back_as_torch_reads_it(cuda):
    kc, vc, ke, ve = empty_cache(F8, 1, 4, 1, 64, cuda)
    kc.view(torch.uint8).copy_(torch.arange(256, dtype=torch.uint8, device=cuda).view(1, 4, 1, 64))
    vc.view(torch.uint8).copy_(255 - torch.arange(256, dtype=torch.uint8, device=cuda).view(1, 4, 1, 64))
    ke.fill_(127 + 3)
    ve.fill_(127 - 9)
    for dtype in (BF, FP):
        k, v = kv_cache_read(kc, vc, torch.arange(4, device=cuda), dtype=dtype, k_exp=ke, v_exp=ve)
        for got, c, s in ((k, kc, 8.0), (v, vc, 2.0 ** -9)):
            assert torch.equal(got.nan_to_num(7.0), (c[0].float() * s).to(dtype).nan_to_num(7.0))


@pytest.mark.gpu
def test_padding_and_foreign_slots(cuda):
    """Negative slots are skipped (and read as zero), one past the cache too, and it sets the status word."""
    key = torch.randn(5, 2, 64, device=cuda).to(BF)
    kc, vc, _, _ = empty_cache(BF, 2, 8, 2, 64, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv_cache_write(key, key, kc, vc, torch.tensor([3, -1, 15, -7, 0], device=cuda), status=status)
    assert status.item() == 0
    at = torch.tensor([3, 15, 0], device=cuda)
    assert torch.equal(kc.view(16, 2, 64)[at], key[[0, 2, 4]]) and int(kc.isnan().sum()) == 13 * 128
    k, _ = kv_cache_read(kc, vc, torch.tensor([15, -1, 0], device=cuda), status=status)
    assert torch.equal(k[[0, 2]], key[[2, 4]]) and (k[1] == 0).all() and status.item() == 0
    before = kc.clone()
    kv_cache_write(key, key, kc, vc, torch.tensor([16, 2 ** 31 - 1, -1, -1, -1], device=cuda), status=status)
    assert status.item() == 1 and torch.equal(kc.nan_to_num(7.0), before.nan_to_num(7.0))
    status.zero_()
    k, v = kv_cache_read(kc, vc, torch.tensor([16, 3], device=cuda), status=status)
    assert status.item() == 1 and (k[0] == 0).all() and (v[0] == 0).all() and torch.equal(k[1], key[0])
    with pytest.raises(ValueError, match="distinct"):
        kv_cache_write(key, key, kc, vc, torch.tensor([1, 2, 3, 2, -1]))
    with pytest.raises(ValueError, match="below 16"):
        kv_cache_write(key, key, kc, vc, torch.tensor([1, 2, 3, 16, -1]))
    kv_cache_write(key[:0], key[:0], kc, vc, torch.zeros(0, dtype=torch.int32, device=cuda))


# ---------------------------------------------------------------- attention
class Case:
    """Sequences of given lengths in shuffled pages of a cache that holds NaN everywhere else."""

    def __init__(self, cuda, dtype, cache, news, lens, H, Hkv, D, page, seed=0, packed=False, qscale=1.5, extra_blocks=2):
        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.page, self.dtype = news, lens, page, dtype
        S, T = len(news), sum(news)
        need = [-(-n // page) for n in lens]
        blocks = sum(need) + extra_blocks
        self.k, self.v, self.ke, self.ve = empty_cache(cache, blocks, page, Hkv, D, cuda, packed)
        perm = torch.randperm(blocks, generator=g).to(torch.int32)
        self.table = torch.full((S, max(need + [1])), -1, dtype=torch.int32)
        self.ok, self.ov, at = [], [], 0
        for s, n in enumerate(lens):
            pages = perm[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = pages
            j = torch.arange(n)
            slots = (pages.long()[j // page] * page + j % page).to(torch.int32).to(cuda)
            k, v = (torch.randn(n, Hkv, D, generator=g).to(dtype).to(cuda) for _ in range(2))
            kv_cache_write(k, v, self.k, self.v, slots, k_exp=self.ke, v_exp=self.ve)
            if cache == F8:
                k, v = kv_cache_read(self.k, self.v, slots, dtype=dtype, k_exp=self.ke, v_exp=self.ve)
            self.ok.append(to64(k))
            self.ov.append(to64(v))
        self.q = (torch.randn(T, H, D, generator=g) * qscale).to(dtype).to(cuda)
        self.cu = np.concatenate([[0], np.cumsum(news)]).astype(int)
        self.scale = D ** -0.5
        self.cuda = cuda

    def run(self, causal=True, **kw):
        kw.setdefault("max_len", max(self.lens + [0]))
        i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(self.cuda)  # noqa: E731
        return paged_attention(kw.pop("q", self.q), self.k, self.v, kw.pop("table", self.table).to(self.cuda),
                               i32(kw.pop("lens", self.lens)), i32(kw.pop("cu", self.cu)), scale=self.scale, causal=causal,
                               k_exp=self.ke, v_exp=self.ve, **kw)

    def check(self, out, lse, causal=True, rows=None):
        ref, rlse, weight, reach = okv.attention(to64(self.q), self.ok, self.ov, self.lens, self.cu, self.scale, causal)
        close(out, lse, ref, rlse, weight, reach, max(self.lens + [1]), self.dtype, rows)


def close(out, lse, ref, rlse, weight, reach, L, dtype, rows=None):
    D = ref.shape[2]
    u = 2.0 ** -8 if dtype == BF else 2.0 ** -11
    score = D * 2.0 ** -24 * reach                                       # [H, T]
    o, e = to64(out), to64(lse)
    rows = slice(None) if rows is None else rows
    bound = u * np.abs(ref) + (u + (2 * score + L * 2.0 ** -23).T[..., None]) * weight + 1e-30
    if dtype == FP:
        bound = bound + 2.0 ** -24
    off = (np.abs(o - ref) / bound)[rows]
    with np.errstate(invalid="ignore"):
        eoff = np.where(rlse == e, 0.0, np.abs(e - rlse) / (score + L * 2.0 ** -24 + 2.0 ** -22 * np.abs(rlse) + 1e-12))[:, rows]
    print(f"  out at {off.max():.3f} of its bound, lse at {eoff.max():.3f}", flush=True)
    assert off.max() <= 1.0 and eoff.max() <= 1.0


ATTN = [
    # dtype, cache, news, lens, H, Hkv, D, page, causal
    (BF, BF, [1], [1], 4, 2, 64, 16, True),
    (BF, BF, [1], [700], 16, 4, 256, 64, True),
    (FP, FP, [1, 1, 1, 1, 1], [1, 63, 64, 65, 513], 8, 1, 128, 16, True),
    (BF, F8, [1, 1, 1], [300, 17, 128], 12, 2, 128, 16, True),
    (FP, F8, [1, 1], [200, 1], 16, 4, 256, 48, True),
    (BF, BF, [40, 21], [333, 150], 8, 2, 256, 16, False),
    (FP, FP, [9], [0], 4, 4, 64, 16, False),
    (BF, BF, [70], [70], 4, 1, 128, 16, True),
    (BF, BF, [130, 1, 33], [200, 129, 33], 6, 1, 64, 7, True),
    (FP, FP, [65, 64], [129, 64], 4, 4, 128, 32, True),
    (BF, F8, [50, 80], [177, 80], 8, 2, 256, 16, True),
    (FP, F8, [33, 7], [100, 7], 3, 3, 64, 1, True),
    (BF, BF, [5, 0, 12, 3], [2, 40, 12, 0], 8, 2, 128, 16, True),      # rows before the first token, empty sequences
    (FP, FP, [150], [260], 16, 2, 256, 64, True),
    (BF, BF, [20], [300], 40, 2, 64, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,news,lens,H,Hkv,D,page,causal", ATTN)
def test_attention_matches_oracle(cuda, dtype, cache, news, lens, H, Hkv, D, page, causal):
    print(f"[paged attn] {dtype} cache {cache} news={news} lens={lens} {H}/{Hkv}x{D} page={page} causal={causal}", flush=True)
    c = Case(cuda, dtype, cache, news, lens, H, Hkv, D, page, packed=cache != F8)
    out, lse = c.run(causal)
    torch.cuda.synchronize()
    c.check(out, lse, causal)
    again = c.run(causal)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    n = c.table.shape[1] * page
    for most in (n, 1):                        # the planning bound changes the split, not the rows
        o2, l2 = c.run(causal, max_len=most)
        c.check(o2, l2, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [BF, F8])
def test_attention_long_prefix_of_one_row(cuda, cache):
    """One row over 20,011 tokens: the long axis is split and joined."""
    c = Case(cuda, BF, cache, [1], [20011], 8, 2, 128, 64, seed=3)
    print(f"[paged attn long] {cache}", flush=True)
    c.check(*c.run())


@pytest.mark.gpu
def test_attention_peaked_and_flat_scores(cuda):
    """Scores in the hundreds (one token takes all the weight) and all equal."""
    for qscale in (40.0, 0.0):
        c = Case(cuda, BF, BF, [3, 80], [400, 80], 4, 2, 128, 16, seed=4, qscale=qscale)
        print(f"[paged attn scores] x{qscale}", flush=True)
        c.check(*c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (FP, FP), (BF, F8)])
@pytest.mark.parametrize("new,length,D", [(40, 40, 128), (70, 200, 128), (1, 90, 128), (70, 200, 64), (70, 200, 256),
                                          (3, 700, 256), (3, 700, 64), (150, 150, 256)])
def test_masked_places_do_not_reach_a_row(cuda, dtype, cache, new, length, D):
    """NaN and infinities in keys and values of later tokens of the chunk: a row that does not see them is what it is
    without them, a row that does is not finite where they are."""
    c = Case(cuda, dtype, cache, [new], [length], 4, 2, D, 16, seed=5)
    clean = c.run()
    at = length - 1                                           # the last token: only the last row sees it
    blk, off = int(c.table[0, at // 16]), at % 16
    if cache == F8:
        c.v.view(torch.uint8)[blk, off, 0, 5] = 0x7F
        c.k.view(torch.uint8)[blk, off, 1, 5] = 0x7F
    else:
        c.v[blk, off, 0, 5], c.v[blk, off, 0, 9], c.k[blk, off, 1, 5] = float("nan"), float("inf"), float("nan")
    print(f"[paged attn NaN] {dtype} {cache} new={new} length={length} D={D}", flush=True)
    out, lse = c.run()
    assert torch.equal(out[:-1], clean[0][:-1]) and torch.equal(lse[:, :-1], clean[1][:, :-1])
    assert out[-1, :2, 5].isnan().all() and out[-1, 2:].isnan().all() and lse[2:, -1].isnan().all()
    if cache != F8:
        assert (out[-1, :2, 9] == float("inf")).all()
    keep = [d for d in range(D) if d not in (5, 9)]
    assert torch.equal(out[-1, :2][:, keep], clean[0][-1, :2][:, keep])


@pytest.mark.gpu
def test_rows_of_no_sequence_stay(cuda):
    """Rows before the first and behind the last sequence are left as they were; a table row wider than needed and
    strided, a strided query and out."""
    c = Case(cuda, BF, BF, [4, 9], [50, 9], 4, 2, 64, 16, seed=6)
    T = 13 + 3 + 5
    q = torch.zeros(T, 6, 64, dtype=BF, device=cuda)
    q[3:16, :4] = c.q
    out = torch.full((T, 5, 64), 7.0, dtype=BF, device=cuda)
    table = torch.full((2, 9), 1 << 30, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table
    o, lse = c.run(q=q[:, :4], out=out[:, :4], table=table, cu=c.cu + 3)
    assert o.data_ptr() == out.data_ptr() and (out[:3] == 7).all() and (out[16:] == 7).all() and (out[:, 4] == 7).all()
    c.check(o[3:16].contiguous(), lse[:, 3:16].contiguous())


@pytest.mark.gpu
def test_bad_tables_and_lengths_give_nan_and_status(cuda):
    """A block outside the cache among those a row sees, a length past the table or below zero: NaN and the status
    word, for that sequence alone; a block past the length is never looked at.  Bounds outside the query: skipped."""
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    c = Case(cuda, BF, BF, [3, 3], [40, 40], 4, 2, 64, 16, seed=7)
    good = c.run(status=status)
    assert status.item() == 0
    for bad in (dict(table=[(0, 1, 99)]), dict(table=[(0, 2, -1)]), dict(lens=[49, 40]), dict(lens=[-1, 40])):
        kw = {k: v for k, v in bad.items() if k == "lens"}
        if "table" in bad:
            kw["table"] = c.table.clone()
            for s, i, b in bad["table"]:
                kw["table"][s, i] = b
        out, lse = c.run(status=status, **kw)
        assert status.item() == 1, bad
        status.zero_()
        assert out[:3].isnan().all() and lse[:, :3].isnan().all(), bad
        assert torch.equal(out[3:], good[0][3:]) and torch.equal(lse[:, 3:], good[1][:, 3:]), bad
    out = torch.full_like(good[0], 7.0)
    c.run(status=status, cu=[0, 3, 7], out=out)
    assert status.item() == 1 and torch.equal(out[:3], good[0][:3]) and (out[3:] == 7).all()
    status.zero_()
    out.fill_(7.0)
    c.run(status=status, cu=[-2, 3, 6], out=out)
    assert status.item() == 1 and torch.equal(out[3:], good[0][3:]) and (out[:3] == 7).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Blocks whose first element lies past 2^31 elements of the cache, and past 2^32 bytes."""
    page, Hkv, D = 64, 4, 256
    blocks = (1 << 31) // (page * Hkv * D) + 40
    kc, vc = (torch.empty(blocks, page, Hkv, D, dtype=BF, device=cuda) for _ in range(2))
    table = torch.tensor([[blocks - 1, blocks - 30]], dtype=torch.int32)
    c = Case(cuda, BF, BF, [2], [100], 8, Hkv, D, page, seed=8)
    j = torch.arange(100)
    new = (table[0].long()[j // page] * page + j % page).to(torch.int32).to(cuda)
    old = (c.table[0].long()[j // page] * page + j % page).to(torch.int32).to(cuda)
    k, v = kv_cache_read(c.k, c.v, old)
    kv_cache_write(k, v, kc, vc, new)
    c.k, c.v, c.table = kc, vc, table
    print(f"[paged attn] blocks={blocks}", flush=True)
    c.check(*c.run())
    assert torch.equal(kv_cache_read(kc, vc, new)[1], v)


@pytest.mark.gpu
def test_prefix_half_and_tree_half_are_one_attention(cuda):
    """A verify step: the prefix's rows written, the tree nodes' attention over the pages, merged with their own
    suffix: each node gets the attention over the prefix and its ancestors."""
    S, N, H, Hkv, D, page = 2, 17, 8, 2, 128, 16
    c = Case(cuda, BF, BF, [N, N], [91, 200], H, Hkv, D, page, seed=9)
    g = torch.Generator().manual_seed(10)
    tk, tv = (torch.randn(S * N, Hkv, D, generator=g).to(BF) for _ in range(2))
    parent = [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, N)]
    not_anc = torch.ones(S, N, N, dtype=torch.bool)
    for n in range(N):
        m = n
        while m >= 0:
            not_anc[:, n, m] = False
            m = parent[m]
    pout, plse = c.run(causal=False)
    out = torch.empty_like(c.q)
    tree_attn_merge(c.q, tk.to(cuda), tv.to(cuda), out, pout, plse, torch.arange(S * N).view(S, N), not_anc, c.scale)
    worst = 0.0
    q = to64(c.q)
    for s in range(S):
        for n in range(N):
            see = np.nonzero(~not_anc[s, n].numpy())[0] + s * N
            for h in range(H):
                hk = h * Hkv // H
                k = np.concatenate([c.ok[s][:, hk], to64(tk)[see, hk]])
                v = np.concatenate([c.ov[s][:, hk], to64(tv)[see, hk]])
                x = c.scale * (k @ q[s * N + n, h])
                p = np.exp(x - x.max())
                p /= p.sum()
                # each half rounded to bf16, its probabilities too, and the merge once more
                bound = 3 * 2.0 ** -8 * (p @ np.abs(v)) + 1e-5
                worst = max(worst, float((np.abs(to64(out[s * N + n, h]) - p @ v) / bound).max()))
    print(f"[verify step] worst {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [BF, F8])
def test_written_and_attended_in_one_graph(cuda, cache):
    """Write, read and attention captured together; replays on new contents, with eager work between, equal the
    eager calls."""
    news, lens, H, Hkv, D, page = [1, 1, 1], [600, 37, 1], 8, 2, 128, 16
    c = Case(cuda, BF, cache, news, lens, H, Hkv, D, page, seed=11)
    key, value = (torch.randn(3, Hkv, D, device=cuda).to(BF) for _ in range(2))
    last = torch.tensor([int(c.table[s, (n - 1) // page]) * page + (n - 1) % page for s, n in enumerate(lens)],
                        dtype=torch.int32, device=cuda)
    table, tl, tc = c.table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), torch.arange(4, dtype=torch.int32, device=cuda)

    def step():
        kv_cache_write(key, value, c.k, c.v, last, k_exp=c.ke, v_exp=c.ve)
        rows = kv_cache_read(c.k, c.v, last, dtype=BF, k_exp=c.ke, v_exp=c.ve)
        return (*paged_attention(c.q, c.k, c.v, table, tl, tc, scale=c.scale, k_exp=c.ke, v_exp=c.ve), *rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        key.copy_(torch.randn(key.shape, device=cuda))
        value.copy_(torch.randn(key.shape, device=cuda))
        c.q.copy_(torch.randn(c.q.shape, device=cuda))
        graph.replay()
        got = [o.clone() for o in outs]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Calls on two streams together give what each gives alone (workspaces are the call's own)."""
    cases = [Case(cuda, BF, BF, [1] * 4, [3000, 2000, 100, 900], 8, 2, 128, 16, seed=20 + i) for i in range(2)]
    alone = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i][0]) and torch.equal(e, alone[i][1]) for o, e in got[i])


@pytest.mark.gpu
def test_index_tensors_of_64_bits(cuda):
    """int64 slots, tables, lengths and bounds; a slot past 32 bits is outside the cache, not what its low half says;
    floats are refused."""
    c = Case(cuda, BF, BF, [2, 1], [40, 9], 4, 2, 64, 16, seed=21)
    ref = c.run()
    i64 = lambda x: torch.as_tensor(x).long().to(cuda)  # noqa: E731
    got = paged_attention(c.q, c.k, c.v, i64(c.table), i64(c.lens), i64(c.cu), scale=c.scale)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    before = c.k.clone()
    key = torch.ones(2, 2, 64, dtype=BF, device=cuda)
    kv_cache_write(key, key, c.k, c.v, i64([2 ** 32, -2 ** 40]), status=status)
    assert status.item() == 1 and torch.equal(c.k.nan_to_num(7.0), before.nan_to_num(7.0))
    with pytest.raises(ValueError, match="integers"):
        kv_cache_write(key, key, c.k, c.v, torch.zeros(2, device=cuda))


@pytest.mark.gpu
def test_attention_in_place_of_the_query(cuda):
    """out may be the query itself: every row and head is read by the workgroups that write it, before they do."""
    for news, lens in (([1, 1], [3000, 40]), ([100], [300])):
        c = Case(cuda, BF, BF, news, lens, 8, 2, 128, 16, seed=22)
        ref = c.run()
        got = c.run(out=c.q)
        assert got[0].data_ptr() == c.q.data_ptr() and torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.gpu
def test_attention_mixed_batch_of_few_and_many_rows(cuda):
    """Decode rows and chunks in one call: each sequence by the kernel for its row count."""
    c = Case(cuda, BF, BF, [1, 90, 1, 4, 33, 0, 1], [500, 200, 1, 70, 33, 20, 64], 8, 2, 128, 16, seed=23)
    print("[paged attn mixed]", flush=True)
    c.check(*c.run())
    c = Case(cuda, FP, F8, [1] * 20 + [200], [30 + 7 * i for i in range(20)] + [250], 16, 4, 256, 64, seed=24)
    c.check(*c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [-1.0, 0.0, -30.0])
@pytest.mark.parametrize("news,lens", [([1, 3], [600, 40]), ([70], [200])])
def test_attention_of_negative_and_zero_scales(cuda, factor, news, lens):
    """The largest score is the smallest product under a negative scale; under zero every visible token counts alike."""
    c = Case(cuda, BF, BF, news, lens, 8, 2, 128, 16, seed=25)
    c.scale *= factor
    c.check(*c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("news,lens", [([1], [900]), ([1, 1, 1], [30, 200, 64]), ([5, 40], [333, 90])])
def test_attention_of_many_heads_on_one(cuda, news, lens):
    """64 query heads on one kv head: a token's rows are more than a tile of 16."""
    for dtype, cache, D in ((BF, BF, 64), (FP, F8, 256)):
        c = Case(cuda, dtype, cache, news, lens, 64, 1, D, 16, seed=26)
        c.check(*c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("S,many", [(70, 0), (70, 60), (5000, 0), (4200, 150)])
def test_attention_of_many_sequences(cuda, S, many):
    """More sequences than a wave has lanes, and than it has pairs of them: each row finds its own."""
    g = torch.Generator().manual_seed(27)
    news = torch.randint(0, 2, (S,), generator=g).tolist()
    if many:
        news[S // 3] = many
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 40, (S,), generator=g))]
    c = Case(cuda, BF, BF, news, [0] * S, 2, 1, 64, 8, seed=27)          # (the pages are filled here, in one call)
    need = [-(-n // 8) for n in lens]
    blocks = sum(need) + 1
    c.k, c.v, _, _ = empty_cache(BF, blocks, 8, 1, 64, cuda)
    perm, at, slots = torch.randperm(blocks, generator=g), 0, []
    c.table = torch.full((S, max(need)), -1, dtype=torch.int32)
    for s, n in enumerate(lens):
        c.table[s, :need[s]] = perm[at:at + need[s]]
        j = torch.arange(n)
        slots.append(perm[at:at + need[s]][j // 8] * 8 + j % 8)
        at += need[s]
    k, v = (torch.randn(sum(lens), 1, 64, generator=g).to(BF) for _ in range(2))
    kv_cache_write(k.to(cuda), v.to(cuda), c.k, c.v, torch.cat(slots).to(cuda))
    c.ok, c.ov = ([to64(x) for x in t.split(lens)] for t in (k, v))
    c.lens = lens
    c.check(*c.run())


@pytest.mark.gpu
def test_bad_tables_and_values_in_a_split_call(cuda):
    """As above where the tokens are cut into pieces: a bad block, length or value in one piece decides for the row."""
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for news, lens in (([1, 1], [6000, 5000]), ([40, 1], [3000, 2000])):
        c = Case(cuda, BF, BF, news, lens, 4, 2, 64, 16, seed=28)
        n = news[0]
        good = c.run(status=status)
        assert status.item() == 0
        table = c.table.clone()
        table[0, 100] = 1 << 20
        for kw in (dict(table=table), dict(lens=[c.table.shape[1] * 16 + 1, lens[1]])):
            out, lse = c.run(status=status, **kw)
            assert status.item() == 1 and out[:n].isnan().all() and lse[:, :n].isnan().all()
            assert torch.equal(out[n:], good[0][n:]) and torch.equal(lse[:, n:], good[1][:, n:])
            status.zero_()
        c.v[int(c.table[0, 100]), 3, 1, 5] = float("nan")
        out, lse = c.run(status=status)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[:n, 2:, 5] = True
        assert torch.equal(out.isnan(), hit) and torch.equal(out[~hit], good[0][~hit]) and torch.equal(lse, good[1])
        assert status.item() == 0


@pytest.mark.gpu
def test_attention_over_an_empty_table(cuda):
    """A table of no blocks: every row sees nothing; a length past it is refused."""
    c = Case(cuda, BF, BF, [2, 30], [0, 0], 4, 2, 64, 16, seed=29)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = c.run(table=c.table[:, :0], status=status)
    assert (out == 0).all() and (lse == -float("inf")).all() and status.item() == 0
    out, lse = c.run(table=c.table[:, :0], lens=[1, 0], status=status)
    assert out[:2].isnan().all() and (out[2:] == 0).all() and status.item() == 1
    for q, cu in ((c.q[:0], [0, 0, 0]), (c.q[:0], [0])):                  # no rows; no sequences
        S = len(cu) - 1
        out, lse = c.run(q=q, cu=cu, lens=[0] * S, table=c.table[:S])
        assert out.shape == (0, 4, 64) and lse.shape == (4, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [BF, F8])
@pytest.mark.parametrize("D,T", [(64, 33000), (256, 8301)])
def test_many_rows_are_what_few_are(cuda, cache, D, T):
    """Calls large enough for several rows a lane against the same rows in small calls, with padding among them."""
    Hkv, page = 4, 16
    g = torch.Generator().manual_seed(30)
    key, value = (torch.randn(T, Hkv, D, generator=g).to(BF).to(cuda) for _ in range(2))
    blocks = -(-T // page) + 3
    slots = torch.randperm(blocks * page, generator=g)[:T].to(torch.int32)
    slots[torch.randperm(T, generator=g)[:50]] = -1
    slots = slots.to(cuda)
    bits = lambda t: t.view(torch.uint8)  # noqa: E731
    one, two = empty_cache(cache, blocks, page, Hkv, D, cuda), empty_cache(cache, blocks, page, Hkv, D, cuda)
    kv_cache_write(key, value, one[0], one[1], slots, k_exp=one[2], v_exp=one[3])
    for i in range(0, T, 3000):
        kv_cache_write(key[i:i + 3000], value[i:i + 3000], two[0], two[1], slots[i:i + 3000], k_exp=two[2], v_exp=two[3])
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(one, two) if a is not None)
    whole = kv_cache_read(one[0], one[1], slots, k_exp=one[2], v_exp=one[3])
    for i in range(0, T, 3000):
        part = kv_cache_read(one[0], one[1], slots[i:i + 3000], k_exp=one[2], v_exp=one[3])
        assert torch.equal(whole[0][i:i + 3000], part[0]) and torch.equal(whole[1][i:i + 3000], part[1])
    if cache == BF:
        used = slots >= 0
        assert torch.equal(whole[0][used], key[used]) and (whole[0][~used] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,length,H", [(40, 1300, 16), (2, 6000, 4), (40, 3000, 16), (37, 2900, 16)])
def test_joins_of_few_and_many_pieces(cuda, D, new, length, H):
    """Up to eight pieces of a row; more, of few rows and heads; more, of many: each joined by its own form."""
    for dtype, cache in ((BF, BF), (FP, F8)):
        c = Case(cuda, dtype, cache, [new, 1], [length, 40], H, 1, D, 16, seed=31)
        c.check(*c.run())
        c.check(*c.run(causal=False), causal=False)
