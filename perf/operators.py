"""The committed prefix's operators as timed cases: the paged key/value cache of a target's attention
layers, and the recurrent state of its gated-delta-net layers.

Every case is a dict of plain values with a ``kind``:

* ``write``: ``kv_cache_write`` -- new keys and values into the slots of a paged cache, as they are or
  quantised to 8 bits with one power-of-two scale per token and head;
* ``read``: ``kv_cache_read`` -- slots of the cache back as rows of the model's type;
* ``attn``: ``paged_attention`` -- new rows (a chunk, a single token, a draft tree's nodes) over each
  sequence's pages, with the log-sum-exp that the tree attention merges by;
* ``prefill``: ``gdn_prefill`` -- the gated delta rule over whole chunks of ragged sequences;
* ``decode``: ``gdn_decode`` -- one token a sequence, the states updated in their slots.

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form.  ``exact`` restates
each in float64.
"""
from __future__ import annotations

import math
import sys
import zlib
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "chain-flow_amd"))

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
TOP = {"bf16": 120, "fp16": 8}      # the exponent at which 256 times the scale is above the type's largest


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # a decode step of 32 requests: one new token each, the smallest calls of the cache
        dict(name="write_t32_fp8", kind="write", tokens=32, kvheads=4, dim=256, dtype="bf16", cache="fp8", page=16),
        # the prompts of a prefill batch, quantised as they are written
        dict(name="write_t16000_fp8", kind="write", tokens=16000, kvheads=4, dim=256, dtype="bf16", cache="fp8", page=64),
        # one request's prefix read back for another layout: an odd length, 2-byte pages
        dict(name="read_t1777_fp16", kind="read", tokens=1777, kvheads=2, dim=128, dtype="fp16", cache="fp16", page=16),
        # long prefixes out of an 8-bit cache
        dict(name="read_t40000_fp8", kind="read", tokens=40000, kvheads=4, dim=256, dtype="bf16", cache="fp8", page=64),
        # one request's next token over a long prefix
        dict(name="attn_b1_l30011", kind="attn", seqs=1, new=1, length=30011, heads=16, kvheads=4, dim=256,
             dtype="bf16", cache="bf16", page=64, causal=True),
        # a decode step of 48 requests of unequal lengths over an 8-bit cache
        dict(name="attn_b48_l9000_fp8", kind="attn", seqs=48, new=1, length=9000, heads=16, kvheads=2, dim=128,
             dtype="bf16", cache="fp8", page=16, causal=True),
        # the prefix half of four requests' 40-node draft trees
        dict(name="attn_tree_s4_n40", kind="attn", seqs=4, new=40, length=5003, heads=16, kvheads=4, dim=256,
             dtype="bf16", cache="bf16", page=16, causal=False),
        # a prefill step: chunks of two prompts, the longer over 9,001 tokens of which 2,500 are new
        dict(name="attn_chunk_l9001", kind="attn", seqs=2, new=2500, length=9001, heads=16, kvheads=4, dim=256,
             dtype="bf16", cache="bf16", page=64, causal=True),
        # the recurrent step of one request, 16-bit state
        dict(name="decode_b1", kind="decode", seqs=1, heads=16, vheads=32, state="bf16"),
        # and of a serving batch with 32-bit states
        dict(name="decode_b61_fp32", kind="decode", seqs=61, heads=16, vheads=32, state="fp32"),
        # short prompts of unequal lengths, 16-bit states
        dict(name="prefill_s5_n300", kind="prefill", seqs=5, new=300, heads=16, vheads=32, state="bf16"),
        # one long prompt
        dict(name="prefill_s1_n8000", kind="prefill", seqs=1, new=8000, heads=16, vheads=32, state="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "decode", "prefill", "prefill"])
    if kind in ("write", "read"):
        kvheads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        most = (16000 if kind == "write" else 40000) * 1024 // max(kvheads * dim, 512)
        dtype = rng.choice(["bf16", "fp16"])
        return dict(kind=kind, tokens=_log(rng, 1, most), kvheads=kvheads, dim=dim, dtype=dtype,
                    cache=rng.choice([dtype, "fp8"]), page=rng.choice([16, 32, 48, 64, 128]))
    if kind == "attn":
        kvheads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        heads = kvheads * rng.choice([1, 2, 4, 6, 8])
        dtype = rng.choice(["bf16", "fp16"])
        case = dict(kind="attn", heads=heads, kvheads=kvheads, dim=dim, dtype=dtype, cache=rng.choice([dtype, dtype, "fp8"]),
                    page=rng.choice([16, 32, 48, 64, 128]))
        form = rng.choice(["decode", "tree", "chunk"])
        if form == "decode":
            seqs = _log(rng, 1, 64)
            case.update(seqs=seqs, new=1, length=_log(rng, 1, min(40000, 100000000 // (seqs * kvheads * dim))), causal=True)
        elif form == "tree":
            seqs = rng.randint(1, 8)
            case.update(seqs=seqs, new=rng.randint(2, 60), length=_log(rng, 1, min(10000, 100000000 // (seqs * kvheads * dim))),
                        causal=False)
        else:
            seqs = rng.randint(1, 4)
            new = _log(rng, 2, min(2500, 2500 * 4096 // (heads * dim)) // seqs)
            case.update(seqs=seqs, new=new, length=new + _log(rng, 1, 6500) // seqs, causal=True)
        return case
    heads = rng.choice([2, 4, 8, 16])
    vheads = heads * rng.choice([1, 2, 4]) if heads < 16 else heads * rng.choice([1, 2])
    state = rng.choice(["bf16", "fp32"])
    if kind == "decode":
        return dict(kind="decode", seqs=_log(rng, 1, 61), heads=heads, vheads=vheads, state=state)
    seqs = rng.randint(1, 6)
    return dict(kind="prefill", seqs=seqs, new=_log(rng, 2, 4000 // seqs), heads=heads, vheads=vheads, state=state)


# ---------------------------------------------------------------- inputs
def _gen(name, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed((zlib.crc32(name.encode()) * 2654435761 + seed * 0x9E3779B97F4A7C15) % 2 ** 63)
    return g


def _normal(name, seed, shape, scale=1.0, dtype=torch.float32, mean=0.0):
    return (torch.randn(shape, generator=_gen(name, seed), device=DEV) * scale + mean).to(dtype)


def _perm(name, seed, n):
    return torch.randperm(n, generator=_gen(name, seed), device=DEV).to(torch.int32)


def _spread(most, n):
    """n unequal sizes, the first `most`, the others from it down to a quarter of it."""
    return [max(1, int(most * (1.0 - 0.75 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]


def _lengths(case):
    """(new rows, tokens in the cache) of each sequence of an attention case."""
    news = _spread(case["new"], case["seqs"])
    past = _spread(max(case["length"] - case["new"], 0), case["seqs"]) if case["causal"] else None
    if past is None:
        return news, _spread(case["length"], case["seqs"])
    return news, [n + p if case["length"] > case["new"] else n for n, p in zip(news, past)]


def _two_to(e):
    """2^e as float32, e in [-126, 127], from its bits (powers by multiplication or pow may round)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(rows, dtype):
    """Rows of a 2-byte type as (e4m3 elements, bytes e + 127 of their scales 2^e): the least power of two, from
    2^-126 up, that brings the row's largest magnitude to 448 or below."""
    x = rows.float()
    m, e = torch.frexp(x.abs().amax(-1) / 448)                  # m in [0.5, 1): a power of two has m = 0.5
    e = torch.where(m == 0.5, e - 1, e).masked_fill(m == 0, -126).clamp(min=-126)
    most = torch.where(e == TOP[dtype], 240.0, 448.0)[..., None]
    q = (x * _two_to(-e)[..., None]).clamp(-most, most).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8)


def _cache_inputs(case, seed, blocks):
    """A paged cache holding values of the model's type (or what they quantise to)."""
    shape = (blocks, case["page"], case["kvheads"], case["dim"])
    st = {}
    for n, scale in (("k", 1.0), ("v", 1.0)):
        x = _normal(n + "_cache", seed, shape, scale, TYPES[case["dtype"]])
        st[n + "_exp"] = None
        if case["cache"] == "fp8":
            x, st[n + "_exp"] = _quantise(x, case["dtype"])
        st[n + "_cache"] = x
    return st


def _kv_inputs(case, seed):
    T, Hkv, D = case["tokens"], case["kvheads"], case["dim"]
    blocks = (T + T // 8 + 2 * case["page"]) // case["page"]
    st = _cache_inputs(case, seed, blocks)
    if case["kind"] == "write":
        # keys and values as a projection leaves them, side by side in one row; token magnitudes vary
        kv = _normal("kv", seed, (T, 2 * Hkv * D)) * torch.exp2(_normal("size", seed, (T, 1)))
        kv = kv.to(TYPES[case["dtype"]]).view(T, 2, Hkv, D)
        st["key"], st["value"] = kv[:, 0], kv[:, 1]
    # whole pages in a shuffled order, the last one used in part
    pages = _perm("pages", seed, blocks).long()
    i = torch.arange(T, device=DEV)
    st["slots"] = (pages[i // case["page"]] * case["page"] + i % case["page"]).to(torch.int32)
    return st


def _attn_inputs(case, seed):
    news, lens = _lengths(case)
    S, page, H, D = case["seqs"], case["page"], case["heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + 3
    st = _cache_inputs(case, seed, blocks)
    pages = _perm("pages", seed, blocks)
    table = torch.zeros(S, max(need), dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = pages[at:at + n]
        at += n
    T = sum(news)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    st.update(q=_normal("q", seed, (T, H, D), 1.5, TYPES[case["dtype"]]), table=table,
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV), cu=torch.tensor(cu, dtype=torch.int32, device=DEV),
              seq=torch.repeat_interleave(torch.arange(S), torch.tensor(news)).to(DEV), max_new=max(news), max_len=max(lens))
    st["row"] = torch.arange(T, device=DEV) - st["cu"].long()[st["seq"]]
    return st


def _gdn_inputs(case, seed):
    H, HV, K, V = case["heads"], case["vheads"], 128, 128
    news = [1] * case["seqs"] if case["kind"] == "decode" else _spread(case["new"], case["seqs"])
    S, T = case["seqs"], sum(news)
    # rows as the convolution before them leaves them (SiLU of something normal): keys share a direction
    x = _normal("qkv", seed, (T, 2 * H * K + HV * V))
    x = (x * torch.sigmoid(x)).to(torch.bfloat16)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    st = dict(qkv=x, a=_normal("a", seed, (T, HV), 1.0, torch.bfloat16), b=_normal("b", seed, (T, HV), 1.5, torch.bfloat16),
              A_log=torch.log(1.0 + 15.0 * torch.rand(HV, generator=_gen("A", seed), device=DEV)),
              dt=_normal("dt", seed, (HV,), 1.0, mean=-4.5),
              state=_normal("state", seed, (S + 2, HV, V, K), 0.2, TYPES[case["state"]]),
              slots=_perm("slots", seed, S + 2)[:S].contiguous(), cu=torch.tensor(cu, dtype=torch.int32, device=DEV),
              seq=torch.repeat_interleave(torch.arange(S), torch.tensor(news)).to(DEV), max_new=max(news))
    st["row"] = torch.arange(T, device=DEV) - st["cu"].long()[st["seq"]]
    return st


def _inputs(case, seed):
    if case["kind"] in ("write", "read"):
        return _kv_inputs(case, seed)
    return _attn_inputs(case, seed) if case["kind"] == "attn" else _gdn_inputs(case, seed)


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---------------------------------------------------------------- the plain forms
def _plain_write(st):
    case = st["case"]
    slots = st["slots"].long()
    page = case["page"]
    for n, rows in (("k", st["key"]), ("v", st["value"])):
        exps = None
        if case["cache"] == "fp8":
            rows, exps = _quantise(rows, case["dtype"])
            st[n + "_exp"][slots // page, slots % page] = exps
        st[n + "_cache"][slots // page, slots % page] = rows
    return _cache_outputs(st)


def _cache_outputs(st):
    return {n: st[n] for n in ("k_cache", "v_cache", "k_exp", "v_exp") if st[n] is not None}


def _rows_of(st, n, block, at):
    """Cache rows as float32."""
    x = st[n + "_cache"][block, at].float()
    if st[n + "_exp"] is not None:
        x = x * _two_to(st[n + "_exp"][block, at].int() - 127)[..., None]
    return x


def _plain_read(st):
    slots, page = st["slots"].long(), st["case"]["page"]
    t = TYPES[st["case"]["dtype"]]
    return tuple(_rows_of(st, n, slots // page, slots % page).to(t) for n in ("k", "v"))


def _plain_attn(st):
    case = st["case"]
    S, H, Hkv, D = case["seqs"], case["heads"], case["kvheads"], case["dim"]
    G, N, L = H // Hkv, st["max_new"], st["max_len"]
    pos = torch.arange(L, device=DEV)
    block = st["table"].long()[:, pos // case["page"]]
    k, v = (_rows_of(st, n, block, (pos % case["page"]).expand(S, L)).permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    q = torch.zeros(S, N, H, D, device=DEV)
    q[st["seq"], st["row"]] = st["q"].float()
    q = q.view(S, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * N, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, H, N, L) * D ** -0.5
    lens = st["lens"].long()
    last = lens[:, None].expand(S, N)
    if case["causal"]:
        new = (st["cu"][1:] - st["cu"][:-1]).long()
        last = lens[:, None] - new[:, None] + torch.arange(1, N + 1, device=DEV)
        last = torch.minimum(last, lens[:, None])
    s = s.masked_fill(pos >= last[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, Hkv, G * N, L), v).view(S, H, N, D) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (m + torch.log(total))[..., 0]
    o, lse = o.permute(0, 2, 1, 3)[st["seq"], st["row"]], lse.permute(0, 2, 1)[st["seq"], st["row"]]
    return o.to(TYPES[case["dtype"]]), lse.t().contiguous()


def _plain_gdn(st):
    case = st["case"]
    S, H, HV, K, V, N = case["seqs"], case["heads"], case["vheads"], 128, 128, st["max_new"]
    # the gates in 64 bits: small decays add up over thousands of tokens
    x = st["a"].double() + st["dt"].double()
    g = -torch.exp(st["A_log"].double()) * torch.log1p(torch.exp(x))
    decay = torch.ones(S, N, HV, device=DEV)
    beta = torch.zeros(S, N, HV, device=DEV)
    decay[st["seq"], st["row"]] = torch.exp(g).float()
    beta[st["seq"], st["row"]] = (1 / (1 + torch.exp(-st["b"].double()))).to(torch.bfloat16).float()
    rows = torch.zeros(S, N, 2 * H * K + HV * V, device=DEV)
    rows[st["seq"], st["row"]] = st["qkv"].float()
    q, k, v = rows.split([H * K, H * K, HV * V], -1)
    q, k = (t.view(S, N, H, K) for t in (q, k))
    q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = (t.repeat_interleave(HV // H, 2) for t in (q * K ** -0.5, k))
    v = v.view(S, N, HV, V)
    slots = st["slots"].long()
    state = st["state"][slots].float()
    out = torch.empty(S, N, HV, V, device=DEV)
    for t in range(N):
        kt = k[:, t, :, None, :]
        state = state * decay[:, t, :, None, None]
        d = (v[:, t] - (state * kt).sum(-1)) * beta[:, t, :, None]
        state = state + d[..., None] * kt
        out[:, t] = (state * q[:, t, :, None, :]).sum(-1)
    st["state"][slots] = state.to(st["state"].dtype)
    return out[st["seq"], st["row"]].to(torch.bfloat16), st["state"]


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn}.get(kind, _plain_gdn)(st)
    if kind == "write":
        from chain_flow_amd.kv_cache import kv_cache_write
        kv_cache_write(st["key"], st["value"], st["k_cache"], st["v_cache"], st["slots"], k_exp=st["k_exp"],
                       v_exp=st["v_exp"])
        return _cache_outputs(st)
    if kind == "read":
        from chain_flow_amd.kv_cache import kv_cache_read
        return kv_cache_read(st["k_cache"], st["v_cache"], st["slots"], dtype=TYPES[case["dtype"]], k_exp=st["k_exp"],
                             v_exp=st["v_exp"])
    if kind == "attn":
        from chain_flow_amd.kv_cache import paged_attention
        return paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["cu"],
                               scale=case["dim"] ** -0.5, causal=case["causal"], k_exp=st["k_exp"], v_exp=st["v_exp"],
                               max_len=st["max_len"])
    if kind == "decode":
        from chain_flow_amd.gdn import gdn_decode
        o = gdn_decode(st["qkv"], st["a"], st["b"], st["A_log"], st["dt"], st["state"], st["slots"],
                       num_q_heads=case["heads"])
        return o, st["state"]
    from chain_flow_amd.gdn import gdn_prefill
    o = gdn_prefill(st["qkv"], st["a"], st["b"], st["A_log"], st["dt"], st["state"], st["slots"], st["cu"],
                    num_q_heads=case["heads"])
    return o, st["state"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("write", "read"):
        row = case["kvheads"] * (case["dim"] + 1 if case["cache"] == "fp8" else 2 * case["dim"])
        return {"bytes": 2.0 * case["tokens"] * (row + 2 * case["kvheads"] * case["dim"]) + 4.0 * case["tokens"], "flops": 0.0}
    if kind == "attn":
        news, lens = _lengths(case)
        H, Hkv, D = case["heads"], case["kvheads"], case["dim"]
        row = Hkv * (D + 1 if case["cache"] == "fp8" else 2 * D)
        pairs = sum(n * m - (n * (n - 1) / 2 if case["causal"] else 0) for n, m in zip(news, lens))
        tables = 4.0 * sum(-(-m // case["page"]) for m in lens)
        return {"bytes": 2.0 * sum(lens) * row + sum(news) * H * (4.0 * D + 4) + tables, "flops": 4.0 * pairs * H * D}
    H, HV, K, V = case["heads"], case["vheads"], 128, 128
    rows = case["seqs"] if kind == "decode" else sum(_spread(case["new"], case["seqs"]))
    state = 2.0 * case["seqs"] * HV * K * V * (2 if case["state"] == "bf16" else 4)
    # a token: decay, S k, the rank-1 update and S q over the state of each value head
    return {"bytes": state + rows * (2.0 * (2 * H * K + 2 * HV * V) + 4.0 * HV), "flops": 7.0 * rows * HV * K * V}


# ---------------------------------------------------------------- the definitions in 64 bits
def _power(e):
    """2^e in float64, exactly, e in [-200, 200]."""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=DEV)[e.long() + 200]


def _grid_e4m3(x):
    """Float64 values rounded to the e4m3 grid (3 mantissa bits, steps of 2^-9 below 2^-6), ties to even."""
    _, e = torch.frexp(x)
    step = _power((e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_write(case, st):
    out = {}
    slots = st["slots"].long()
    for n, rows in (("k", st["key"]), ("v", st["value"])):
        flat = st[n + "_cache"].double().flatten(0, 1)
        x = rows.double()
        if case["cache"] == "fp8":
            amax = x.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / 448))
            e = torch.where(amax > 448 * _power(e), e + 1, e)               # (log2 rounds)
            e = torch.where(amax <= 448 * _power(e - 1), e - 1, e)
            e = torch.where(amax > 0, e, torch.full_like(e, -126.0)).clamp(min=-126.0)
            x = _grid_e4m3(x / _power(e))
            x = torch.where((x.abs() > 240) & (e == TOP[case["dtype"]]), torch.sign(x) * 240, x)
        flat[slots] = x
        out[n + "_cache"] = flat.view(st[n + "_cache"].shape)
        if case["cache"] == "fp8":
            out[n + "_exp"] = None
    return out


def _exact_rows(st, n):
    x = st[n + "_cache"].double().flatten(0, 1)
    if st[n + "_exp"] is not None:
        x = x * _power(st[n + "_exp"].int().flatten(0, 1) - 127)[..., None]
    return x


def _exact_read(case, st):
    return tuple(_exact_rows(st, n)[st["slots"].long()] for n in ("k", "v"))


def _exact_attn(case, st):
    H, Hkv, D, page = case["heads"], case["kvheads"], case["dim"], case["page"]
    news, lens = _lengths(case)
    kc, vc = _exact_rows(st, "k"), _exact_rows(st, "v")
    outs, lses, at = [], [], 0
    for s, (n, m) in enumerate(zip(news, lens)):
        i = torch.arange(m, device=DEV)
        slots = st["table"][s].long()[i // page] * page + i % page
        hidden = i[None] > (m - n + torch.arange(n, device=DEV))[:, None] if case["causal"] else None
        o, e = [], []
        for h in range(H):
            k, v = kc[slots, h * Hkv // H], vc[slots, h * Hkv // H]
            x = torch.mm(st["q"][at:at + n, h].double(), k.t()) / math.sqrt(D)
            if hidden is not None:
                x[hidden] = -math.inf
            e.append(torch.logsumexp(x, -1))
            o.append(torch.mm(torch.exp(x - e[-1][:, None]), v))
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(e, 0))
        at += n
    return torch.cat(outs), torch.cat(lses, 1)


def _exact_gdn(case, st):
    """Chunk by chunk: the updates of 32 rows as the solution of one triangular system."""
    H, HV, K, V, C = case["heads"], case["vheads"], 128, 128, 32
    state = st["state"].double().clone()
    q, k, v = st["qkv"].double().split([H * K, H * K, HV * V], -1)
    g = torch.nn.functional.softplus(st["a"].double() + st["dt"].double(), threshold=40.0) * -torch.exp(st["A_log"].double())
    beta = torch.sigmoid(st["b"].double()).to(torch.bfloat16).double()
    out = torch.empty(q.shape[0], HV, V, dtype=torch.float64, device=DEV)
    heads = torch.arange(HV, device=DEV) * H // HV
    cu = st["cu"].tolist()
    for s, slot in enumerate(st["slots"].tolist()):
        S = state[slot]                                                       # [HV, V, K]
        for lo in range(cu[s], cu[s + 1], C):
            r = slice(lo, min(lo + C, cu[s + 1]))
            n = r.stop - r.start
            kk, qq = (t[r].view(n, H, K).transpose(0, 1)[heads] for t in (k, q))   # [HV, n, K]
            kk = kk * torch.rsqrt((kk * kk).sum(-1, keepdim=True) + 1e-6)
            qq = qq * torch.rsqrt((qq * qq).sum(-1, keepdim=True) + 1e-6) / math.sqrt(K)
            vv, bb, G = v[r].view(n, HV, V).transpose(0, 1), beta[r].t()[..., None], torch.cumsum(g[r], 0).t()
            ratio = torch.exp((G[:, :, None] - G[:, None, :]).tril())
            low = (bb * ratio * torch.matmul(kk, kk.transpose(1, 2).contiguous())).tril(-1)
            start = torch.exp(G)[..., None]
            rhs = bb * (vv - start * torch.matmul(kk, S.transpose(1, 2).contiguous()))
            d = torch.linalg.solve_triangular(low + torch.eye(n, dtype=torch.float64, device=DEV), rhs, upper=False,
                                              unitriangular=True)
            att = (ratio * torch.matmul(qq, kk.transpose(1, 2).contiguous())).tril()
            out[r] = (start * torch.matmul(qq, S.transpose(1, 2).contiguous()) + torch.matmul(att, d)).transpose(0, 1)
            tail = torch.exp(G[:, -1:] - G)[..., None]
            S = start[:, -1:] * S + torch.matmul((tail * d).transpose(1, 2).contiguous(), kk)
        state[slot] = S
    return out, state


def exact(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    return {"write": _exact_write, "read": _exact_read, "attn": _exact_attn}.get(kind, _exact_gdn)(case, st)
