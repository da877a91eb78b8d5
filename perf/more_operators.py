"""What a sampled speculative step adds around the target's verify, as timed cases: the drafter's head at 4
bits, the acceptance of drafted tokens from given random numbers, the accepted rows' place in the paged
cache, and the cache's pages.

Every case is a dict of plain values with a ``kind``:

* ``accept``: ``tree_sample_accept`` -- each row's target token drawn from its filtered softmax by a given
  uniform number, and the walk down the drafted tree;
* ``commit``: ``kv_cache_commit`` -- the accepted nodes' rows moved to the front of the tree's rows;
* ``resize``: ``kv_pages_resize`` twice -- room for the drafted nodes, then only for what was accepted;
* ``fork``: ``kv_pages_fork`` and the first ``kv_pages_resize`` behind it, which copies shared last pages;
* ``matvec4``: ``matvec4`` -- rows times a matrix of 4-bit weights with a scale for each group of columns.

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form.  ``exact`` restates
each in float64 or in whole numbers.
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
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one request's chain of five drafted tokens, temperature alone: the smallest verify
        dict(name="accept_b1_chain5", kind="accept", seqs=1, nodes=5, tree=False, vocab=248320, dtype="bf16", mixed=False),
        # four requests' 40-node trees, each with its own temperature, top-k and top-p
        dict(name="accept_b4_tree40", kind="accept", seqs=4, nodes=40, tree=True, vocab=248320, dtype="bf16", mixed=True),
        # a serving batch's trees over a smaller vocabulary, fp16 logits
        dict(name="accept_b48_tree40_v32000", kind="accept", seqs=48, nodes=40, tree=True, vocab=32000, dtype="fp16",
             mixed=True),
        # one request's accepted path in the caches of eight layers
        dict(name="commit_s1_l8", kind="commit", seqs=1, nodes=40, length=1201, layers=8, kvheads=4, dim=256, cache="bf16",
             page=16),
        # a batch's accepted paths, 8-bit caches
        dict(name="commit_s48_l16_fp8", kind="commit", seqs=48, nodes=40, length=401, layers=16, kvheads=2, dim=128,
             cache="fp8", page=64),
        # room for 41 rows and back to the accepted ones: a serving batch ...
        dict(name="resize_s48", kind="resize", seqs=48, nodes=41, length=9000, blocks=40000, page=16),
        # ... and the largest one, over a pool of a quarter of a million pages
        dict(name="resize_s1000", kind="resize", seqs=1000, nodes=41, length=3500, blocks=250000, page=16),
        # one prompt answered eight times
        dict(name="fork_p1_n8", kind="fork", parents=1, children=8, length=30011, new=1, layers=4, kvheads=4, dim=256,
             cache="bf16", page=64),
        # a batch of prompts answered four times each, all layers' last pages copied
        dict(name="fork_p24_n4", kind="fork", parents=24, children=4, length=777, new=41, layers=8, kvheads=4, dim=256,
             cache="bf16", page=64),
        # one beam row over the shortlisted head of the shipped latent drafter
        dict(name="matvec4_m1_k2560", kind="matvec4", rows=1, cols=2560, out=62642, group=128),
        # four beams over the shortlisted head and its markov columns at d = 5120
        dict(name="matvec4_m4_k5376", kind="matvec4", rows=4, cols=5376, out=62642, group=64),
        # sixteen rows over an odd count of candidate rows
        dict(name="matvec4_m16_k4096", kind="matvec4", rows=16, cols=4096, out=8191, group=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["accept", "accept", "commit", "resize", "fork", "matvec4", "matvec4"])
    if kind == "accept":
        tree = rng.random() < 0.6
        nodes = rng.randint(2, 60) if tree else rng.randint(1, 8)
        vocab = _log(rng, 1000, 248320)
        seqs = _log(rng, 1, min(64, 40000000 // (vocab * (nodes + 1))))
        return dict(kind=kind, seqs=seqs, nodes=nodes, tree=tree, vocab=vocab, dtype=rng.choice(["bf16", "fp16"]),
                    mixed=rng.random() < 0.7)
    if kind == "commit":
        layers, kvheads, dim = rng.choice([1, 3, 8, 16]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        length = _log(rng, 1, 1200)
        seqs = _log(rng, 1, min(64, 200000000 // (layers * kvheads * dim * (length + 200))))
        return dict(kind=kind, seqs=seqs, nodes=rng.randint(2, 60), length=length, layers=layers, kvheads=kvheads, dim=dim,
                    cache=rng.choice(["bf16", "fp16", "fp8"]), page=rng.choice([16, 32, 48, 64]))
    if kind == "resize":
        seqs, page = _log(rng, 1, 1000), rng.choice([16, 32, 48, 64])
        length = _log(rng, 1, min(30000, 3500000 // seqs))
        most = 250000
        need = seqs * (-(-(length + 100) // page) + 1)
        return dict(kind=kind, seqs=seqs, nodes=rng.randint(1, 61), length=length, blocks=_log(rng, need, max(need, most)),
                    page=page)
    if kind == "fork":
        layers, kvheads, dim = rng.choice([1, 4, 8]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        parents, children = rng.randint(1, 24), rng.randint(1, 8)
        length = _log(rng, 1, min(30000, 100000000 // (parents * layers * kvheads * dim)))
        return dict(kind=kind, parents=parents, children=children, length=length, new=rng.randint(1, 60), layers=layers,
                    kvheads=kvheads, dim=dim, cache=rng.choice(["bf16", "fp16", "fp8"]), page=rng.choice([16, 32, 48, 64]))
    group = rng.choice([32, 64, 128])
    cols = 128 * rng.randint(5, 42)
    return dict(kind=kind, rows=rng.choice([1, 2, 3, 4, 8, 11, 16]), cols=cols, out=_log(rng, 500, 62642), group=group)


# ---------------------------------------------------------------- inputs
def _gen(name, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed((zlib.crc32(name.encode()) * 2654435761 + seed * 0x9E3779B97F4A7C15) % 2 ** 63)
    return g


def _normal(name, seed, shape, scale=1.0, dtype=torch.float32, mean=0.0):
    return (torch.randn(shape, generator=_gen(name, seed), device=DEV) * scale + mean).to(dtype)


def _uniform(name, seed, shape):
    return torch.rand(shape, generator=_gen(name, seed), device=DEV)


def _perm(name, seed, n):
    return torch.randperm(n, generator=_gen(name, seed), device=DEV).to(torch.int32)


def _spread(most, n):
    """n unequal sizes, the first `most`, the others from it down to a quarter of it."""
    return [max(1, int(most * (1.0 - 0.75 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _tree_of(nodes, tree, which):
    """Parents of a drafted tree in breadth-first order (-1: the root) and each node's place among its siblings: a
    chain, or levels of up to eight nodes under the first ones of the level before."""
    if not tree:
        return [i - 1 for i in range(nodes)], [0] * nodes
    parents, places, level = [], [], [-1]
    while len(parents) < nodes:
        here = []
        for j in range(min(8, nodes - len(parents))):
            p = level[(j * j // 3 + which) % min(len(level), 3)]
            places.append(sum(1 for i in here if parents[i] == p))
            here.append(len(parents))
            parents.append(p)
        level = here
    return parents, places


def _accept_inputs(case, seed):
    B, n, V = case["seqs"], case["nodes"], case["vocab"]
    R = B * (n + 1)
    # a row of a target: most of the vocabulary far below a few likely tokens
    x = _normal("logits", seed, (R, V), 2.5)
    top = torch.randint(0, V, (R, 8), generator=_gen("top", seed), device=DEV)
    x.scatter_add_(1, top, _uniform("lift", seed, (R, 8)) * 4 + 13 - torch.arange(8, device=DEV))
    x = x.to(TYPES[case["dtype"]])
    parents, places = zip(*(_tree_of(n, case["tree"], b) for b in range(B)))
    par, place = torch.tensor(parents, device=DEV), torch.tensor(places, device=DEV)
    # a node holds one of its parent row's likely tokens
    row = torch.arange(B, device=DEV)[:, None] * (n + 1) + par + 1
    ids = torch.topk(x[:, :].float(), 8, dim=1).indices
    draft = ids[row, (place + (torch.arange(B, device=DEV)[:, None] % 2)) % 8]
    cyc = lambda vals: torch.tensor([vals[b % len(vals)] for b in range(B)], device=DEV)    # noqa: E731
    mixed = case["mixed"]
    return dict(logits=x, parents=par.flatten().to(torch.int32), draft=draft.flatten().to(torch.int32),
                cu_draft=_ints([n * (b + 1) for b in range(B)]), cu_rows=_ints([(n + 1) * (b + 1) for b in range(B)]),
                u=_uniform("u", seed, (R,)),
                T=cyc([0.7, 1.0, 0.6, 0.0, 1.3]).float() if mixed else torch.ones(B, device=DEV),
                top_k=cyc([20, 0, 50, 0, 0, 7]).to(torch.int32) if mixed else None,
                top_p=cyc([0.95, 1.0, 0.8, 1.0, 0.9, 0.99, 1.0]).float() if mixed else None)


def _values(seed, name, shape, cache):
    """Cache elements: normal values of the type; 8-bit ones with a byte e + 127 of each row's scale 2^e."""
    if cache != "fp8":
        return _normal(name, seed, shape, 1.0, TYPES[cache]), None
    x = _normal(name, seed, shape, 60.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return x, torch.randint(120, 126, shape[:-1], generator=_gen(name + "_exp", seed), device=DEV).to(torch.uint8)


def _cache_inputs(case, seed, blocks):
    shape = (case["layers"], blocks, case["page"], case["kvheads"], case["dim"])
    st = {}
    st["k_cache"], st["k_exp"] = _values(seed, "k", shape, case["cache"])
    st["v_cache"], st["v_exp"] = _values(seed, "v", shape, case["cache"])
    return st


def _tables(seed, held, width, blocks):
    """A block table of rows with `held` pages each, out of a shuffled pool of `blocks` (unheld entries: -1), and the
    count of holders of every page."""
    pages = _perm("pages", seed, blocks)
    table = torch.full((len(held), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = pages[at:at + n]
        at += n
    ref = torch.zeros(blocks, dtype=torch.int32, device=DEV)
    ref[pages[:at].long()] = 1
    return table, ref


def _path_of(nodes, s):
    """The accepted nodes of sequence s: strictly ascending, up to six of them."""
    out, at = [], (s + 1) % 3
    while at < nodes and len(out) < 1 + (5 * s + 4) % 6:
        out.append(at)
        at += 1 + (3 * s + 5 * len(out)) % 9
    return out


def _commit_inputs(case, seed):
    S, page = case["seqs"], case["page"]
    lens = _spread(case["length"], S)
    held = [-(-(m + case["nodes"]) // page) for m in lens]
    blocks = sum(held) + 2
    st = _cache_inputs(case, seed, blocks)
    st["table"], _ = _tables(seed, held, max(held), blocks)
    paths = [_path_of(case["nodes"], s) for s in range(S)]
    st.update(lens=_ints(lens), path=_ints([p + [-1] * (8 - len(p)) for p in paths]), count=_ints([len(p) for p in paths]))
    return st


def _resize_rooms(case):
    """Tokens that each sequence has room for: before, with the drafted nodes, with the accepted ones."""
    now = _spread(case["length"], case["seqs"])
    return now, [m + case["nodes"] for m in now], [m + 1 + (7 * s) % case["nodes"] if case["nodes"] > 1 else m + 1
                                                   for s, m in enumerate(now)]


def _resize_inputs(case, seed):
    page = case["page"]
    now, most, kept = _resize_rooms(case)
    held = [-(-m // page) for m in now]
    width = -(-max(most) // page) + 1
    st = {}
    st["table"], st["ref"] = _tables(seed, held, width, case["blocks"])
    st.update(room=_ints(now), most=_ints(most), kept=_ints(kept))
    return st


def _fork_inputs(case, seed):
    P, C, page = case["parents"], case["children"], case["page"]
    now = _spread(case["length"], P)
    held = [-(-m // page) for m in now]
    width = -(-(max(now) + case["new"]) // page)
    # each child's own pages behind the shared ones, its last shared page copied, and two pages nobody takes
    blocks = sum(held) + P * C * (-(-case["new"] // page) + 1) + 2
    st = _cache_inputs(case, seed, blocks)
    st["table"], st["ref"] = _tables(seed, held + [0] * (P * C), width, blocks)
    src = [p for p in range(P) for _ in range(C)]
    st.update(room=_ints(now + [0] * (P * C)), src=_ints(src), dst=_ints([P + i for i in range(P * C)]),
              new_room=_ints(now + [now[p] + case["new"] for p in src]))
    return st


def _matvec_inputs(case, seed):
    n, K = case["out"], case["cols"]
    # a byte holds two weights, the even column's in its low half; scales of rows of unequal size
    q = torch.randint(0, 256, (n, K // 2), generator=_gen("q", seed), device=DEV, dtype=torch.int16).to(torch.uint8)
    s = (torch.exp2(_normal("s", seed, (n, K // case["group"]), 0.5)) * 0.01).to(torch.float16)
    return dict(q=q, scale=s, x=_normal("x", seed, (case["rows"], K), 1.0, torch.float16))


def _inputs(case, seed):
    return {"accept": _accept_inputs, "commit": _commit_inputs, "resize": _resize_inputs, "fork": _fork_inputs,
            "matvec4": _matvec_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---------------------------------------------------------------- the plain forms
def _plain_accept(st):
    case = st["case"]
    B, n, V = case["seqs"], case["nodes"], case["vocab"]
    R = B * (n + 1)
    per_row = lambda t: t.repeat_interleave(n + 1)[:, None]                                   # noqa: E731
    xs, ids = torch.sort(st["logits"].float() + 0.0, dim=1, descending=True, stable=True)
    T = per_row(st["T"]).double()
    # sums in 64 bits: a draw next to a border has to fall on its own side
    w = torch.exp((xs.double() - xs[:, :1].double()) / torch.where(T > 0, T, torch.ones_like(T)))
    pos = torch.arange(V, device=DEV)
    w = torch.where((T > 0) | (pos == 0), w, torch.zeros_like(w))
    if st["top_k"] is not None:
        k = per_row(st["top_k"])
        w = w.masked_fill((pos >= k) & (k > 0), 0.0)
    cum = torch.cumsum(w, 1)
    kept = cum[:, -1:]
    if st["top_p"] is not None:
        p = per_row(st["top_p"]).double()
        before = torch.cat([torch.zeros(R, 1, dtype=torch.float64, device=DEV), cum[:, :-1]], 1)
        w = w.masked_fill((before >= p * kept) & (p < 1) & (pos > 0), 0.0)
        cum = torch.cumsum(w, 1)
        kept = cum[:, -1:]
    at = torch.minimum((cum <= st["u"].double()[:, None] * kept).sum(1), (w > 0).sum(1) - 1)[:, None]
    tok = torch.gather(ids, 1, at).view(B, n + 1)
    lp = torch.log(torch.gather(w, 1, at) / kept).view(B, n + 1)
    # the walk: a level a step, all requests at once
    par, draft = st["parents"].view(B, n).long(), st["draft"].view(B, n).long()
    out = torch.full((B, n + 1), -1, dtype=torch.int32, device=DEV)
    path = torch.full((B, n), -1, dtype=torch.int32, device=DEV)
    lps = torch.zeros(B, n + 1, dtype=torch.float32, device=DEV)
    cur = torch.full((B, 1), -1, dtype=torch.int64, device=DEV)
    live = torch.ones(B, 1, dtype=torch.bool, device=DEV)
    count = torch.zeros(B, dtype=torch.int32, device=DEV)
    nodes = torch.arange(n, device=DEV)
    for d in range(n + 1):
        t = torch.gather(tok, 1, cur + 1)
        out[:, d:d + 1] = torch.where(live, t, torch.full_like(t, -1)).int()
        lps[:, d:d + 1] = torch.where(live, torch.gather(lp, 1, cur + 1), torch.zeros_like(live).double()).float()
        hit = (par == cur) & (draft == t) & live
        first = torch.where(hit, nodes, torch.full_like(nodes, n)).amin(1, keepdim=True)
        live = first < n
        if d < n:
            path[:, d:d + 1] = torch.where(live, first, torch.full_like(first, -1)).int()
        count += live[:, 0].int()
        cur = torch.where(live, first, cur)
    return out, path, count, lps


def _slots_of(table, pos, page):
    return table.gather(1, pos // page).long() * page + pos % page


def _caches(st):
    return [st[n].flatten(1, 2) for n in ("k_cache", "v_cache", "k_exp", "v_exp") if st[n] is not None]


def _plain_commit(st):
    page = st["case"]["page"]
    d = torch.arange(8, device=DEV)
    live = d < st["count"][:, None]
    to = st["lens"].long()[:, None] + torch.where(live, d, torch.zeros_like(d))
    at = st["lens"].long()[:, None] + torch.where(live, st["path"].long(), st["path"][:, :1].long())
    src, dst = (_slots_of(st["table"], p, page).flatten() for p in (at, to))
    for c in _caches(st):
        rows = c.view(torch.uint8)[:, src]
        c.view(torch.uint8)[:, dst] = rows
    return {n: st[n] for n in ("k_cache", "v_cache", "k_exp", "v_exp") if st[n] is not None}


def _plain_resize(table, room, ref, new_room, page, st=None):
    S, W = table.shape
    blocks = ref.shape[0]
    j = torch.arange(W, device=DEV)
    had, want = ((r.long() + page - 1) // page for r in (room, new_room))
    # pages behind the new room are let go of
    gone = (j >= want[:, None]) & (j < had[:, None])
    ref.index_add_(0, torch.where(gone, table, torch.zeros_like(table)).flatten().long(), -gone.flatten().int())
    table.masked_fill_(gone, -1)
    had = torch.minimum(had, want)
    # a last page that is filled in part and shared is copied before its sequence grows: by all but the last of those
    # that hold it, in order
    part = torch.where(new_room > room, room % page, torch.zeros_like(room))
    tail = table.gather(1, (had - 1).clamp(min=0)[:, None])[:, 0]
    grows = (part > 0) & (had > 0)
    before = ((tail[:, None] == tail[None]) & grows[:, None] & grows[None]).tril(-1).sum(1)
    copied = grows & (ref[tail.clamp(min=0).long()] - before > 1)
    ref.index_add_(0, tail.clamp(min=0).long(), -copied.int())
    need = want - had + copied
    first = torch.cumsum(need, 0) - need
    # the lowest free pages, in order of the sequences and of their places
    free = torch.sort((ref > 0).to(torch.uint8), stable=True).indices
    k = j - had[:, None] + copied[:, None]
    fresh = (k >= 0) & (j < want[:, None])
    given = free[(first[:, None] + k).clamp(0, blocks - 1)]
    ref.index_add_(0, torch.where(fresh, given, torch.zeros_like(given)).flatten(), fresh.flatten().int())
    table.copy_(torch.where(fresh, given.to(torch.int32), table))
    if st is not None:
        new = table.gather(1, (had - 1).clamp(min=0)[:, None])[:, 0]
        i = torch.arange(page, device=DEV)
        moved = copied[:, None] & (i < part[:, None])
        src = tail.clamp(min=0).long()[:, None] * page + i
        dst = torch.where(moved, new.clamp(min=0).long()[:, None] * page + i, src)
        for c in _caches(st):
            rows = c.view(torch.uint8)[:, src.flatten()]
            c.view(torch.uint8)[:, dst.flatten()] = rows
    room.copy_(new_room)


def _plain_fork(st):
    page, table, room, ref = st["case"]["page"], st["table"], st["room"], st["ref"]
    src, dst = st["src"].long(), st["dst"].long()
    j = torch.arange(table.shape[1], device=DEV)
    for rows, sign in ((dst, -1), (src, 1)):
        held = j < ((room[rows] + page - 1) // page)[:, None]
        ref.index_add_(0, torch.where(held, table[rows], torch.zeros_like(table[rows])).flatten().long(),
                       sign * held.flatten().int())
    table[dst] = table[src]
    room[dst] = room[src]


def _pages(st, more=()):
    return {n: st[n] for n in ("table", "room", "ref") + tuple(more) if st[n] is not None}


def _plain_pages(st):
    case = st["case"]
    if case["kind"] == "resize":
        _plain_resize(st["table"], st["room"], st["ref"], st["most"], case["page"])
        mid = st["table"].clone()
        _plain_resize(st["table"], st["room"], st["ref"], st["kept"], case["page"])
        return {"grown": mid, **_pages(st)}
    _plain_fork(st)
    _plain_resize(st["table"], st["room"], st["ref"], st["new_room"], case["page"], st)
    return _pages(st, ("k_cache", "v_cache", "k_exp", "v_exp"))


def _plain_matvec4(st):
    case = st["case"]
    q = torch.stack([st["q"] & 15, st["q"] >> 4], -1).view(case["out"], -1, case["group"])
    w = ((q.float() - 8.0) * st["scale"].float()[..., None]).view(case["out"], case["cols"])
    return torch.matmul(st["x"].float(), w.t()).to(torch.float16)


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"accept": _plain_accept, "commit": _plain_commit, "matvec4": _plain_matvec4}.get(kind, _plain_pages)(st)
    if kind == "accept":
        from chain_flow_amd.tree_verify import tree_sample_accept
        return tree_sample_accept(st["logits"], st["cu_draft"], st["cu_rows"], st["draft"], st["parents"], case["nodes"],
                                  st["u"], st["T"], top_k=st["top_k"], top_p=st["top_p"])
    if kind == "commit":
        from chain_flow_amd.kv_cache import kv_cache_commit
        kv_cache_commit(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["path"], st["count"], k_exp=st["k_exp"],
                        v_exp=st["v_exp"])
        return {n: st[n] for n in ("k_cache", "v_cache", "k_exp", "v_exp") if st[n] is not None}
    if kind == "resize":
        from chain_flow_amd.kv_pages import kv_pages_resize
        kv_pages_resize(st["table"], st["room"], st["ref"], st["most"], page=case["page"])
        mid = st["table"].clone()
        kv_pages_resize(st["table"], st["room"], st["ref"], st["kept"], page=case["page"])
        return {"grown": mid, **_pages(st)}
    if kind == "fork":
        from chain_flow_amd.kv_pages import kv_pages_fork, kv_pages_resize
        kv_pages_fork(st["table"], st["room"], st["ref"], st["src"], st["dst"], page=case["page"])
        kv_pages_resize(st["table"], st["room"], st["ref"], st["new_room"], page=case["page"], k_cache=st["k_cache"],
                        v_cache=st["v_cache"], k_exp=st["k_exp"], v_exp=st["v_exp"])
        return _pages(st, ("k_cache", "v_cache", "k_exp", "v_exp"))
    from chain_flow_amd.head import matvec4
    return matvec4(st["x"], st["q"], st["scale"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "accept":
        B, n, V = case["seqs"], case["nodes"], case["vocab"]
        # every row read once; its uniform number, the tree, the outputs.  A row's counts and sums: one addition a logit
        return {"bytes": B * (n + 1) * (2.0 * V + 4) + B * n * 8.0 + B * (n * 12.0 + 12), "flops": 1.0 * B * (n + 1) * V}
    if kind == "commit":
        row = case["kvheads"] * (case["dim"] + 1 if case["cache"] == "fp8" else 2 * case["dim"])
        moved = sum(sum(p != d for d, p in enumerate(_path_of(case["nodes"], s))) for s in range(case["seqs"]))
        return {"bytes": 2.0 * 2 * moved * row * case["layers"] + case["seqs"] * 80.0, "flops": 0.0}
    if kind == "resize":
        now, most, kept = _resize_rooms(case)
        page = case["page"]
        taken = sum(-(-m // page) - -(-n // page) for n, m in zip(now, most))
        back = sum(-(-m // page) - -(-n // page) for n, m in zip(kept, most))
        # an entry and a count for every page that changes hands, the rooms, one look at the counts for free pages; the copy
        # of the table between the calls
        width = -(-max(most) // page) + 1
        return {"bytes": 12.0 * (taken + back) + 16.0 * case["seqs"] + 4.0 * case["blocks"] + 8.0 * case["seqs"] * width,
                "flops": 0.0}
    if kind == "fork":
        P, C, page = case["parents"], case["children"], case["page"]
        now = _spread(case["length"], P)
        row = case["kvheads"] * (case["dim"] + 1 if case["cache"] == "fp8" else 2 * case["dim"])
        shared = sum(C * -(-m // page) for m in now)
        copied = sum(C * (m % page) for m in now)
        blocks = sum(-(-m // page) for m in now) + P * C * (-(-case["new"] // page) + 1) + 2
        return {"bytes": 16.0 * shared + 2.0 * 2 * copied * row * case["layers"] + 4.0 * blocks + 16.0 * P * C, "flops": 0.0}
    M, K, n = case["rows"], case["cols"], case["out"]
    return {"bytes": n * (K / 2 + 2.0 * K / case["group"]) + 2.0 * M * (K + n), "flops": 2.0 * M * n * K}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_row(x, T, k, P, u):
    """One row's drawn token and the log of its probability, from the distinct values and how often each occurs."""
    if T <= 0:
        return int(torch.nonzero(x == x.max())[0]), 0.0
    vals, counts = torch.unique(x.double(), return_counts=True)
    vals, counts = vals.flip(0), counts.flip(0)
    cum = torch.cumsum(counts, 0)
    if k > 0:
        counts = (counts - (cum - k).clamp(min=0)).clamp(min=0)
    w = torch.exp((vals - vals[0]) / T)
    mass = torch.cumsum(counts * w, 0)
    if P < 1:
        goal = P * mass[-1]
        i = int((mass < goal).sum())
        i = min(i, len(vals) - 1)
        over = (goal - (mass[i] - counts[i] * w[i])) / w[i]
        counts[i] = torch.minimum(counts[i], torch.ceil(over).clamp(min=1).long())
        counts[i + 1:] = 0
        mass = torch.cumsum(counts * w, 0)
    goal = u * mass[-1]
    i = min(int((mass <= goal).sum()), int((counts > 0).sum()) - 1)
    r = int(torch.floor((goal - (mass[i] - counts[i] * w[i])) / w[i]).clamp(min=0))
    r = min(r, int(counts[i]) - 1)
    return int(torch.nonzero(x.double() == vals[i])[r]), float(torch.log(w[i] / mass[-1]))


def _exact_accept(case, st):
    B, n = case["seqs"], case["nodes"]
    lps = torch.zeros(B, n + 1, dtype=torch.float64)
    par, draft = st["parents"].view(B, n).tolist(), st["draft"].view(B, n).tolist()
    for b in range(B):
        T = float(st["T"][b])
        k = 0 if st["top_k"] is None else int(st["top_k"][b])
        P = 1.0 if st["top_p"] is None else float(st["top_p"][b])
        cur, d = -1, 0
        while True:
            row = b * (n + 1) + cur + 1
            tok, lps[b, d] = _exact_row(st["logits"][row], T, k, P, float(st["u"][row]))
            nxt = [i for i in range(n) if par[b][i] == cur and draft[b][i] == tok]
            if not nxt:
                break
            cur, d = nxt[0], d + 1
    return None, None, None, lps.to(DEV)


def _exact_commit(case, st):
    page, out = case["page"], {}
    table, path, lens = (st[n].tolist() for n in ("table", "path", "lens"))
    for n in ("k_cache", "v_cache"):
        c = st[n].double()
        old = c.clone()
        for s, m in enumerate(st["count"].tolist()):
            for d in range(m):
                a, b = lens[s] + path[s][d], lens[s] + d
                c[:, table[s][b // page], b % page] = old[:, table[s][a // page], a % page]
        out[n] = c
    if st["k_exp"] is not None:
        out["k_exp"] = out["v_exp"] = None
    return out


def _exact_fork(case, st):
    """Cache contents: each child's last shared page, where it is filled in part, stands copied in the next free page."""
    P, C, page = case["parents"], case["children"], case["page"]
    now, out = _spread(case["length"], P), {}
    free = [i for i, r in enumerate(st["ref"].tolist()) if r == 0]
    table = st["table"].tolist()
    copies = []
    for p in range(P):
        for _ in range(C):
            used = -(-(now[p] + case["new"]) // page) - now[p] // page
            if now[p] % page:
                copies.append((table[p][now[p] // page], free[0], now[p] % page))
            free = free[used:]
    for n in ("k_cache", "v_cache"):
        c = st[n].double()
        for a, b, m in copies:
            c[:, b, :m] = c[:, a, :m]
        out[n] = c
    return {"table": None, "room": None, "ref": None, **out, **({} if st["k_exp"] is None else {"k_exp": None, "v_exp": None})}


def _exact_matvec4(case, st):
    out, x = [], st["x"].double()
    for lo in range(0, case["out"], 4096):
        q = st["q"][lo:lo + 4096].to(torch.int64)
        w = torch.empty(q.shape[0], case["cols"], dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (q % 16 - 8).double(), (q // 16 - 8).double()
        w *= st["scale"][lo:lo + 4096].double().repeat_interleave(case["group"], 1)
        out.append(torch.mm(x, w.t()))
    return torch.cat(out, 1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "resize":
        return None                                 # whole numbers alone
    st = _inputs(case, seed)
    return {"accept": _exact_accept, "commit": _exact_commit, "fork": _exact_fork, "matvec4": _exact_matvec4}[kind](case, st)
