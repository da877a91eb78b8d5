"""Sampled speculative steps as a server takes them, everything on the device: two prompts shared by three sequences each, trees drafted
by the 4-bit head, room for their rows, the rows written, tokens drawn and accepted, accepted rows moved together and the
rooms cut back -- eagerly, on a side stream and as one captured graph.  After each step the emitted tokens equal the float64
oracle's, the cache holds each sequence's tokens and no page is lost."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.head import QuantHead
from chain_flow_amd.kv_cache import kv_cache_commit, kv_cache_read, kv_cache_write, paged_attention
from chain_flow_amd.kv_pages import kv_pages_fork, kv_pages_resize
from chain_flow_amd.tree_verify import tree_sample_accept
from oracle import tree_verify as otv

V, S, N, PAGE, HKV, D, LAYERS, WIDTH = 640, 6, 7, 4, 2, 64, 2, 14
PARENTS = [-1, -1, 0, 0, 1, 2, 4]              # of a tree's nodes: two children of the root, two and one of theirs, ..


class _Server:
    def __init__(self, dev, kind):
        g = torch.Generator().manual_seed(5)
        rand = lambda *s: torch.randn(*s, generator=g)                                   # noqa: E731
        self.dev, f8 = dev, kind == "fp8"
        self.hidden = rand(V, 256).half().to(dev)
        self.head = QuantHead((rand(V, 256) * 0.2).half().to(dev), None, rand(V, 128).half(), (rand(V, 128) * 0.2).half())
        everyone = torch.arange(V, dtype=torch.int32, device=dev)
        self.target = self.head.logits(self.hidden, everyone).to(torch.bfloat16)         # a token's next token's logits
        self.rows = [rand(LAYERS, V, HKV, D).to(torch.bfloat16).to(dev) for _ in range(2)]
        blocks = S * WIDTH
        shape = (LAYERS, blocks, PAGE, HKV, D)
        kinds = torch.float8_e4m3fn if f8 else torch.bfloat16
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device=dev).to(kinds) for _ in range(2))
        self.exps = [torch.full(shape[:-1], 127, dtype=torch.uint8, device=dev) for _ in range(2)] if f8 else [None, None]
        self.table = torch.full((S, WIDTH), -1, dtype=torch.int32, device=dev)
        self.room, self.lens, self.root = (torch.zeros(S, dtype=torch.int32, device=dev) for _ in range(3))
        self.ref = torch.zeros(blocks, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.u = torch.zeros(S * (N + 1), device=dev)
        self.T = torch.tensor([0.0, 0.8, 1.0, 1.3, 0.0, 0.6], device=dev)
        self.top_k = torch.tensor([0, 40, 0, 300, 5, 0], dtype=torch.int32, device=dev)
        self.top_p = torch.tensor([1.0, 0.95, 0.9, 1.0, 1.0, 0.8], device=dev)
        self.cu_d, self.cu_r = (torch.arange(1, S + 1, dtype=torch.int32, device=dev) * n for n in (N, N + 1))
        self.parents = torch.tensor(PARENTS * S, dtype=torch.int32, device=dev)
        self.draft = torch.zeros(S, N, dtype=torch.int32, device=dev)
        self.out = torch.zeros(S, N + 1, dtype=torch.int32, device=dev)
        self.count = torch.zeros(S, dtype=torch.int32, device=dev)
        self.logprobs = torch.zeros(S, N + 1, device=dev)

    def _cache(self, layer=None):
        at = lambda t: t if t is None or layer is None else t[layer]                     # noqa: E731
        return dict(k_cache=at(self.k), v_cache=at(self.v), k_exp=at(self.exps[0]), v_exp=at(self.exps[1]))

    def _write(self, tokens, slots):
        for layer in range(LAYERS):
            key, value = (r[layer][tokens.long()] for r in self.rows)
            kv_cache_write(key, value, slots=slots.to(torch.int32), status=self.status, **self._cache(layer))

    def prompts(self, texts):
        """Sequence 0 and 3 read them, the others share."""
        room = [len(texts[0]), 0, 0, len(texts[1]), 0, 0]
        kv_pages_resize(self.table, self.room, self.ref, torch.tensor(room), page=PAGE, status=self.status)
        for s, text in ((0, texts[0]), (3, texts[1])):
            pos = torch.arange(len(text), device=self.dev)
            self._write(torch.tensor(text, device=self.dev), self.table[s][pos // PAGE] * PAGE + pos % PAGE)
        kv_pages_fork(self.table, self.room, self.ref, torch.tensor([0, 0, 3, 3]), torch.tensor([1, 2, 4, 5]), page=PAGE,
                      status=self.status)
        self.lens.copy_(self.room)

    def step(self):
        tops = lambda prev, n: self.head.topk(self.hidden[prev.long()], n, prev)[1].to(torch.int32)      # noqa: E731
        d = self.draft
        d[:, :2] = tops(self.root, 2)
        d[:, 2:4] = tops(d[:, 0].contiguous(), 2)
        d[:, 4:5] = tops(d[:, 1].contiguous(), 1)
        d[:, 5:6] = tops(d[:, 2].contiguous(), 1)
        d[:, 6:7] = tops(d[:, 4].contiguous(), 1)
        kv_pages_resize(self.table, self.room, self.ref, self.lens + (N + 1), page=PAGE, status=self.status, **self._cache())
        tokens = torch.cat([self.root[:, None], d], 1).reshape(-1)
        pos = (self.lens[:, None] + torch.arange(N + 1, device=self.dev)).long()
        self._write(tokens, (self.table.gather(1, pos // PAGE) * PAGE + pos % PAGE).reshape(-1))
        out, path, count, lps = tree_sample_accept(
            self.target[tokens.long()], self.cu_d, self.cu_r, d.reshape(-1), self.parents, N, self.u, self.T, top_k=self.top_k,
            top_p=self.top_p, status=self.status)
        kv_cache_commit(block_table=self.table, seq_lens=self.lens + 1, path=path, path_len=count, status=self.status, **self._cache())
        self.lens.add_(count + 1)
        kv_pages_resize(self.table, self.room, self.ref, self.lens, page=PAGE, status=self.status, **self._cache())
        self.root.copy_(out.gather(1, count.long()[:, None])[:, 0])
        self.out.copy_(out)
        self.count.copy_(count)
        self.logprobs.copy_(lps)

    def check(self, texts, roots):
        """Against the oracle; texts and roots (host) move on."""
        assert int(self.status) == 0
        tokens = np.concatenate([np.array(roots)[:, None], self.draft.cpu().numpy()], 1).reshape(-1)
        f64 = lambda t: t.double().cpu().numpy()                                          # noqa: E731
        out, path, count, lps = otv.sampled_descent(
            f64(self.target)[tokens], self.cu_d.cpu().numpy(), self.cu_r.cpu().numpy(), self.draft.cpu().numpy().reshape(-1),
            np.array(PARENTS * S), N, f64(self.u), f64(self.T), self.top_k.cpu().numpy(), f64(self.top_p))
        assert np.array_equal(self.out.cpu().numpy(), out) and np.array_equal(self.count.cpu().numpy(), count)
        assert (np.abs(f64(self.logprobs) - lps) <= np.abs(lps) * 2.0 ** -24 + V * 2.0 ** -51).all()
        for s in range(S):
            texts[s] += [roots[s]] + [int(t) for t in out[s, :count[s]]]
            roots[s] = int(out[s, count[s]])
        lens, table, ref = self.lens.tolist(), self.table.cpu().numpy(), np.zeros(S * WIDTH, dtype=int)
        assert lens == [len(t) for t in texts] == self.room.tolist() and self.root.tolist() == roots
        for s in range(S):
            held = -(-lens[s] // PAGE)
            assert (table[s, held:] == -1).all()
            np.add.at(ref, table[s, :held], 1)
            pos = np.arange(lens[s])
            slots = torch.tensor(table[s][pos // PAGE] * PAGE + pos % PAGE, dtype=torch.int32, device=self.dev)
            ids = torch.tensor(texts[s], device=self.dev)
            for layer in range(LAYERS):
                plain = {n: None if t is None else torch.zeros_like(t) for n, t in self._cache(layer).items()}
                kv_cache_write(*(r[layer][ids] for r in self.rows), slots=torch.arange(lens[s]), **plain)
                want = kv_cache_read(slots=torch.arange(lens[s]), dtype=torch.bfloat16, **plain)
                got = kv_cache_read(slots=slots, dtype=torch.bfloat16, **self._cache(layer))
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert np.array_equal(self.ref.cpu().numpy(), ref)
        return int(count.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("how", ["eager", "stream", "graph"])
def test_sampled_steps(cuda, how, kind):
    server = _Server(cuda, kind)
    rng = np.random.default_rng(11)
    texts = [[int(t) for t in rng.integers(0, V, n)] for n in (6, 9)]
    print(f"[sampled steps] {how} {kind}", flush=True)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if how == "stream" else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        server.prompts(texts)
    stream.synchronize()
    texts = [list(texts[s // 3]) for s in range(S)]
    roots = [int(t) for t in rng.integers(0, V, S)]
    server.root.copy_(torch.tensor(roots))
    graph, accepted = None, 0
    for i in range(5):
        server.u.copy_(torch.tensor(rng.random(S * (N + 1)), dtype=torch.float32))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            if how == "graph" and i == 1:          # (the first step is an eager one; capturing runs nothing)
                graph = torch.cuda.CUDAGraph()
                with torch.inference_mode(), torch.cuda.graph(graph):    # (as the draft graphs: captures of one mode go together)
                    server.step()
            if graph is not None:
                graph.replay()
            else:
                server.step()
        stream.synchronize()
        print(f"[sampled steps] step {i} lengths {server.lens.tolist()}", flush=True)
        accepted += server.check(texts, roots)
    # greedy requests' drafts are the target's own first choices, but where a rounding makes two of them one
    assert accepted > 0 and int(server.ref.max()) == 3
    # attention over the pages as they ended, one token a sequence
    q = torch.randn(S, 4, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    cu = torch.arange(S + 1, dtype=torch.int32, device=cuda)
    got, lse = paged_attention(q, block_table=server.table, seq_lens=server.lens, cu_q=cu, scale=0.125, **server._cache(1))
    for s in range(S):
        pos = np.arange(len(texts[s]))
        slots = torch.tensor(server.table[s].cpu().numpy()[pos // PAGE] * PAGE + pos % PAGE, dtype=torch.int32)
        k, v = (t.double().cpu() for t in kv_cache_read(slots=slots, dtype=torch.bfloat16, **server._cache(1)))
        for h in range(4):
            x = (k[:, h // 2] @ q[s, h].double().cpu()) * 0.125
            want = torch.softmax(x, 0) @ v[:, h // 2]
            # weights are rounded to bf16 on their way into the second product (2^-8), the result once more (2^-8)
            tol = 2.0 ** -7 * (torch.softmax(x, 0) @ v[:, h // 2].abs()) + 2.0 ** -8 * want.abs() + 1e-6
            assert ((got[s, h].double().cpu() - want).abs() <= tol).all()
            assert abs(float(lse[h, s]) - float(torch.logsumexp(x, 0))) < 1e-4
    # requests end: every page is free again
    kv_pages_resize(server.table, server.room, server.ref, torch.zeros(S, dtype=torch.int32), page=PAGE, status=server.status)
    assert int(server.ref.abs().sum()) == 0 and (server.table == -1).all() and int(server.status) == 0


@pytest.mark.gpu
def test_two_servers_at_once(cuda):
    """Two of them on streams of their own, steps in turn and no waiting in between: neither finds the other's workspaces."""
    rng = np.random.default_rng(3)
    servers, texts, roots, streams = [], [], [], [torch.cuda.Stream() for _ in range(2)]
    print("[sampled steps] two at once", flush=True)
    for i in range(2):
        servers.append(_Server(cuda, ("bf16", "fp8")[i]))
        prompts = [[int(t) for t in rng.integers(0, V, n)] for n in (5 + i, 8)]
        servers[i].prompts(prompts)
        texts.append([list(prompts[s // 3]) for s in range(S)])
        roots.append([int(t) for t in rng.integers(0, V, S)])
        servers[i].root.copy_(torch.tensor(roots[i]))
    for step in range(3):
        draws = [torch.tensor(rng.random(S * (N + 1)), dtype=torch.float32).to(cuda) for _ in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                servers[i].u.copy_(draws[i])
                servers[i].step()
        torch.cuda.synchronize()
        for i in range(2):
            servers[i].check(texts[i], roots[i])
        print(f"[sampled steps] step {step}", flush=True)
