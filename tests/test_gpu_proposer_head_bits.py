"""The proposer over the 4-bit head (CF_HEAD_BITS=4), with and without draft graphs."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from chain_flow_amd.drafter import front_pad
from chain_flow_amd.head import QuantHead
from chain_flow_amd.vllm_plugin import flow_proposer as fp
from test_gpu_proposer import _ckpt


@pytest.mark.gpu
@pytest.mark.parametrize("graph", ["1", "0"])
def test_proposer_over_the_4_bit_head(cuda, tmp_path, monkeypatch, graph):
    """Steps of one to three requests give the drafts of the eager Drafter with head_bits=4 on the same history."""
    cfg, W, slv = _ckpt(tmp_path)
    for k in ("VLLM_SPEC_TREE", "CF_SHORTLIST", "CF_FLOW_STEPS", "CF_DRAFT_BUCKETS", "CF_ASYNC_SPEC", "CF_TWOPASS_M",
              "CF_TWOPASS_SHARED", "CF_TWOPASS_SEED"):
        monkeypatch.delenv(k, raising=False)
    monkeypatch.setenv("CF_DRAFTER_DIR", str(tmp_path))
    monkeypatch.setenv("CF_CUDAGRAPH", graph)
    monkeypatch.setenv("CF_HEAD_BITS", "4")
    p = fp.FlowDrafterProposer(SimpleNamespace(speculative_config=SimpleNamespace(num_speculative_tokens=5),
                                               scheduler_config=SimpleNamespace(max_num_seqs=4)))
    p.bind_target(W["embed_tokens.weight"].to(cuda), W["lm_head.weight"].to(cuda))
    rng = np.random.default_rng(6)
    hist = {i: [] for i in range(3)}
    for step, live in enumerate((1, 3, 2, 3)):
        toks = [[int(t) for t in slv[rng.integers(0, len(slv), size=int(rng.integers(1, 4)))]] for _ in range(live)]
        hid = torch.randn(sum(map(len, toks)), 512, generator=torch.Generator().manual_seed(90 + step)).half()
        off = 0
        for i, t in enumerate(toks):
            hist[i] += [hid[off + j] for j in range(len(t))]
            off += len(t)
        for i in range(live, 3):
            hist[i] = []                                           # (a request that leaves takes its history with it)
        out = p.propose(toks, hidden_states=hid.to(cuda), req_ids=[f"r{i}.{step if i else 0}" for i in range(live)])
        for i in range(1, live):                                   # (all but the first are new requests each step)
            hist[i] = hist[i][-len(toks[i]):]
        torch.cuda.synchronize()
        assert isinstance(p.drafter.head, QuantHead)
        ctx = torch.stack([front_pad(torch.stack(hist[i])[None], cfg.context_size)[0] for i in range(live)]).to(cuda)
        want = p.drafter.beam_chains(ctx, torch.tensor([t[-1] for t in toks], device=cuda), 5, 4).cpu().tolist()
        print(f"[proposer, 4-bit head] step {step} graph={graph} {out} eager {want}", flush=True)
        assert [list(o) for o in out] == want
