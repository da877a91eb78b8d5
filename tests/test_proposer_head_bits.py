"""The proposer's CF_HEAD_BITS (host logic, no GPU)."""
from __future__ import annotations

import pytest

from chain_flow_amd.drafter import Drafter
from chain_flow_amd.vllm_plugin import flow_proposer as fp
from test_proposer import _env, _vcfg, ckpt  # noqa: F401


def _proposer(monkeypatch, folder, **env):
    _env(monkeypatch, CF_DRAFTER_DIR=folder)
    for k in ("CF_TWOPASS_M", "CF_TWOPASS_SHARED", "CF_TWOPASS_SEED", "CF_HEAD_BITS"):
        monkeypatch.delenv(k, raising=False)
    for k, v in env.items():
        monkeypatch.setenv(k, v)
    return fp.FlowDrafterProposer(_vcfg())


def test_head_bits(monkeypatch, ckpt):  # noqa: F811
    """16 by default, with the two-pass head; 4 searches in one pass, and what cannot go with it is refused."""
    for env in ({}, {"CF_HEAD_BITS": ""}, {"CF_HEAD_BITS": "16"}):
        p = _proposer(monkeypatch, ckpt[0], **env)
        assert (p.head_bits, p.twopass_m, p.twopass_shared) == (16, 8192, True)
    for env in ({}, {"CF_TWOPASS_M": "0"}):
        p = _proposer(monkeypatch, ckpt[0], CF_HEAD_BITS="4", **env)
        assert (p.head_bits, p.twopass_m, p.twopass_shared) == (4, 0, False)
    with pytest.raises(ValueError, match="CF_HEAD_BITS=8 is not 16 or 4"):
        _proposer(monkeypatch, ckpt[0], CF_HEAD_BITS="8")
    with pytest.raises(ValueError, match="does not go with CF_TWOPASS_M"):
        _proposer(monkeypatch, ckpt[0], CF_HEAD_BITS="4", CF_TWOPASS_M="64")


def test_head_bits_reach_the_drafter(monkeypatch, ckpt):  # noqa: F811
    """The choice is handed on; a drafter of other widths is refused before it touches the device."""
    with pytest.raises(ValueError, match="head_bits=8 is not 16 or 4"):
        Drafter(ckpt[1], ckpt[2], None, device="cpu", head_bits=8)
    with pytest.raises(ValueError, match="one pass"):
        Drafter(ckpt[1], ckpt[2], None, device="cpu", head_bits=4, twopass_m=32)
    import torch
    seen = {}

    class Stop(Exception):
        pass

    def drafter(*args, **kw):
        seen.update(kw)
        raise Stop
    monkeypatch.setattr(fp, "Drafter", drafter)
    p = _proposer(monkeypatch, ckpt[0], CF_HEAD_BITS="4", CF_SHORTLIST="")
    emb = torch.zeros(64, 512, dtype=torch.float16)
    p.bind_target(emb, emb.clone())
    with pytest.raises(Stop):
        p._build()
    assert seen["head_bits"] == 4 and seen["twopass_m"] == 0 and not seen["twopass_shared"]
