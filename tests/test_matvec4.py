"""The 4-bit head's oracle against its rules, and the calls' refusals (CPU only)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd import _lib
from chain_flow_amd.drafter import Drafter
from chain_flow_amd.head import QuantHead, matvec4, quantize4, row_topk
from oracle import head as ohead


def test_oracle_is_off_by_half_a_scale_at_most():
    rng = np.random.default_rng(0)
    w = (rng.normal(size=(40, 256)) * np.exp(rng.normal(size=(40, 1)) * 3)).astype(np.float16).astype(np.float64)
    w[3, 64:128] = 0
    w[4] = 6e-8                                                       # (the least fp16 values: scales round up)
    for group in (32, 64, 128):
        q, s = ohead.quantize4(w, group)
        assert q.min() >= 1 and q.max() <= 15
        assert (np.abs(ohead.dequant4(q, s) - w) <= np.repeat(s, group, 1) / 2 * (1 + 1e-12)).all()
        assert (s[3, 64 // group: 128 // group] == 0).all() if group <= 64 else True
    assert np.array_equal(ohead.unpack4(np.array([[0x21, 0xf0]])), [[1, 2, 0, 15]])


def test_refusals_without_a_device():
    x = torch.zeros(2, 256, dtype=torch.float16)
    w, s = torch.zeros(5, 128, dtype=torch.uint8), torch.zeros(5, 4, dtype=torch.float16)
    for args in ((x.float(), w, s), (x[0], w, s), (x, w.int(), s), (x, w, s.float()), (x, w, s[:4]), (x, w, s[:, :3]),
                 (x, w, torch.zeros(5, 16, dtype=torch.float16)), (x, w[:, :96], torch.zeros(5, 3, dtype=torch.float16)),
                 (x[:, :128], w, s), (x, w, s[:, :0])):
        with pytest.raises(ValueError):
            matvec4(*args)
    t, ids = torch.zeros(7, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    for kw in (dict(table=t), dict(ids=ids), dict(table=t, ids=ids.long()), dict(table=t.float(), ids=ids), dict(table=t, ids=ids[:1]),
               dict(table=t, ids=ids, ids_stride=2), dict(table=t, ids=ids, ids_stride=0), dict(table=t[:, :64], ids=ids)):
        with pytest.raises(ValueError):
            matvec4(x[:, :128], w, s, **kw)
    with pytest.raises(ValueError, match="one GPU"):
        matvec4(x, w, s)
    for args in ((x.float(),), (x, 48), (x[:, :192], 128), (x[:, :64], 64), (x, 64, None, x[:1]), (x, 64, None, t[:2, :32])):
        with pytest.raises(ValueError):
            quantize4(*args)
    with pytest.raises(ValueError, match="CUDA"):
        QuantHead(x, None)
    with pytest.raises(ValueError, match="head_bits"):
        Drafter(None, {}, None, head_bits=8)
    with pytest.raises(ValueError, match="one pass"):
        Drafter(None, {}, None, head_bits=4, twopass_m=64)
    L, p = _lib.lib(), 4096      # stand-in addresses: never dereferenced, the checks fail first

    def mv(x=p, ld_x=256, M=2, d=256, w=p, ld_w=128, s=p, ld_s=4, group=64, n=5, a=None, rows=0, ids=None, r=0, y=p, ld_y=5):
        return L.cfh_matvec4(x, ld_x, M, d, w, ld_w, s, ld_s, group, n, a, rows, ids, 1, r, y, ld_y, None)
    assert mv(M=0) == mv(n=0) == 0
    assert mv(x=None) == mv(x=p + 2) == mv(ld_x=252) == mv(ld_x=248) == mv(w=p + 4) == mv(ld_w=112) == mv(ld_w=136) == mv(s=p + 2) == 1
    assert mv(ld_s=3) == mv(ld_s=5) == mv(group=16) == mv(ld_y=4) == mv(y=None) == mv(M=-1) == mv(d=0) == mv(r=-1) == 1
    more = dict(d=128, r=128, a=p, rows=3, ids=p)
    assert mv(**{**more, "a": None}) == mv(**{**more, "ids": None}) == mv(**{**more, "rows": 0}) == mv(**{**more, "a": p + 8}) == 1
    assert mv(d=192) == mv(d=130, r=126, a=p, rows=3, ids=p) == mv(d=65536 + 128, ld_x=1 << 17, ld_w=1 << 17, ld_s=4096) == 2

    def qt(w=p, w2=None, n=3, d=256, r=0, group=64, q=p, s=p):
        return L.cfh_quantize4(w, w2, None, n, d, r, group, q, s, None)
    assert qt(n=0) == 0 and qt(w=None) == qt(w=p + 2) == qt(q=None) == qt(s=None) == qt(group=0) == qt(r=64, d=192) == 1
    assert qt(d=96) == qt(d=192) == qt(d=160, r=96, w2=p) == 2


@pytest.mark.parametrize("split", [False, True])
def test_row_topk_refusals(split):
    x = torch.zeros(2, 256, dtype=torch.float16)
    for bad in (x, x.bfloat16(), x.float(), x[0]):                    # (host memory, other types, one row)
        with pytest.raises(ValueError, match="logits"):
            row_topk(bad, 4, split=split)
