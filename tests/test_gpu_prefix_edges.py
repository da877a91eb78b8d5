"""Edges of the committed prefix's calls on the GPU: saturated bounds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from chain_flow_amd.kv_cache import paged_attention
from conftest import to64
from oracle import kv_cache as okv
from test_gpu_kv_cache import BF, Case, close


def check_first(c, out, lse, S, causal=True):
    """The rows of the first S sequences of an attention case against the oracle."""
    T = c.cu[S]
    ref = okv.attention(to64(c.q[:T]), c.ok[:S], c.ov[:S], c.lens[:S], c.cu[:S + 1], c.scale, causal)
    close(out[:T].contiguous(), lse[:, :T].contiguous(), *ref, max(c.lens[:S] + [1]), c.dtype)


# ---------------------------------------------------------------- saturated bounds
@pytest.mark.gpu
@pytest.mark.parametrize("H,bounds", [(256, [0, 5, 2 ** 40, 2 ** 40]),                             # many rows a sequence
                                      (32, [0, 1, 2, 3, 3, 3, 3, 3, 3, 3, 3, 2 ** 40, 2 ** 40])])  # few
def test_attention_bounds_past_32_bits_skip_their_sequences_only(cuda, H, bounds):
    """Bounds that 32 bits do not hold, times many heads a kv head: those sequences are skipped, the others are not."""
    S, good = len(bounds) - 1, next(i for i, b in enumerate(bounds) if b > 100) - 1
    news = np.diff(np.minimum(bounds, bounds[good] + 1)).tolist()
    c = Case(cuda, BF, BF, news, [40 + 3 * i for i in range(S)], H, 1, 64, 16, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(c.q, 7.0)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(cuda)  # noqa: E731
    o, lse = paged_attention(c.q, c.k, c.v, i32(c.table), i32(c.lens), torch.tensor(bounds), scale=c.scale, out=out, status=status)
    assert status.item() == 1 and (o[bounds[good]:] == 7).all()
    check_first(c, o, lse, good)
