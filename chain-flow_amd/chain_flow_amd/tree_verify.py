"""Host side of the rest of the tree verify (the forked vLLM's tree arm) on the HIP kernels:

* ``tree_conv`` -- ``tree_scan_causal_conv1d`` (``cf/vllm_tree/tree_ssm.py:393-438``): the GDN
  layers' width-4 causal conv over the draft tree (bf16);
* ``tree_attn_merge`` -- the suffix half of ``_tree_attention_fixup`` plus the merge
  (``_tree_suffix_eager`` / ``fused_suffix_merge``, patch lines 403-575, 2793-3121): the tree rows'
  ancestor-masked attention merged into ``output`` with the prefix half by log-sum-exp;
* ``tree_greedy_accept`` -- ``tree_rejection_sample`` (patch lines 510-550): row argmax + greedy
  descent;
* ``tree_sample_accept`` -- the same walk with every row's token drawn from the target's filtered
  probabilities by a given uniform number (temperature, top-k, top-p a request).
"""
from __future__ import annotations

import torch

from chain_flow_amd import _lib


def _i32(t, dev):
    return torch.as_tensor(t).to(dev, torch.int32).contiguous()


def _host(t):
    """The values of a host-side index argument (None for a device tensor: not read back)."""
    if isinstance(t, torch.Tensor):
        return None if t.is_cuda else t.cpu().numpy()
    import numpy as np
    return np.asarray(t)


# Every device tensor handed to a launch is kept in a local until the launch is queued: a temporary
# freed after .data_ptr() returns its block to the caching allocator, and the next temporary of
# the same size would then alias it.


def tree_conv(x, conv_state, weight, bias, node_slots, parent, *, prefix_slot: int = 1, activation="silu",
              out=None):
    """x [N, dim] bf16 (rows may be strided), conv_state [slots, dim, 4] bf16 (node slots written in
    place), weight [dim, 4] bf16, bias [dim] or None; parent [N] node indices (BFS, -1 = root).
    Returns out [N, dim] bf16."""
    if x.dtype != torch.bfloat16 or conv_state.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError("tree_conv runs on bf16 tensors")
    N, dim = x.shape
    if x.stride(1) != 1 or conv_state.shape[1:] != (dim, 4) or not conv_state.is_contiguous():
        raise ValueError("x rows must be contiguous; conv_state [slots, dim, 4] contiguous")
    if activation not in ("silu", None, "none"):
        raise ValueError(f"activation {activation!r}")
    dev = x.device
    slots = conv_state.shape[0]
    hs, hp = _host(node_slots), _host(parent)
    if hs is not None and (len(hs) != N or hs.min() < 0 or hs.max() >= slots):
        raise ValueError(f"node_slots must be {N} slots in [0, {slots})")
    if hp is not None and (len(hp) != N or any(not (-1 <= int(hp[i]) < i) for i in range(N))):
        raise ValueError("parent[i] must be -1 or an earlier node (BFS order)")
    if not 0 <= prefix_slot < slots:
        raise ValueError(f"prefix_slot {prefix_slot} outside [0, {slots})")
    if out is None:
        out = torch.empty(N, dim, dtype=torch.bfloat16, device=dev)
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    ns, par = _i32(node_slots, dev), _i32(parent, dev)
    _lib.check(_lib.lib().cfh_tree_conv(
        x.data_ptr(), x.stride(0), conv_state.data_ptr(), w.data_ptr(), _lib.ptr(b), ns.data_ptr(),
        par.data_ptr(), prefix_slot, N, dim, 1 if activation == "silu" else 0, out.data_ptr(), out.stride(0),
        _lib.stream_handle()), "cfh_tree_conv")
    return out


def tree_attn_merge(query, key, value, output, prefix_out, prefix_lse, idx_pad, not_anc, scale: float):
    """query/key/value/output [T, heads, D] (bf16 or fp16, head dims contiguous), prefix_out
    [S*N, H, D], prefix_lse [H, S*N] fp32, idx_pad [S, N] forward rows of the tree nodes, not_anc
    [S, N, N] bool.  Writes the merged tree rows into ``output`` in place."""
    S, N = idx_pad.shape
    T, H, D = query.shape
    Hkv = key.shape[1]
    dt = query.dtype
    if dt not in (torch.bfloat16, torch.float16) or any(t.dtype != dt for t in (key, value, output, prefix_out)):
        raise ValueError("q/k/v/output/prefix_out must share one 2-byte dtype")
    for t in (query, key, value, output):
        if t.stride(2) != 1 or t.stride(1) != D:
            raise ValueError("head rows must be [.][heads][D] with contiguous heads")
    dev = query.device
    if prefix_out.shape != (S * N, H, D) or prefix_lse.shape != (H, S * N) or tuple(not_anc.shape) != (S, N, N):
        raise ValueError("prefix_out [S*N, H, D], prefix_lse [H, S*N], not_anc [S, N, N]")
    hi = _host(idx_pad)
    if hi is not None and (hi.min() < 0 or hi.max() >= min(T, key.shape[0], value.shape[0], output.shape[0])):
        raise ValueError("idx_pad rows outside the q/k/v/output rows")
    pout = prefix_out.contiguous()
    plse = prefix_lse.to(torch.float32).contiguous()
    idx = _i32(idx_pad, dev)
    # (a bool mask's bytes are 0 and 1 already: reinterpreted, not converted by a launch)
    mask = torch.as_tensor(not_anc).to(dev).contiguous()
    mask = mask.view(torch.uint8) if mask.dtype == torch.bool else mask.to(torch.uint8)
    _lib.check(_lib.lib().cfh_tree_attn_merge(
        query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0),
        output.data_ptr(), output.stride(0), pout.data_ptr(), plse.data_ptr(), idx.data_ptr(), mask.data_ptr(),
        float(scale), S, N, H, Hkv, D, 1 if dt == torch.bfloat16 else 0, _lib.stream_handle()),
        "cfh_tree_attn_merge")
    return output


def tree_greedy_accept(logits, cu_num_draft_tokens, cu_num_sampled_tokens, draft_token_ids, tree_parents,
                       max_spec_len: int):
    """logits [rows, V] (bf16 / fp16); cumulative (inclusive) per-request draft and row counts;
    draft ids and local parents (-1 = root) per draft token.  Returns (output_token_ids [B,
    max_spec_len + 1] int32, -1 padded; accepted_path [B, max_spec_len]; accepted_len [B])."""
    if logits.dtype not in (torch.bfloat16, torch.float16) or logits.stride(1) != 1:
        raise ValueError("logits must be bf16 / fp16 with contiguous rows")
    dev = logits.device
    B = len(cu_num_draft_tokens)
    R, V = logits.shape
    out = torch.empty(B, max_spec_len + 1, dtype=torch.int32, device=dev)
    path = torch.empty(B, max(max_spec_len, 1), dtype=torch.int32, device=dev)
    ln = torch.empty(B, dtype=torch.int32, device=dev)
    ra = torch.empty(R, dtype=torch.int32, device=dev)
    ws = torch.empty(int(_lib.lib().cfh_tree_accept_ws_bytes(R)), dtype=torch.uint8, device=dev)
    cd, cs = _host(cu_num_draft_tokens), _host(cu_num_sampled_tokens)
    if cd is not None and cs is not None:
        import numpy as np
        nd = np.diff(np.concatenate([[0], cd]))
        if (nd < 0).any() or nd.max(initial=0) > max_spec_len or int(cs[-1]) > R or \
                not np.array_equal(np.diff(np.concatenate([[0], cs])), nd + 1) or int(cd[-1]) > len(draft_token_ids):
            raise ValueError("cumulative draft / row counts inconsistent with the logits rows and max_spec_len")
    draft = _i32(draft_token_ids, dev) if len(draft_token_ids) else torch.zeros(1, dtype=torch.int32, device=dev)
    par = _i32(tree_parents, dev) if len(tree_parents) else torch.zeros(1, dtype=torch.int32, device=dev)
    cdg, csg = _i32(cu_num_draft_tokens, dev), _i32(cu_num_sampled_tokens, dev)
    _lib.check(_lib.lib().cfh_tree_greedy_accept(
        logits.data_ptr(), logits.stride(0), V, R, 1 if logits.dtype == torch.bfloat16 else 0, cdg.data_ptr(),
        csg.data_ptr(), draft.data_ptr(), par.data_ptr(), B, max_spec_len, out.data_ptr(), path.data_ptr(),
        ln.data_ptr(), ra.data_ptr(), ws.data_ptr(), _lib.stream_handle()), "cfh_tree_greedy_accept")
    return out, path[:, :max_spec_len], ln


def _counts_fit(cd, cs, R, D, max_spec_len):
    """Whether host-side cumulative draft and row counts describe requests of n drafts and n + 1 rows (or none of either)."""
    import numpy as np
    nd, ns = (np.diff(np.concatenate([[0], np.asarray(c, dtype=np.int64)])) for c in (cd, cs))
    return not ((nd < 0).any() or nd.max(initial=0) > max_spec_len or ((ns != nd + 1) & ((ns != 0) | (nd != 0))).any()
                or int(cs[-1]) > R or int(cd[-1]) > D)


def tree_sample_accept(logits, cu_num_draft_tokens, cu_num_sampled_tokens, draft_token_ids, tree_parents,
                       max_spec_len: int, uniforms, temperature, *, top_k=None, top_p=None, status=None):
    """``tree_greedy_accept`` for sampled requests: row r's target token is drawn by uniforms[r] in [0, 1) from its logits
    under its request's ``temperature`` [B] (fp32; 0: the largest logit), ``top_k`` [B] (int32; 0, or None: off) and
    ``top_p`` [B] (fp32; 1, or None: off); the walk from a request's root row steps to the first child that holds the
    drawn token and ends with the token that no child holds.  Drafts count as certain (a beam search's are), so that what is
    emitted is distributed as the target's own samples.

    A row's tokens are ordered by logit, ties by the lower index; NaN and -inf are none.  Of exp((x - max) / temperature) the
    first top_k are kept, of those the shortest prefix that has top_p of their sum (one token at least), and the token
    is the first at which the running sum exceeds uniforms[r] times what is kept.  Sums are held in 64 bits.  A row
    without any token gives none: its walk ends there.  Uniforms outside [0, 1) count as the nearest in it, NaN as 0; a
    temperature that is not above 0 as 0.

    logits [rows, V] (bf16 / fp16; rows may be strided); cumulative (inclusive) draft and row counts a request (n drafts have n + 1
    rows; a request of no rows and drafts is padding); draft ids and local parents (-1 = root).  -> (output_token_ids
    [B, max_spec_len + 1] int32, -1 padded; accepted_path [B, max_spec_len]; accepted_len [B]; logprobs [B, max_spec_len
    + 1] fp32, 0 padded: the log of what each emitted token's probability was, after the filters).  Counts are
    read on the device only (host ones are checked here): a request whose counts do not fit the rows or drafts, and all
    behind counts that fall, emit nothing and set ``status`` (int32 [1] on the device, zeroed by the caller), if given, to 1."""
    if logits.dtype not in (torch.bfloat16, torch.float16) or logits.dim() != 2 or logits.numel() == 0:
        raise ValueError("logits must be bf16 / fp16 [rows, V]")
    R, V = logits.shape
    ld = logits.stride(0) if R > 1 else V
    if (V > 1 and logits.stride(1) != 1) or ld < V:
        raise ValueError("logits must have contiguous rows")
    max_spec_len = int(max_spec_len)
    if max_spec_len < 0:
        raise ValueError(f"max_spec_len {max_spec_len} is negative")
    B, D = len(cu_num_draft_tokens), len(draft_token_ids)
    if len(cu_num_sampled_tokens) != B or len(tree_parents) != D:
        raise ValueError("draft and row counts must be of one length, and draft ids and parents of another")
    dev = _lib.device_of(logits, status=status)
    for name, t, n, kinds in (("uniforms", uniforms, R, (torch.float32,)), ("temperature", temperature, B, (torch.float32,)),
                              ("top_k", top_k, B, (torch.int32, torch.int64)), ("top_p", top_p, B, (torch.float32,))):
        if t is None and name[:3] == "top":
            continue
        if not isinstance(t, torch.Tensor) or t.shape != (n,) or t.dtype not in kinds or t.get_device() != dev:
            raise ValueError(f"{name} must be {' or '.join(str(k) for k in kinds)} [{n}] on cuda:{dev}")
    cd, cs = _host(cu_num_draft_tokens), _host(cu_num_sampled_tokens)
    if B and cd is not None and cs is not None and not _counts_fit(cd, cs, R, D, max_spec_len):
        raise ValueError("cumulative draft / row counts inconsistent with the logits rows, the drafts and max_spec_len")
    index = lambda t: _lib.index32(t if isinstance(t, torch.Tensor) else torch.as_tensor(t, dtype=torch.int64), dev)  # noqa: E731
    draft, par, cdg, csg = (index(t) for t in (draft_token_ids, tree_parents, cu_num_draft_tokens, cu_num_sampled_tokens))
    uniforms, temperature = uniforms.contiguous(), temperature.contiguous()
    top_k = None if top_k is None else _lib.index32(top_k, dev)
    top_p = None if top_p is None else top_p.contiguous()
    out = torch.empty(B, max_spec_len + 1, dtype=torch.int32, device=logits.device)
    path = torch.empty(B, max_spec_len, dtype=torch.int32, device=logits.device)
    ln = torch.empty(B, dtype=torch.int32, device=logits.device)
    lps = torch.empty(B, max_spec_len + 1, dtype=torch.float32, device=logits.device)
    L = _lib.lib()
    ws = torch.empty(int(L.cfh_tree_sample_ws_bytes(R, V)), dtype=torch.uint8, device=logits.device)
    _lib.check(L.cfh_tree_sample_accept(
        logits.data_ptr(), ld, V, R, logits.dtype == torch.bfloat16, cdg.data_ptr(), csg.data_ptr(), _lib.ptr(draft),
        _lib.ptr(par), D, B, max_spec_len, uniforms.data_ptr(), temperature.data_ptr(), _lib.ptr(top_k), _lib.ptr(top_p),
        out.data_ptr(), path.data_ptr(), ln.data_ptr(), lps.data_ptr(), ws.data_ptr(), _lib.ptr(status),
        _lib.stream_of(dev)), "cfh_tree_sample_accept")
    return out, path, ln, lps
