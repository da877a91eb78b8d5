"""chain-flow drafting hot path on MI355X: PyTorch-ROCm host code over libcfhip.so (HIP/gfx950).

Modules: ``config`` (TreeFlowConfig), ``weights`` (seeded synthetic state), ``shortlist`` (the
shortlist file format and vocabulary guard), ``flow`` (fused predict_hidden), ``head`` (shortlisted
lm_head + top-k, at fp16 or 4 bits, path residual), ``drafter`` (chain/tree beam drafts), ``gdn`` (gated delta net over
draft trees, prefill chunks and decode rows), ``kv_cache`` (the committed prefix's paged cache, the attention
over it and the accepted rows' way into it), ``kv_pages`` (the cache's pages: taken, given back, shared),
``tree_verify`` (tree conv, attention merge, greedy and sampled accept), ``vllm_plugin.flow_proposer`` (the
``FlowDrafterProposer`` custom_class surface).
"""

__version__ = "0.1.0"
