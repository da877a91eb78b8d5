"""chain-flow drafting hot path on MI355X: PyTorch-ROCm host code over libcfhip.so (HIP/gfx950).

Modules: ``config`` (TreeFlowConfig), ``weights`` (seeded synthetic state), ``shortlist`` (the
shortlist file format and vocabulary guard), ``flow`` (fused predict_hidden), ``head`` (shortlisted
lm_head + top-k, path residual), ``drafter`` (chain/tree beam drafts), ``gdn`` (gated delta net over
draft trees, prefill chunks and decode rows), ``kv_cache`` (the committed prefix's paged cache and the attention
over it), ``tree_verify`` (tree conv, attention merge, greedy accept), ``vllm_plugin.flow_proposer`` (the
``FlowDrafterProposer`` custom_class surface).
"""

__version__ = "0.1.0"
