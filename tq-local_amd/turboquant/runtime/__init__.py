"""Runtime: libtq kernel wrappers, packed cache, attention backend, generation loop."""

from turboquant.runtime.attention import (
    block_sparse_attention,
    chunked_turboquant_attention,
    fused_attention,
    prompt_attention,
    shared_prefix_attention,
    tree_attention,
    triton_available,
)
from turboquant.runtime.shared_prefix import SharedPrefixLayer, share_prefix

__all__ = ["fused_attention", "triton_available", "chunked_turboquant_attention", "prompt_attention",
           "tree_attention", "block_sparse_attention", "shared_prefix_attention", "share_prefix", "SharedPrefixLayer"]
