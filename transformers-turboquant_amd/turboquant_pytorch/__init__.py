"""MI355X-native TurboQuant KV-cache compression (gfx950 HIP kernels behind a C ABI).

Public objects keep the reference's names (src/turboquant_pytorch/__init__.py:3).
"""

from .compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2
from .drafts import append_tree_attention, tree_attention, verify_drafts
from .fused import compressed_attention
from .pages import PagePool
from .prefix import append_prefix_attention, prefix_attention, prefix_groups
from .sampling import filter_probs, sample_tokens

__all__ = ["TurboQuantCompressorV2", "TurboQuantCompressorMSE", "compressed_attention", "PagePool",
           "append_prefix_attention", "append_tree_attention", "filter_probs", "prefix_attention", "prefix_groups",
           "sample_tokens", "tree_attention", "verify_drafts"]
